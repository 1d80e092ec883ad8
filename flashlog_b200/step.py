"""One sparse DRUM training step on static buffers, with no host synchronization.

This is src/model_DRUM_kernel_sp.py:92-204 (T hops of c1 selection,
expansion with the c2 budget, coalesce-sum and row normalization), the
channel readout and log loss of src/utils.py:36-47, their backward and an
SGD update of a per-query-relation attention table, written against buffers
allocated once.  Every buffer is sized by a static bound:

  selected entries of hop t   S_t = min(C_t, ceil(rows * c1 * zero_slack))
  fact slots of hop t         F_t = min(S_t * k_max, rows * K)
  outputs of hop t            C_{t+1} = min(F_t, rows * E)

where k(e) = min(deg_ori(e), c2//2) + min(deg_inv(e), c2//2) + 1 is the slot
capacity of entity e, k_max its maximum, K its sum over the entities (a row
holds every entity at most once) and C_0 = rows.  zero_slack is 1 without
dropout: a row keeps at most c1 entries unless it has at most c1 nonzero
values, and then all of them.  Such a row also keeps its explicit zeros
(flashlog_kernel.py:1114-1117).  With dropout p, a row of n entries holds
about n (1 - p) nonzero values, so the rows kept whole hold up to about
c1 / (1 - p) entries: zero_slack defaults to 1 / (1 - p) + 0.25 (see
default_zero_slack; p = 1 leaves the selection unbounded).  The kernels
read the live counts from the device (row_ptr[-1]), so nothing is read back
to the host and one step can be captured in a CUDA graph and replayed.  A
device status word flags any capacity overflow (it cannot happen under these
bounds without dropout) and `check` reads it.

The autograd path of engine.drum_propagate computes the same step with one
host synchronization per hop.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib as L
from . import muon, ops
from .ops import Graph, _p, _stream, check, lib


def _buf(n, dtype, dev):
    return torch.empty(max(int(n), 1), dtype=dtype, device=dev)


def default_zero_slack(p: float) -> float:
    """Selection slack for dropout p: rows kept whole hold up to about
    c1 / (1 - p) entries (their explicit zeros included), plus a margin."""
    if p <= 0.0:
        return 1.0
    if p >= 1.0:
        return math.inf
    return 1.0 / (1.0 - p) + 0.25


def capacities(rows: int, T: int, c1, k_max: int, K: int, E: int, zero_slack: float = 1.0):
    """Static bounds of the step's buffers per hop, as lists (C, S, F, U):
    C_t inputs, S_t selected entries, F_t fact slots, U_t = C_{t+1} outputs,
    with C_0 = rows, S_t = min(C_t, ceil(rows * c1 * zero_slack)) (C_t
    without c1, or with an infinite slack), F_t = min(S_t * k_max, rows * K),
    U_t = min(F_t, rows * E)."""
    Cs, Ss, Fs, Us = [], [], [], []
    C = rows
    for _ in range(T):
        S = min(C, math.ceil(rows * c1 * zero_slack)) if (c1 is not None and math.isfinite(zero_slack)) else C
        F = min(S * k_max, rows * K)
        Cs.append(C)
        Ss.append(S)
        Fs.append(F)
        C = min(F, rows * E)
        Us.append(C)
    return Cs, Ss, Fs, Us


class DrumTrainStep:
    """Static-buffer DRUM step: forward (T hops), loss, backward, SGD.

    table: [2R, T, N, n] attention logits (the parameter); a query with
    relation r uses table[r].  Inputs per step are copied into the static
    tensors heads, tails, rels (i64[Q]) and hide (i64[H], triple ids hidden
    during the step) with `load`.  With apply_update the step ends with the
    SGD update table[rels] -= lr * d loss / d logits (only the batch's rows
    are touched); without it the dense gradient of the table is left in
    `grad` (for an all-reduce across ranks before the caller's update),
    hop by hop in grad_hop[t] as the backward reaches it (see `parts`).
    dropout > 0 applies the training dropout of each hop's values
    (src/model_DRUM_kernel_sp.py:189-192) in place; replay k (from 1) draws
    hop t's keep bits from (dropout_seed, k, t), counted on the device.
    A step whose forward overflowed a buffer (status word nonzero) leaves
    the table and the gradient untouched (the gradient is scaled by 0 on the
    device); `check` then raises.

    head (weight [n, H], bias [n] or None): the table is [2R, T, N, H] hidden
    states, and a hop's logits are attention.linear of the queries' rows; the
    head is trained too (its gradients in grad_head).  rules
    (attention.OperatorRules): what the weights may take; its bias is not
    trained.  optimizer "muon": the table's T N matrices [2R, n or H] and the
    head's weight take muon.muon_update_ steps (muon_options: beta, nesterov,
    weight_decay, scale, steps, coefficients, eps) with momentum kept here,
    the whole table each step; a head's bias takes the SGD step.  `update`
    is the last part by itself, for a caller that reduced the gradients.
    """

    def __init__(self, graph: Graph, r_size: int, Q: int, T: int, N: int, c1, c2: int, table: torch.Tensor,
                 n_hide: int, lr: float = 0.01, eps: float = 1e-7, thr: float = 1e-7, stats: bool = True,
                 apply_update: bool = True, dropout: float = 0.0, dropout_seed: int = 0, zero_slack=None,
                 record_grad_w: bool = False, head=None, rules=None, optimizer: str = "sgd", muon_options=None):
        dev = table.device
        self.dev, self.graph, self.r_size, self.Q, self.T, self.N = dev, graph, r_size, Q, T, N
        self.n = 2 * r_size + 1
        self.c1 = None if c1 is None or c1 < 0 else int(c1)
        self.topk = c2 // 2 if c2 and c2 > 0 else L.NO_BUDGET
        self.flags = L.FL_SKIP_NONPOS_W | L.FL_DROP_MASKED
        self.eps, self.thr, self.lr = eps, thr, lr
        self.apply_update = apply_update
        if optimizer not in ("sgd", "muon"):
            raise ValueError(f"optimizer must be sgd or muon, got {optimizer!r}")
        width = self.n if head is None else head[0].shape[-1]
        # a table of more hops serves a step that keeps only gradients
        hops = table.shape[1] if table.dim() == 4 else -1
        if table.dim() != 4 or tuple(table.shape[2:]) != (N, width) or hops < T or (
                hops > T and (apply_update or optimizer != "sgd")):
            raise ValueError(f"table must be [2R, {T}, {N}, {width}], got {tuple(table.shape)}")
        if head is not None:
            if tuple(head[0].shape) != (self.n, width) or (head[1] is not None and tuple(head[1].shape) != (self.n,)):
                raise ValueError(f"head must be a weight [{self.n}, H] and a bias [{self.n}] or None")
            if any(t is not None and (t.dtype != torch.float32 or t.device != dev or not t.is_contiguous())
                   for t in head):
                raise ValueError("head must be contiguous float32 tensors on the table's device")
        if rules is not None:
            rules.check(T, Q, self.n)
        self.head, self.rules, self.optimizer, self.width = head, rules, optimizer, width
        self.muon_options = dict(muon_options or {})
        if not 0.0 <= float(dropout) <= 1.0:
            raise ValueError(f"dropout probability must lie in [0, 1], got {dropout}")
        self.dropout, self.dropout_seed = float(dropout), int(dropout_seed) & 0xFFFFFFFFFFFFFFFF
        self.drop_counter = torch.zeros(1, dtype=torch.int64, device=dev)  # replays so far
        self.zero_slack = default_zero_slack(self.dropout) if zero_slack is None else float(zero_slack)
        self.table = table
        # without the update: the dense table gradient, one contiguous [2R, N, n]
        # block per hop (grad_hop[t]); grad views it as the table's [2R, T, N, n]
        keep_grad = not apply_update or optimizer == "muon"
        self.grad_hop = torch.zeros((T,) + tuple(table.shape[:1]) + tuple(table.shape[2:]), dtype=table.dtype,
                                    device=dev) if keep_grad else None
        self.grad = self.grad_hop.permute(1, 0, 2, 3) if keep_grad else None
        self.grad_head = None if head is None else tuple(None if t is None else torch.zeros_like(t) for t in head)
        # momentum of the table's matrices, hop by hop as grad_hop, and of the head's weight
        self.momentum = torch.zeros_like(self.grad_hop) if optimizer == "muon" else None
        self.momentum_head = torch.zeros_like(head[0]) if optimizer == "muon" and head is not None else None
        rows = Q * N
        self.rows = rows
        csr = graph.csr
        M = csr[1].numel()
        E = graph.E
        d_o = (csr[0][1:] - csr[0][:-1]).to(torch.int64).clamp_max(self.topk)
        d_i = (csr[4][1:] - csr[4][:-1]).to(torch.int64).clamp_max(self.topk)
        k = d_o + d_i + 1
        k_max, K = (int(k.max().item()), int(k.sum().item())) if E > 0 else (1, 1)
        self.C, self.S, self.F, self.U = capacities(rows, T, self.c1, k_max, K, E, self.zero_slack)
        i64, i32, f32, u8, i16 = torch.int64, torch.int32, torch.float32, torch.uint8, torch.int16
        # inputs
        self.heads = _buf(Q, i64, dev)
        self.tails = _buf(Q, i64, dev)
        self.rels = _buf(Q, i64, dev)
        self.hide = _buf(n_hide, i64, dev)
        self.n_hide = n_hide
        # visibility in CSR order, with the position of every triple on each side
        self.vis = (torch.ones(M, dtype=u8, device=dev), torch.ones(M, dtype=u8, device=dev))
        self.pos = []
        for order in (csr[3], csr[7]):
            p = torch.empty(M, dtype=i64, device=dev)
            p[order.to(i64)] = torch.arange(M, dtype=i64, device=dev)
            self.pos.append(p)
        # hop-1 state
        self.rp0 = torch.arange(rows + 1, dtype=i64, device=dev)
        self.ent0 = _buf(rows, i32, dev)
        self.val0 = torch.ones(rows, dtype=f32, device=dev)
        # per hop: what the backward needs
        self.w = [_buf(rows * self.n, f32, dev) for _ in range(T)]
        self.rp_sel = [_buf(rows + 1, i64, dev) for _ in range(T)]
        self.val_sel = [_buf(self.S[t], f32, dev) for t in range(T)]
        self.src_sel = [_buf(self.S[t], i64, dev) for t in range(T)]
        self.slot_base = [_buf(self.S[t] + 1, i64, dev) for t in range(T)]
        self.entry_count = [_buf(self.S[t], i32, dev) for t in range(T)]
        self.fact_rel = [_buf(self.F[t], i16, dev) for t in range(T)]
        self.fact_pos = [_buf(self.F[t], i32, dev) for t in range(T)]
        self.out_rp = [_buf(rows + 1, i64, dev) for _ in range(T)]
        self.out_ent = [_buf(self.U[t], i32, dev) for t in range(T)]
        self.out_x = [_buf(self.U[t], f32, dev) for t in range(T)]
        self.out_y = [_buf(self.U[t], f32, dev) for t in range(T)]
        self.out_denom = [_buf(rows, f32, dev) for _ in range(T)]
        self.g_y = [_buf(self.U[t], f32, dev) for t in range(T)]
        # transient, shared by the hops
        Smax, Fmax = max(self.S), max(self.F)
        self.ent_sel = _buf(Smax, i32, dev)
        self.entry_info = _buf(L.FL_ENTRY_INFO_INTS * Smax, i32, dev)
        self.use_rank = 0 < r_size <= 16384 and self.topk < L.NO_BUDGET
        self.rel_rank = _buf(rows * 2 * r_size, i16, dev) if self.use_rank else None
        # rows of queries with one relation have one w: they share the first such row's ranks
        self.rank_row = _buf(rows, i32, dev) if self.use_rank else None
        self.chan = torch.arange(N, dtype=torch.int64, device=dev)
        # per hop: rows by descending slot count, the reduction's and the backward's block order
        self.row_order = [_buf(rows, i32, dev) for _ in range(T)]
        self.fact_dst = _buf(Fmax, i32, dev)
        self.fact_val = _buf(Fmax, f32, dev)
        self.grad_sel = _buf(Smax, f32, dev)
        # d loss / d w of the hop being differentiated; with record_grad_w one slice per hop is kept
        self.record_grad_w = bool(record_grad_w)
        self.grad_w = _buf((T if self.record_grad_w else 1) * rows * self.n, f32, dev)
        self.work = _buf(2, i32, dev)  # the expansion's two work queues
        self.status = torch.zeros(1, dtype=i32, device=dev)
        self.ok = torch.ones(1, dtype=f32, device=dev)  # 1 while the status word is clear
        self.scores = _buf(Q, f32, dev)
        self.loss = torch.zeros((), dtype=f32, device=dev)
        # gradient of the batch's table rows: of the logits, or with a head of the hidden states
        self.grad_logits = torch.empty((Q, T, N, width), dtype=f32, device=dev)
        # with a head or rules the backward wants the hops' hidden states and logits again
        self.hidden = None if head is None else [torch.empty((rows, width), dtype=f32, device=dev) for _ in range(T)]
        # (the logits' signs, under a repetition penalty; without rules one buffer serves all hops)
        self.logits = None
        if rules is not None or head is not None:
            each = [torch.empty((rows, self.n), dtype=f32, device=dev) for _ in range(1 if rules is None else T)]
            self.logits = each * T if rules is None else each
        # the queries' histories by row, for all hops and the backward of a run
        self.history = None
        if rules is not None and rules.history is not None and rules.history.shape[1] > 0:
            self.history = torch.empty((rows, rules.history.shape[1]), dtype=torch.int64, device=dev)
        ws = 0
        for t in range(T):
            ws = max(ws, lib().fl_topc_workspace(rows, self.C[t]), lib().fl_hop_workspace(rows, self.S[t]),
                     lib().fl_reduce_workspace(rows, self.F[t]))
        ws = max(ws, lib().fl_hop_backward_workspace(rows, self.n))
        self.ws = _buf(ws, u8, dev)
        self.stats = torch.zeros(4, dtype=i64, device=dev) if stats else None
        self.timer = None  # optional: per hop (start, after expand, after reduce) external events

    # ------------------------------------------------------------------
    def memory_bytes(self) -> int:
        seen, total = set(), 0
        for v in vars(self).values():
            for t in (v if isinstance(v, (list, tuple)) else [v]):
                if isinstance(t, torch.Tensor) and t.is_cuda and t.data_ptr() not in seen:
                    seen.add(t.data_ptr())
                    total += t.numel() * t.element_size()
        return total

    def load(self, heads, tails, rels, hide):
        """Copy one step's inputs (device tensors) into the static buffers."""
        if hide.numel() != self.n_hide or heads.numel() != self.Q:
            raise ValueError("inputs must have the static sizes given at construction")
        self.heads.copy_(heads)
        self.tails.copy_(tails)
        self.rels.copy_(rels)
        self.hide.copy_(hide)

    def grad_w_of(self, t):
        """d loss / d w of hop t as [Q, N, n] (kept for every hop only with record_grad_w)."""
        k = t if self.record_grad_w else 0
        m = self.rows * self.n
        return self.grad_w[k * m:(k + 1) * m].view(self.Q, self.N, self.n)

    def _params(self, t, flags):
        return L.fl_hop_params(self.rows, self.N, self.n, self.r_size, self.graph.E, int(self.topk), int(flags), -1,
                               float(self.eps), int(self.F[t]), self.status.data_ptr(), self.entry_info.data_ptr(),
                               self.vis[0].data_ptr(), self.vis[1].data_ptr(), self.work.data_ptr(),
                               self.rel_rank.data_ptr() if self.use_rank else None,
                               self.rank_row.data_ptr() if self.use_rank else None,
                               self.row_order[t].data_ptr())

    # ------------------------------------------------------------------
    def run(self):
        """Forward, loss, backward and (optionally) the SGD update; returns the loss tensor."""
        for part in self.parts():
            part()
        return self.loss

    def parts(self):
        """The step as T + 1 stream-ordered callables, run in order: the
        forward, the loss and the backward of hop T-1; then the backward of
        hops T-2, ..., 0, one per part; last the update.  After part k < T the
        gradient of hop T-1-k is complete (in grad_hop[T-1-k] when the step
        does not apply the update itself), so a caller can start that hop's
        collective while the later parts run; each part can be captured in a
        CUDA graph of its own."""
        T = self.T
        return [self._part_forward] + [lambda t=t: self._backward_hop(t) for t in reversed(range(T - 1))] + \
            [self._finish]

    def _part_forward(self):
        lb, st, g = lib(), _stream(), self.graph
        rows, N, Q, T = self.rows, self.N, self.Q, self.T
        ws, wsn = _p(self.ws), self.ws.numel()
        if self.dropout > 0:
            self.drop_counter.add_(1)
        if self.head is not None:
            for g_head in self.grad_head:
                if g_head is not None:
                    g_head.zero_()
        # hide the batch's own triples (src/main.py:888), remembering what was there
        hid = [self.pos[k][self.hide] for k in range(2)]
        old = [self.vis[k][hid[k]] for k in range(2)]
        for k in range(2):
            self.vis[k].index_fill_(0, hid[k], 0)
        if self.use_rank:
            # first query with the same relation (argmax returns the first maximum)
            first = (self.rels[:, None] == self.rels[None, :]).to(torch.int32).argmax(dim=1)
            self.rank_row.view(Q, N).copy_(first[:, None] * N + self.chan[None, :])
        self.ent0[:rows].view(Q, N).copy_(self.heads.view(Q, 1).expand(Q, N))
        rp_in, ent_in, val_in = self.rp0, self.ent0, self.val0
        for t in range(T):
            self._weights(t)
            # c1
            if self.c1 is not None:
                check(lb.fl_topc_select(_p(rp_in), _p(ent_in), _p(val_in), rows, self.C[t], self.c1, None,
                                        _p(self.rp_sel[t]), _p(self.ent_sel), _p(self.val_sel[t]),
                                        _p(self.src_sel[t]), self.S[t], _p(self.status), ws, wsn, st), "topc_select")
                rp_s, ent_s, val_s = self.rp_sel[t], self.ent_sel, self.val_sel[t]
            else:
                rp_s, ent_s, val_s = rp_in, ent_in, val_in
                self.rp_sel[t].copy_(rp_in)
                self.val_sel[t][:self.S[t]].copy_(val_in[:self.S[t]])
            if self.use_rank:
                check(lb.fl_relation_rank(_p(self.w[t]), rows, self.r_size, _p(self.rank_row), _p(self.rel_rank), st),
                      "relation_rank")
            params = self._params(t, self.flags)
            check(lb.fl_hop_plan(ctypes.byref(params), _p(rp_s), _p(ent_s), self.S[t], g.ori, g.inv,
                                 _p(self.slot_base[t]), None, ws, wsn, st), "hop_plan")
            # rows by descending slot count: the reduction and the backward take the heaviest first
            if rows <= 16384:
                check(lb.fl_row_order(_p(rp_s), _p(self.slot_base[t]), rows, _p(self.row_order[t]), st), "row_order")
            else:
                rows_facts = self.slot_base[t][rp_s[1:]] - self.slot_base[t][rp_s[:-1]]
                self.row_order[t].copy_(torch.argsort(rows_facts, descending=True, stable=True))
            if self.timer is not None:
                self.timer[t][0].record()
            check(lb.fl_hop_expand(ctypes.byref(params), _p(rp_s), _p(ent_s), _p(val_s), self.S[t], _p(self.w[t]),
                                   g.ori, g.inv, None, None, None, None, _p(self.slot_base[t]), _p(self.fact_dst),
                                   _p(self.fact_val), _p(self.fact_rel[t]), None, _p(self.entry_count[t]), st),
                  "hop_expand")
            if self.timer is not None and len(self.timer[t]) > 2:
                self.timer[t][1].record()
            check(lb.fl_row_reduce(_p(rp_s), rows, g.E, _p(self.slot_base[t]), _p(self.entry_count[t]),
                                   _p(self.fact_dst), _p(self.fact_val), self.F[t], _p(self.fact_pos[t]),
                                   ctypes.c_float(self.eps), _p(self.out_rp[t]), _p(self.out_ent[t]),
                                   _p(self.out_x[t]), _p(self.out_y[t]), _p(self.out_denom[t]), _p(self.status),
                                   _p(self.row_order[t]), ws, wsn, self._drop(t), st), "row_reduce")
            if self.timer is not None:
                self.timer[t][-1].record()
            if self.stats is not None:
                check(lb.fl_hop_stats(_p(rp_s), rows, _p(ent_s), self.S[t], g.ori, g.inv, _p(self.entry_count[t]),
                                      _p(self.out_rp[t]), 0, _p(self.stats), st), "hop_stats")
            rp_in, ent_in, val_in = self.out_rp[t], self.out_ent[t], self.out_y[t]
        # the backward reads no visibility: restore what the batch hid
        for k in range(2):
            self.vis[k].index_put_((hid[k],), old[k])
        # readout + loss (src/utils.py:36-47)
        check(lb.fl_readout(_p(rp_in), _p(ent_in), _p(val_in), N, _p(self.tails), Q, _p(self.scores), st), "readout")
        score = self.scores[:Q]
        self.loss.copy_(-torch.mean(torch.log(torch.clamp_min(score, self.thr))))
        g_score = torch.where(score > self.thr, -1.0 / (Q * torch.clamp_min(score, self.thr)),
                              torch.zeros_like(score))
        check(lb.fl_readout_backward(_p(rp_in), _p(ent_in), N, _p(self.tails), Q, _p(g_score), _p(self.g_y[T - 1]),
                                     self.U[T - 1], _p(self.out_rp[T - 1][rows:]), self._drop(T - 1), st),
              "readout_backward")
        # a forward that overflowed a buffer updates nothing: its gradient is scaled by 0
        self.ok.copy_(self.status == 0)
        self._backward_hop(T - 1)

    def _weights(self, t):
        """Hop t's attention rows [Q, N, n] into w[t]: gathered contiguous, through the head, then softmax."""
        Q, N, rows, n = self.Q, self.N, self.rows, self.n
        w = self.w[t][:rows * n]
        if self.head is None and self.rules is None:
            w.view(Q, N, n).copy_(torch.softmax(self.table[:, t].index_select(0, self.rels), dim=-1))
            return
        kept = self.hidden[t] if self.head is not None else self.logits[t]
        torch.index_select(self.table[:, t], 0, self.rels, out=kept.view(Q, N, self.width))
        if self.head is not None:
            ops.linear_forward(kept, self.head[0], self.head[1], out=self.logits[t])
        if self.history is not None and t == 0:
            self.history.view(Q, N, -1).copy_(self.rules.history[:, None, :].expand(-1, N, -1))
        kw = {} if self.rules is None else self.rules.rows(t, N, self.history)
        ops.relation_weights(self.logits[t], out=w.view(rows, n), **kw)

    def _weights_backward(self, t):
        """From grad_w to the gradient of hop t's table rows (and of the head)."""
        Q, N, rows, n = self.Q, self.N, self.rows, self.n
        wt, gw = self.w[t][:rows * n].view(Q, N, n), self.grad_w_of(t)
        if self.head is None and self.rules is None:
            # softmax backward, d logits = w * (g - sum(g * w)): torch's own kernel
            dz = torch._softmax_backward_data(gw, wt, -1, torch.float32)
        else:
            dz, _ = ops.relation_weights_backward(wt.view(rows, n), gw.view(rows, n), self.logits[t],
                                                  history=self.history,
                                                  repetition=1.0 if self.rules is None else self.rules.repetition)
            dz = dz.view(Q, N, n)
        if self.head is None:
            torch.mul(dz, self.ok, out=self.grad_logits[:, t])
            return
        dz = dz.view(rows, n) * self.ok
        dx, dw, db = ops.linear_backward(self.hidden[t], self.head[0], None, dz,
                                         want=(True, True, self.head[1] is not None))
        self.grad_logits[:, t].copy_(dx.view(Q, N, self.width))
        self.grad_head[0].add_(dw)
        if db is not None:
            self.grad_head[1].add_(db)

    def _backward_hop(self, t):
        """Backward of hop t; g_y[t] arrived through hop t's dropout (the same
        keep bits and scale), applied where it is written."""
        lb, st = lib(), _stream()
        rows, N, Q = self.rows, self.N, self.Q
        ws, wsn = _p(self.ws), self.ws.numel()
        params = self._params(t, self.flags)
        check(lb.fl_hop_backward(ctypes.byref(params), _p(self.rp_sel[t]), _p(self.val_sel[t]), self.S[t],
                                 _p(self.w[t]), _p(self.slot_base[t]), _p(self.entry_count[t]),
                                 _p(self.fact_pos[t]), _p(self.fact_rel[t]), None, _p(self.out_rp[t]),
                                 _p(self.out_x[t]), _p(self.out_denom[t]), _p(self.g_y[t]), _p(self.grad_sel),
                                 _p(self.grad_w_of(t)), ws, wsn, st), "hop_backward")
        if t > 0:
            src = self.src_sel[t] if self.c1 is not None else None
            if src is not None:
                check(lb.fl_scatter_grad(_p(self.grad_sel), _p(src), self.S[t], _p(self.rp_sel[t][rows:]),
                                         _p(self.g_y[t - 1]), self.U[t - 1], _p(self.out_rp[t - 1][rows:]),
                                         self._drop(t - 1), st),
                      "scatter_grad")
            else:
                self.g_y[t - 1][:self.S[t]].copy_(self.grad_sel[:self.S[t]])
                if self.dropout > 0:
                    self._dropout(self.g_y[t - 1], t - 1, st)
        self._weights_backward(t)
        if self.grad_hop is not None:
            # hop t's dense table gradient, complete once this part has run
            self.grad_hop[t].zero_()
            self.grad_hop[t].index_add_(0, self.rels, self.grad_logits[:, t])

    def _finish(self):
        if self.apply_update:
            self.update()

    def update(self):
        """The optimizer's step from this run's gradients (in place; what parts() ends with under apply_update)."""
        if self.optimizer == "sgd":
            if self.grad_hop is None:
                # SGD on the rows of the batch's relations only: no dense gradient
                self.table.index_add_(0, self.rels, self.grad_logits, alpha=-self.lr)
            else:
                self.table.sub_(self.grad, alpha=self.lr)
        else:
            # matrices [2R, n or H] of every hop and channel: strided views of the table
            muon.muon_update_(self.table.permute(1, 2, 0, 3), self.grad_hop.permute(0, 2, 1, 3),
                              self.momentum.permute(0, 2, 1, 3), lr=self.lr, gate=self.ok, **self.muon_options)
        if self.head is not None:
            weight, bias = self.head
            if self.optimizer == "sgd":
                weight.sub_(self.grad_head[0], alpha=self.lr)
            else:
                muon.muon_update_(weight, self.grad_head[0], self.momentum_head, lr=self.lr, gate=self.ok,
                                  **self.muon_options)
            if bias is not None:
                bias.addcmul_(self.grad_head[1], self.ok, value=-self.lr)

    def _drop(self, t):
        """fl_dropout of hop t for the kernels that write its values or their gradient (None: no dropout)."""
        if self.dropout <= 0:
            return None
        return ctypes.byref(L.fl_dropout(self.dropout, self.dropout_seed, self.drop_counter.data_ptr(), t))

    def _dropout(self, x, t, st):
        check(lib().fl_value_dropout(_p(x), _p(x), self.U[t], _p(self.out_rp[t][self.rows:]),
                                     ctypes.c_double(self.dropout), self.dropout_seed, _p(self.drop_counter), t, st),
              "value_dropout")

    def check(self):
        """Raise if any hop ran out of its buffers (one host read), or a wait of the head's or the update's products
        ran out (the step's results hold NaN)."""
        if int(self.status.item()) & L.FL_STATUS_SLOT_OVERFLOW:
            raise RuntimeError("a hop exceeded its static capacity")
        if self.head is not None or self.optimizer == "muon":
            with torch.cuda.device(self.dev):
                if ops.gemm_fault():
                    raise RuntimeError("a wait of a matrix product ran out")

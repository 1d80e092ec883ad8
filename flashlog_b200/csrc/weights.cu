// weights.cu -- the hops' weights from the relation logits, and the gradient:
//
//   u = z / theta (z > 0) or z * theta (z <= 0) for operators in the row's
//       history, z otherwise;  u -= frequency * count + presence * [count > 0]
//   u += bias;  u = -inf where the mask row of the row's state forbids it
//   w = softmax(u / tau), all 0 for a row with nothing left
//
//   du = w (g - sum g w) / tau;  dz = du * (theta, 1 / theta or 1);  dbias = sum of du
//
// One pass over the row: its values stay in registers, and one joint reduction
// gives the maximum and the sum, each thread having summed relative to its own
// maximum.  A row wider than one block's registers is spread over a cluster of
// up to eight blocks, which send each other their (maximum, sum) pairs.  The operation is bound by HBM: a value is read once and written once.
//
// The history's counts live in shared memory next to one "seen" bit per
// column; a warp's 32 columns share one word of bits, so columns without
// history cost nothing per column.  Counts are cleared by walking the
// history again, not by clearing the row.
#include "gemm.cuh"

namespace fl {

namespace {

struct WeightsArgs {
    const void *logits;
    int64_t ld;
    const void *bias;        // [n] (bias_ld 0) or [rows, n], or NULL
    int64_t bias_ld;
    const uint8_t *mask;     // [n_states, n] or NULL
    int64_t mask_ld, n_states;
    const int64_t *states;   // [rows], or NULL: row r has state min(r, n_states - 1)
    const int64_t *history;  // [rows, hist] or NULL; entries outside [0, n) do not count
    int64_t hist_ld, hist;
    int64_t rows, n;
    float theta, frequency, presence, inv_tau;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t smem_u32(const void *p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// The blocks of a cluster exchange one 8-byte value each per row: every block
// sends its own to all (itself too) with a store that counts on the receiver's
// barrier, so no fence has to wait for the rows written to global memory.  Two
// slots alternate: a block can only send for row r + 2 after it has received
// everything for row r + 1, which the others send after reading row r.
struct Exchange {
    uint64_t bar[2];
    float2 slot[2][8];
};
constexpr uint64_t kWaitLimitNs = 4000000000ull;

__device__ __forceinline__ void exchange_init(Exchange &x) {
    if (threadIdx.x < 2)
        asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;\n fence.mbarrier_init.release.cluster;" ::"r"(
                         smem_u32(&x.bar[threadIdx.x])) : "memory");
    __syncthreads();
    cluster_barrier();
}
// Called by warp 0 after the block's value is known; `round` counts rows.
__device__ __forceinline__ void exchange_send(Exchange &x, int flip, uint32_t rank, uint32_t ranks, float a, float b) {
    const int lane = threadIdx.x & 31;
    if (lane == 0)
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(&x.bar[flip])),
                     "r"(ranks * 8) : "memory");
    __syncwarp();
    if (lane < static_cast<int>(ranks)) {
        const uint64_t v = static_cast<uint64_t>(__float_as_uint(a)) | (static_cast<uint64_t>(__float_as_uint(b)) << 32);
        asm volatile(
            "{\n .reg .b32 d, m;\n mapa.shared::cluster.u32 d, %0, %2;\n mapa.shared::cluster.u32 m, %1, %2;\n"
            " st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [d], %3, [m];\n}" ::"r"(
                smem_u32(&x.slot[flip][rank])), "r"(smem_u32(&x.bar[flip])), "r"(lane), "l"(v) : "memory");
    }
}
// All blocks' values, lane r holding block r's.  A wait that runs out (which no
// healthy run does) gives NaN.
__device__ __forceinline__ float2 exchange_receive(Exchange &x, int flip, uint32_t parity, uint32_t ranks) {
    const int lane = threadIdx.x & 31;
    const uint32_t bar = smem_u32(&x.bar[flip]);
    uint64_t start = 0, now = 0;
    for (int i = 0;; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
            " selp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) break;
        if ((i & 63) == 63) {
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
            if (start == 0) start = now;
            if (now - start > kWaitLimitNs) {
                const float nan = __int_as_float(0x7fc00000);
                return make_float2(nan, nan);
            }
        }
    }
    return lane < static_cast<int>(ranks) ? x.slot[flip][lane] : make_float2(-INFINITY, 0.0f);
}

// A thread's columns of its block are i * THREADS + threadIdx.x.  The seen bits
// of a warp's 32 columns form one word; the words of a warp lie together, so
// one load and a ballot tell a warp which of its VPT words are not empty.
template <int THREADS, int VPT>
__device__ __forceinline__ int word_of(int c) {  // column of the block -> word
    const int i = c / THREADS, w = (c % THREADS) >> 5;
    return w * VPT + i;
}

// History counts of one row for the block's columns: add (or clear).
template <int THREADS, int VPT, bool ADD>
__device__ __forceinline__ void history_pass(const WeightsArgs &a, int64_t row, int c0, unsigned *seen,
                                             unsigned *count) {
    const int64_t *h = a.history + row * a.hist_ld;
    const int hist = static_cast<int>(a.hist);
    for (int j = threadIdx.x; j < hist; j += THREADS) {
        const int64_t v = h[j];
        const int64_t c = v - c0;
        if (v < 0 || v >= a.n || c < 0 || c >= THREADS * VPT) continue;
        const int k = static_cast<int>(c);
        if (ADD) {
            atomicAdd(count + k, 1u);
            atomicOr(seen + word_of<THREADS, VPT>(k), 1u << (k & 31));
        } else {
            count[k] = 0u;
            seen[word_of<THREADS, VPT>(k)] = 0u;
        }
    }
}

// exp((from - to) * k / log2 e): the rescaling of a part summed relative to
// `from`.  Equal (both -inf too): nothing to do.
__device__ __forceinline__ float rescale(float from, float to, float k) {
    return from == to ? 1.0f : exp2f((from - to) * k);
}

// 1024 threads per SM with up to 64 registers each: enough rows in flight to
// cover the loads' latency while other rows are in their reductions.
template <typename T, int THREADS, int VPT, bool CL>
__global__ __launch_bounds__(THREADS, 1024 / THREADS) void weights_forward_kernel(const WeightsArgs a, float *out) {
    extern __shared__ unsigned dyn[];
    constexpr int kChunk = THREADS * VPT, kWarps = THREADS / 32;
    unsigned *seen = dyn, *count = dyn + kChunk / 32;
    __shared__ float warp_m[2][kWarps], warp_s[2][kWarps];
    __shared__ Exchange ex;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rank = CL ? cluster_rank() : 0, ranks = CL ? cluster_size() : 1;
    const int c0 = static_cast<int>(rank) * kChunk;
    const int left = static_cast<int>(a.n) - c0 - tid;  // the thread's column i exists iff i * THREADS < left
    const bool hist = a.hist > 0;
    const float k = a.inv_tau * 1.4426950408889634f;
    if (hist)
        for (int i = tid; i < kChunk / 32 + kChunk; i += THREADS) dyn[i] = 0u;
    if (CL) exchange_init(ex);
    __syncthreads();
    int flip = 0;
    uint32_t parity = 0;
    for (int64_t row = blockIdx.x / ranks; row < a.rows; row += gridDim.x / ranks) {
        // all of the row's loads first: they are in flight together
        const T *z = static_cast<const T *>(a.logits) + row * a.ld + c0 + tid;
        T raw[VPT];
#pragma unroll
        for (int i = 0; i < VPT; ++i) raw[i] = i * THREADS < left ? z[i * THREADS] : from_f32<T>(0.0f);
        unsigned allowed = 0u;
        if (a.mask == nullptr) {
#pragma unroll
            for (int i = 0; i < VPT; ++i) allowed |= (i * THREADS < left ? 1u : 0u) << i;
        } else {
            const int64_t state = a.states != nullptr ? a.states[row] : (row < a.n_states ? row : a.n_states - 1);
            if (state >= 0 && state < a.n_states) {
                const uint8_t *mask = a.mask + state * a.mask_ld + c0 + tid;
                uint8_t ok[VPT];
#pragma unroll
                for (int i = 0; i < VPT; ++i) ok[i] = i * THREADS < left ? mask[i * THREADS] : 0;
#pragma unroll
                for (int i = 0; i < VPT; ++i) allowed |= (ok[i] != 0 ? 1u : 0u) << i;
            }
        }
        float u[VPT], m = -INFINITY;
        if (a.bias != nullptr) {
            const T *bias = static_cast<const T *>(a.bias) + row * a.bias_ld + c0 + tid;
#pragma unroll
            for (int i = 0; i < VPT; ++i) u[i] = i * THREADS < left ? to_f32<T>(bias[i * THREADS]) : 0.0f;
        } else {
#pragma unroll
            for (int i = 0; i < VPT; ++i) u[i] = 0.0f;
        }
        unsigned word = 0u, any = 0u;
        if (hist) {
            history_pass<THREADS, VPT, true>(a, row, c0, seen, count);
            __syncthreads();
            word = lane < VPT ? seen[warp * VPT + lane] : 0u;
            any = __ballot_sync(kFull, word != 0u);
        }
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            float v = to_f32<T>(raw[i]);
            if ((any >> i) & 1u) {  // the same for the whole warp
                if ((__shfl_sync(kFull, word, i) >> lane) & 1u) {
                    v = v > 0.0f ? v / a.theta : v * a.theta;
                    v = v - a.frequency * static_cast<float>(count[i * THREADS + tid]) - a.presence;
                }
            }
            u[i] = (allowed >> i) & 1u ? v + u[i] : -INFINITY;
            m = fmaxf(m, u[i]);
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            // -inf contributes nothing even where it is also the maximum; a NaN stays one
            u[i] = u[i] == -INFINITY ? 0.0f : exp2f((u[i] - m) * k);
            s += u[i];
        }
        const float wm = warp_max(m);
        const float ws = warp_sum(s * rescale(m, wm, k));
        float top = wm, total = ws;
        if (kWarps > 1) {
            if (lane == 0) {
                warp_m[flip][warp] = wm;
                warp_s[flip][warp] = ws;
            }
            __syncthreads();
            const float bm = lane < kWarps ? warp_m[flip][lane] : -INFINITY;
            const float bs = lane < kWarps ? warp_s[flip][lane] : 0.0f;
            top = warp_max(bm);
            total = warp_sum(bs * rescale(bm, top, k));
        }
        if (CL) {
            if (warp == 0) exchange_send(ex, flip, rank, ranks, top, total);
            const float2 b = exchange_receive(ex, flip, parity, ranks);
            top = warp_max(b.x);
            total = warp_sum(b.y * rescale(b.x, top, k));
        }
        const float f = total == 0.0f ? 0.0f : rescale(m, top, k) / total;
        float *w = out + row * a.n + c0 + tid;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            if (i * THREADS < left) w[i * THREADS] = u[i] * f;
        if (hist) {
            if (kWarps == 1) __syncwarp();  // otherwise the reduction's barrier lies behind every read of the counts
            history_pass<THREADS, VPT, false>(a, row, c0, seen, count);
            __syncthreads();
        }
        flip ^= 1;
        if (flip == 0) parity ^= 1;
    }
    if (CL) cluster_barrier();  // no block leaves while another may write to its slots
}

// dbias_partial: [blocks / ranks, n] sums of du over the rows each cluster took (a fixed set), or NULL;
// du: [rows, n] for a bias of the logits' shape, or NULL.
template <typename T, int THREADS, int VPT, bool CL>
__global__ __launch_bounds__(THREADS, 1024 / THREADS) void weights_backward_kernel(const WeightsArgs a, const float *w,
                                                                                   const float *g, int64_t ld_g, T *dz,
                                                                                   T *du, float *dbias_partial) {
    extern __shared__ unsigned dyn[];
    constexpr int kChunk = THREADS * VPT, kWarps = THREADS / 32;
    unsigned *seen = dyn, *count = dyn + kChunk / 32;
    __shared__ float warp_s[2][kWarps];
    __shared__ Exchange ex;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rank = CL ? cluster_rank() : 0, ranks = CL ? cluster_size() : 1;
    const int c0 = static_cast<int>(rank) * kChunk;
    const int left = static_cast<int>(a.n) - c0 - tid;
    const bool hist = a.hist > 0 && a.theta != 1.0f && dz != nullptr;  // only the repetition penalty has a slope
    if (hist)
        for (int i = tid; i < kChunk / 32 + kChunk; i += THREADS) dyn[i] = 0u;
    if (CL) exchange_init(ex);
    __syncthreads();
    float acc[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) acc[i] = 0.0f;
    int flip = 0;
    uint32_t parity = 0;
    for (int64_t row = blockIdx.x / ranks; row < a.rows; row += gridDim.x / ranks) {
        const float *pw = w + row * a.n + c0 + tid, *pg = g + row * ld_g + c0 + tid;
        float p[VPT], q[VPT], s = 0.0f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) p[i] = i * THREADS < left ? pw[i * THREADS] : 0.0f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) q[i] = i * THREADS < left ? pg[i * THREADS] : 0.0f;
        unsigned word = 0u, any = 0u;
        if (hist) {
            history_pass<THREADS, VPT, true>(a, row, c0, seen, count);
            __syncthreads();
            word = lane < VPT ? seen[warp * VPT + lane] : 0u;
            any = __ballot_sync(kFull, word != 0u);
        }
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            if (p[i] == 0.0f) q[i] = 0.0f;  // a weight of 0 passes nothing on, whatever the gradient there
            s = fmaf(p[i], q[i], s);
        }
        float dot = warp_sum(s);
        if (kWarps > 1) {
            if (lane == 0) warp_s[flip][warp] = dot;
            __syncthreads();
            dot = warp_sum(lane < kWarps ? warp_s[flip][lane] : 0.0f);
        }
        if (CL) {
            if (warp == 0) exchange_send(ex, flip, rank, ranks, dot, 0.0f);
            const float2 b = exchange_receive(ex, flip, parity, ranks);
            dot = warp_sum(lane < static_cast<int>(ranks) ? b.x : 0.0f);
        }
        const int64_t at = row * a.n + c0 + tid;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const float d = p[i] == 0.0f ? 0.0f : p[i] * (q[i] - dot) * a.inv_tau;
            p[i] = d;
            acc[i] += d;
        }
        if (du != nullptr) {
#pragma unroll
            for (int i = 0; i < VPT; ++i)
                if (i * THREADS < left) du[at + i * THREADS] = from_f32<T>(p[i]);
        }
        if (dz != nullptr) {
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                if ((any >> i) & 1u) {
                    if (((__shfl_sync(kFull, word, i) >> lane) & 1u) && i * THREADS < left) {
                        const T *z = static_cast<const T *>(a.logits) + row * a.ld + c0 + tid;
                        p[i] = to_f32<T>(z[i * THREADS]) > 0.0f ? p[i] / a.theta : p[i] * a.theta;
                    }
                }
                if (i * THREADS < left) dz[at + i * THREADS] = from_f32<T>(p[i]);
            }
        }
        if (hist) {
            // the seen words were read before the reduction's barrier
            if (kWarps == 1) __syncwarp();
            history_pass<THREADS, VPT, false>(a, row, c0, seen, count);
            __syncthreads();
        }
        flip ^= 1;
        if (flip == 0) parity ^= 1;
    }
    if (dbias_partial != nullptr) {
        float *po = dbias_partial + (blockIdx.x / ranks) * a.n + c0 + tid;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            if (i * THREADS < left) po[i * THREADS] = acc[i];
    }
    if (CL) cluster_barrier();
}

// Column sums of [parts, n] in a fixed order: 32 columns x 32 groups of parts per block.
template <typename T>
__global__ void column_sum_kernel(const float *partial, int64_t parts, int64_t n, T *out) {
    __shared__ float part[32][33];
    const int64_t c = blockIdx.x * int64_t(32) + threadIdx.x;
    float s = 0.0f;
    if (c < n)
        for (int64_t p = threadIdx.y; p < parts; p += 32) s += partial[p * n + c];
    part[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && c < n) {
#pragma unroll
        for (int i = 1; i < 32; ++i) s += part[i][threadIdx.x];
        out[c] = from_f32<T>(s);
    }
}

// How a row is laid over threads: the narrowest form that holds it.  The
// counts of the widest (8192 columns) take 33 KB of shared memory.
struct Layout {
    int threads, vpt, ranks;
    int64_t clusters;  // rows in flight
};

constexpr int64_t kMaxColumns = 65536;

Layout layout(int64_t rows, int64_t n) {
    const int sms = fl_device_sm_count() > 0 ? fl_device_sm_count() : 148;
    Layout l{512, 16, 1, 0};
    if (n <= 128) l = {32, 4, 1, 0};
    else if (n <= 512) l = {64, 8, 1, 0};
    else if (n <= 1024) l = {128, 8, 1, 0};
    else if (n <= 2048) l = {256, 8, 1, 0};
    else if (n <= 4096) l = {512, 8, 1, 0};
    else {
        // few rows: eight narrow blocks per row put more SMs to work on each
        const int vpt = rows * 4 < sms ? 8 : 16;
        while (l.ranks < 8 && static_cast<int64_t>(l.ranks) * 512 * vpt < n) l.ranks *= 2;
        l.vpt = static_cast<int64_t>(l.ranks) * 512 * vpt >= n ? vpt : 16;
    }
    const int64_t fit = static_cast<int64_t>(sms) * (1024 / l.threads) / l.ranks;  // rows in flight
    l.clusters = rows < fit ? rows : fit;
    return l;
}

template <typename K, typename... Args>
int launch_rows(K kernel, const Layout &l, size_t smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(l.clusters * l.ranks));
    cfg.blockDim = dim3(l.threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = l.ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = l.ranks > 1 ? 1 : 0;
    note_launch();
    FL_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    return check_launch("relation weights");
}

size_t history_smem(const Layout &l, bool hist) {
    const size_t chunk = static_cast<size_t>(l.threads) * l.vpt;
    return hist ? (chunk / 32 + chunk) * sizeof(unsigned) : 0;
}

#define FL_LAYOUTS(F)                                                             \
    if (l.threads == 32) F(32, 4, false);                                         \
    else if (l.threads == 64) F(64, 8, false);                                    \
    else if (l.threads == 128) F(128, 8, false);                                  \
    else if (l.threads == 256) F(256, 8, false);                                  \
    else if (l.ranks == 1 && l.vpt == 8) F(512, 8, false);                        \
    else if (l.ranks == 1) F(512, 16, false);                                     \
    else if (l.vpt == 8) F(512, 8, true);                                         \
    else F(512, 16, true);

template <typename T>
int forward_t(const WeightsArgs &a, float *w, cudaStream_t st) {
    const Layout l = layout(a.rows, a.n);
    const size_t smem = history_smem(l, a.hist > 0);
    int rc = FL_OK;
#define F(TH, V, C) rc = launch_rows(weights_forward_kernel<T, TH, V, C>, l, smem, st, a, w)
    FL_LAYOUTS(F)
#undef F
    return rc;
}

template <typename T>
int backward_t(const WeightsArgs &a, const float *w, const float *g, int64_t ld_g, T *dz, T *du, T *dbias, Carve &ws,
               cudaStream_t st) {
    const Layout l = layout(a.rows, a.n);
    float *partial = nullptr;
    if (dbias != nullptr) {
        partial = ws.take<float>(l.clusters * a.n);
        FL_REQUIRE(partial != nullptr, "relation weights: workspace too small");
    }
    const size_t smem = history_smem(l, a.hist > 0 && a.theta != 1.0f && dz != nullptr);
    int rc = FL_OK;
#define F(TH, V, C) \
    rc = launch_rows(weights_backward_kernel<T, TH, V, C>, l, smem, st, a, w, g, ld_g, dz, du, partial)
    FL_LAYOUTS(F)
#undef F
    if (rc || dbias == nullptr) return rc;
    launch(column_sum_kernel<T>, static_cast<unsigned>((a.n + 31) / 32), dim3(32, 32), 0, st, partial, l.clusters, a.n,
           dbias);
    return check_launch("relation weights bias");
}

int weights_args(const fl_weights *p, WeightsArgs *a) {
    FL_REQUIRE(p != nullptr, "relation weights: null parameters");
    FL_REQUIRE(p->dtype == FL_F32 || p->dtype == FL_F16 || p->dtype == FL_BF16, "relation weights: bad dtype %d", p->dtype);
    FL_REQUIRE(p->rows >= 0 && p->n > 0 && p->n <= kMaxColumns, "relation weights: need 1 to %lld columns",
               static_cast<long long>(kMaxColumns));
    FL_REQUIRE(p->rows == 0 || (p->logits != nullptr && p->ld >= p->n), "relation weights: bad logits");
    FL_REQUIRE(p->tau > 0.0 && p->repetition > 0.0, "relation weights: tau and repetition must be positive");
    FL_REQUIRE(p->mask == nullptr || (p->n_states > 0 && (p->n_states == 1 || p->mask_ld >= p->n)),
               "relation weights: bad mask");
    FL_REQUIRE(p->hist >= 0 && (p->hist == 0 || p->history != nullptr), "relation weights: bad history");
    *a = WeightsArgs{p->logits, p->ld, p->bias, p->bias_ld, static_cast<const uint8_t *>(p->mask), p->mask_ld,
                     p->mask != nullptr ? p->n_states : 0, p->states, p->history, p->hist_ld, p->hist, p->rows, p->n,
                     static_cast<float>(p->repetition), static_cast<float>(p->frequency),
                     static_cast<float>(p->presence), static_cast<float>(1.0 / p->tau)};
    return FL_OK;
}

}  // namespace
}  // namespace fl

using namespace fl;

extern "C" {

int fl_relation_weights(const fl_weights *p, float *w, fl_stream_t stream) {
    WeightsArgs a;
    int rc = weights_args(p, &a);
    if (rc) return rc;
    if (p->rows == 0) return FL_OK;
    FL_REQUIRE(w != nullptr, "relation weights: null output");
    cudaStream_t st = as_stream(stream);
    if (p->dtype == FL_F32) return forward_t<float>(a, w, st);
    if (p->dtype == FL_F16) return forward_t<__half>(a, w, st);
    return forward_t<__nv_bfloat16>(a, w, st);
}

size_t fl_relation_weights_workspace(int64_t rows, int64_t n) {
    if (rows <= 0 || n <= 0 || n > kMaxColumns) return 0;
    return carve_bytes<float>(layout(rows, n).clusters * n);
}

int fl_relation_weights_backward(const fl_weights *p, const float *w, const float *g, int64_t ld_g, void *dlogits,
                                 void *dbias, void *ws, size_t ws_bytes, fl_stream_t stream) {
    WeightsArgs a;
    int rc = weights_args(p, &a);
    if (rc) return rc;
    cudaStream_t st = as_stream(stream);
    const size_t es = p->dtype == FL_F32 ? 4 : 2;
    if (p->rows == 0) {
        if (dbias != nullptr && p->bias_ld == 0) FL_CUDA(cudaMemsetAsync(dbias, 0, p->n * es, st));
        return FL_OK;
    }
    FL_REQUIRE(w != nullptr && g != nullptr && ld_g >= 0, "relation weights: null gradient");
    Carve carve(ws, ws_bytes);
    void *du = p->bias_ld != 0 ? dbias : nullptr, *db = p->bias_ld == 0 ? dbias : nullptr;
    if (p->dtype == FL_F32)
        return backward_t<float>(a, w, g, ld_g, static_cast<float *>(dlogits), static_cast<float *>(du),
                                 static_cast<float *>(db), carve, st);
    if (p->dtype == FL_F16)
        return backward_t<__half>(a, w, g, ld_g, static_cast<__half *>(dlogits), static_cast<__half *>(du),
                                  static_cast<__half *>(db), carve, st);
    return backward_t<__nv_bfloat16>(a, w, g, ld_g, static_cast<__nv_bfloat16 *>(dlogits),
                                     static_cast<__nv_bfloat16 *>(du), static_cast<__nv_bfloat16 *>(db), carve, st);
}

}  // extern "C"

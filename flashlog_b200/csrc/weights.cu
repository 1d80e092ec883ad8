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
// maximum.  A few long rows are spread over a cluster of eight blocks each,
// which send each other their (maximum, sum) pairs; the widest rows take two
// passes.  A value has to be read once and written once: 382 MB and 58 us for
// 1536 x 29649 with masks and histories of 200, which take 118 us (the two-pass
// form 134 us): a row's barriers and its 40 instructions a value are what the
// copies do not cover.
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
    float theta, inv_theta, frequency, presence, inv_tau;
    float k;                 // log2 e / tau, rounded once: w is a power of 2 of (u - max) k.  (From 1 / tau and
                             // log2 e, each rounded, the weights were off by 2.0e-7 at tau = 0.9, now by 0.8e-7;
                             // a softmax by divisions and expf is off by 1.6e-7.)
};

// A thread's columns of its block are i * THREADS + threadIdx.x.  The seen bits
// of a warp's 32 columns form one word; the words of a warp lie together, so
// one load and a ballot tell a warp which of its VPT words are not empty.
template <int THREADS, int VPT>
__device__ __forceinline__ int word_of(int c) {  // column of the block -> word
    const int i = c / THREADS, w = (c % THREADS) >> 5;
    return w * VPT + i;
}

// History counts of a row for the block's columns.  `token` is the thread's
// first entry, loaded a row ahead; longer histories are read here.  Three
// buffers rotate: between two of the row loop's barriers the counts of the next
// row are added while those of the row before are cleared, by walking its
// history again.
template <int THREADS, int VPT, bool ADD>
__device__ __forceinline__ void history_entry(const WeightsArgs &a, int64_t v, unsigned *buf) {
    if (v < 0 || v >= a.n) return;
    const int k = static_cast<int>(v);
    unsigned *seen = buf + word_of<THREADS, VPT>(k), *count = buf + THREADS * VPT / 32 + k;
    if (ADD) {
        atomicAdd(count, 1u);
        atomicOr(seen, 1u << (k & 31));
    } else {
        *count = 0u;
        *seen = 0u;
    }
}
template <int THREADS, int VPT, bool ADD>
__device__ __forceinline__ void history_pass(const WeightsArgs &a, int64_t row, int64_t token, unsigned *buf) {
    history_entry<THREADS, VPT, ADD>(a, token, buf);
    const int64_t *h = a.history + row * a.hist_ld;
    for (int64_t j0 = threadIdx.x + THREADS; j0 < a.hist; j0 += 8 * THREADS) {
        int64_t v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = j0 + q * THREADS < a.hist ? h[j0 + q * THREADS] : -1;
#pragma unroll
        for (int q = 0; q < 8; ++q) history_entry<THREADS, VPT, ADD>(a, v[q], buf);
    }
}
__device__ __forceinline__ int64_t first_token(const WeightsArgs &a, int64_t row) {
    return static_cast<int64_t>(threadIdx.x) < a.hist ? a.history[row * a.hist_ld + threadIdx.x] : -1;
}
__device__ __forceinline__ int64_t state_of(const WeightsArgs &a, int64_t row) {
    return a.states != nullptr ? a.states[row] : (row < a.n_states ? row : a.n_states - 1);
}

// A logit of an operator that is `count` times in the row's history.  (A division
// in the place of the rounded 1 / theta would save half a step of the logit and
// cost 1536 x 29649 16 of 136 us: its code keeps registers from the row.)
__device__ __forceinline__ float penalised(const WeightsArgs &a, float v, unsigned count) {
    v *= v > 0.0f ? a.inv_theta : a.theta;
    return v - a.frequency * static_cast<float>(count) - a.presence;
}
// 2^x, to 2^-22, a fourth of what the exponent's own rounding moves a weight of
// e^-16; results below 2^-126 are 0
__device__ __forceinline__ float power2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// exp((from - to) * k / log2 e): the rescaling of a part summed relative to
// `from`.  Equal (both -inf too): nothing to do.
__device__ __forceinline__ float rescale(float from, float to, float k) {
    return from == to ? 1.0f : power2((from - to) * k);
}
// Blocks per SM to compile for: 16 values a thread with their prefetched
// successors want about 90 registers (640 threads per SM; with 768, 4608 x 1645
// took 16.8 us instead of 15.7).
constexpr int kBackwardThreads = 512;
constexpr int min_blocks(int threads, int vpt) {
    const int b = (vpt > 8 ? 640 : 1024) / threads;
    return b > 24 ? 24 : b;
}

// The backward's sixteen values, gradients, their successors and the sums for
// the bias want 110: with 768 threads per SM it spilled, and 4608 x 1645 took 41
// us instead of 25 (30 instead of 15 without history and bias).
constexpr int min_blocks_backward(int threads, int vpt) {
    return vpt > 8 ? kBackwardThreads / threads : min_blocks(threads, vpt);
}

// What a thread holds of a row before its turn.
template <typename T, int VPT>
struct RowInputs {
    T logit[VPT];
    uint8_t ok[VPT];
    int64_t token;
};
template <typename T, int THREADS, int VPT>
__device__ __forceinline__ void load_inputs(const WeightsArgs &a, int64_t row, int64_t state, int left,
                                            RowInputs<T, VPT> &in) {
    const T *z = static_cast<const T *>(a.logits) + row * a.ld + threadIdx.x;
#pragma unroll
    for (int i = 0; i < VPT; ++i) in.logit[i] = i * THREADS < left ? z[i * THREADS] : from_f32<T>(0.0f);
    const bool legal = state >= 0 && state < a.n_states;
    if (a.mask != nullptr && legal) {
        const uint8_t *mask = a.mask + state * a.mask_ld + threadIdx.x;
#pragma unroll
        for (int i = 0; i < VPT; ++i) in.ok[i] = i * THREADS < left ? mask[i * THREADS] : 0;
    } else {
#pragma unroll
        for (int i = 0; i < VPT; ++i) in.ok[i] = a.mask == nullptr && i * THREADS < left ? 1 : 0;
    }
    in.token = first_token(a, row);
}

// A row's loads are issued while the row before it is reduced and written (and
// its state a row earlier still): one barrier per row, and the block never
// waits for memory that it has only just asked for.
template <typename T, int THREADS, int VPT>
__global__ __launch_bounds__(THREADS, min_blocks(THREADS, VPT)) void weights_forward_kernel(const WeightsArgs a, float *out) {
    extern __shared__ unsigned dyn[];
    constexpr int kChunk = THREADS * VPT, kWarps = THREADS / 32, kCounts = kChunk / 32 + kChunk;
    __shared__ float warp_m[2][kWarps], warp_s[2][kWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int left = static_cast<int>(a.n) - tid;  // the thread's column i exists iff i * THREADS < left
    const bool hist = a.hist > 0;
    const float k = a.k;
    const int64_t step = gridDim.x;
    int64_t row = blockIdx.x;
    RowInputs<T, VPT> in;
    int64_t state = 0;
    if (row < a.rows) {
        load_inputs<T, THREADS, VPT>(a, row, state_of(a, row), left, in);
        if (row + step < a.rows) state = state_of(a, row + step);
    }
    if (hist) {
        for (int i = tid; i < 3 * kCounts; i += THREADS) dyn[i] = 0u;
        __syncthreads();
        if (row < a.rows) history_pass<THREADS, VPT, true>(a, row, in.token, dyn);
    }
    __syncthreads();
    int flip = 0, buf = 0;
    for (; row < a.rows; row += step) {
        const unsigned *seen = dyn + buf * kCounts, *count = seen + kChunk / 32;
        unsigned word = 0u, any = 0u;
        if (hist) {
            word = lane < VPT ? seen[warp * VPT + lane] : 0u;
            any = __ballot_sync(kFull, word != 0u);
        }
        float u[VPT], m = -INFINITY;
        if (a.bias != nullptr) {
            const T *bias = static_cast<const T *>(a.bias) + row * a.bias_ld + tid;
#pragma unroll
            for (int i = 0; i < VPT; ++i) u[i] = i * THREADS < left ? to_f32<T>(bias[i * THREADS]) : 0.0f;
        } else {
#pragma unroll
            for (int i = 0; i < VPT; ++i) u[i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            float v = to_f32<T>(in.logit[i]);
            if ((any >> i) & 1u) {  // the same for the whole warp
                if ((__shfl_sync(kFull, word, i) >> lane) & 1u) v = penalised(a, v, count[i * THREADS + tid]);
            }
            u[i] = in.ok[i] != 0 ? v + u[i] : -INFINITY;
            m = fmaxf(m, u[i]);
        }
        // the next row's inputs, and the state after it
        const int64_t token = in.token;
        if (row + step < a.rows) {
            load_inputs<T, THREADS, VPT>(a, row + step, state, left, in);
            if (row + 2 * step < a.rows) state = state_of(a, row + 2 * step);
        }
        // -inf contributes nothing even where it is also the maximum; a NaN stays one
        const float from = m == -INFINITY ? 0.0f : m;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            u[i] = power2((u[i] - from) * k);
            s += u[i];
        }
        const float wm = warp_max(m);
        const float ws = warp_sum(s * rescale(m, wm, k));
        if (lane == 0) {
            warp_m[flip][warp] = wm;
            warp_s[flip][warp] = ws;
        }
        const int next = buf == 2 ? 0 : buf + 1;
        if (hist && row + step < a.rows)
            history_pass<THREADS, VPT, true>(a, row + step, in.token, dyn + next * kCounts);
        __syncthreads();
        const float bm = lane < kWarps ? warp_m[flip][lane] : -INFINITY;
        const float bs = lane < kWarps ? warp_s[flip][lane] : 0.0f;
        const float top = warp_max(bm);
        const float total = warp_sum(bs * rescale(bm, top, k));
        if (hist) history_pass<THREADS, VPT, false>(a, row, token, dyn + buf * kCounts);
        const float f = total == 0.0f ? 0.0f : rescale(m, top, k) / total;
        float *w = out + row * a.n + tid;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            if (i * THREADS < left) w[i * THREADS] = u[i] * f;
        flip ^= 1;
        buf = next;
    }
}

// dbias_partial: [blocks, n] sums of du over the rows each block took (a fixed set), or NULL;
// du: [rows, n] for a bias of the logits' shape, or NULL.
template <typename T, int THREADS, int VPT>
__global__ __launch_bounds__(THREADS, min_blocks_backward(THREADS, VPT)) void weights_backward_kernel(const WeightsArgs a, const float *w,
                                                                                   const float *g, int64_t ld_g, T *dz,
                                                                                   T *du, float *dbias_partial) {
    extern __shared__ unsigned dyn[];
    constexpr int kChunk = THREADS * VPT, kWarps = THREADS / 32, kCounts = kChunk / 32 + kChunk;
    __shared__ float warp_s[2][kWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int left = static_cast<int>(a.n) - tid;
    const bool hist = a.hist > 0 && a.theta != 1.0f && dz != nullptr;  // only the repetition penalty has a slope
    const int64_t step = gridDim.x;
    int64_t row = blockIdx.x, token = -1;
    float acc[VPT], p_next[VPT], q_next[VPT];
    auto load = [&](int64_t r) {
        const float *pw = w + r * a.n + tid, *pg = g + r * ld_g + tid;
#pragma unroll
        for (int i = 0; i < VPT; ++i) p_next[i] = i * THREADS < left ? pw[i * THREADS] : 0.0f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) q_next[i] = i * THREADS < left ? pg[i * THREADS] : 0.0f;
        if (hist) token = first_token(a, r);
    };
    if (row < a.rows) load(row);
#pragma unroll
    for (int i = 0; i < VPT; ++i) acc[i] = 0.0f;
    if (hist) {
        for (int i = tid; i < 3 * kCounts; i += THREADS) dyn[i] = 0u;
        __syncthreads();
        if (row < a.rows) history_pass<THREADS, VPT, true>(a, row, token, dyn);
    }
    __syncthreads();
    int flip = 0, buf = 0;
    for (; row < a.rows; row += step) {
        unsigned word = 0u, any = 0u;
        if (hist) {
            word = lane < VPT ? dyn[buf * kCounts + warp * VPT + lane] : 0u;
            any = __ballot_sync(kFull, word != 0u);
        }
        float p[VPT], q[VPT], s = 0.0f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            p[i] = p_next[i];
            q[i] = p[i] == 0.0f ? 0.0f : q_next[i];  // a weight of 0 passes nothing on, whatever the gradient there
            s = fmaf(p[i], q[i], s);
        }
        const int64_t old_token = token;
        const int next = buf == 2 ? 0 : buf + 1;
        if (row + step < a.rows) load(row + step);
        const float ws = warp_sum(s);
        if (lane == 0) warp_s[flip][warp] = ws;
        if (hist && row + step < a.rows)
            history_pass<THREADS, VPT, true>(a, row + step, token, dyn + next * kCounts);
        __syncthreads();
        const float dot = warp_sum(lane < kWarps ? warp_s[flip][lane] : 0.0f);
        if (hist) history_pass<THREADS, VPT, false>(a, row, old_token, dyn + buf * kCounts);
        const int64_t at = row * a.n + tid;
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
                        const T *z = static_cast<const T *>(a.logits) + row * a.ld + tid;
                        p[i] = to_f32<T>(z[i * THREADS]) > 0.0f ? p[i] / a.theta : p[i] * a.theta;
                    }
                }
                if (i * THREADS < left) dz[at + i * THREADS] = from_f32<T>(p[i]);
            }
        }
        flip ^= 1;
        buf = next;
    }
    if (dbias_partial != nullptr) {
        float *po = dbias_partial + blockIdx.x * a.n + tid;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            if (i * THREADS < left) po[i * THREADS] = acc[i];
    }
}

// ---- rows of 4097 columns and more (row_form says up to where) ---------------
// A row's 32 values a thread stay in registers, while the next row lands in
// shared memory by asynchronous copies of 16 bytes.  A landed row keeps its
// position within 16 bytes: column c lies at element c + lead.  A thread copies
// the same pieces of 16 bytes that it reads, so it asks for a piece of the next
// row as soon as it has read this row's.  The mask row follows behind a barrier:
// its pieces are cut elsewhere.  The counts take 16 bits each (no history has
// more than 65535 entries); one set of them, with one "seen" bit per element, is
// cleared and filled again between a row's barriers.
constexpr int kRowValues = 32;

template <typename T>
__device__ __forceinline__ int lead_of(const T *p) {
    return static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15) / static_cast<int>(sizeof(T));
}
template <int THREADS, bool ADD>
__device__ __forceinline__ void row_history(const WeightsArgs &a, int64_t row, int64_t token, int lead, unsigned *seen,
                                            unsigned *count) {
    const int64_t *h = a.history + row * a.hist_ld;
    for (int64_t j = threadIdx.x; j < a.hist; j += THREADS) {
        const int64_t v = j == threadIdx.x ? token : h[j];
        if (v < 0 || v >= a.n) continue;
        const int e = static_cast<int>(v) + lead;
        if (ADD) {
            atomicAdd(count + (e >> 1), 1u << (16 * (e & 1)));
            atomicOr(seen + (e >> 5), 1u << (e & 31));
        } else {
            count[e >> 1] = 0u;
            seen[e >> 5] = 0u;
        }
    }
}

__device__ __forceinline__ void copy16(const void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
                 "l"(src) : "memory");
}
// The elements of a landing row before its first and after its last whole piece: one a thread.
template <typename T>
__device__ __forceinline__ int edge_column(const T *src, int n) {  // or -1
    constexpr int kPer = 16 / sizeof(T);
    const int lead = lead_of(src), head = lead == 0 ? 0 : kPer - lead, tail = (n - head) % kPer;
    const int t = threadIdx.x;
    return t < head ? t : t >= 16 && t - 16 < tail ? n - tail + t - 16 : -1;
}
template <typename T>
__device__ __forceinline__ T edge_load(const T *src, int n) {
    const int c = edge_column(src, n);
    return c >= 0 ? src[c] : T(0.0f);
}
template <typename T>
__device__ __forceinline__ void edge_store(unsigned char *dst, const T *src, int n, T edge) {
    const int c = edge_column(src, n);
    if (c >= 0) reinterpret_cast<T *>(dst)[lead_of(src) + c] = edge;
}
// The whole pieces of a mask row.
template <int THREADS>
__device__ __forceinline__ void land_mask(unsigned char *dst, const uint8_t *src, int n) {
    const int lead = lead_of(src), head = (16 - lead) & 15, pieces = (n - head) / 16;
    for (int i = threadIdx.x; i < pieces; i += THREADS) copy16(dst + lead + head + 16 * i, src + head + 16 * i);
}
// room for n elements at any position within 16 bytes
__host__ __device__ constexpr int landing_bytes(int n, int size) { return (n * size + 15) / 16 * 16 + 16; }
// words of counts: one half for each element of whole pieces, up to seven before the row and seven after it
__host__ __device__ constexpr int count_words(int n) { return (n + 16) / 2; }

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) weights_row_kernel(const WeightsArgs a, float *out) {
    extern __shared__ uint4 rows_raw[];
    constexpr int kWarps = THREADS / 32, kPer = 16 / sizeof(T), kPieces = kRowValues / kPer;
    __shared__ float warp_m[kWarps], warp_s[kWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = static_cast<int>(a.n);
    unsigned char *const zs = reinterpret_cast<unsigned char *>(rows_raw);
    unsigned char *const ms = zs + landing_bytes(n, sizeof(T));
    unsigned *const seen = reinterpret_cast<unsigned *>(a.mask != nullptr ? ms + landing_bytes(n, 1) + 16 : ms);
    unsigned *const count = seen + THREADS;
    const bool hist = a.hist > 0;
    const float k = a.k;
    const int64_t step = gridDim.x;
    int64_t row = blockIdx.x;
    if (row >= a.rows) return;  // for the whole block
    const T *z = static_cast<const T *>(a.logits) + row * a.ld;
    int64_t state = state_of(a, row), state_next = row + step < a.rows ? state_of(a, row + step) : 0;
    bool legal = state >= 0 && state < a.n_states;
    const uint8_t *mask = a.mask != nullptr && legal ? a.mask + state * a.mask_ld : nullptr;
    T edge = edge_load(z, n);
    uint8_t mask_edge = mask != nullptr ? edge_load(mask, n) : 0;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int e = kPer * (i * THREADS + tid);
        if (e >= lead_of(z) && e + kPer <= lead_of(z) + n) copy16(zs + 16 * (i * THREADS + tid), z + e - lead_of(z));
    }
    if (mask != nullptr) land_mask<THREADS>(ms, mask, n);
    int64_t token = -1, token_next = -1;
    if (hist) {
        if (tid < a.hist) token = a.history[row * a.hist_ld + tid];
        for (int i = tid; i < THREADS + count_words(n); i += THREADS) seen[i] = 0u;
        __syncthreads();
        row_history<THREADS, true>(a, row, token, lead_of(z), seen, count);
    }
    edge_store<T>(zs, z, n, edge);
    if (mask != nullptr) edge_store<uint8_t>(ms, mask, n, mask_edge);
    for (; row < a.rows; row += step) {
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();  // the row has landed, its counts are complete
        const bool more = row + step < a.rows;
        const int lead = lead_of(z), end = lead + n;
        const T *zn = more ? z + step * a.ld : z;
        const int lead_n = lead_of(zn), end_n = more ? lead_n + n : 0;
        const T *from_n = zn - lead_n;  // element 0, on 16 bytes
        // mask byte of element e: ms + (mask mod 16) + e - lead (the bytes before it are the landing place of the logits)
        const int mask_at = (mask != nullptr ? lead_of(mask) : 0) - lead + 8;
        const unsigned *mr = reinterpret_cast<const unsigned *>(ms - 8 + (mask_at & ~3));
        const int turn = 8 * (mask_at & 3);
        const unsigned all = a.mask != nullptr && !legal ? 0u : 0xffffffffu;  // no such state: nothing is allowed
        const T *bias = a.bias != nullptr ? static_cast<const T *>(a.bias) + row * a.bias_ld - lead : nullptr;
        float u[kRowValues], m = -INFINITY;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int e = kPer * (i * THREADS + tid);
            float *v = u + i * kPer;
            if (e < end) {
                union { uint4 w; T t[kPer]; } x;
                x.w = rows_raw[i * THREADS + tid];
                const unsigned bits = hist ? (seen[e >> 5] >> (e & 31)) & ((1u << kPer) - 1u) : 0u;
#pragma unroll
                for (int q = 0; q < kPer; ++q) v[q] = to_f32<T>(x.t[q]);
                if (bits != 0u) {
#pragma unroll
                    for (int q = 0; q < kPer; ++q) {
                        const unsigned cnt = (count[(e + q) >> 1] >> (16 * (q & 1))) & 65535u;
                        if ((bits >> q) & 1u) v[q] = penalised(a, v[q], cnt);
                    }
                }
                if (bias != nullptr) {
#pragma unroll
                    for (int q = 0; q < kPer; ++q)
                        if (e + q >= lead && e + q < end) v[q] += to_f32<T>(bias[e + q]);
                }
#pragma unroll
                for (int h = 0; h < kPer; h += 4) {
                    unsigned ok = all;  // a byte per element
                    if (mask != nullptr) ok = __funnelshift_r(mr[(e + h) / 4], mr[(e + h) / 4 + 1], turn);
#pragma unroll
                    for (int q = h; q < h + 4; ++q)
                        if ((ok & (255u << (8 * (q - h)))) == 0u) v[q] = -INFINITY;
                }
                if (e < lead || e + kPer > end) {
#pragma unroll
                    for (int q = 0; q < kPer; ++q)
                        if (e + q < lead || e + q >= end) v[q] = -INFINITY;
                }
#pragma unroll
                for (int q = 0; q < kPer; ++q) m = fmaxf(m, v[q]);
            } else {
#pragma unroll
                for (int q = 0; q < kPer; ++q) v[q] = -INFINITY;
            }
            // the values above are in registers: the piece's place is free
            if (e >= lead_n && e + kPer <= end_n) copy16(zs + 16 * (i * THREADS + tid), from_n + e);
        }
        if (hist && more && tid < a.hist) token_next = a.history[(row + step) * a.hist_ld + tid];
        __syncthreads();  // the mask row and the counts have been read
        if (more) {
            z = zn;
            state = state_next;
            legal = state >= 0 && state < a.n_states;
            mask = a.mask != nullptr && legal ? a.mask + state * a.mask_ld : nullptr;
            edge = edge_load(z, n);
            if (mask != nullptr) {
                land_mask<THREADS>(ms, mask, n);
                mask_edge = edge_load(mask, n);
            }
            if (row + 2 * step < a.rows) state_next = state_of(a, row + 2 * step);
        }
        if (hist) row_history<THREADS, false>(a, row, token, lead, seen, count);
        // -inf contributes nothing even where it is also the maximum; a NaN stays one
        const float from = m == -INFINITY ? 0.0f : m;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kRowValues; ++i) {
            u[i] = power2((u[i] - from) * k);
            s += u[i];
        }
        const float wm = warp_max(m);
        const float ws = warp_sum(s * rescale(m, wm, k));
        if (lane == 0) {
            warp_m[warp] = wm;
            warp_s[warp] = ws;
        }
        __syncthreads();  // the counts are clear, the warps' sums are there
        if (hist && more) {
            token = token_next;
            row_history<THREADS, true>(a, row + step, token, lead_of(z), seen, count);
        }
        const float bm = lane < kWarps ? warp_m[lane] : -INFINITY;
        const float bs = lane < kWarps ? warp_s[lane] : 0.0f;
        const float top = warp_max(bm);
        const float total = warp_sum(bs * rescale(bm, top, k));
        const float f = total == 0.0f ? 0.0f : rescale(m, top, k) / total;
        float *w = out + row * a.n - lead;  // of element 0, which may lie before the row
        const bool aligned = (reinterpret_cast<uintptr_t>(w) & 15) == 0;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int e = kPer * (i * THREADS + tid);
            if (aligned && e >= lead && e + kPer <= end) {
#pragma unroll
                for (int q = i * kPer; q < (i + 1) * kPer; q += 4)
                    *reinterpret_cast<float4 *>(w + e + q - i * kPer) =
                        make_float4(u[q] * f, u[q + 1] * f, u[q + 2] * f, u[q + 3] * f);
            } else {
#pragma unroll
                for (int q = 0; q < kPer; ++q)
                    if (e + q >= lead && e + q < end) w[e + q] = u[i * kPer + q] * f;
            }
        }
        if (more) {
            edge_store<T>(zs, z, n, edge);
            if (mask != nullptr) edge_store<uint8_t>(ms, mask, n, mask_edge);
        }
    }
}

// ---- rows of more columns ----------------------------------------------------
// Two passes by one block: the first stores u where w will lie and keeps the
// running maximum and the sum relative to it, the second reads u back (from L2:
// the rows in flight fit) and writes w.
constexpr int kStreamThreads = 512, kStreamUnroll = 8, kStreamBlocks = 2;

// Counts of a long row: 16 bits each, two to a word (no history has more than
// 65535 entries), behind one seen bit per column.
template <bool ADD>
__device__ __forceinline__ void stream_history(const WeightsArgs &a, int64_t row, unsigned *seen, unsigned *count) {
    const int64_t *h = a.history + row * a.hist_ld;
    for (int64_t j = threadIdx.x; j < a.hist; j += kStreamThreads) {
        const int64_t v = h[j];
        if (v < 0 || v >= a.n) continue;
        const int c = static_cast<int>(v);
        if (ADD) {
            atomicAdd(count + (c >> 1), 1u << (16 * (c & 1)));
            atomicOr(seen + (c >> 5), 1u << (c & 31));
        } else {
            count[c >> 1] = 0u;
            seen[c >> 5] = 0u;
        }
    }
}

// u of U columns a thread, kStreamThreads apart, from column `base` on; the
// running maximum and sum take them in.  FULL: all columns exist, and one load
// and a ballot tell a warp which of its U words of seen bits are not empty.
template <typename T, int U, bool FULL>
__device__ __forceinline__ void stream_group(const WeightsArgs &a, const T *z, const T *bias, const uint8_t *mask,
                                             float *w, int base, int left, const unsigned *seen, const unsigned *count,
                                             float k, float &m, float &s) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T raw[U], extra[U];
    uint8_t ok[U];
#pragma unroll
    for (int i = 0; i < U; ++i) raw[i] = FULL || i * kStreamThreads < left ? z[i * kStreamThreads] : from_f32<T>(0.0f);
    if (mask != nullptr) {
#pragma unroll
        for (int i = 0; i < U; ++i) ok[i] = FULL || i * kStreamThreads < left ? mask[i * kStreamThreads] : 0;
    } else {
#pragma unroll
        for (int i = 0; i < U; ++i) ok[i] = FULL || i * kStreamThreads < left ? 1 : 0;
    }
    if (bias != nullptr) {
#pragma unroll
        for (int i = 0; i < U; ++i) extra[i] = FULL || i * kStreamThreads < left ? bias[i * kStreamThreads] : from_f32<T>(0.0f);
    }
    unsigned word = 0u, any = 0u;
    if (seen != nullptr) {
        const int at = (base >> 5) + warp + lane * (kStreamThreads / 32);
        word = lane < U && (FULL || 32 * at < a.n) ? seen[at] : 0u;
        any = __ballot_sync(kFull, word != 0u);
    }
    float u[U], top = m;
#pragma unroll
    for (int i = 0; i < U; ++i) {
        float v = to_f32<T>(raw[i]);
        if ((any >> i) & 1u) {  // the same for the whole warp
            if ((__shfl_sync(kFull, word, i) >> lane) & 1u) {
                const int c = base + i * kStreamThreads + threadIdx.x;
                v = penalised(a, v, (count[c >> 1] >> (16 * (c & 1))) & 65535u);
            }
        }
        if (bias != nullptr) v += to_f32<T>(extra[i]);
        u[i] = ok[i] != 0 ? v : -INFINITY;
        top = fmaxf(top, u[i]);
        if (FULL || i * kStreamThreads < left) w[i * kStreamThreads] = u[i];
    }
    const float from = top == -INFINITY ? 0.0f : top;
    s *= rescale(m, top, k);
    m = top;
#pragma unroll
    for (int i = 0; i < U; ++i) s += power2((u[i] - from) * k);
}

template <typename T>
__global__ void __launch_bounds__(kStreamThreads, kStreamBlocks) weights_stream_kernel(const WeightsArgs a, float *out) {
    extern __shared__ unsigned dyn[];
    constexpr int kWarps = kStreamThreads / 32, U = kStreamUnroll, kGroup = U * kStreamThreads;
    __shared__ float warp_m[2][kWarps], warp_s[2][kWarps];
    const int n = static_cast<int>(a.n), words = (n + 31) / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool hist = a.hist > 0;
    unsigned *seen = hist ? dyn : nullptr, *count = dyn + words;
    const float k = a.k;
    if (hist)
        for (int i = tid; i < words + (n + 1) / 2; i += kStreamThreads) dyn[i] = 0u;
    int flip = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, flip ^= 1) {
        if (hist) {
            __syncthreads();  // the counts are clear
            stream_history<true>(a, row, seen, count);
            __syncthreads();
        }
        const int64_t state = state_of(a, row);
        const bool legal = state >= 0 && state < a.n_states;
        const T *z = static_cast<const T *>(a.logits) + row * a.ld + tid;
        const T *bias = a.bias != nullptr ? static_cast<const T *>(a.bias) + row * a.bias_ld + tid : nullptr;
        const uint8_t *mask = a.mask != nullptr && legal ? a.mask + state * a.mask_ld + tid : nullptr;
        float *w = out + row * a.n + tid;
        float m = -INFINITY, s = 0.0f;
        if (a.mask != nullptr && !legal) {
            // no such state: nothing is allowed
            for (int c = tid; c < n; c += kStreamThreads) w[c - tid] = -INFINITY;
        } else {
            int base = 0;
            for (; base + kGroup <= n; base += kGroup)
                stream_group<T, U, true>(a, z + base, bias != nullptr ? bias + base : nullptr,
                                         mask != nullptr ? mask + base : nullptr, w + base, base, 0, seen, count, k, m, s);
            if (base < n)
                stream_group<T, U, false>(a, z + base, bias != nullptr ? bias + base : nullptr,
                                          mask != nullptr ? mask + base : nullptr, w + base, base, n - base - tid, seen,
                                          count, k, m, s);
        }
        const float wm = warp_max(m);
        const float ws = warp_sum(s * rescale(m, wm, k));
        if (lane == 0) {
            warp_m[flip][warp] = wm;
            warp_s[flip][warp] = ws;
        }
        __syncthreads();
        const float bm = lane < kWarps ? warp_m[flip][lane] : -INFINITY;
        const float bs = lane < kWarps ? warp_s[flip][lane] : 0.0f;
        const float top = warp_max(bm);
        const float total = warp_sum(bs * rescale(bm, top, k));
        if (hist) stream_history<false>(a, row, seen, count);
        const float from = top == -INFINITY ? 0.0f : top;
        const float f = total == 0.0f ? 0.0f : 1.0f / total;
        int base = 0;
        for (; base + kGroup <= n; base += kGroup) {
            float u[U];
#pragma unroll
            for (int i = 0; i < U; ++i) u[i] = w[base + i * kStreamThreads];
#pragma unroll
            for (int i = 0; i < U; ++i) w[base + i * kStreamThreads] = power2((u[i] - from) * k) * f;
        }
        for (base += tid; base < n; base += kStreamThreads) w[base - tid] = power2((w[base - tid] - from) * k) * f;
    }
}

// The gradient of long rows: the sum w g first, then both are read again.
// dbias_partial [blocks, n] holds zeros, or is NULL.
template <typename T>
__global__ void __launch_bounds__(kStreamThreads) weights_stream_backward_kernel(const WeightsArgs a, const float *w,
                                                                                 const float *g, int64_t ld_g, T *dz,
                                                                                 T *du, float *dbias_partial) {
    extern __shared__ unsigned dyn[];
    constexpr int kWarps = kStreamThreads / 32, U = kStreamUnroll;
    __shared__ float warp_s[2][kWarps];
    const int n = static_cast<int>(a.n), words = (n + 31) / 32;
    unsigned *seen = dyn;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool hist = a.hist > 0 && a.theta != 1.0f && dz != nullptr;  // only the repetition penalty has a slope
    float *partial = dbias_partial != nullptr ? dbias_partial + blockIdx.x * a.n : nullptr;
    int flip = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, flip ^= 1) {
        if (hist) {
            __syncthreads();
            for (int i = tid; i < words; i += kStreamThreads) seen[i] = 0u;
            __syncthreads();
            const int64_t *h = a.history + row * a.hist_ld;
            for (int64_t j = tid; j < a.hist; j += kStreamThreads) {
                const int64_t v = h[j];
                if (v >= 0 && v < a.n) atomicOr(seen + (v >> 5), 1u << (v & 31));
            }
        }
        const float *pw = w + row * a.n, *pg = g + row * ld_g;
        float s = 0.0f;
        for (int base = tid; base < n; base += U * kStreamThreads) {
            float p[U], q[U];
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int c = base + i * kStreamThreads;
                p[i] = c < n ? pw[c] : 0.0f;
                q[i] = c < n ? pg[c] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < U; ++i) s = fmaf(p[i], p[i] == 0.0f ? 0.0f : q[i], s);
        }
        const float ws = warp_sum(s);
        if (lane == 0) warp_s[flip][warp] = ws;
        __syncthreads();
        const float dot = warp_sum(lane < kWarps ? warp_s[flip][lane] : 0.0f);
        const T *z = static_cast<const T *>(a.logits) + row * a.ld;
        const int64_t at = row * a.n;
        for (int base = tid; base < n; base += U * kStreamThreads) {
            float p[U], q[U], r[U];
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int c = base + i * kStreamThreads;
                p[i] = c < n ? pw[c] : 0.0f;
                q[i] = c < n ? pg[c] : 0.0f;
                r[i] = partial != nullptr && c < n ? partial[c] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int c = base + i * kStreamThreads;
                if (c >= n) continue;
                // a weight of 0 gets and passes nothing
                float d = p[i] == 0.0f ? 0.0f : p[i] * (q[i] - dot) * a.inv_tau;
                if (partial != nullptr) partial[c] = r[i] + d;
                if (du != nullptr) du[at + c] = from_f32<T>(d);
                if (dz != nullptr) {
                    if (hist && (seen[c >> 5] >> (c & 31)) & 1u) d = to_f32<T>(z[c]) > 0.0f ? d / a.theta : d * a.theta;
                    dz[at + c] = from_f32<T>(d);
                }
            }
        }
    }
}

// ---- a few long rows: eight blocks to a row ----------------------------------
// One row would leave all SMs but one idle: a cluster of eight blocks holds it
// in registers (19 us -> 7 us for one row of 29649).  The blocks read each
// other's sums from shared memory, once.
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float peer_float(const float *p, uint32_t rank) {
    float v;
    asm volatile(
        "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %1, %2;\n ld.shared::cluster.f32 %0, [a];\n}"
        : "=f"(v) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank) : "memory");
    return v;
}
constexpr int kWideBlocks = 8;

// Which of a block's columns are in the row's history, and how often.
template <int VPT>
__device__ __forceinline__ void wide_history(const WeightsArgs &a, int64_t row, int c0, unsigned *seen,
                                             unsigned *count) {
    constexpr int kChunk = kStreamThreads * VPT;
    for (int i = threadIdx.x; i < kChunk / 32 + kChunk; i += kStreamThreads) seen[i] = 0u;
    __syncthreads();
    const int64_t *h = a.history + row * a.hist_ld;
    for (int64_t j = threadIdx.x; j < a.hist; j += kStreamThreads) {
        const int64_t v = h[j];
        const int64_t c = v - c0;
        if (v < 0 || v >= a.n || c < 0 || c >= kChunk) continue;
        atomicAdd(count + c, 1u);
        atomicOr(seen + (c >> 5), 1u << (c & 31));
    }
    __syncthreads();
}

template <typename T, int VPT>
__global__ void __launch_bounds__(kStreamThreads) __cluster_dims__(kWideBlocks, 1, 1)
    weights_wide_kernel(const WeightsArgs a, float *out) {
    extern __shared__ unsigned dyn[];
    constexpr int kChunk = kStreamThreads * VPT, kWarps = kStreamThreads / 32;
    __shared__ float warp_m[kWarps], warp_s[kWarps], block_m, block_s;
    unsigned *seen = dyn, *count = dyn + kChunk / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int c0 = static_cast<int>(cluster_rank()) * kChunk, left = static_cast<int>(a.n) - c0 - tid;
    const int64_t row = blockIdx.x / kWideBlocks;
    const bool hist = a.hist > 0;
    const float k = a.k;
    const T *z = static_cast<const T *>(a.logits) + row * a.ld + c0 + tid;
    const T *bias = static_cast<const T *>(a.bias) + row * a.bias_ld + c0 + tid;
    T raw[VPT], extra[VPT];
    uint8_t ok[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) raw[i] = i * kStreamThreads < left ? z[i * kStreamThreads] : from_f32<T>(0.0f);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
        extra[i] = a.bias != nullptr && i * kStreamThreads < left ? bias[i * kStreamThreads] : from_f32<T>(0.0f);
    const int64_t state = state_of(a, row);
    const bool legal = state >= 0 && state < a.n_states;
    const uint8_t *mask = a.mask + (legal ? state * a.mask_ld : 0) + c0 + tid;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        ok[i] = i * kStreamThreads < left ? 1 : 0;
        if (a.mask != nullptr) ok[i] = legal && ok[i] ? mask[i * kStreamThreads] : 0;
    }
    if (hist) wide_history<VPT>(a, row, c0, seen, count);
    float u[VPT], m = -INFINITY;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = i * kStreamThreads + tid;
        float v = to_f32<T>(raw[i]);
        if (hist && (seen[c >> 5] >> (c & 31)) & 1u) v = penalised(a, v, count[c]);
        if (a.bias != nullptr) v += to_f32<T>(extra[i]);
        u[i] = ok[i] != 0 ? v : -INFINITY;
        m = fmaxf(m, u[i]);
    }
    const float from = m == -INFINITY ? 0.0f : m;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        u[i] = power2((u[i] - from) * k);
        s += u[i];
    }
    const float wm = warp_max(m);
    const float ws = warp_sum(s * rescale(m, wm, k));
    if (lane == 0) {
        warp_m[warp] = wm;
        warp_s[warp] = ws;
    }
    __syncthreads();
    float bm = lane < kWarps ? warp_m[lane] : -INFINITY;
    float bs = lane < kWarps ? warp_s[lane] : 0.0f;
    float top = warp_max(bm);
    float total = warp_sum(bs * rescale(bm, top, k));
    if (tid == 0) {
        block_m = top;
        block_s = total;
    }
    cluster_barrier();
    bm = lane < kWideBlocks ? peer_float(&block_m, lane) : -INFINITY;
    bs = lane < kWideBlocks ? peer_float(&block_s, lane) : 0.0f;
    top = warp_max(bm);
    total = warp_sum(bs * rescale(bm, top, k));
    const float f = total == 0.0f ? 0.0f : rescale(m, top, k) / total;
    float *w = out + row * a.n + c0 + tid;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
        if (i * kStreamThreads < left) w[i * kStreamThreads] = u[i] * f;
    cluster_barrier();  // no block leaves while another may read its sums
}

// dbias_partial: [rows, n], or NULL.
template <typename T, int VPT>
__global__ void __launch_bounds__(kStreamThreads) __cluster_dims__(kWideBlocks, 1, 1)
    weights_wide_backward_kernel(const WeightsArgs a, const float *w, const float *g, int64_t ld_g, T *dz, T *du,
                                 float *dbias_partial) {
    extern __shared__ unsigned dyn[];
    constexpr int kChunk = kStreamThreads * VPT, kWarps = kStreamThreads / 32;
    __shared__ float warp_s[kWarps], block_s;
    unsigned *seen = dyn, *count = dyn + kChunk / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int c0 = static_cast<int>(cluster_rank()) * kChunk, left = static_cast<int>(a.n) - c0 - tid;
    const int64_t row = blockIdx.x / kWideBlocks, at = row * a.n + c0 + tid;
    const bool hist = a.hist > 0 && a.theta != 1.0f && dz != nullptr;  // only the repetition penalty has a slope
    float p[VPT], q[VPT], s = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) p[i] = i * kStreamThreads < left ? w[at + i * kStreamThreads] : 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) q[i] = i * kStreamThreads < left ? g[row * ld_g + c0 + tid + i * kStreamThreads] : 0.0f;
    if (hist) wide_history<VPT>(a, row, c0, seen, count);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        if (p[i] == 0.0f) q[i] = 0.0f;  // a weight of 0 passes nothing on, whatever the gradient there
        s = fmaf(p[i], q[i], s);
    }
    const float ws = warp_sum(s);
    if (lane == 0) warp_s[warp] = ws;
    __syncthreads();
    float dot = warp_sum(lane < kWarps ? warp_s[lane] : 0.0f);
    if (tid == 0) block_s = dot;
    cluster_barrier();
    dot = warp_sum(lane < kWideBlocks ? peer_float(&block_s, lane) : 0.0f);
    const T *z = static_cast<const T *>(a.logits) + row * a.ld + c0 + tid;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        if (i * kStreamThreads >= left) continue;
        const int c = i * kStreamThreads + tid;
        float d = p[i] == 0.0f ? 0.0f : p[i] * (q[i] - dot) * a.inv_tau;
        if (dbias_partial != nullptr) dbias_partial[at + i * kStreamThreads] = d;
        if (du != nullptr) du[at + i * kStreamThreads] = from_f32<T>(d);
        if (dz != nullptr) {
            if (hist && (seen[c >> 5] >> (c & 31)) & 1u)
                d = to_f32<T>(z[i * kStreamThreads]) > 0.0f ? d / a.theta : d * a.theta;
            dz[at + i * kStreamThreads] = from_f32<T>(d);
        }
    }
    cluster_barrier();
}

// Column sums of [parts, n] in a fixed order: 32 columns x 32 groups of parts per block.
template <typename T>
__global__ void column_sum_kernel(const float *partial, int64_t parts, int64_t n, T *out) {
    __shared__ float part[32][33];
    const int64_t c = blockIdx.x * int64_t(32) + threadIdx.x;
    float s = 0.0f;
    if (c < n) {
        float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int64_t p0 = threadIdx.y; p0 < parts; p0 += 128)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (p0 + 32 * q < parts) t[q] += partial[(p0 + 32 * q) * n + c];
        s = (t[0] + t[1]) + (t[2] + t[3]);
    }
    part[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && c < n) {
#pragma unroll
        for (int i = 1; i < 32; ++i) s += part[i][threadIdx.x];
        out[c] = from_f32<T>(s);
    }
}

// How a row is laid over threads: the narrowest form that holds it.  The counts
// of 4096 columns (three rows) take 51 KB of shared memory.
struct Layout {
    int threads, vpt;  // vpt 0: the two-pass form
    int wide;          // values a thread of the cluster form, or 0
    int64_t blocks;    // rows in flight
    int sms;
};

constexpr int64_t kMaxColumns = 65536, kMaxHistory = 65535;

Layout layout(int64_t rows, int64_t n) {
    const int sms = fl_device_sm_count() > 0 ? fl_device_sm_count() : 148;
    Layout l{256, 16, 0, 0, sms};
    // Sixteen values a thread: what a row costs each thread besides (the
    // reductions, the history) is then spread far enough (12288 x 4096: 113 us
    // with eight, 80 us with sixteen).
    if (n <= 128) l = {32, 4, 0, 0, sms};
    else if (n <= 512) l = {32, 16, 0, 0, sms};
    else if (n <= 1024) l = {64, 16, 0, 0, sms};
    else if (n <= 2048) l = {128, 16, 0, 0, sms};
    else if (n > 4096) l = {kStreamThreads, 0, 0, 0, sms};
    if (l.vpt == 0 && rows * kWideBlocks <= 2 * sms) l.wide = n <= 8 * kWideBlocks * kStreamThreads ? 8 : 16;
    const int64_t fit = static_cast<int64_t>(sms) * (l.vpt ? min_blocks(l.threads, l.vpt) : 3);
    l.blocks = rows < fit ? rows : fit;
    return l;
}

// The form that holds a row in registers while the next one lands: its shared
// memory, and its threads or 0.  Against the two-pass form, 40 million values
// with masks and histories of 200: 90 us and 137 us at n = 8000, 90 and 115 at
// 16000 (bf16: 94 and 138, 96 and 113).  A block of 1024 threads is alone on its
// SM and nothing covers its barriers: it wins with most of its values in use
// (92 us and 106 us at n = 32000, 115 and 109 at 20000) and in 32 bits (bf16:
// 113 and 100 at 32000).
size_t row_smem(int64_t n, size_t size, bool mask, bool hist, int threads) {
    const int c = static_cast<int>(n);
    return landing_bytes(c, static_cast<int>(size)) + (mask ? landing_bytes(c, 1) + 16 : 0) +
           (hist ? (threads + count_words(c)) * sizeof(unsigned) : 0);
}
int row_form(int64_t n, size_t size, bool mask, bool hist) {
    const int64_t elements = n + 7;  // a row that starts 7 elements after a 16-byte boundary
    if (n <= 4096 || elements > 1024 * kRowValues) return 0;
    const int threads = elements <= 256 * kRowValues ? 256 : elements <= 512 * kRowValues ? 512 : 1024;
    if (threads == 1024 && (size != 4 || n < 24 * 1024)) return 0;
    return row_smem(n, size, mask, hist, threads) <= 226 * 1024 ? threads : 0;
}

template <typename K, typename... Args>
int launch_rows(K kernel, const Layout &l, size_t smem, cudaStream_t st, Args... args) {
    // 48 KB need no permission, for this and what a kernel holds anyway (256 bytes at most) together
    if (smem > 40 * 1024)
        FL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    const int64_t grid = l.wide ? l.blocks * kWideBlocks : l.blocks;
    launch(kernel, static_cast<unsigned>(grid), l.threads, smem, st, args...);
    return check_launch("relation weights");
}

size_t history_smem(const Layout &l, int64_t n, bool hist, bool counts) {
    if (!hist) return 0;
    if (l.wide) return (l.threads * l.wide / 32 + l.threads * l.wide) * sizeof(unsigned);
    if (l.vpt == 0) return ((n + 31) / 32 + (counts ? (n + 1) / 2 : 0)) * sizeof(unsigned);
    const size_t chunk = static_cast<size_t>(l.threads) * l.vpt;
    return 3 * (chunk / 32 + chunk) * sizeof(unsigned);
}

#define FL_LAYOUTS(F)                            \
    if (l.vpt == 4) F(32, 4);                    \
    else if (l.threads == 32) F(32, 16);         \
    else if (l.threads == 64) F(64, 16);         \
    else if (l.threads == 128) F(128, 16);       \
    else F(256, 16);

template <typename T>
int forward_t(const WeightsArgs &a, float *w, cudaStream_t st) {
    Layout l = layout(a.rows, a.n);
    const size_t smem = history_smem(l, a.n, a.hist > 0, true);
    if (l.wide == 8) return launch_rows(weights_wide_kernel<T, 8>, l, smem, st, a, w);
    if (l.wide == 16) return launch_rows(weights_wide_kernel<T, 16>, l, smem, st, a, w);
    const int row_threads = row_form(a.n, sizeof(T), a.mask != nullptr, a.hist > 0);
    if (row_threads != 0) {
        l.threads = row_threads;
        const size_t bytes = row_smem(a.n, sizeof(T), a.mask != nullptr, a.hist > 0, row_threads);
        const int64_t room = static_cast<int64_t>(228 * 1024 / (bytes + 1280));  // blocks whose memory an SM has
        const int64_t fit = l.sms * (room < 1024 / row_threads ? room : 1024 / row_threads);
        l.blocks = a.rows < fit ? a.rows : fit;
        if (row_threads == 256) return launch_rows(weights_row_kernel<T, 256>, l, bytes, st, a, w);
        if (row_threads == 512) return launch_rows(weights_row_kernel<T, 512>, l, bytes, st, a, w);
        if constexpr (sizeof(T) == 4) return launch_rows(weights_row_kernel<T, 1024>, l, bytes, st, a, w);
    }
    if (l.vpt == 0 && a.rows < (1ll << 31)) l.blocks = a.rows;  // a block per row: the hardware balances them
    if (l.vpt == 0) return launch_rows(weights_stream_kernel<T>, l, smem, st, a, w);
    int rc = FL_OK;
#define F(TH, V) rc = launch_rows(weights_forward_kernel<T, TH, V>, l, smem, st, a, w)
    FL_LAYOUTS(F)
#undef F
    return rc;
}

template <typename T>
int backward_t(const WeightsArgs &a, const float *w, const float *g, int64_t ld_g, T *dz, T *du, T *dbias, Carve &ws,
               cudaStream_t st) {
    Layout l = layout(a.rows, a.n);
    if (l.vpt != 0) {
        const int64_t fit = static_cast<int64_t>(l.sms) * min_blocks_backward(l.threads, l.vpt);
        if (l.blocks > fit) l.blocks = fit;  // (no more than the workspace was sized for)
    }
    float *partial = nullptr;
    if (dbias != nullptr) {
        partial = ws.take<float>(l.blocks * a.n);
        FL_REQUIRE(partial != nullptr, "relation weights: workspace too small");
    }
    const size_t smem = history_smem(l, a.n, a.hist > 0 && a.theta != 1.0f && dz != nullptr, false);
    int rc = FL_OK;
    if (l.wide == 8) {
        rc = launch_rows(weights_wide_backward_kernel<T, 8>, l, smem, st, a, w, g, ld_g, dz, du, partial);
    } else if (l.wide == 16) {
        rc = launch_rows(weights_wide_backward_kernel<T, 16>, l, smem, st, a, w, g, ld_g, dz, du, partial);
    } else if (l.vpt == 0) {
        if (partial != nullptr) FL_CUDA(cudaMemsetAsync(partial, 0, l.blocks * a.n * sizeof(float), st));
        rc = launch_rows(weights_stream_backward_kernel<T>, l, smem, st, a, w, g, ld_g, dz, du, partial);
    } else {
#define F(TH, V) rc = launch_rows(weights_backward_kernel<T, TH, V>, l, smem, st, a, w, g, ld_g, dz, du, partial)
        FL_LAYOUTS(F)
#undef F
    }
    if (rc || dbias == nullptr) return rc;
    launch(column_sum_kernel<T>, static_cast<unsigned>((a.n + 31) / 32), dim3(32, 32), 0, st, partial, l.blocks, a.n,
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
    FL_REQUIRE(p->hist >= 0 && p->hist <= kMaxHistory && (p->hist == 0 || p->history != nullptr),
               "relation weights: bad history (at most %lld entries)", static_cast<long long>(kMaxHistory));
    *a = WeightsArgs{p->logits, p->ld, p->bias, p->bias_ld, static_cast<const uint8_t *>(p->mask), p->mask_ld,
                     p->mask != nullptr ? p->n_states : 0, p->states, p->history, p->hist_ld, p->hist, p->rows, p->n,
                     static_cast<float>(p->repetition), static_cast<float>(1.0 / p->repetition),
                     static_cast<float>(p->frequency), static_cast<float>(p->presence), static_cast<float>(1.0 / p->tau),
                     static_cast<float>(1.4426950408889634 / p->tau)};
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
    return carve_bytes<float>(layout(rows, n).blocks * n);
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

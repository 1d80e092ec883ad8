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
// up to eight blocks, which exchange their (maximum, sum) pairs through shared
// memory.  The operation is bound by HBM: a value is read once and written once.
//
// The history's counts live in shared memory next to one "seen" bit per
// column; a warp's 32 columns share one word of bits, so columns without
// history cost one broadcast read per warp.  Counts are cleared by walking the
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
__device__ __forceinline__ float peer_float(const float *p, uint32_t rank) {
    float v;
    asm volatile(
        "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %1, %2;\n ld.shared::cluster.f32 %0, [a];\n}"
        : "=f"(v) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank) : "memory");
    return v;
}

// History counts of one row for the columns [c0, c0 + chunk): add (or clear).
template <int THREADS, bool ADD>
__device__ __forceinline__ void history_pass(const WeightsArgs &a, int64_t row, int64_t c0, int chunk, unsigned *seen,
                                             unsigned *count) {
    const int64_t *h = a.history + row * a.hist_ld;
    for (int64_t j = threadIdx.x; j < a.hist; j += THREADS) {
        const int64_t v = h[j];
        if (v < 0 || v >= a.n) continue;
        const int64_t c = v - c0;
        if (c < 0 || c >= chunk) continue;
        if (ADD) {
            atomicAdd(count + c, 1u);
            atomicOr(seen + (c >> 5), 1u << (c & 31));
        } else {
            count[c] = 0u;
            seen[c >> 5] = 0u;
        }
    }
}

// (max, sum relative to it) of two parts
__device__ __forceinline__ float rescale(float m, float to, float inv_tau) {
    return m == to ? 1.0f : expf((m - to) * inv_tau);  // equal (both -inf too): nothing to do
}

// 1024 threads per SM with up to 64 registers each: enough rows in flight to
// cover the loads' latency while other rows are in their reductions.
template <typename T, int THREADS, int VPT, bool CL>
__global__ __launch_bounds__(THREADS, 1024 / THREADS) void weights_forward_kernel(const WeightsArgs a, float *out) {
    extern __shared__ unsigned dyn[];
    constexpr int kChunk = THREADS * VPT, kWarps = THREADS / 32;
    unsigned *seen = dyn, *count = dyn + kChunk / 32;
    __shared__ float warp_m[2][kWarps], warp_s[2][kWarps], block_m[2], block_s[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rank = CL ? cluster_rank() : 0, ranks = CL ? cluster_size() : 1;
    const int64_t c0 = static_cast<int64_t>(rank) * kChunk;
    if (a.hist > 0) {
        for (int i = tid; i < kChunk / 32 + kChunk; i += THREADS) dyn[i] = 0u;
        __syncthreads();
    }
    int flip = 0;
    for (int64_t row = blockIdx.x / ranks; row < a.rows; row += gridDim.x / ranks, flip ^= 1) {
        if (a.hist > 0) {
            history_pass<THREADS, true>(a, row, c0, kChunk, seen, count);
            __syncthreads();
        }
        const T *z = static_cast<const T *>(a.logits) + row * a.ld;
        const T *bias = static_cast<const T *>(a.bias) + row * a.bias_ld;
        const int64_t state = a.states != nullptr ? a.states[row] : (row < a.n_states ? row : a.n_states - 1);
        const bool legal = state >= 0 && state < a.n_states;
        const uint8_t *mask = a.mask + (legal ? state * a.mask_ld : 0);
        // all of the row's loads first: they are in flight together
        float u[VPT], m = -INFINITY;
        T raw[VPT];
        unsigned allowed = 0u;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int64_t col = c0 + i * THREADS + tid;
            raw[i] = col < a.n ? z[col] : from_f32<T>(0.0f);
        }
        if (a.mask == nullptr) {
#pragma unroll
            for (int i = 0; i < VPT; ++i) allowed |= (c0 + i * THREADS + tid < a.n ? 1u : 0u) << i;
        } else if (legal) {
            uint8_t ok[VPT];
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                const int64_t col = c0 + i * THREADS + tid;
                ok[i] = col < a.n ? mask[col] : 0;
            }
#pragma unroll
            for (int i = 0; i < VPT; ++i) allowed |= (ok[i] != 0 ? 1u : 0u) << i;
        }
        if (a.bias != nullptr) {
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                const int64_t col = c0 + i * THREADS + tid;
                u[i] = col < a.n ? to_f32<T>(bias[col]) : 0.0f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < VPT; ++i) u[i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = i * THREADS + tid;
            float v = to_f32<T>(raw[i]);
            if (a.hist > 0 && (seen[c >> 5] >> (c & 31)) & 1u) {
                v = v > 0.0f ? v / a.theta : v * a.theta;
                v = v - a.frequency * static_cast<float>(count[c]) - a.presence;
            }
            v = (allowed >> i) & 1u ? v + u[i] : -INFINITY;
            u[i] = v;
            m = fmaxf(m, v);
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            // -inf contributes nothing even where it is also the maximum; a NaN stays one
            u[i] = u[i] == -INFINITY ? 0.0f : expf((u[i] - m) * a.inv_tau);
            s += u[i];
        }
        const float wm = warp_max(m);
        const float ws = warp_sum(s * rescale(m, wm, a.inv_tau));
        if (lane == 0) {
            warp_m[flip][warp] = wm;
            warp_s[flip][warp] = ws;
        }
        __syncthreads();
        float bm = lane < kWarps ? warp_m[flip][lane] : -INFINITY;
        float bs = lane < kWarps ? warp_s[flip][lane] : 0.0f;
        float top = warp_max(bm);
        float total = warp_sum(bs * rescale(bm, top, a.inv_tau));
        if (CL) {
            if (tid == 0) {
                block_m[flip] = top;
                block_s[flip] = total;
            }
            cluster_barrier();
            bm = lane < static_cast<int>(ranks) ? peer_float(&block_m[flip], lane) : -INFINITY;
            bs = lane < static_cast<int>(ranks) ? peer_float(&block_s[flip], lane) : 0.0f;
            top = warp_max(bm);
            total = warp_sum(bs * rescale(bm, top, a.inv_tau));
        }
        const float f = total == 0.0f ? 0.0f : rescale(m, top, a.inv_tau) / total;
        float *w = out + row * a.n;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int64_t col = c0 + i * THREADS + tid;
            if (col < a.n) w[col] = u[i] * f;
        }
        if (a.hist > 0) {
            // every thread read its counts before the reduction's barrier
            history_pass<THREADS, false>(a, row, c0, kChunk, seen, count);
            __syncthreads();
        }
    }
    if (CL) cluster_barrier();  // no block leaves while another may read its pair
}

// dbias_partial: [blocks / ranks, n] sums of du over the rows each cluster took (a fixed set), or NULL;
// du: [rows, n] for a bias of the logits' shape, or NULL.
template <typename T, int THREADS, int VPT, bool CL>
__global__ __launch_bounds__(THREADS, 1024 / THREADS) void weights_backward_kernel(const WeightsArgs a, const float *w, const float *g,
                                                                   int64_t ld_g, T *dz, T *du, float *dbias_partial) {
    extern __shared__ unsigned dyn[];
    constexpr int kChunk = THREADS * VPT, kWarps = THREADS / 32;
    unsigned *seen = dyn, *count = dyn + kChunk / 32;
    __shared__ float warp_s[2][kWarps], block_s[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rank = CL ? cluster_rank() : 0, ranks = CL ? cluster_size() : 1;
    const int64_t c0 = static_cast<int64_t>(rank) * kChunk;
    const bool hist = a.hist > 0 && a.theta != 1.0f && dz != nullptr;  // only the repetition penalty has a slope
    if (hist) {
        for (int i = tid; i < kChunk / 32 + kChunk; i += THREADS) dyn[i] = 0u;
        __syncthreads();
    }
    float acc[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) acc[i] = 0.0f;
    int flip = 0;
    for (int64_t row = blockIdx.x / ranks; row < a.rows; row += gridDim.x / ranks, flip ^= 1) {
        if (hist) {
            history_pass<THREADS, true>(a, row, c0, kChunk, seen, count);
            __syncthreads();
        }
        float p[VPT], q[VPT], s = 0.0f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int64_t col = c0 + i * THREADS + tid;
            p[i] = col < a.n ? w[row * a.n + col] : 0.0f;
            q[i] = col < a.n ? g[row * ld_g + col] : 0.0f;
            if (p[i] == 0.0f) q[i] = 0.0f;  // a weight of 0 passes nothing on, whatever the gradient there
            s = fmaf(p[i], q[i], s);
        }
        s = warp_sum(s);
        if (lane == 0) warp_s[flip][warp] = s;
        __syncthreads();
        float dot = warp_sum(lane < kWarps ? warp_s[flip][lane] : 0.0f);
        if (CL) {
            if (tid == 0) block_s[flip] = dot;
            cluster_barrier();
            dot = warp_sum(lane < static_cast<int>(ranks) ? peer_float(&block_s[flip], lane) : 0.0f);
        }
        const T *z = static_cast<const T *>(a.logits) + row * a.ld;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = i * THREADS + tid;
            const int64_t col = c0 + c;
            if (col < a.n) {
                const float d = p[i] == 0.0f ? 0.0f : p[i] * (q[i] - dot) * a.inv_tau;
                acc[i] += d;
                if (du != nullptr) du[row * a.n + col] = from_f32<T>(d);
                if (dz != nullptr) {
                    float x = d;
                    if (hist && (seen[c >> 5] >> (c & 31)) & 1u)
                        x = to_f32<T>(z[col]) > 0.0f ? d / a.theta : d * a.theta;
                    dz[row * a.n + col] = from_f32<T>(x);
                }
            }
        }
        if (hist) {
            __syncthreads();  // the seen bits were read after the reduction's barrier
            history_pass<THREADS, false>(a, row, c0, kChunk, seen, count);
            __syncthreads();
        }
    }
    if (dbias_partial != nullptr) {
        float *out = dbias_partial + (blockIdx.x / ranks) * a.n;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int64_t col = c0 + i * THREADS + tid;
            if (col < a.n) out[col] = acc[i];
        }
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
    // 2048 threads per SM bound the rows in flight
    int64_t fit = static_cast<int64_t>(sms) * (2048 / l.threads < 32 ? 2048 / l.threads : 32) / l.ranks;
    if (l.vpt == 16) fit = fit / 2 > 0 ? fit / 2 : 1;
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

// muon.cu -- orthogonalised updates by Newton-Schulz products.
//
// X = U / (|U|_F + eps), then `steps` times X <- a X + (b A + c A^2) X with
// A = X X^T (the shorter side first): every singular value goes through the odd
// polynomial a s + b s^3 + c s^5.  The Muon step applies it to
// U = g + beta m' (or m'), m' = beta m + g:  p <- p (1 - lr wd) - lr scale O.
//
// All products run on the tensor cores with both operands as two fp16 planes
// (22 bits): what a product rounds off is amplified by up to a^steps in the
// directions of small singular values, so single 16-bit planes would lose two
// to three digits of the result on matrices whose spectrum decays (7% error
// measured on a rank-3 matrix with 0.1% noise, 2e-5 with two planes).  The
// planes are scaled by powers of two: |X| <= 1.3 entries by 2^13, A and
// b A + c A^2 by 2^12.
//
// Two forms, by the sides' ratio r = long / short, in units of 2 short^3
// operations with symmetric products at half:
//   direct: X is multiplied in every step:    steps (1.5 r + 0.5)
//   Gram:   everything but the first and last product of a segment of steps is
//           short x short: with P = a I + b A + c A^2, A <- P A P and Q <- P Q,
//           at the end X <- Q X:  1.5 r + 2 steps - 1.5 for each segment
// All the short matrices are polynomials of the first A: symmetric, so only
// their lower triangles are computed.
//
// The Gram form works with squared singular values: what A is rounded by grows
// by up to a^2 a step in the directions of small ones, and Q holds factors of up
// to a^steps beside factors of 1.  Where the singular values fall as 1 / i^2 (128
// x 256), five steps in one segment are off by 2.7e-4 and seven by 2e-2; plain
// fp32 steps by 1.0e-5 and 4.5e-5.  So a segment has at most three steps, then X
// is formed and squared again: 7.7e-6 and 3.1e-5.  Five steps cost 3 r + 7.
// Measured, Gram and direct form: 1024 x 1536 274 and 258 us, x 2048 287 and 284,
// x 4096 356 and 429, x 29649 907 and 2188; 9 x 474 x 711 281 and 235, x 950 291
// and 266, x 1422 323 and 316; 3 x 1645 x 3290 1343 and 1523.  Taken from r = 2.
//
// Matrices too small to fill a tile run whole in one block, in fp32
// multiply-adds from shared memory: 9 matrices of 24 x 25 take 15 us.
//
// Measured: 29649 x 1024 in bf16 845 us (norm 18, planes 51; two segments, each A
// in parts 98 and its product with X 186; their short products 129 and 80); a
// Muon step of 9 matrices of 1644 x 1645 2.5 ms, 2.3 ms of it products at 1.06
// PFLOP/s of matrix instructions; of 9 matrices of 474 x 475 230 us, 15 dependent
// phases of 14 us.
#include <math.h>

#include "gemm.cuh"

namespace fl {

namespace {

constexpr float kScaleX = 8192.0f, kScaleA = 4096.0f;
constexpr int kMaxParts = 1024;
constexpr int64_t kNormalizeBlocks = 888;

// What the update is made of, in the caller's orientation [m, n].
struct Source {
    Strided u;          // the update itself (dtype), or the gradient of a Muon step (fp32)
    Strided mom;        // momentum in (no pointer: a plain update)
    Strided mom_out;
    const float *gate;  // where it holds 0, momentum and parameter stay as they are; or NULL
    float beta;
    int nesterov, dtype;
    int64_t batch, nb2, m, n;
};

// The update's element (i, j); FIRST: also writes the new momentum, which the
// later passes then read.  UNIT: columns are neighbours.
template <typename T, bool MUON, bool FIRST, bool UNIT = false>
__device__ __forceinline__ float update_at(const Source &s, int64_t ub, int64_t mb, int64_t ob, int64_t i, int64_t j) {
    const float g = to_f32(static_cast<const T *>(s.u.ptr)[ub + i * s.u.i + (UNIT ? j : j * s.u.j)]);
    if (!MUON) return g;
    float *out = static_cast<float *>(s.mom_out.ptr) + ob + i * s.mom_out.i + (UNIT ? j : j * s.mom_out.j);
    float v;
    if (FIRST) {
        const float old = static_cast<const float *>(s.mom.ptr)[mb + i * s.mom.i + j * s.mom.j];
        v = s.gate != nullptr && *s.gate == 0.0f ? old : fmaf(s.beta, old, g);
        *out = v;
    } else {
        v = *out;
    }
    return s.nesterov ? fmaf(s.beta, v, g) : v;
}

// Sum of squares over the block in 64 bits, the same on every run.
__device__ __forceinline__ double block_sum(double v, double *scratch) {
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    double r = 0.0;
    for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) r += scratch[i];
    __syncthreads();
    return r;
}

// Pass 1: new momentum, and partial sums of squares of the update: grid (parts,
// batch).  Four columns a thread are in flight; the sums run in 64 bits, where
// no square of an fp32 value overflows.
// UNIT: columns are neighbours in all tensors, whose addresses then cost no
// products: 9 matrices of 1644 x 1645 (292 MB) 87 -> 56 us, 5.2 TB/s.
template <typename T, bool MUON, bool UNIT>
__global__ void __launch_bounds__(256) square_sum_kernel(const Source s, double *partial, int *counts, int n_counts) {
    const int64_t step_u = UNIT ? 1 : s.u.j, step_m = UNIT ? 1 : s.mom.j, step_o = UNIT ? 1 : s.mom_out.j;
    __shared__ double scratch[8];
    const int64_t b = blockIdx.y;
    if (blockIdx.x == 0 && b == 0)  // the products' counters of finished tiles
        for (int i = threadIdx.x; i < n_counts; i += blockDim.x) counts[i] = 0;
    const bool closed = s.gate != nullptr && *s.gate == 0.0f;
    const int64_t ub = s.u.at(b, s.nb2), mb = s.mom.at(b, s.nb2), ob = s.mom_out.at(b, s.nb2);
    double sum[4] = {0.0, 0.0, 0.0, 0.0};
    for (int64_t i = blockIdx.x; i < s.m; i += gridDim.x) {
        const T *pu = static_cast<const T *>(s.u.ptr) + ub + i * s.u.i;
        const float *pm = MUON ? static_cast<const float *>(s.mom.ptr) + mb + i * s.mom.i : nullptr;
        float *po = MUON ? static_cast<float *>(s.mom_out.ptr) + ob + i * s.mom_out.i : nullptr;
        for (int64_t j0 = threadIdx.x; j0 < s.n; j0 += 1024) {
            float g[4], v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int64_t j = j0 + 256 * q;
                const bool in = j < s.n;
                g[q] = in ? to_f32(pu[j * step_u]) : 0.0f;
                v[q] = MUON && in ? pm[j * step_m] : 0.0f;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int64_t j = j0 + 256 * q;
                float u = g[q];
                if (MUON) {
                    if (!closed) v[q] = fmaf(s.beta, v[q], g[q]);
                    if (j < s.n) po[j * step_o] = v[q];
                    u = s.nesterov ? fmaf(s.beta, v[q], g[q]) : v[q];
                }
                sum[q] = fma(static_cast<double>(u), static_cast<double>(u), sum[q]);
            }
        }
    }
    const double total = block_sum((sum[0] + sum[1]) + (sum[2] + sum[3]), scratch);
    if (threadIdx.x == 0) partial[b * gridDim.x + blockIdx.x] = total;
}

// Pass 1 of a plain update whose rows are contiguous and start on 16 bytes: a
// warp per row, four 16-byte loads in flight per lane.
template <typename T>
__global__ void __launch_bounds__(256) square_sum_rows_kernel(const Source s, double *partial, int *counts, int n_counts) {
    constexpr int kPer = 16 / sizeof(T);
    __shared__ double scratch[8];
    const int64_t b = blockIdx.y;
    if (blockIdx.x == 0 && b == 0)
        for (int i = threadIdx.x; i < n_counts; i += blockDim.x) counts[i] = 0;
    const int lane = threadIdx.x & 31;
    const T *base = static_cast<const T *>(s.u.ptr) + s.u.at(b, s.nb2);
    const int pieces = static_cast<int>(s.n / kPer);
    double sum[2] = {0.0, 0.0};
    for (int64_t i = blockIdx.x * int64_t(8) + (threadIdx.x >> 5); i < s.m; i += gridDim.x * int64_t(8)) {
        const T *row = base + i * s.u.i;
        for (int q0 = lane; q0 < pieces; q0 += 128) {
            union { uint4 u; T t[kPer]; } x[4];
#pragma unroll
            for (int q = 0; q < 4; ++q)
                x[q].u = q0 + 32 * q < pieces ? reinterpret_cast<const uint4 *>(row)[q0 + 32 * q] : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int e = 0; e < kPer; ++e) {
                    const double v = to_f32(x[q].t[e]);
                    sum[e & 1] = fma(v, v, sum[e & 1]);
                }
        }
        for (int64_t j = pieces * kPer + lane; j < s.n; j += 32) {
            const double v = to_f32(row[j]);
            sum[0] = fma(v, v, sum[0]);
        }
    }
    const double total = block_sum(sum[0] + sum[1], scratch);
    if (threadIdx.x == 0) partial[b * gridDim.x + blockIdx.x] = total;
}

// Pass 2: planes of X * 2^13, turned to [short, long]: 64 x 64 tiles, grid
// (blocks, batch); a lane holds two neighbours, so rows are written in whole
// cache lines.  9 matrices of 1644 x 1645 55 us (292 MB), 29649 x 1024 turned
// 49 us (182 MB).
template <typename T, bool MUON, bool TURNED>
__global__ void __launch_bounds__(256) normalize_kernel(const Source s, const double *partial, int parts, double eps,
                                                        double growth, int *shift, __half *out, int64_t ld, int64_t plane) {
    __shared__ double scratch[8];
    // rows of 66 words, pairs of columns exchanged in every other 16 rows: pairs are written in one
    // access, and a column is read with at most two rows to a bank
    __shared__ __align__(8) float tile[TURNED ? 64 * 66 : 1];
    auto at = [](int r, int c) { return r * 66 + (c ^ (((r >> 4) & 1) << 1)); };
    const int64_t b = blockIdx.y;
    const int64_t ub = s.u.at(b, s.nb2), ob = s.mom_out.at(b, s.nb2);
    double sum = 0.0;
    for (int p = threadIdx.y * 32 + threadIdx.x; p < parts; p += 256) sum += partial[b * parts + p];
    sum = warp_sum(sum);
    if (threadIdx.x == 0) scratch[threadIdx.y] = sum;
    __syncthreads();
    sum = 0.0;
    for (int i = 0; i < 8; ++i) sum += scratch[i];
    const double norm = sqrt(sum);
    double scale = static_cast<double>(kScaleX) / (norm + eps);
    // |X| is below 1 where eps counts; as long as the steps cannot bring it there (growth is the most they do),
    // a power of two keeps its values away from the planes' smallest
    int e = 0;
    const double room = (norm + eps) / (norm * growth);
    if (norm > 0.0 && room >= 2.0) {
        e = static_cast<int>(floor(log2(room)));
        e = e > 60 ? 60 : e;
        scale = ldexp(scale, e);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0 && threadIdx.y == 0) shift[b] = e;
    // the product in 32 bits where the scale is far from their ends
    const bool far = !(scale > 1e-30 && scale < 1e30);
    const float scale_f = far ? 0.0f : static_cast<float>(scale);
    auto scaled = [&](float v) { return far ? static_cast<float>(v * scale) : v * scale_f; };
    __half *hi = out + b * 2 * plane;
    const int64_t tiles_j = (s.n + 63) / 64, tiles = tiles_j * ((s.m + 63) / 64);
    constexpr bool kApart = TURNED && sizeof(T) == 4;
    const bool pairs = sizeof(T) == 2 && s.u.j == 1 && ((reinterpret_cast<uintptr_t>(s.u.ptr) | s.u.i * 2 | ub * 2) & 3) == 0;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int64_t i0 = t / tiles_j * 64, j0 = t % tiles_j * 64;
        float v[8][2];
        // a whole tile's loads have no conditions between them: all are in flight together
        const bool whole = i0 + 64 <= s.m && j0 + 64 <= s.n;
        if (pairs && whole) {
            const T *p = static_cast<const T *>(s.u.ptr) + ub + (i0 + threadIdx.y) * s.u.i + j0 + 2 * threadIdx.x;
            union { unsigned u; T t[4 / sizeof(T)]; } x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k].u = *reinterpret_cast<const unsigned *>(p + 8 * k * s.u.i);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[k][0] = to_f32(x[k].t[0]);
                v[k][1] = to_f32(x[k].t[sizeof(T) == 2 ? 1 : 0]);
            }
        } else {
            // two neighbours a lane; turned 32-bit tiles a lane per element (they turn in shared memory)
            const int64_t i = i0 + threadIdx.y, j = j0 + (kApart ? threadIdx.x : 2 * threadIdx.x);
            if (whole && s.u.j == 1 && (!MUON || s.mom_out.j == 1)) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
#pragma unroll
                    for (int w = 0; w < 2; ++w)
                        v[k][w] = update_at<T, MUON, false, true>(s, ub, 0, ob, i + 8 * k, j + (kApart ? 32 * w : w));
            } else if (whole) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
#pragma unroll
                    for (int w = 0; w < 2; ++w)
                        v[k][w] = update_at<T, MUON, false>(s, ub, 0, ob, i + 8 * k, j + (kApart ? 32 * w : w));
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const int64_t c = j + (kApart ? 32 * w : w);
                        v[k][w] = i + 8 * k < s.m && c < s.n ? update_at<T, MUON, false>(s, ub, 0, ob, i + 8 * k, c) : 0.0f;
                    }
            }
        }
        if (TURNED) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int r = threadIdx.y + 8 * k;
                const float x = scaled(v[k][0]), y = scaled(v[k][1]);
                if (kApart) {
                    tile[at(r, threadIdx.x)] = x;
                    tile[at(r, threadIdx.x + 32)] = y;
                } else {
                    *reinterpret_cast<float2 *>(&tile[at(r, 2 * threadIdx.x)]) = make_float2(x, y);
                }
            }
            __syncthreads();
        }
        const int64_t rows = TURNED ? s.n : s.m, cols = TURNED ? s.m : s.n, r0 = TURNED ? j0 : i0, c0 = TURNED ? i0 : j0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int64_t r = r0 + threadIdx.y + 8 * k, c = c0 + 2 * threadIdx.x;
            const float a = TURNED ? tile[at(2 * threadIdx.x, threadIdx.y + 8 * k)] : scaled(v[k][0]);
            const float z = TURNED ? tile[at(2 * threadIdx.x + 1, threadIdx.y + 8 * k)] : scaled(v[k][1]);
            if (r >= rows || c >= cols) continue;
            __half2 h, l;
            split_pair(a, z, h, l);
            // the pitch is a multiple of 8 and at least cols: the pair fits in the row
            *reinterpret_cast<__half2 *>(hi + r * ld + c) = h;
            *reinterpret_cast<__half2 *>(hi + plane + r * ld + c) = l;
        }
        if (TURNED) __syncthreads();
    }
}

template <typename T, bool MUON>
int normalize(const Source &s, bool turned, double eps, double growth, double *partial, int parts, int *counts,
              int n_counts, int *shift, __half *x, int64_t ld, int64_t plane, cudaStream_t st) {
    const int64_t size = sizeof(T);
    const bool rows = !MUON && s.u.j == 1 && reinterpret_cast<uintptr_t>(s.u.ptr) % 16 == 0 && s.u.i * size % 16 == 0 &&
                      s.u.b1 * size % 16 == 0 && s.u.b2 * size % 16 == 0;
    const dim3 parts_grid(parts, static_cast<unsigned>(s.batch));
    if (rows) launch(square_sum_rows_kernel<T>, parts_grid, 256, 0, st, s, partial, counts, n_counts);
    else if (s.u.j == 1 && (!MUON || (s.mom.j == 1 && s.mom_out.j == 1)))
        launch(square_sum_kernel<T, MUON, true>, parts_grid, 256, 0, st, s, partial, counts, n_counts);
    else launch(square_sum_kernel<T, MUON, false>, parts_grid, 256, 0, st, s, partial, counts, n_counts);
    // about six blocks per SM in all, each of several tiles: the norm is put together once per block
    const int64_t tiles = ((s.n + 63) / 64) * ((s.m + 63) / 64), most = (kNormalizeBlocks + s.batch - 1) / s.batch;
    const dim3 grid(static_cast<unsigned>(tiles < most ? tiles : most), static_cast<unsigned>(s.batch));
    if (turned) launch(normalize_kernel<T, MUON, true>, grid, dim3(32, 8), 0, st, s, partial, parts, eps, growth, shift, x, ld, plane);
    else launch(normalize_kernel<T, MUON, false>, grid, dim3(32, 8), 0, st, s, partial, parts, eps, growth, shift, x, ld, plane);
    return check_launch("newton-schulz normalize");
}

struct Finish {
    Strided out, base;  // out = factor * O + keep * base, or base where the gate is closed
    const float *gate;
    float factor, keep;
    int dtype;
};

__device__ __forceinline__ void store_any(void *p, int64_t at, float v, int dtype) {
    if (dtype == kOutF32) static_cast<float *>(p)[at] = v;
    else if (dtype == kOutF16) static_cast<__half *>(p)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p)[at] = __float2bfloat16_rn(v);
}

// C[i, j] = sum_k A[i, k] * (B_T ? B[j, k] : B[k, j]) from shared memory: 2 x 2
// outputs a thread, rows and columns strided so that neighbours read neighbours.
template <bool B_T, typename F>
__device__ __forceinline__ void small_product(const float *A, int lda, const float *B, int ldb, int rows, int cols,
                                              int depth, F store) {
    const int rh = (rows + 1) / 2, ch = (cols + 1) / 2;
    for (int t = threadIdx.x; t < rh * ch; t += blockDim.x) {
        const int i0 = t / ch, j0 = t - i0 * ch, i1 = i0 + rh, j1 = j0 + ch;
        const int i1c = i1 < rows ? i1 : i0, j1c = j1 < cols ? j1 : j0;
        float s00 = 0.0f, s01 = 0.0f, s10 = 0.0f, s11 = 0.0f;
#pragma unroll 8
        for (int k = 0; k < depth; ++k) {
            const float a0 = A[i0 * lda + k], a1 = A[i1c * lda + k];
            const float b0 = B_T ? B[j0 * ldb + k] : B[k * ldb + j0], b1 = B_T ? B[j1c * ldb + k] : B[k * ldb + j1c];
            s00 = fmaf(a0, b0, s00);
            s01 = fmaf(a0, b1, s01);
            s10 = fmaf(a1, b0, s10);
            s11 = fmaf(a1, b1, s11);
        }
        store(i0, j0, s00);
        if (j1 < cols) store(i0, j1, s01);
        if (i1 < rows) store(i1, j0, s10);
        if (i1 < rows && j1 < cols) store(i1, j1, s11);
    }
}

// The whole step of one small matrix in one block.
template <typename T, bool MUON>
__global__ void __launch_bounds__(512) small_kernel(const Source s, const Finish f, int turned, int lo, int hi,
                                                    int steps, float ca, float cb, float cc, double eps) {
    extern __shared__ float sm[];
    __shared__ double scratch[16];
    const int ldx = hi | 1, lda = lo | 1;  // odd pitches: columns fall into different banks
    float *X = sm, *Y = X + lo * ldx, *A = Y + lo * ldx, *B = A + lo * lda;
    const int64_t b = blockIdx.x;
    const int64_t ub = s.u.at(b, s.nb2), mb = s.mom.at(b, s.nb2), ob = s.mom_out.at(b, s.nb2);
    const int m = static_cast<int>(s.m), n = static_cast<int>(s.n);
    double sum = 0.0;
    for (int t = threadIdx.x; t < m * n; t += blockDim.x) {
        const int i = t / n, j = t - i * n;
        const float v = update_at<T, MUON, true>(s, ub, mb, ob, i, j);
        sum = fma(static_cast<double>(v), static_cast<double>(v), sum);
        X[turned ? j * ldx + i : i * ldx + j] = v;
    }
    sum = block_sum(sum, scratch);
    const double scale = 1.0 / (sqrt(sum) + eps);
    for (int t = threadIdx.x; t < lo * hi; t += blockDim.x) {
        const int i = t / hi, j = t - i * hi;
        X[i * ldx + j] = static_cast<float>(X[i * ldx + j] * scale);
    }
    __syncthreads();
    for (int k = 0; k < steps; ++k) {
        small_product<true>(X, ldx, X, ldx, lo, lo, hi, [&](int i, int j, float v) { A[i * lda + j] = v; });
        __syncthreads();
        small_product<true>(A, lda, A, lda, lo, lo, lo,
                            [&](int i, int j, float v) { B[i * lda + j] = fmaf(cc, v, cb * A[i * lda + j]); });
        __syncthreads();
        small_product<false>(B, lda, X, ldx, lo, hi, lo,
                             [&](int i, int j, float v) { Y[i * ldx + j] = fmaf(ca, X[i * ldx + j], v); });
        __syncthreads();
        float *t = X;
        X = Y;
        Y = t;
    }
    const int64_t fb = f.out.at(b, s.nb2), bb = f.base.at(b, s.nb2);
    for (int t = threadIdx.x; t < m * n; t += blockDim.x) {
        const int i = t / n, j = t - i * n;
        float v = f.factor * X[turned ? j * ldx + i : i * ldx + j];
        if (f.base.ptr != nullptr) {
            const float old = static_cast<const float *>(f.base.ptr)[bb + i * f.base.i + j * f.base.j];
            v = f.gate != nullptr && *f.gate == 0.0f ? old : fmaf(f.keep, old, v);
        }
        store_any(f.out.ptr, fb + i * f.out.i + j * f.out.j, v, f.dtype);
    }
}

size_t small_smem(int64_t lo, int64_t hi) { return (2 * lo * (hi | 1) + 2 * lo * (lo | 1)) * sizeof(float); }

// One block holds the matrix, and its products (fp32 multiply-adds on one SM)
// take no longer than the tensor path's launches.
bool is_small(int64_t lo, int64_t hi, int steps) {
    return small_smem(lo, hi) <= 200 * 1024 && steps * lo * lo * (2 * hi + lo) <= 2500000;
}

bool use_gram(int64_t lo, int64_t hi, int steps) {
    const double r = static_cast<double>(hi) / static_cast<double>(lo);
    return r >= 2.0 && ns_segments(steps, 1) * (1.5 * r - 1.5) + 2.0 * steps < steps * (1.5 * r + 0.5);
}

int parts_of(int64_t batch, int64_t m) {
    int64_t p = (148 * 8 + batch - 1) / batch;
    if (p > m) p = m;
    if (p > kMaxParts) p = kMaxParts;
    return static_cast<int>(p);
}

// Largest |x|, |A|, |b A + c A^2|, |A P| and |Q| (the factor of a segment of the
// Gram form) over singular values in [0, 1]: what the fp16 planes have to hold.
// growth: the largest factor of all steps.
struct Range {
    double x, a, b, ap, q, growth;
};
Range polynomial_range(double ca, double cb, double cc, int steps) {
    // a function of four numbers that a program hardly ever changes: the last answer is kept
    thread_local double key[4] = {0, 0, 0, -1};
    thread_local Range r;
    if (key[0] == ca && key[1] == cb && key[2] == cc && key[3] == steps) return r;
    key[0] = ca;
    key[1] = cb;
    key[2] = cc;
    key[3] = steps;
    r = Range{0, 0, 0, 0, 0, 0};
    const int segments = ns_segments(steps, 1);
    for (int i = 0; i <= 4096; ++i) {
        double x = i / 4096.0, q = 1.0, growth = 1.0;
        for (int k = 0, segment = 0, left = 0; k < steps; ++k, --left) {
            if (left == 0) {
                left = ns_segment_steps(steps, segments, segment++);
                q = 1.0;
            }
            const double t = x * x, bt = cb * t + cc * t * t, p = ca + bt;
            r.x = fmax(r.x, fabs(x));
            r.a = fmax(r.a, t);
            r.b = fmax(r.b, fabs(bt));
            r.ap = fmax(r.ap, fabs(t * p));
            x *= p;
            q *= p;
            growth *= p;
            r.q = fmax(r.q, fabs(q));
            r.growth = fmax(r.growth, fabs(growth));
            if (!(fabs(x) < 1e6)) { r.x = 1e6; return r; }
        }
        r.x = fmax(r.x, fabs(x));
    }
    return r;
}

NsBuffer take_planes(Carve &ws, int64_t batch, int64_t rows, int64_t cols) {
    NsBuffer b;
    b.ld = pitch_of(cols);
    b.plane = rows * b.ld;
    b.p = ws.take<__half>(batch * 2 * b.plane);
    return b;
}
size_t planes_bytes(int64_t batch, int64_t rows, int64_t cols) {
    return carve_bytes<__half>(batch * 2 * rows * pitch_of(cols));
}

Strided turn(Strided s, bool turned) {
    if (turned) { const int64_t t = s.i; s.i = s.j; s.j = t; }
    return s;
}

template <typename T, bool MUON>
int run_small(const Source &s, const Finish &f, bool turned, int64_t lo, int64_t hi, int steps, float a, float b, float c,
              double eps, cudaStream_t st) {
    auto kernel = small_kernel<T, MUON>;
    FL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
    launch(kernel, static_cast<unsigned>(s.batch), lo * hi >= 2048 ? 512 : 256, small_smem(lo, hi), st, s, f,
           static_cast<int>(turned), static_cast<int>(lo), static_cast<int>(hi), steps, a, b, c, eps);
    return check_launch("newton-schulz");
}

int newton_schulz(const Source &s, const Finish &f, int steps, double ca, double cb, double cc, double eps, void *wsp,
                  size_t ws_bytes, cudaStream_t st) {
    const bool turned = s.m > s.n;
    const int64_t lo = turned ? s.n : s.m, hi = turned ? s.m : s.n;
    const Range r = polynomial_range(ca, cb, cc, steps);
    FL_REQUIRE(r.x <= 3.0 && r.b <= 12.0 && r.ap <= 12.0 && r.q < 1e9,
               "newton-schulz: these coefficients do not keep singular values of [0, 1] within 3");
    const float fa = static_cast<float>(ca), fb = static_cast<float>(cb), fc = static_cast<float>(cc);
    if (is_small(lo, hi, steps)) {
        if (s.mom_out.ptr != nullptr) return run_small<float, true>(s, f, turned, lo, hi, steps, fa, fb, fc, eps, st);
        if (s.dtype == FL_F32) return run_small<float, false>(s, f, turned, lo, hi, steps, fa, fb, fc, eps, st);
        if (s.dtype == FL_F16) return run_small<__half, false>(s, f, turned, lo, hi, steps, fa, fb, fc, eps, st);
        return run_small<__nv_bfloat16, false>(s, f, turned, lo, hi, steps, fa, fb, fc, eps, st);
    }
    FL_REQUIRE(s.batch <= 65535, "newton-schulz: at most 65535 matrices that one block cannot hold");
    Carve ws(wsp, ws_bytes);
    const int parts = parts_of(s.batch, s.m);
    const bool gram = use_gram(lo, hi, steps);
    const int n_counts = ns_phases(steps, gram) * static_cast<int>(s.batch);
    double *partial = ws.take<double>(s.batch * parts);
    int *counts = ws.take<int>(n_counts), *shift = ws.take<int>(s.batch);
    NsBuffer buf[kNsBuffers] = {};
    bool fits = partial != nullptr && counts != nullptr && shift != nullptr;
    for (int i = 0; i < kNsBuffers; ++i) {
        if (gram ? i == kNsX2 && ns_segments(steps, 1) == 1 : i >= kNsQ) continue;
        buf[i] = take_planes(ws, s.batch, lo, i <= kNsX2 ? hi : lo);
        fits = fits && buf[i].p != nullptr;
    }
    const size_t part_bytes = gram ? ns_parts_bytes(lo, hi, s.batch) : 0;
    float *outer_parts = part_bytes ? ws.take<float>(part_bytes / sizeof(float)) : nullptr;
    FL_REQUIRE(fits && (part_bytes == 0 || outer_parts != nullptr), "newton-schulz: workspace too small");
    const NsBuffer &x = buf[kNsX];
    int rc;
    if (s.mom_out.ptr != nullptr)
        rc = normalize<float, true>(s, turned, eps, r.growth, partial, parts, counts, n_counts, shift, x.p, x.ld, x.plane, st);
    else if (s.dtype == FL_F32)
        rc = normalize<float, false>(s, turned, eps, r.growth, partial, parts, counts, n_counts, shift, x.p, x.ld, x.plane, st);
    else if (s.dtype == FL_F16)
        rc = normalize<__half, false>(s, turned, eps, r.growth, partial, parts, counts, n_counts, shift, x.p, x.ld, x.plane, st);
    else
        rc = normalize<__nv_bfloat16, false>(s, turned, eps, r.growth, partial, parts, counts, n_counts, shift, x.p, x.ld, x.plane, st);
    if (rc) return rc;
    NsProgram p{};
    p.lo = static_cast<int>(lo);
    p.hi = static_cast<int>(hi);
    p.batch = static_cast<int>(s.batch);
    p.steps = steps;
    p.gram = gram;
    p.shift = shift;
    p.a = fa;
    p.b = fb;
    p.c = fc;
    p.scale_x = kScaleX;
    p.scale_a = kScaleA;
    // Q's scale leaves room for its largest factor (a^steps of a segment in the null space)
    p.scale_q = exp2f(floorf(log2f(32768.0f / static_cast<float>(r.q))));
    p.factor = f.factor;
    p.final.out = turn(f.out, turned);
    p.final.base = turn(f.base, turned);
    p.final.gate = f.gate;
    p.final.keep = f.keep;
    p.final.nb2 = s.nb2;
    p.final.dtype = f.dtype;
    return ns_products(p, buf, counts, outer_parts, st);
}

Strided strided(const fl_matrices *t) {
    if (t == nullptr) return Strided{nullptr, 0, 0, 0, 0};
    return Strided{t->ptr, t->stride_b1, t->stride_b2, t->stride_i, t->stride_j};
}

int check_batch(int64_t b1, int64_t b2, int64_t m, int64_t n, int steps) {
    FL_REQUIRE(b1 >= 0 && b2 >= 0 && m > 0 && n > 0 && m < (1 << 24) && n < (1 << 24), "newton-schulz: bad shape");
    FL_REQUIRE(steps >= 1 && steps <= 64, "newton-schulz: 1 to 64 steps");
    return FL_OK;
}

}  // namespace
}  // namespace fl

using namespace fl;

extern "C" {

size_t fl_newton_schulz_workspace(int64_t batch, int64_t m, int64_t n, int steps) {
    if (batch <= 0 || m <= 0 || n <= 0) return 0;
    const int64_t lo = m < n ? m : n, hi = m < n ? n : m;
    if (is_small(lo, hi, steps)) return 0;
    const bool gram = use_gram(lo, hi, steps);
    size_t b = carve_bytes<double>(batch * parts_of(batch, m)) + carve_bytes<int>(ns_phases(steps, gram) * batch) +
               carve_bytes<int>(batch);
    b += (gram && ns_segments(steps, 1) == 1 ? 1 : 2) * planes_bytes(batch, lo, hi) +
         (gram ? 5 : 2) * planes_bytes(batch, lo, lo);
    return b + (gram ? ns_parts_bytes(lo, hi, batch) + 512 : 0);
}

int fl_orthogonalize(const fl_matrices *in, const fl_matrices *out, int64_t b1, int64_t b2, int64_t m, int64_t n,
                     int dtype, int steps, double a, double b, double c, double eps, void *ws, size_t ws_bytes,
                     fl_stream_t stream) {
    int rc = check_batch(b1, b2, m, n, steps);
    if (rc) return rc;
    FL_REQUIRE(dtype == FL_F32 || dtype == FL_F16 || dtype == FL_BF16, "orthogonalize: bad dtype %d", dtype);
    if (b1 * b2 == 0) return FL_OK;
    FL_REQUIRE(in != nullptr && out != nullptr && in->ptr != nullptr && out->ptr != nullptr, "orthogonalize: null matrix");
    Source s{};
    s.u = strided(in);
    s.dtype = dtype;
    s.batch = b1 * b2;
    s.nb2 = b2;
    s.m = m;
    s.n = n;
    Finish f{};
    f.out = strided(out);
    f.factor = 1.0f;
    f.dtype = dtype;
    return newton_schulz(s, f, steps, a, b, c, eps, ws, ws_bytes, as_stream(stream));
}

int fl_muon_update(const fl_matrices *param, const fl_matrices *grad, const fl_matrices *momentum,
                   const fl_matrices *param_out, const fl_matrices *momentum_out, int64_t b1, int64_t b2, int64_t m,
                   int64_t n, double lr, double beta, int nesterov, double weight_decay, double scale, int steps,
                   double a, double b, double c, double eps, const float *gate, void *ws, size_t ws_bytes,
                   fl_stream_t stream) {
    int rc = check_batch(b1, b2, m, n, steps);
    if (rc) return rc;
    if (b1 * b2 == 0) return FL_OK;
    FL_REQUIRE(param && grad && momentum && param_out && momentum_out && param->ptr && grad->ptr && momentum->ptr &&
                   param_out->ptr && momentum_out->ptr,
               "muon_update: null matrix");
    Source s{};
    s.u = strided(grad);
    s.mom = strided(momentum);
    s.mom_out = strided(momentum_out);
    s.gate = gate;
    s.beta = static_cast<float>(beta);
    s.nesterov = nesterov;
    s.dtype = FL_F32;
    s.batch = b1 * b2;
    s.nb2 = b2;
    s.m = m;
    s.n = n;
    Finish f{};
    f.out = strided(param_out);
    f.base = strided(param);
    f.gate = gate;
    f.factor = static_cast<float>(-lr * scale);
    f.keep = static_cast<float>(1.0 - lr * weight_decay);
    f.dtype = FL_F32;
    return newton_schulz(s, f, steps, a, b, c, eps, ws, ws_bytes, as_stream(stream));
}

}  // extern "C"

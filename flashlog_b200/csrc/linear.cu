// linear.cu -- the relation head: y = act(x W^T + bias) + residual and its
// gradients, on the tcgen05 product of gemm.cu.
//
// fp32 operands are split into two fp16 planes, hi + lo, after scaling each
// line of the uncontracted index by a power of two that brings its largest
// value to [2^14, 2^15): no line can lose bits to another line's size.  lo is
// held 2048 times as large, where it reaches as far down as hi: a value keeps 22
// bits down to 2^-29 of its line's largest, and is off by at most 2^-50 of that
// below.  Scale and exponents are undone in the product's epilogue; the cross
// products have an accumulator of their own anyway.
#include "gemm.cuh"

namespace fl {

namespace {

constexpr int kSumRows = 128;  // rows per partial column sum
constexpr float kLoScale = 2048.0f;

int elem_size(int dtype) { return dtype == FL_F32 ? 4 : 2; }

// exponent e with max * 2^-e in [2^14, 2^15); 0 for a zero or non-finite line
__device__ __forceinline__ int line_exponent(float absmax) {
    if (!(absmax > 0.0f) || !(absmax <= 3.402823466e38f)) return 0;
    int e = ((__float_as_int(absmax) >> 23) & 255) - 127;
    if (e < -100) e = -100;  // subnormal or tiny lines: 2^-e stays representable
    return e - 14;
}

__device__ __forceinline__ void split_scaled(float v, int e, __half &hi, __half &lo) {
    const float s = scale_pow2(v, -e);
    hi = __float2half_rn(s);
    lo = __float2half_rn((s - __half2float(hi)) * kLoScale);
}

__device__ __forceinline__ float block_max(float v, float *scratch) {
    v = warp_max(v);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    float r = scratch[0];
    for (int i = 1; i < static_cast<int>(blockDim.x >> 5); ++i) r = fmaxf(r, scratch[i]);
    __syncthreads();
    return r;
}

// One block per row: the row's exponent, then its planes (second read from
// L1/L2).  One or two matrices per launch.
struct PackRows {
    const float *src;
    int64_t ld, rows;
    __half *out;
    int64_t plane;
    int *exps;
};
__global__ void pack_rows_kernel(const PackRows a, const PackRows b, int64_t cols, int64_t ldp) {
    __shared__ float scratch[32];
    const bool second = static_cast<int64_t>(blockIdx.x) >= a.rows;
    const PackRows &p = second ? b : a;
    const int64_t r = second ? blockIdx.x - a.rows : blockIdx.x, ld = p.ld, plane = p.plane;
    const float *src = p.src, *row = src + r * ld;
    __half *out = p.out;
    int *exps = p.exps;
    const bool vec = ((reinterpret_cast<uintptr_t>(src) & 15) == 0) && (ld & 3) == 0;
    const int64_t quads = vec ? cols >> 2 : 0;
    float mx = 0.0f;
    for (int64_t q = threadIdx.x; q < quads; q += blockDim.x) {
        const float4 v = reinterpret_cast<const float4 *>(row)[q];
        mx = fmaxf(fmaxf(fmaxf(mx, fabsf(v.x)), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
    }
    for (int64_t c = quads * 4 + threadIdx.x; c < cols; c += blockDim.x) mx = fmaxf(mx, fabsf(row[c]));
    const int e = line_exponent(block_max(mx, scratch));
    if (threadIdx.x == 0) exps[r] = e;
    __half *hi = out + r * ldp, *lo = hi + plane;
    for (int64_t q = threadIdx.x; q < quads; q += blockDim.x) {
        const float4 v = reinterpret_cast<const float4 *>(row)[q];
        union { __half h[4]; uint2 u; } a, b;
        split_scaled(v.x, e, a.h[0], b.h[0]);
        split_scaled(v.y, e, a.h[1], b.h[1]);
        split_scaled(v.z, e, a.h[2], b.h[2]);
        split_scaled(v.w, e, a.h[3], b.h[3]);
        reinterpret_cast<uint2 *>(hi)[q] = a.u;
        reinterpret_cast<uint2 *>(lo)[q] = b.u;
    }
    for (int64_t c = quads * 4 + threadIdx.x; c < cols; c += blockDim.x) {
        __half x, y;
        split_scaled(row[c], e, x, y);
        hi[c] = x;
        lo[c] = y;
    }
}

// Rows of at most 1024 values that start on 16 bytes: a warp per row, which
// stays in its registers, and nothing to wait for but its loads (4608 + 1645
// rows of 1024: 9 us, the block form 14 us).
constexpr int kWarpCols = 1024;
__global__ void __launch_bounds__(128) pack_short_rows_kernel(const PackRows a, const PackRows b, int64_t cols, int64_t ldp) {
    int64_t r = blockIdx.x * int64_t(4) + (threadIdx.x >> 5);
    const bool second = r >= a.rows;
    const PackRows &p = second ? b : a;
    if (second) r -= a.rows;
    if (second && r >= b.rows) return;
    const int lane = threadIdx.x & 31, quads = static_cast<int>(cols >> 2), rest = static_cast<int>(cols & 3);
    const float *row = p.src + r * p.ld;
    float4 v[kWarpCols / 128];
#pragma unroll
    for (int i = 0; i < kWarpCols / 128; ++i)
        v[i] = lane + 32 * i < quads ? reinterpret_cast<const float4 *>(row)[lane + 32 * i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float tail = lane < rest ? row[quads * 4 + lane] : 0.0f;
    float mx = fabsf(tail);
#pragma unroll
    for (int i = 0; i < kWarpCols / 128; ++i)
        mx = fmaxf(fmaxf(fmaxf(mx, fabsf(v[i].x)), fabsf(v[i].y)), fmaxf(fabsf(v[i].z), fabsf(v[i].w)));
    const int e = line_exponent(warp_max(mx));
    if (lane == 0) p.exps[r] = e;
    __half *hi = p.out + r * ldp, *lo = hi + p.plane;
#pragma unroll
    for (int i = 0; i < kWarpCols / 128; ++i) {
        union { __half h[4]; uint2 u; } x, y;
        split_scaled(v[i].x, e, x.h[0], y.h[0]);
        split_scaled(v[i].y, e, x.h[1], y.h[1]);
        split_scaled(v[i].z, e, x.h[2], y.h[2]);
        split_scaled(v[i].w, e, x.h[3], y.h[3]);
        if (lane + 32 * i < quads) {
            reinterpret_cast<uint2 *>(hi)[lane + 32 * i] = x.u;
            reinterpret_cast<uint2 *>(lo)[lane + 32 * i] = y.u;
        }
    }
    if (lane < rest) split_scaled(tail, e, hi[quads * 4 + lane], lo[quads * 4 + lane]);
}

int pack_rows(const PackRows &a, const PackRows &b, int64_t cols, int64_t ldp, cudaStream_t st) {
    auto ready = [](const PackRows &p) { return (reinterpret_cast<uintptr_t>(p.src) & 15) == 0 && (p.ld & 3) == 0; };
    const int64_t rows = a.rows + b.rows;
    FL_REQUIRE(rows < (1ll << 31), "linear: bad shape");
    if (cols <= kWarpCols && ready(a) && (b.rows == 0 || ready(b)))
        launch(pack_short_rows_kernel, static_cast<unsigned>((rows + 3) / 4), 128, 0, st, a, b, cols, ldp);
    else
        launch(pack_rows_kernel, static_cast<unsigned>(rows), cols > 2048 ? 512 : 128, 0, st, a, b, cols, ldp);
    return check_launch("linear pack");
}

// Largest |value| of each column, as fp32 bits (order-independent): a block
// takes 32 columns x a range of rows.
__global__ void col_absmax_kernel(const float *src, int64_t ld, int64_t rows, int64_t cols, int64_t chunk,
                                  unsigned *out) {
    __shared__ float part[8][33];
    const int64_t c = blockIdx.x * int64_t(32) + threadIdx.x;
    const int64_t r0 = blockIdx.y * chunk, r1 = min(rows, r0 + chunk);
    float mx = 0.0f;
    if (c < cols)
        for (int64_t r = r0 + threadIdx.y; r < r1; r += 8) mx = fmaxf(mx, fabsf(src[r * ld + c]));
    part[threadIdx.y][threadIdx.x] = mx;
    __syncthreads();
    if (threadIdx.y == 0 && c < cols) {
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = fmaxf(mx, part[i][threadIdx.x]);
        atomicMax(out + c, __float_as_uint(mx));
    }
}

// Planes of a matrix scaled per column; 64 columns x 32 rows per block.  The
// first rows' blocks also write the exponents.
__global__ void pack_cols_kernel(const float *src, int64_t ld, int64_t rows, int64_t cols, const unsigned *bits, int *exps,
                                 __half *out, int64_t ldp, int64_t plane) {
    const int64_t c = blockIdx.x * int64_t(64) + 2 * threadIdx.x;
    if (c >= cols) return;
    const int e0 = line_exponent(__uint_as_float(bits[c]));
    const int e1 = c + 1 < cols ? line_exponent(__uint_as_float(bits[c + 1])) : 0;
    if (exps != nullptr && blockIdx.y == 0 && threadIdx.y == 0) {
        exps[c] = e0;
        if (c + 1 < cols) exps[c + 1] = e1;
    }
    const bool vec = ((reinterpret_cast<uintptr_t>(src) & 7) == 0) && (ld & 1) == 0 && c + 1 < cols;
    const int64_t r1 = min(rows, (blockIdx.y + int64_t(1)) * 32);
    for (int64_t r = blockIdx.y * int64_t(32) + threadIdx.y; r < r1; r += 8) {
        const float *p = src + r * ld + c;
        float2 v;
        if (vec) v = *reinterpret_cast<const float2 *>(p);
        else v = make_float2(p[0], c + 1 < cols ? p[1] : 0.0f);
        union { __half h[2]; unsigned u; } a, b;
        split_scaled(v.x, e0, a.h[0], b.h[0]);
        split_scaled(v.y, e1, a.h[1], b.h[1]);
        // the pitch is a multiple of 8 and at least cols: the pair fits in the row
        *reinterpret_cast<unsigned *>(out + r * ldp + c) = a.u;
        *reinterpret_cast<unsigned *>(out + plane + r * ldp + c) = b.u;
    }
}

// 16-bit rows copied to an aligned pitch (rows whose pitch or base TMA cannot
// take): a warp per row, two values a lane, eight such pairs in flight (23734 x
// 572: 12.6 us; a block per row took 28.7).
__global__ void __launch_bounds__(256) pack16_kernel(const uint16_t *src, int64_t ld, int64_t rows, int64_t cols,
                                                     uint16_t *out, int64_t ldp) {
    constexpr int U = 8;
    const int64_t r = blockIdx.x * int64_t(8) + (threadIdx.x >> 5);
    if (r >= rows) return;
    const uint16_t *p = src + r * ld;
    uint16_t *o = out + r * ldp;
    for (int64_t c0 = 2 * (threadIdx.x & 31); c0 < cols; c0 += 64 * U) {
        unsigned a[U], b[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int64_t c = c0 + 64 * i;
            a[i] = c < cols ? p[c] : 0u;
            b[i] = c + 1 < cols ? p[c + 1] : 0u;
        }
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (c0 + 64 * i < cols) *reinterpret_cast<unsigned *>(o + c0 + 64 * i) = a[i] | (b[i] << 16);
    }
}

// Eight values from p on.  Rows need not start on 16 bytes: a lane reads the
// aligned 16-byte pieces around its values (pieces_load) and turns them into
// place (pieces_turn).
template <typename T>
struct Pieces {
    static constexpr int kCount = 8 * sizeof(T) / 16 + 1;
    uint4 w[kCount];
};
template <typename T>
__device__ __forceinline__ const char *pieces_at(const T *p) {
    return reinterpret_cast<const char *>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(15));
}
template <typename T>
__device__ __forceinline__ void pieces_load(const T *p, Pieces<T> &x) {
    const uint4 *base = reinterpret_cast<const uint4 *>(pieces_at(p));
    const bool aligned = (reinterpret_cast<uintptr_t>(p) & 15) == 0;  // then the last piece is not needed
#pragma unroll
    for (int i = 0; i < Pieces<T>::kCount; ++i) x.w[i] = base[aligned && i == Pieces<T>::kCount - 1 ? i - 1 : i];
}
template <typename T>
__device__ __forceinline__ void pieces_turn(const T *p, const Pieces<T> &x, float (&d)[8]) {
    constexpr int kWords = 4 * Pieces<T>::kCount, kPer = 4 / sizeof(T);
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15);
    unsigned c[kWords];
#pragma unroll
    for (int i = 0; i < Pieces<T>::kCount; ++i)
        c[4 * i] = x.w[i].x, c[4 * i + 1] = x.w[i].y, c[4 * i + 2] = x.w[i].z, c[4 * i + 3] = x.w[i].w;
    if ((off & 4) != 0) {
#pragma unroll
        for (int i = 0; i < kWords - 1; ++i) c[i] = c[i + 1];
    }
    if ((off & 8) != 0) {
#pragma unroll
        for (int i = 0; i < kWords - 2; ++i) c[i] = c[i + 2];
    }
#pragma unroll
    for (int i = 0; i < 8 / kPer; ++i) {
        union { unsigned u; T t[kPer]; } y;
        y.u = sizeof(T) == 2 ? __funnelshift_r(c[i], c[i + 1], 8 * (off & 3)) : c[i];
#pragma unroll
        for (int k = 0; k < kPer; ++k) d[i * kPer + k] = to_f32<T>(y.t[k]);
    }
}

// dz of a 16-bit head with an activation, as the products take it: two planes of
// the operands' type, dz = first * hi + second * lo.  One plane would add a
// rounding of 2^-8 (2^-11 in fp16, and more below its smallest normal value) to
// each term of both products, as much as the result's own: the error of dx and
// dweight 1.4 times as large.  fp16 holds half of dz, which may pass its largest
// value, and 2048 times what is left, which then lies as far above its smallest
// as hi does.  The product takes the planes in turn: twice its matrix
// instructions (a step of 4608 x 1024 -> 29649 with SiLU 1394 -> 1802 us).
template <typename T> struct DzPlanes { static constexpr float first = 1.0f, second = 1.0f; };
template <> struct DzPlanes<__half> { static constexpr float first = 2.0f, second = 1.0f / 1024.0f; };
template <typename T>
__device__ __forceinline__ void dz_split(float d, T &hi, T &lo) {
    const float s = d * (1.0f / DzPlanes<T>::first);
    hi = from_f32<T>(s);
    const float rest = s - to_f32<T>(hi);  // NaN where hi is not finite: lo adds nothing there
    lo = from_f32<T>(rest == rest ? rest * (DzPlanes<T>::first / DzPlanes<T>::second) : 0.0f);
}

// dz = gy * act'(z), written as T with pitch ldo (or not at all; in two planes,
// `plane` elements apart, where plane is not 0), and its column sums over
// kSumRows rows at a time, taken before the rounding.  A lane takes eight neighbouring columns of four rows, all in flight, and stores whole
// pieces: 4608 x 29649 in bf16, copied to an aligned pitch, 120 us (546 MB, 4.6
// TB/s), where single 16-bit loads and stores took 405 us and single loads alone
// 167 us.
template <typename T>
__global__ void __launch_bounds__(256) dz_kernel(const T *gy, int64_t ld_gy, const float *z, int64_t rows, int64_t n, int act,
                                                 T *out, int64_t ldo, int64_t plane, float *partial) {
    __shared__ float part[8][256];
    constexpr int U = 4;  // rows in flight
    const int64_t c0 = blockIdx.x * int64_t(256) + 8 * threadIdx.x;
    const int64_t r0 = blockIdx.y * int64_t(kSumRows), r1 = min(rows, r0 + kSumRows);
    const int left = c0 < n ? static_cast<int>(min(static_cast<int64_t>(8), n - c0)) : 0;
    const char *const first = reinterpret_cast<const char *>(gy);
    const char *const last = reinterpret_cast<const char *>(gy + (rows - 1) * ld_gy + n);
    float sum[8] = {};
    for (int64_t r = r0 + threadIdx.y; r < r1; r += 8 * U) {
        const T *p = gy + r * ld_gy + c0;
        float d[U][8];
        // eight columns of all rows exist, and no piece leaves the array
        if (left == 8 && r + 8 * (U - 1) < r1 && pieces_at(p) >= first &&
            pieces_at(p + 8 * (U - 1) * ld_gy) + 16 * Pieces<T>::kCount <= last) {
            Pieces<T> x[U];
#pragma unroll
            for (int k = 0; k < U; ++k) pieces_load(p + 8 * k * ld_gy, x[k]);
#pragma unroll
            for (int k = 0; k < U; ++k) pieces_turn(p + 8 * k * ld_gy, x[k], d[k]);
        } else {
#pragma unroll
            for (int k = 0; k < U; ++k)
#pragma unroll
                for (int w = 0; w < 8; ++w) d[k][w] = r + 8 * k < r1 && w < left ? to_f32<T>(p[8 * k * ld_gy + w]) : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            if (r + 8 * k >= r1 || left <= 0) continue;
            if (act != kActNone) {
                const float *pz = z + (r + 8 * k) * n + c0;
#pragma unroll
                for (int w = 0; w < 8; ++w)
                    if (w < left) d[k][w] *= act_slope(pz[w], act);
            }
            if (out != nullptr) {
                // the pitch is a multiple of 8: the whole piece lies in the row
                struct alignas(16) Vec { T t[8]; } v, lo;
                if (sizeof(T) == 2 && plane != 0) {
#pragma unroll
                    for (int w = 0; w < 8; ++w) dz_split<T>(d[k][w], v.t[w], lo.t[w]);
                    *reinterpret_cast<Vec *>(out + plane + (r + 8 * k) * ldo + c0) = lo;
                } else {
#pragma unroll
                    for (int w = 0; w < 8; ++w) v.t[w] = from_f32<T>(d[k][w]);
                }
                *reinterpret_cast<Vec *>(out + (r + 8 * k) * ldo + c0) = v;
            }
#pragma unroll
            for (int w = 0; w < 8; ++w) sum[w] += d[k][w];
        }
    }
    if (partial == nullptr) return;
#pragma unroll
    for (int w = 0; w < 8; ++w) part[threadIdx.y][8 * threadIdx.x + w] = sum[w];
    __syncthreads();
    const int c = threadIdx.y * 32 + threadIdx.x;
    if (blockIdx.x * int64_t(256) + c < n) {
        float s = part[0][c];
#pragma unroll
        for (int i = 1; i < 8; ++i) s += part[i][c];
        partial[blockIdx.y * n + blockIdx.x * int64_t(256) + c] = s;
    }
}

template <typename T>
__global__ void sum_partials_kernel(const float *partial, int64_t parts, int64_t n, T *out) {
    const int64_t c = blockIdx.x * int64_t(blockDim.x) + threadIdx.x;
    if (c >= n) return;
    float s = 0.0f;
    for (int64_t p = 0; p < parts; ++p) s += partial[p * n + c];
    out[c] = from_f32<T>(s);
}

// ---- small products in fp32 multiply-adds ------------------------------------
// Up to a few hundred million operations the tensor path's launches (two packs
// and a product, about 12 us for fp32) cost more than the arithmetic: these
// kernels read the operands as they are and take one launch.

// Few rows: a warp takes four columns of W for all R rows, its lanes along k.
// Every element of W is read once and used R times from registers; the rows of
// x come from L1.
template <typename T, int R, int V>
__global__ void __launch_bounds__(256) few_rows_kernel(const fl_linear p, void *y, int64_t ld_y, float *z) {
    const int lane = threadIdx.x & 31;
    const int64_t j0 = (blockIdx.x * int64_t(8) + (threadIdx.x >> 5)) * 4;
    if (j0 >= p.n) return;
    const int64_t r0 = blockIdx.y * int64_t(R);
    const T *x = static_cast<const T *>(p.x), *w = static_cast<const T *>(p.w);
    const T *wj[4], *xr[R];
#pragma unroll
    for (int c = 0; c < 4; ++c) wj[c] = w + (j0 + c < p.n ? j0 + c : p.n - 1) * p.ld_w;  // columns past n repeat the last
#pragma unroll
    for (int r = 0; r < R; ++r) xr[r] = x + (r0 + r < p.rows ? r0 + r : p.rows - 1) * p.ld_x;
    float acc[R][4];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[r][c] = 0.0f;
    struct alignas(V * sizeof(T)) Vec { T t[V]; };
    for (int64_t k = lane * V; k < p.k; k += 32 * V) {
        float b[4][V];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const Vec v = *reinterpret_cast<const Vec *>(wj[c] + k);
#pragma unroll
            for (int e = 0; e < V; ++e) b[c][e] = to_f32(v.t[e]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const Vec v = *reinterpret_cast<const Vec *>(xr[r] + k);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float a = to_f32(v.t[e]);
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[r][c] = fmaf(a, b[c][e], acc[r][c]);
            }
        }
    }
    float mine[(R * 4 + 31) / 32];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float v = warp_sum(acc[r][c]);
            if (lane == ((r * 4 + c) & 31)) mine[(r * 4 + c) >> 5] = v;
        }
#pragma unroll
    for (int q = 0; q < (R * 4 + 31) / 32; ++q) {
        const int o = q * 32 + lane;
        const int64_t row = r0 + (o >> 2), col = j0 + (o & 3);
        if (o >= R * 4 || row >= p.rows || col >= p.n) continue;
        float v = mine[q];
        if (p.bias != nullptr) v += to_f32(static_cast<const T *>(p.bias)[col]);
        if (z != nullptr) z[row * p.n + col] = v;
        v = act_value(v, p.act);
        if (p.residual != nullptr) v += to_f32(static_cast<const T *>(p.residual)[row * p.ld_res + col]);
        static_cast<T *>(y)[row * ld_y + col] = from_f32<T>(v);
    }
}

// D[i, j] = sum_k A(i, k) B(j, k) in 32 x 32 tiles; 128 threads of 2 x 4
// outputs, the next tile's loads in registers under the products of this one.
//   kForward:  A = x, B = W                      D = z -> y
//   kGradX:    A = dz, B = W^T (k runs over n)   D = dx
//   kGradW:    A = dz^T, B = x^T (k over rows)   D = dw, and the sums of A over k are dbias
// dz = gy * act'(z) is formed as it is loaded and not rounded.  With more than
// one split of k the sums go to `partial` [splits, m, n + 1] (the last column:
// dbias) and reduce_kernel adds them in order.
enum { kForward = 0, kGradX = 1, kGradW = 2 };
struct SmallArgs {
    const void *a, *b;
    int64_t ld_a, ld_b;
    const float *z;         // of dz (pitch ld_z), or NULL
    int64_t ld_z, m, n, k, chunk;
    const void *bias, *residual;
    int64_t ld_res;
    void *out;
    int64_t ld_out;
    float *z_out;
    void *sum_out;
    float *partial;
    int act;
};

constexpr int kT = 32, kPitch = 36;

template <typename T, int MODE>
__device__ __forceinline__ void small_tile(const SmallArgs &p, int bx, int by, int bz, float (&As)[kT][kPitch],
                                           float (&Bs)[kT][kPitch]) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t i0 = by * int64_t(kT), j0 = bx * int64_t(kT);
    const int64_t k0 = bz * p.chunk, k1 = min(p.k, k0 + p.chunk);
    constexpr bool kAT = MODE == kGradW, kBT = MODE != kForward;  // the output index is contiguous
    constexpr bool kDz = MODE != kForward;
    // line e of the thread's eight is 4 e lines on; a tile further in k is one step
    const int64_t step_a = kAT ? kT * p.ld_a : kT, step_b = kBT ? kT * p.ld_b : kT, step_z = kAT ? kT * p.ld_z : kT;
    const int64_t la = kAT ? k0 + warp : i0 + warp, ca = kAT ? i0 + lane : k0 + lane;
    const T *pa = static_cast<const T *>(p.a) + la * p.ld_a + ca;
    const float *pz = p.z != nullptr ? p.z + la * p.ld_z + ca : nullptr;
    const T *pb = static_cast<const T *>(p.b) + (kBT ? k0 + warp : j0 + warp) * p.ld_b + (kBT ? j0 : k0) + lane;
    unsigned ok_a = 0u, ok_b = 0u;  // which of the eight lie inside as to the output index
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        ok_a |= (i0 + (kAT ? lane : warp + 4 * e) < p.m ? 1u : 0u) << e;
        ok_b |= (j0 + (kBT ? lane : warp + 4 * e) < p.n ? 1u : 0u) << e;
    }
    const bool slope = kDz && p.act != kActNone;
    T ra[8], rb[8];
    float rz[8];
    auto load = [&](int left) {  // left: how much of k is left at this tile
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int s = warp + 4 * e;
            ra[e] = ((ok_a >> e) & 1u) && (kAT ? s : lane) < left ? pa[e * 4 * p.ld_a] : from_f32<T>(0.0f);
            rb[e] = ((ok_b >> e) & 1u) && (kBT ? s : lane) < left ? pb[e * 4 * p.ld_b] : from_f32<T>(0.0f);
            if (slope) rz[e] = ((ok_a >> e) & 1u) && (kAT ? s : lane) < left ? pz[e * 4 * p.ld_z] : 0.0f;
        }
        pa += step_a;
        pb += step_b;
        if (slope) pz += step_z;
    };
    const int ti = (tid >> 3) * 2, tj = (tid & 7) * 4;
    float acc[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}}, sums[2] = {0, 0};
    int left = static_cast<int>(k1 - k0);
    load(left);
    for (; left > 0; left -= kT) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int s = warp + 4 * e;
            float v = to_f32(ra[e]);
            if (slope) v *= act_slope(rz[e], p.act);
            As[kAT ? s : lane][kAT ? lane : s] = v;
            Bs[kBT ? s : lane][kBT ? lane : s] = to_f32(rb[e]);
        }
        __syncthreads();
        if (left > kT) load(left - kT);
#pragma unroll
        for (int k = 0; k < kT; ++k) {
            const float2 a = *reinterpret_cast<const float2 *>(&As[k][ti]);
            const float4 b = *reinterpret_cast<const float4 *>(&Bs[k][tj]);
            const float av[2] = {a.x, a.y}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if (MODE == kGradW) sums[u] += av[u];
#pragma unroll
                for (int v = 0; v < 4; ++v) acc[u][v] = fmaf(av[u], bv[v], acc[u][v]);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int64_t i = i0 + ti + u;
        if (i >= p.m) continue;
        const bool owns_sum = MODE == kGradW && bx == 0 && tj == 0;
        if (p.partial != nullptr) {
            float *q = p.partial + (bz * p.m + i) * (p.n + 1);
#pragma unroll
            for (int v = 0; v < 4; ++v)
                if (j0 + tj + v < p.n) q[j0 + tj + v] = acc[u][v];
            if (owns_sum) q[p.n] = sums[u];
            continue;
        }
        if (owns_sum && p.sum_out != nullptr) static_cast<T *>(p.sum_out)[i] = from_f32<T>(sums[u]);
        if (p.out == nullptr) continue;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int64_t j = j0 + tj + v;
            if (j >= p.n) continue;
            float x = acc[u][v];
            if (MODE == kForward) {
                if (p.bias != nullptr) x += to_f32(static_cast<const T *>(p.bias)[j]);
                if (p.z_out != nullptr) p.z_out[i * p.n + j] = x;
                x = act_value(x, p.act);
                if (p.residual != nullptr) x += to_f32(static_cast<const T *>(p.residual)[i * p.ld_res + j]);
            }
            static_cast<T *>(p.out)[i * p.ld_out + j] = from_f32<T>(x);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(128) small_forward_kernel(const SmallArgs p) {
    __shared__ __align__(16) float As[kT][kPitch], Bs[kT][kPitch];
    const int tiles_n = static_cast<int>((p.n + kT - 1) / kT), by = blockIdx.x / tiles_n;
    small_tile<T, kForward>(p, blockIdx.x - by * tiles_n, by, 0, As, Bs);
}

// Both gradients in one launch: the blocks below `split` are dx's tiles.
struct GradGrid {
    int tiles_x, tiles_w, per_x, per_w, split;  // tiles along the output's columns, tiles per part of k
};
template <typename T>
__global__ void __launch_bounds__(128) small_backward_kernel(const SmallArgs x, const SmallArgs w, const GradGrid g) {
    __shared__ __align__(16) float As[kT][kPitch], Bs[kT][kPitch];
    const int b = blockIdx.x;
    if (b < g.split) {
        const int r = b % g.per_x;
        small_tile<T, kGradX>(x, r % g.tiles_x, r / g.tiles_x, b / g.per_x, As, Bs);
    } else {
        const int c = b - g.split, r = c % g.per_w;
        small_tile<T, kGradW>(w, r % g.tiles_w, r / g.tiles_w, c / g.per_w, As, Bs);
    }
}

// The parts of both gradients, added in order: elements below `count_x` are dx's.
template <typename T>
__device__ __forceinline__ void reduce_one(const SmallArgs &p, int64_t splits, int64_t t) {
    const int64_t i = t / (p.n + 1), j = t - i * (p.n + 1);
    float s = 0.0f;
    for (int64_t q = 0; q < splits; ++q) s += p.partial[q * p.m * (p.n + 1) + t];
    if (j < p.n) {
        if (p.out != nullptr) static_cast<T *>(p.out)[i * p.n + j] = from_f32<T>(s);
    } else if (p.sum_out != nullptr) {
        static_cast<T *>(p.sum_out)[i] = from_f32<T>(s);
    }
}
template <typename T>
__global__ void reduce_kernel(const SmallArgs x, int64_t splits_x, int64_t count_x, const SmallArgs w, int64_t splits_w,
                              int64_t count_w) {
    const int64_t t = blockIdx.x * int64_t(blockDim.x) + threadIdx.x;
    if (t < count_x) reduce_one<T>(x, splits_x, t);
    else if (t - count_x < count_w) reduce_one<T>(w, splits_w, t - count_x);
}

// ---- host side -------------------------------------------------------------
struct Split {
    int64_t splits, chunk;
};
// Splits of the contraction: enough blocks for four per SM, at least 64 long.
Split split_of(int64_t m, int64_t n, int64_t k) {
    const int64_t tiles = ((m + 31) / 32) * ((n + 31) / 32);
    int64_t s = (4 * 148 + tiles - 1) / tiles;
    const int64_t most = k / 64 > 1 ? k / 64 : 1;
    if (s > most) s = most;
    if (s > 64) s = 64;
    Split r;
    r.chunk = ((k + s - 1) / s + 31) / 32 * 32;
    r.splits = (k + r.chunk - 1) / r.chunk;
    return r;
}
size_t split_bytes(int64_t m, int64_t n, int64_t k) {
    const Split s = split_of(m, n, k);
    return s.splits > 1 ? carve_bytes<float>(s.splits * m * (n + 1)) : 0;
}

// Which path: microseconds as measured.  A small product takes 2.5 and, for
// every 32 of k, 0.8, or its operations at 12 TFLOP/s where there are many.  The
// tensor path takes 12 in fp32 (the packing and the product) on the device and
// 19 to launch; 5.5 in 16 bits when TMA takes the operands as they are and 9 when
// it does not; for the gradients 55 and 22 in all.
bool is_few_rows(int64_t rows, int dtype) { return rows <= (dtype == FL_F32 ? 16 : 8); }
double small_us(int64_t m, int64_t n, int64_t k, int64_t chunk, bool reduced) {
    const double steps = 0.8 * static_cast<double>((chunk + 31) / 32);
    const double ops = 2.0 * static_cast<double>(m) * static_cast<double>(n) * static_cast<double>(k) / 12e6;
    return 2.5 + (steps > ops ? steps : ops) + (reduced ? 3.0 : 0.0);
}
bool is_small(int64_t rows, int64_t n, int64_t k, int dtype) {
    return small_us(rows, n, k, k, false) <= (dtype == FL_F32 ? 16.0 : k % 8 == 0 ? 5.5 : 9.0);
}
bool is_small_backward(int64_t rows, int64_t n, int64_t k, int dtype) {
    const Split x = split_of(rows, k, n), w = split_of(n, k, rows);
    return small_us(rows, k, n, x.chunk, x.splits > 1) + small_us(n, k, rows, w.chunk, w.splits > 1) <=
           (dtype == FL_F32 ? 55.0 : 22.0);
}

bool tma_ready(const void *p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0; }

size_t operand_bytes(int64_t lines, int64_t inner, int64_t exps, int dtype) {
    if (dtype != FL_F32) return carve_bytes<__half>(lines * pitch_of(inner));
    return carve_bytes<__half>(2 * lines * pitch_of(inner)) + carve_bytes<int>(exps) + carve_bytes<unsigned>(exps);
}

// Readies the matrix src [lines, inner] as a product operand.  by_line: the
// uncontracted index is the line (K-major), else the inner index (MN-major).
int make_operand(const void *src, int64_t ld, int64_t lines, int64_t inner, bool by_line, int dtype, Carve &ws,
                 GemmOperand *op, const int **exps, cudaStream_t st, PackRows *pending = nullptr) {
    op->batch = 0;
    op->in_turn = 0;
    op->mn_major = by_line ? 0 : 1;
    *exps = nullptr;
    if (dtype != FL_F32) {
        op->planes = 1;
        op->plane = 0;
        if (tma_ready(src, ld)) {
            op->ptr = src;
            op->ld = ld;
            return FL_OK;
        }
        const int64_t ldp = pitch_of(inner);
        uint16_t *out = ws.take<uint16_t>(lines * ldp);
        FL_REQUIRE(out != nullptr, "linear: workspace too small");
        FL_REQUIRE(lines < (1ll << 31), "linear: bad shape");
        launch(pack16_kernel, static_cast<unsigned>((lines + 7) / 8), 256, 0, st, static_cast<const uint16_t *>(src), ld,
               lines, inner, out, ldp);
        op->ptr = out;
        op->ld = ldp;
        return check_launch("linear pack");
    }
    const int64_t ldp = pitch_of(inner), plane = lines * ldp;
    __half *out = ws.take<__half>(2 * plane);
    int *ex = ws.take<int>(by_line ? lines : inner);
    FL_REQUIRE(out != nullptr && ex != nullptr, "linear: workspace too small");
    const float *x = static_cast<const float *>(src);
    if (by_line) {
        const PackRows a{x, ld, lines, out, plane, ex};
        if (pending != nullptr) {
            *pending = a;  // the caller packs it together with another
        } else if (int rc = pack_rows(a, PackRows{}, inner, ldp, st)) {
            return rc;
        }
    } else {
        unsigned *bits = ws.take<unsigned>(inner);
        FL_REQUIRE(bits != nullptr, "linear: workspace too small");
        FL_CUDA(cudaMemsetAsync(bits, 0, inner * sizeof(unsigned), st));
        int64_t chunk = 256;
        while ((lines + chunk - 1) / chunk > 65535) chunk *= 2;
        launch(col_absmax_kernel, dim3(static_cast<unsigned>((inner + 31) / 32),
                                       static_cast<unsigned>((lines + chunk - 1) / chunk)),
               dim3(32, 8), 0, st, x, ld, lines, inner, chunk, bits);
        for (int64_t r = 0; r < lines; r += 65535 * 32) {
            const int64_t cnt = lines - r < 65535 * 32 ? lines - r : 65535 * 32;
            launch(pack_cols_kernel, dim3(static_cast<unsigned>((inner + 63) / 64), static_cast<unsigned>((cnt + 31) / 32)),
                   dim3(32, 8), 0, st, x + r * ld, ld, cnt, inner, bits, r == 0 ? ex : nullptr, out + r * ldp, ldp, plane);
        }
    }
    op->ptr = out;
    op->ld = ldp;
    op->plane = plane;
    op->planes = 2;
    *exps = ex;
    return check_launch("linear pack");
}

int check_linear(const fl_linear *p) {
    FL_REQUIRE(p != nullptr, "linear: null parameters");
    FL_REQUIRE(p->dtype == FL_F32 || p->dtype == FL_F16 || p->dtype == FL_BF16, "linear: bad dtype %d", p->dtype);
    FL_REQUIRE(p->act >= FL_ACT_NONE && p->act <= FL_ACT_GELU, "linear: bad activation %d", p->act);
    FL_REQUIRE(p->rows >= 0 && p->n > 0 && p->k > 0 && p->rows < (1ll << 30) && p->n < (1ll << 30) && p->k < (1ll << 30),
               "linear: bad shape");
    FL_REQUIRE((p->x != nullptr || p->rows == 0) && p->w != nullptr && p->ld_x >= p->k && p->ld_w >= p->k &&
                   (p->residual == nullptr || p->ld_res >= p->n),
               "linear: bad operand");
    return FL_OK;
}

GemmShape shape(int64_t m, int64_t n, int64_t k, int dtype) {
    GemmShape s;
    s.m = m;
    s.n = n;
    s.k = k;
    s.batch = 1;
    s.symmetric = 0;
    s.kind = dtype == FL_BF16 ? kBF16 : kF16;
    return s;
}

LinearEpilogue plain_epilogue(void *out, int64_t ld, int dtype, const int *re, const int *ce) {
    LinearEpilogue e{};
    e.row_exp = re;
    e.col_exp = ce;
    e.out = out;
    e.ld_out = ld;
    e.dtype = dtype;
    e.act = kActNone;
    e.second = 1.0f / kLoScale;
    return e;
}

template <typename T>
int linear_dz(const fl_linear *p, const float *z, const void *gy, int64_t ld_gy, T *out, int64_t ldo, int64_t plane,
              float *partial, cudaStream_t st) {
    // grid.y (row groups) is limited to 65535: 8 million rows
    const int64_t parts = (p->rows + kSumRows - 1) / kSumRows;
    FL_REQUIRE(parts <= 65535, "linear: more than %d rows in a backward pass", 65535 * kSumRows);
    launch(dz_kernel<T>, dim3(static_cast<unsigned>((p->n + 255) / 256), static_cast<unsigned>(parts)), dim3(32, 8), 0, st,
           static_cast<const T *>(gy), ld_gy, z, p->rows, p->n, p->act, out, ldo, plane, partial);
    return check_launch("linear dz");
}

template <typename T, int R>
void few_rows(const fl_linear *p, void *y, int64_t ld_y, float *z, cudaStream_t st) {
    const dim3 grid(static_cast<unsigned>((p->n + 31) / 32), static_cast<unsigned>((p->rows + R - 1) / R));
    auto ready = [](const void *q, int64_t ld) {
        return (reinterpret_cast<uintptr_t>(q) % (4 * sizeof(T))) == 0 && ld % 4 == 0;
    };
    if (p->k % 4 == 0 && ready(p->x, p->ld_x) && ready(p->w, p->ld_w))
        launch(few_rows_kernel<T, R, 4>, grid, 256, 0, st, *p, y, ld_y, z);
    else
        launch(few_rows_kernel<T, R, 1>, grid, 256, 0, st, *p, y, ld_y, z);
}

template <typename T>
int small_forward(const fl_linear *p, void *y, int64_t ld_y, float *z, cudaStream_t st) {
    if (is_few_rows(p->rows, p->dtype)) {
        if (p->rows == 1) few_rows<T, 1>(p, y, ld_y, z, st);
        else if (p->rows <= 4) few_rows<T, 4>(p, y, ld_y, z, st);
        else few_rows<T, 8>(p, y, ld_y, z, st);
        return check_launch("linear");
    }
    SmallArgs a{};
    a.a = p->x;
    a.ld_a = p->ld_x;
    a.b = p->w;
    a.ld_b = p->ld_w;
    a.m = p->rows;
    a.n = p->n;
    a.k = a.chunk = p->k;
    a.bias = p->bias;
    a.residual = p->residual;
    a.ld_res = p->ld_res;
    a.out = y;
    a.ld_out = ld_y;
    a.z_out = z;
    a.act = p->act;
    const int64_t tiles = ((a.m + kT - 1) / kT) * ((a.n + kT - 1) / kT);  // (a small product has few, whatever its sides)
    FL_REQUIRE(tiles < (1ll << 31), "linear: too many tiles");
    launch(small_forward_kernel<T>, static_cast<unsigned>(tiles), 128, 0, st, a);
    return check_launch("linear");
}

template <typename T>
int small_backward(const fl_linear *p, const float *z, const void *gy, int64_t ld_gy, void *dx, void *dw, void *dbias,
                   Carve &ws, cudaStream_t st) {
    SmallArgs a{};
    a.a = gy;
    a.ld_a = ld_gy;
    a.z = z;
    a.ld_z = p->n;
    a.act = p->act;
    SmallArgs x = a, w = a;
    GradGrid g{1, 1, 1, 1, 0};
    Split sx{1, 0}, sw{1, 0};
    int64_t blocks_w = 0;
    const bool want_w = dw != nullptr || dbias != nullptr;
    auto plan = [&](SmallArgs &q, Split &s, int &tiles, int &per) -> int {
        s = split_of(q.m, q.n, q.k);
        q.chunk = s.chunk;
        tiles = static_cast<int>((q.n + kT - 1) / kT);
        const int64_t all = tiles * ((q.m + kT - 1) / kT);
        FL_REQUIRE(all * s.splits < (1ll << 30), "linear backward: too many tiles");
        per = static_cast<int>(all);
        if (s.splits > 1) {
            q.partial = ws.take<float>(s.splits * q.m * (q.n + 1));
            FL_REQUIRE(q.partial != nullptr, "linear backward: workspace too small");
        }
        return FL_OK;
    };
    int rc = FL_OK;
    if (dx != nullptr) {
        x.b = p->w;
        x.ld_b = p->ld_w;
        x.m = p->rows;
        x.n = p->k;
        x.k = p->n;
        x.out = dx;
        x.ld_out = p->k;
        rc = plan(x, sx, g.tiles_x, g.per_x);
        if (rc) return rc;
        g.split = static_cast<int>(g.per_x * sx.splits);
    }
    if (want_w) {
        w.b = p->x;
        w.ld_b = p->ld_x;
        w.m = p->n;
        w.n = p->k;
        w.k = p->rows;
        w.out = dw;
        w.ld_out = p->k;
        w.sum_out = dbias;
        rc = plan(w, sw, g.tiles_w, g.per_w);
        if (rc) return rc;
        blocks_w = g.per_w * sw.splits;
    }
    if (g.split + blocks_w == 0) return FL_OK;
    launch(small_backward_kernel<T>, static_cast<unsigned>(g.split + blocks_w), 128, 0, st, x, w, g);
    const int64_t count_x = dx != nullptr && sx.splits > 1 ? x.m * (x.n + 1) : 0;
    const int64_t count_w = want_w && sw.splits > 1 ? w.m * (w.n + 1) : 0;
    if (count_x + count_w > 0)
        launch(reduce_kernel<T>, static_cast<unsigned>((count_x + count_w + 255) / 256), 256, 0, st, x, sx.splits, count_x, w,
               sw.splits, count_w);
    return check_launch("linear backward");
}

}  // namespace

size_t linear_workspace(int64_t rows, int64_t n, int64_t k, int dtype) {
    if (rows <= 0 || n <= 0 || k <= 0 || is_few_rows(rows, dtype) || is_small(rows, n, k, dtype)) return 0;
    return operand_bytes(rows, k, rows, dtype) + operand_bytes(n, k, n, dtype);
}

int linear_forward(const fl_linear *p, void *y, int64_t ld_y, float *z, void *wsp, size_t ws_bytes, cudaStream_t st) {
    int rc = check_linear(p);
    if (rc) return rc;
    if (p->rows == 0) return FL_OK;
    FL_REQUIRE(y != nullptr && ld_y >= p->n, "linear: bad output");
    if (is_small(p->rows, p->n, p->k, p->dtype) || is_few_rows(p->rows, p->dtype)) {
        if (p->dtype == FL_F32) return small_forward<float>(p, y, ld_y, z, st);
        if (p->dtype == FL_F16) return small_forward<__half>(p, y, ld_y, z, st);
        return small_forward<__nv_bfloat16>(p, y, ld_y, z, st);
    }
    Carve ws(wsp, ws_bytes);
    GemmOperand a, b;
    const int *ea, *eb;
    PackRows px{}, pw{};
    rc = make_operand(p->x, p->ld_x, p->rows, p->k, true, p->dtype, ws, &a, &ea, st, &px);
    if (!rc) rc = make_operand(p->w, p->ld_w, p->n, p->k, true, p->dtype, ws, &b, &eb, st, &pw);
    if (rc) return rc;
    if (p->dtype == FL_F32) {
        rc = pack_rows(px, pw, p->k, pitch_of(p->k), st);
        if (rc) return rc;
    }
    LinearEpilogue e = plain_epilogue(y, ld_y, p->dtype, ea, eb);
    e.bias = p->bias;
    e.residual = p->residual;
    e.ld_res = p->ld_res;
    e.z = z;
    e.ld_z = p->n;
    e.act = p->act;
    return gemm_linear(shape(p->rows, p->n, p->k, p->dtype), a, b, e, st);
}

size_t linear_backward_workspace(int64_t rows, int64_t n, int64_t k, int dtype, int act) {
    if (rows <= 0 || n <= 0 || k <= 0) return 0;
    if (is_small_backward(rows, n, k, dtype)) return split_bytes(rows, k, n) + split_bytes(n, k, rows) + 256;
    size_t b = carve_bytes<float>(((rows + kSumRows - 1) / kSumRows) * n);  // column sums
    // dz: of an activation, and of 16-bit gradients whose rows TMA cannot take
    const int planes = act != FL_ACT_NONE && dtype != FL_F32 ? 2 : 1;
    if (act != FL_ACT_NONE || dtype != FL_F32) b += carve_bytes<char>(planes * rows * pitch_of(n) * elem_size(dtype));
    if (dtype == FL_F32) b += operand_bytes(rows, n, rows, dtype) + operand_bytes(rows, n, n, dtype);  // its two scalings
    return b + operand_bytes(n, k, k, dtype) + operand_bytes(rows, k, k, dtype);
}

int linear_backward(const fl_linear *p, const float *z, const void *gy, int64_t ld_gy, void *dx, void *dw, void *dbias,
                    void *wsp, size_t ws_bytes, cudaStream_t st) {
    int rc = check_linear(p);
    if (rc) return rc;
    const int es = elem_size(p->dtype);
    if (p->rows == 0) {
        if (dw != nullptr) FL_CUDA(cudaMemsetAsync(dw, 0, p->n * p->k * es, st));
        if (dbias != nullptr) FL_CUDA(cudaMemsetAsync(dbias, 0, p->n * es, st));
        return FL_OK;
    }
    FL_REQUIRE(gy != nullptr && ld_gy >= p->n, "linear backward: bad gradient");
    FL_REQUIRE(p->act == FL_ACT_NONE || z != nullptr, "linear backward: an activation needs the pre-activation");
    Carve ws(wsp, ws_bytes);
    if (is_small_backward(p->rows, p->n, p->k, p->dtype)) {
        if (p->dtype == FL_F32) return small_backward<float>(p, z, gy, ld_gy, dx, dw, dbias, ws, st);
        if (p->dtype == FL_F16) return small_backward<__half>(p, z, gy, ld_gy, dx, dw, dbias, ws, st);
        return small_backward<__nv_bfloat16>(p, z, gy, ld_gy, dx, dw, dbias, ws, st);
    }
    const void *dz = gy;
    int64_t ld_dz = ld_gy;
    // 16-bit gradients whose rows TMA cannot take are copied to an aligned pitch in the same pass
    const bool copies = p->dtype != FL_F32 && !tma_ready(gy, ld_gy) && (dx != nullptr || dw != nullptr);
    const bool in_turn = p->dtype != FL_F32 && p->act != FL_ACT_NONE;  // dz in two planes
    int64_t plane = 0;
    if (p->act != FL_ACT_NONE || dbias != nullptr || copies) {
        void *out = nullptr;
        const int64_t ldo = pitch_of(p->n);
        if (p->act != FL_ACT_NONE || copies) {
            if (in_turn) plane = p->rows * ldo;
            out = ws.take<char>((in_turn ? 2 : 1) * p->rows * ldo * es);
            FL_REQUIRE(out != nullptr, "linear backward: workspace too small");
            dz = out;
            ld_dz = ldo;
        }
        const int64_t parts = (p->rows + kSumRows - 1) / kSumRows;
        float *partial = nullptr;
        if (dbias != nullptr) {
            partial = ws.take<float>(parts * p->n);
            FL_REQUIRE(partial != nullptr, "linear backward: workspace too small");
        }
        const unsigned grid = static_cast<unsigned>((p->n + 127) / 128);
        if (p->dtype == FL_F32) {
            rc = linear_dz<float>(p, z, gy, ld_gy, static_cast<float *>(out), ldo, 0, partial, st);
            if (!rc && dbias) launch(sum_partials_kernel<float>, grid, 128, 0, st, partial, parts, p->n, static_cast<float *>(dbias));
        } else if (p->dtype == FL_F16) {
            rc = linear_dz<__half>(p, z, gy, ld_gy, static_cast<__half *>(out), ldo, plane, partial, st);
            if (!rc && dbias) launch(sum_partials_kernel<__half>, grid, 128, 0, st, partial, parts, p->n, static_cast<__half *>(dbias));
        } else {
            rc = linear_dz<__nv_bfloat16>(p, z, gy, ld_gy, static_cast<__nv_bfloat16 *>(out), ldo, plane, partial, st);
            if (!rc && dbias)
                launch(sum_partials_kernel<__nv_bfloat16>, grid, 128, 0, st, partial, parts, p->n,
                       static_cast<__nv_bfloat16 *>(dbias));
        }
        if (rc) return rc;
    }
    GemmOperand a{}, b{};
    const int *ea, *eb;
    auto planes_in_turn = [&](LinearEpilogue e) {
        if (!in_turn) return e;
        a.planes = 2;
        a.plane = plane;
        a.in_turn = 1;
        e.first = p->dtype == FL_F16 ? DzPlanes<__half>::first : DzPlanes<__nv_bfloat16>::first;
        e.second = p->dtype == FL_F16 ? DzPlanes<__half>::second : DzPlanes<__nv_bfloat16>::second;
        return e;
    };
    if (dx != nullptr) {  // dz [rows, n] contracted over n with W [n, k]
        rc = make_operand(dz, ld_dz, p->rows, p->n, true, p->dtype, ws, &a, &ea, st);
        if (!rc) rc = make_operand(p->w, p->ld_w, p->n, p->k, false, p->dtype, ws, &b, &eb, st);
        if (rc) return rc;
        const LinearEpilogue e = planes_in_turn(plain_epilogue(dx, p->k, p->dtype, ea, eb));
        rc = gemm_linear(shape(p->rows, p->k, p->n, p->dtype), a, b, e, st);
        if (rc) return rc;
    }
    if (dw != nullptr) {  // dz [rows, n] and x [rows, k] contracted over the rows
        if (dx == nullptr || p->dtype == FL_F32) {
            rc = make_operand(dz, ld_dz, p->rows, p->n, false, p->dtype, ws, &a, &ea, st);
            if (rc) return rc;
        } else {
            a.mn_major = 1;  // 16-bit types: the operand that dx used, read along its other index
        }
        rc = make_operand(p->x, p->ld_x, p->rows, p->k, false, p->dtype, ws, &b, &eb, st);
        if (rc) return rc;
        const LinearEpilogue e = planes_in_turn(plain_epilogue(dw, p->k, p->dtype, ea, eb));
        rc = gemm_linear(shape(p->n, p->k, p->rows, p->dtype), a, b, e, st);
        if (rc) return rc;
    }
    return check_launch("linear backward");
}

int gemm_fault(int *fault);
int gemm_wait_limits(int64_t wait_ns, int64_t phase_ns);

}  // namespace fl

using namespace fl;

extern "C" {

size_t fl_linear_workspace(int64_t rows, int64_t n, int64_t k, int dtype) { return linear_workspace(rows, n, k, dtype); }

int fl_linear_forward(const fl_linear *p, void *y, int64_t ld_y, float *z, void *ws, size_t ws_bytes,
                      fl_stream_t stream) {
    return linear_forward(p, y, ld_y, z, ws, ws_bytes, as_stream(stream));
}

size_t fl_linear_backward_workspace(int64_t rows, int64_t n, int64_t k, int dtype, int act) {
    return linear_backward_workspace(rows, n, k, dtype, act);
}

int fl_linear_backward(const fl_linear *p, const float *z, const void *gy, int64_t ld_gy, void *dx, void *dw,
                       void *dbias, void *ws, size_t ws_bytes, fl_stream_t stream) {
    return linear_backward(p, z, gy, ld_gy, dx, dw, dbias, ws, ws_bytes, as_stream(stream));
}

int fl_gemm_fault(int *fault) { return gemm_fault(fault); }

int fl_gemm_wait_limits(int64_t wait_ns, int64_t phase_ns) { return gemm_wait_limits(wait_ns, phase_ns); }

}  // extern "C"

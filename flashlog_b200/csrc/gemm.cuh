// gemm.cuh -- the tcgen05 matrix product behind the linear head and the
// Newton-Schulz products: D[i, j] = sum_k A(i, k) B(j, k), batched.
//
// Operands are 16-bit arrays in global memory, each as 1 or 2 planes.  Two
// fp16 planes hold one fp32 matrix as hi + lo (22 bits); the product is then
// hi*hi + hi*lo + lo*hi in fp32 accumulators (the dropped lo*lo is below
// 2^-22 of each term), three matrix instructions per step on operands that
// were loaded once.  An operand is K-major (its contraction index is
// contiguous) or MN-major (its output index is), so products with a transposed
// operand need no transposing pass.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace fl {

enum { kF16 = 0, kBF16 = 1 };                 // operand type
enum { kOutF32 = 0, kOutF16 = 1, kOutBF16 = 2 };  // fl_dtype values (FL_F32, FL_F16, FL_BF16)

// Elements from line to line of a 16-bit array that a kernel writes for a
// product: lines that are not short start on 128 bytes, so that the writes and
// the product's loads take whole cache lines.
constexpr int64_t pitch_of(int64_t n) { return n < 64 ? (n + 7) & ~int64_t(7) : (n + 63) & ~int64_t(63); }

struct GemmOperand {
    const void *ptr;         // 16-byte aligned
    int64_t ld;              // elements between lines, a multiple of 8
    int64_t plane;           // elements between the planes (multiple of 8)
    int64_t batch;           // elements between the batch's matrices (multiple of 8)
    int planes;              // 1 or 2
    int mn_major;            // 0: lines are output indices, k contiguous; 1: lines are k
    int in_turn;             // A of a product with one plane: its second plane follows the first along k, into a
                             // second accumulator (D = first * (hi B) + second * (lo B))
};

// Epilogue of the linear head: z = acc * 2^(ea[i] + eb[j]) + bias[j],
// y = act(z) + residual[i, j].
struct LinearEpilogue {
    const int *row_exp, *col_exp;  // NULL: 0
    const void *bias;
    const void *residual;
    int64_t ld_res;
    void *out;
    int64_t ld_out;
    float *z;                // pre-activation for the backward, or NULL
    int64_t ld_z;
    int dtype, act;
    int aligned;             // set by gemm_linear: rows of all arrays start on 16 bytes
    int64_t out_batch;       // elements between the outputs of a batch (0: one output)
    float first, second;     // of the accumulators, where A's planes are taken in turn; with two planes an operand,
                             // second is that of the cross products (1 / the scale of the lo planes)
};

// A batch of matrices in a caller's memory: element (b, i, j) lies at
// (b / nb2) * .b1 + (b % nb2) * .b2 + i * .i + j * .j (nb2 is shared by the tensors of a call).
struct Strided {
    void *ptr;
    int64_t b1, b2, i, j;
    __host__ __device__ int64_t at(int64_t b, int64_t nb2) const { return (b / nb2) * b1 + (b % nb2) * b2; }
};

// The last Newton-Schulz product's result: out = v + keep * base.
struct FinalOutput {
    Strided out;             // of `dtype`
    Strided base;            // fp32, or no pointer
    const float *gate;       // where it holds 0, out = base; or NULL
    float keep;
    int64_t nb2;
    int dtype;
};

// The products of a Newton-Schulz run on the two-plane buffers below, in one
// kernel.  X [lo, hi] holds scale_x * X at the start; A, B, Q, T are [lo, lo],
// at scale_a (Q: scale_q).  gram 0: X <- a X + (b A + c A^2) X with A = X X^T,
// X and X2 in turn.  gram 1: see muon.cu; X and X2 in turn from segment to
// segment.  The result is factor * O.
enum { kNsX = 0, kNsX2 = 1, kNsA = 2, kNsB = 3, kNsQ = 4, kNsQ2 = 5, kNsT = 6, kNsBuffers = 7 };
struct NsBuffer {
    __half *p;               // NULL: not used
    int64_t ld, plane;       // the planes of one matrix follow each other, the matrices too
};
struct NsProgram {
    int lo, hi, batch, steps, gram;
    int last;                // this segment's product is the result (set by ns_products)
    const int *shift;        // [batch]: X holds scale_x * 2^shift * X (more than 0 for a matrix far below eps only)
    float a, b, c, scale_x, scale_a, scale_q, factor;
    FinalOutput final;
};

struct GemmShape {
    int64_t m, n, k, batch;
    int symmetric;           // D is symmetric: elements i >= j are computed and mirrored
    int kind;                // kF16 or kBF16
};

int gemm_linear(const GemmShape &s, const GemmOperand &a, const GemmOperand &b, const LinearEpilogue &e,
                cudaStream_t st);
// Phases of the whole run, and how many segments of the Gram form it takes.
int ns_phases(int steps, int gram);
int ns_segments(int steps, int gram);
// Steps of segment i: as many in each, the first ones one more.
inline int ns_segment_steps(int steps, int segments, int i) { return steps / segments + (i < steps % segments ? 1 : 0); }
// Bytes of `parts` (fp32 parts of A = X X^T, where the gram form splits it).
size_t ns_parts_bytes(int64_t lo, int64_t hi, int64_t batch);
// done_count: ns_phases * batch zeros.
int ns_products(const NsProgram &p, const NsBuffer *buffers, int *done_count, float *parts, cudaStream_t st);

// ---- activations -------------------------------------------------------------
enum { kActNone = 0, kActRelu = 1, kActTanh = 2, kActSilu = 3, kActGelu = 4 };

__device__ __forceinline__ float act_value(float z, int act) {
    switch (act) {
        case kActRelu: return z > 0.0f ? z : (z <= 0.0f ? 0.0f : z);  // NaN stays NaN
        case kActTanh: return tanhf(z);
        case kActSilu: return __fdividef(z, 1.0f + expf(-z));
        case kActGelu: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
        default: return z;
    }
}
__device__ __forceinline__ float act_slope(float z, int act) {
    switch (act) {
        case kActRelu: return z > 0.0f ? 1.0f : 0.0f;
        case kActTanh: { const float t = tanhf(z); return (1.0f - t) * (1.0f + t); }
        case kActSilu: { const float t = __fdividef(1.0f, 1.0f + expf(-z)); return t * (1.0f + z * (1.0f - t)); }
        case kActGelu:
            return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * expf(-0.5f * z * z) * 0.39894228040143268f;
        default: return 1.0f;
    }
}

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// two values at a time: one conversion instruction packs both
template <typename T> __device__ __forceinline__ unsigned pack_pair(float a, float b);
template <> __device__ __forceinline__ unsigned pack_pair<__half>(float a, float b) {
    union { __half2 h; unsigned u; } x;
    x.h = __floats2half2_rn(a, b);
    return x.u;
}
template <> __device__ __forceinline__ unsigned pack_pair<__nv_bfloat16>(float a, float b) {
    union { __nv_bfloat162 h; unsigned u; } x;
    x.h = __floats2bfloat162_rn(a, b);
    return x.u;
}
// v = hi + lo to 22 bits
__device__ __forceinline__ void split_pair(float a, float b, __half2 &hi, __half2 &lo) {
    hi = __floats2half2_rn(a, b);
    const float2 h = __half22float2(hi);
    lo = __floats2half2_rn(a - h.x, b - h.y);
}

// v * 2^e without an overflow or underflow on the way: the power is applied in
// two halves of one sign (|e| <= 252 as each side's exponent is within 126)
__device__ __forceinline__ float scale_pow2(float v, int e) {
    const int h = e / 2;
    return v * __int_as_float((h + 127) << 23) * __int_as_float((e - h + 127) << 23);
}

}  // namespace fl

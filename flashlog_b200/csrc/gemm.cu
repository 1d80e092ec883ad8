// gemm.cu -- the persistent tcgen05 matrix product (declared in gemm.cuh).
//
// A pair of CTAs (a cluster of two, cta_group::2) owns one 256 x BN tile at a
// time: each CTA holds 128 rows of A and half of the tile's columns of B in
// shared memory, and the pair's tensor cores read both halves, so an SM loads
// (128 + BN/2) lines for 128 x BN outputs; with one CTA per tile the L2 -> SM
// traffic would be 1.5 times that, above what the L2 delivers at the full
// matrix rate.  Roles per CTA: one warp loads by TMA (128-byte swizzle), one
// warp (of the pair's first CTA) issues the matrix instructions, eight warps
// read the accumulators back (two TMEM buffers, so a tile's epilogue runs
// under the next tile's products).  Waits are bounded: one that runs out marks
// the device fault word, and the tiles left get NaN.
#include <cuda.h>

#include "gemm.cuh"

namespace fl {

namespace {

constexpr int kBM = 128;        // rows of A per CTA
constexpr int kBK = 64;         // contraction per stage: one 128-byte swizzle line
constexpr int kEpiWarps = 8;    // warp w reads TMEM lanes 32 (w % 4).., columns of half w / 4
constexpr int kLoadWarp = kEpiWarps, kMmaWarp = kEpiWarps + 1;
constexpr int kThreads = 32 * (kEpiWarps + 2);
constexpr int kStageBudget = 196 * 1024;
constexpr int kStagePad = 33;   // row pitch (words) of the epilogue's transposing tile
constexpr uint64_t kWaitLimitNs = 4000000000ull;  // four seconds: far above any wait between healthy roles

__device__ int g_gemm_fault;    // set when a bounded wait ran out

__device__ __forceinline__ uint32_t smem_u32(const void *p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive_cta0(uint32_t bar) {
    asm volatile(
        "{\n .reg .b32 r;\n mapa.shared::cluster.u32 r, %0, 0;\n"
        " mbarrier.arrive.release.cluster.shared::cluster.b64 _, [r];\n}" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// false when the wait ran out (or another role of this CTA already failed)
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int *failed) {
    if (bar_try(bar, parity)) return true;
    uint64_t start, now;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(start));
    do {
        for (int i = 0; i < 64; ++i)
            if (bar_try(bar, parity)) return true;
        if (*failed) return false;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    } while (now - start < kWaitLimitNs);
    *failed = 1;
    atomicExch(&g_gemm_fault, 1);
    return false;
}

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1, int c2,
                                         int c3) {
    // the pair's barrier lives in its first CTA: clear the address bit that tells the two apart
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar & 0xFEFFFFFFu), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
        "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"(static_cast<uint16_t>(3)) : "memory");
}
__device__ __forceinline__ void tmem_read32(float (&v)[32], uint32_t addr) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Shared-memory matrix descriptor, 128-byte swizzle (8 lines of 128 bytes per
// 1024-byte atom): `lbo` steps between 64-element column blocks of an MN-major
// operand, `sbo` between groups of 8 lines.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFF) | (static_cast<uint64_t>((lbo >> 4) & 0x3FFF) << 16) |
           (static_cast<uint64_t>((sbo >> 4) & 0x3FFF) << 32) | (1ull << 46) | (2ull << 61);
}

struct TileGrid {
    int tiles_m, tiles_n, per_batch, total, symmetric, n_fast, batch;
};

// tile t -> (batch, row tile, column tile).  A symmetric product takes only the
// tiles that hold an element i >= j.
template <int BN>
__device__ __forceinline__ void tile_of(const TileGrid &g, int t, int &b, int &ti, int &tj) {
    b = t / g.per_batch;
    int r = t - b * g.per_batch;
    if (g.symmetric) {
        ti = 0;
        for (;;) {  // rows of tiles, each with min(tiles_n, (ti + 1) * 256 / BN) tiles
            const int w = min(g.tiles_n, (ti + 1) * (2 * kBM / BN));
            if (r < w) break;
            r -= w;
            ++ti;
        }
        tj = r;
    } else if (g.n_fast) {
        ti = r / g.tiles_n;
        tj = r - ti * g.tiles_n;
    } else {
        tj = r / g.tiles_m;
        ti = r - tj * g.tiles_m;
    }
}

// ---- epilogues: 32 rows x 32 columns per call, lane = row, v[c] = column c -----
template <int N>
__device__ __forceinline__ void apply_act(float (&z)[N], int act) {
    if (act == kActNone) return;
    if (act == kActRelu) {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = act_value(z[i], kActRelu);
    } else if (act == kActTanh) {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = act_value(z[i], kActTanh);
    } else if (act == kActSilu) {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = act_value(z[i], kActSilu);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = act_value(z[i], kActGelu);
    }
}

// Lane = column (or a pair of columns, two rows at a time, for 16-bit types
// whose rows are 4-byte aligned): the warp's stores are whole 64- or 128-byte
// pieces of a row at any alignment.  Eight rows are in flight at once.
template <typename T, bool PAIR>
__device__ __forceinline__ void linear_rows(const LinearEpilogue &e, const float *stage, int64_t row0, int64_t col0,
                                            int rows, int64_t n, int lane, bool exact_scale, int row_exp) {
    constexpr int kW = PAIR ? 2 : 1;              // columns per lane
    const int sub = PAIR ? lane >> 4 : 0;         // which of the two rows
    const int lc = PAIR ? (lane & 15) * 2 : lane;
    const int64_t col = col0 + lc;
    float bias[kW], factor[kW];
    int ce[kW];
    bool in[kW];
#pragma unroll
    for (int w = 0; w < kW; ++w) {
        in[w] = col + w < n;
        bias[w] = in[w] && e.bias != nullptr ? to_f32(static_cast<const T *>(e.bias)[col + w]) : 0.0f;
        ce[w] = in[w] && e.col_exp != nullptr ? e.col_exp[col + w] : 0;
        factor[w] = exact_scale ? 1.0f : __int_as_float((ce[w] + 127) << 23);
    }
    constexpr int kRows = 8;                      // rows per batch (per half warp: 2 kRows in all)
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += kRows * kW) {
        float z[kRows * kW], res[kRows * kW];
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            const int r = r0 + k * kW + sub;
#pragma unroll
            for (int w = 0; w < kW; ++w) {
                z[k * kW + w] = stage[r * kStagePad + lc + w];
                res[k * kW + w] = 0.0f;
            }
        }
        if (e.residual != nullptr) {
#pragma unroll
            for (int k = 0; k < kRows; ++k) {
                const int r = r0 + k * kW + sub;
                const T *p = static_cast<const T *>(e.residual) + (row0 + r) * e.ld_res + col;
                if (PAIR) {
                    if (r < rows && in[kW - 1]) {
                        union { unsigned u; T t[2]; } x;
                        x.u = *reinterpret_cast<const unsigned *>(p);
                        res[k * kW] = to_f32(x.t[0]);
                        res[k * kW + kW - 1] = to_f32(x.t[1]);
                    } else if (r < rows && in[0]) {
                        res[k * kW] = to_f32(p[0]);
                    }
                } else if (r < rows && in[0]) {
                    res[k] = to_f32(p[0]);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kRows; ++k)
#pragma unroll
            for (int w = 0; w < kW; ++w) {
                float x = z[k * kW + w];
                if (exact_scale) {
                    const int re = __shfl_sync(kFull, row_exp, r0 + k * kW + sub);
                    x = scale_pow2(x, re + ce[w]);
                } else {
                    x *= factor[w];
                }
                z[k * kW + w] = x + bias[w];
            }
        if (e.z != nullptr) {
#pragma unroll
            for (int k = 0; k < kRows; ++k) {
                const int r = r0 + k * kW + sub;
                float *p = e.z + (row0 + r) * e.ld_z + col;
#pragma unroll
                for (int w = 0; w < kW; ++w)
                    if (r < rows && in[w]) p[w] = z[k * kW + w];
            }
        }
        apply_act(z, e.act);
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            const int r = r0 + k * kW + sub;
            T *p = static_cast<T *>(e.out) + (row0 + r) * e.ld_out + col;
            if (PAIR && r < rows && in[kW - 1]) {
                union { unsigned u; T t[2]; } x;
                x.t[0] = from_f32<T>(z[k * kW] + res[k * kW]);
                x.t[PAIR ? 1 : 0] = from_f32<T>(z[k * kW + kW - 1] + res[k * kW + kW - 1]);
                *reinterpret_cast<unsigned *>(p) = x.u;
            } else if (r < rows && in[0]) {
                p[0] = from_f32<T>(z[k * kW] + res[k * kW]);
            }
        }
    }
}

template <typename T>
__device__ __forceinline__ void linear_store(const LinearEpilogue &e, float (&v)[32], float *stage, int64_t row0,
                                             int64_t col0, int64_t m, int64_t n, int lane) {
    // exponents within +-60 multiply in two exact steps; larger ones take the slow exact form
    int re = 0, ce = 0;
    if (e.row_exp != nullptr) {
        if (row0 + lane < m) re = e.row_exp[row0 + lane];
        if (col0 + lane < n) ce = e.col_exp[col0 + lane];
    }
    const bool exact_scale = __any_sync(kFull, re > 60 || re < -60 || ce > 60 || ce < -60);
    const float rf = exact_scale ? 1.0f : __int_as_float((re + 127) << 23);
#pragma unroll
    for (int c = 0; c < 32; ++c) stage[lane * kStagePad + c] = v[c] * rf;
    __syncwarp();
    const int rows = static_cast<int>(min(static_cast<int64_t>(32), m - row0));
    if (sizeof(T) == 2 && e.pair) linear_rows<T, sizeof(T) == 2>(e, stage, row0, col0, rows, n, lane, exact_scale, re);
    else linear_rows<T, false>(e, stage, row0, col0, rows, n, lane, exact_scale, re);
    __syncwarp();
}

template <typename T>
struct EpiLinear {
    LinearEpilogue p;
    __device__ __forceinline__ void operator()(float (&v)[32], float *stage, int, int64_t row0, int64_t col0,
                                               int64_t m, int64_t n, int lane) const {
        linear_store<T>(p, v, stage, row0, col0, m, n, lane);
    }
};

__device__ __forceinline__ void split_half(float v, __half &hi, __half &lo) {
    hi = __float2half_rn(v);
    lo = __float2half_rn(v - __half2float(hi));
}

// 32 consecutive columns of one row as two planes; the row's padding (up to ld)
// may be written, it is never read (the tensor maps end at n).
__device__ __forceinline__ void planes_row(__half *hi, int64_t plane, const float (&v)[32], int cols) {
    __half *lo = hi + plane;
    if (cols >= 32) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            union { __half h[8]; uint4 u; } a, b;
#pragma unroll
            for (int c = 0; c < 8; ++c) split_half(v[q * 8 + c], a.h[c], b.h[c]);
            reinterpret_cast<uint4 *>(hi)[q] = a.u;
            reinterpret_cast<uint4 *>(lo)[q] = b.u;
        }
    } else {
#pragma unroll
        for (int c = 0; c < 32; ++c)
            if (c < cols) {
                __half a, b;
                split_half(v[c], a, b);
                hi[c] = a;
                lo[c] = b;
            }
    }
}

template <typename T>
__device__ __forceinline__ void final_store(const PlanesEpilogue &e, const float (&v)[32], float *stage, int b,
                                            int64_t row0, int64_t col0, int64_t m, int64_t n, int lane) {
    T *out = static_cast<T *>(e.fin.ptr) + e.fin.at(b, e.nb2);
    const float *base = e.base.ptr != nullptr ? static_cast<const float *>(e.base.ptr) + e.base.at(b, e.nb2) : nullptr;
    if (e.fin.i == 1) {  // lane = row is the contiguous direction
        const int64_t row = row0 + lane;
        if (row < m) {
#pragma unroll
            for (int c = 0; c < 32; ++c) {
                const int64_t col = col0 + c;
                if (col < n) {
                    float x = v[c];
                    if (base != nullptr) x = fmaf(e.keep, base[row * e.base.i + col * e.base.j], x);
                    out[row + col * e.fin.j] = from_f32<T>(x);
                }
            }
        }
        return;
    }
#pragma unroll
    for (int c = 0; c < 32; ++c) stage[lane * kStagePad + c] = v[c];
    __syncwarp();
    const int64_t col = col0 + lane;
    const int rows = static_cast<int>(min(static_cast<int64_t>(32), m - row0));
    if (col < n) {
        for (int r = 0; r < rows; ++r) {
            const int64_t row = row0 + r;
            float x = stage[r * kStagePad + lane];
            if (base != nullptr) x = fmaf(e.keep, base[row * e.base.i + col * e.base.j], x);
            out[row * e.fin.i + col * e.fin.j] = from_f32<T>(x);
        }
    }
    __syncwarp();
}

template <bool SYM>
struct EpiPlanes {
    PlanesEpilogue p;
    __device__ __forceinline__ void operator()(float (&v)[32], float *stage, int b, int64_t row0, int64_t col0,
                                               int64_t m, int64_t n, int lane) const {
        if (SYM && col0 > row0 + 31) return;  // all of it above the diagonal: its mirror image writes it
        const int64_t row = row0 + lane;
        const int cols = static_cast<int>(min(static_cast<int64_t>(32), n - col0));
        const bool in = row < m;
        if (p.c != nullptr && in) {
            const __half *hi = p.c + b * p.c_batch + row * p.c_ld + col0;
            const __half *lo = hi + p.c_plane;
            // ld is a multiple of 8 and at least n: whole vectors stay within the row
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (q * 8 < cols) {
                    union { uint4 u; __half h[8]; } a, z;
                    a.u = reinterpret_cast<const uint4 *>(hi)[q];
                    z.u = reinterpret_cast<const uint4 *>(lo)[q];
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        v[q * 8 + c] = fmaf(p.alpha, v[q * 8 + c],
                                            p.beta * (__half2float(a.h[c]) + __half2float(z.h[c])));
                }
            }
        } else {
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] *= p.alpha;
        }
        if (p.fin.ptr != nullptr) {
            if (p.dtype == kOutF32) final_store<float>(p, v, stage, b, row0, col0, m, n, lane);
            else if (p.dtype == kOutF16) final_store<__half>(p, v, stage, b, row0, col0, m, n, lane);
            else final_store<__nv_bfloat16>(p, v, stage, b, row0, col0, m, n, lane);
        }
        if (p.out != nullptr && in) write<0>(v, b, row, row0, col0, cols);
        if (p.out2 != nullptr && in) {
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = p.alpha2 * v[c] + (col0 + c == row ? p.diag : 0.0f);
            write<1>(v, b, row, row0, col0, cols);
        }
    }
    template <int WHICH>
    __device__ __forceinline__ void write(const float (&v)[32], int b, int64_t row, int64_t row0, int64_t col0,
                                          int cols) const {
        __half *base = WHICH == 0 ? p.out + b * p.batch : p.out2 + b * p.batch2;
        const int64_t ld = WHICH == 0 ? p.ld : p.ld2, plane = WHICH == 0 ? p.plane : p.plane2;
        __half *hi = base + row * ld + col0;
        if (!SYM) {
            planes_row(hi, plane, v, cols);
            return;
        }
        if (col0 + 31 <= row0) {  // below the diagonal for every lane
            planes_row(hi, plane, v, cols);
        } else {
#pragma unroll
            for (int c = 0; c < 32; ++c)
                if (c < cols && col0 + c <= row) {
                    __half x, y;
                    split_half(v[c], x, y);
                    hi[c] = x;
                    hi[plane + c] = y;
                }
        }
        // the mirror image: lane = row is the contiguous direction
#pragma unroll
        for (int c = 0; c < 32; ++c)
            if (c < cols && col0 + c < row) {
                __half x, y;
                split_half(v[c], x, y);
                __half *t = base + (col0 + c) * ld + row;
                t[0] = x;
                t[plane] = y;
            }
    }
};

template <int BN, int PLANES>
struct Config {
    static constexpr int kA = kBM * kBK * 2;              // bytes of one plane of A per stage
    static constexpr int kB = (BN / 2) * kBK * 2;         // of B (this CTA's half)
    static constexpr int kStage = PLANES * (kA + kB);
    static constexpr int kStages = kStageBudget / kStage > 8 ? 8 : kStageBudget / kStage;
    static constexpr int kSmem = kStages * kStage + kEpiWarps * 32 * kStagePad * 4 + 1024;
};

template <int BN, int PLANES, typename Epi>
__global__ __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1)
void gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, int64_t m,
                 int64_t n, int64_t k, TileGrid grid, int a_mn, int b_mn, uint32_t idesc, const Epi epi) {
    using C = Config<BN, PLANES>;
    extern __shared__ unsigned char raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    float *stage_epi = reinterpret_cast<float *>(smem + C::kStages * C::kStage);
    __shared__ uint64_t bars[2 * C::kStages + 4];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int failed;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t cta;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(cta));
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const uint32_t full = smem_u32(bars), empty = full + 8 * C::kStages, acc_full = empty + 8 * C::kStages,
                   acc_empty = acc_full + 16;

    if (threadIdx.x == 0) {
        failed = 0;
        for (int s = 0; s < C::kStages; ++s) {
            bar_init(full + 8 * s, 1);
            bar_init(empty + 8 * s, 1);
        }
        for (int s = 0; s < 2; ++s) {
            bar_init(acc_full + 8 * s, 1);
            bar_init(acc_empty + 8 * s, 2 * kEpiWarps);  // of both CTAs
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(2 * BN) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;
    const int kblocks = static_cast<int>((k + kBK - 1) / kBK);

    if (warp == kLoadWarp && lane == 0) {
        // ---- loads ----
        int s = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int t = pair; ok && t < grid.total; t += pairs) {
            int b, ti, tj;
            tile_of<BN>(grid, t, b, ti, tj);
            const int row = ti * 2 * kBM + static_cast<int>(cta) * kBM, col = tj * BN + static_cast<int>(cta) * (BN / 2);
            for (int kb = 0; kb < kblocks; ++kb) {
                ok = bar_wait(empty + 8 * s, phase ^ 1, &failed);
                if (!ok) break;
                if (cta == 0) bar_expect(full + 8 * s, 2 * C::kStage);
                const uint32_t sa = smem_u32(smem) + s * C::kStage, sb = sa + PLANES * C::kA;
#pragma unroll
                for (int p = 0; p < PLANES; ++p) {
                    if (a_mn) {
#pragma unroll
                        for (int h = 0; h < kBM / 64; ++h)
                            tma_load(sa + p * C::kA + h * 8192, &map_a, full + 8 * s, row + 64 * h, kb * kBK, p, b);
                    } else {
                        tma_load(sa + p * C::kA, &map_a, full + 8 * s, kb * kBK, row, p, b);
                    }
                    if (b_mn) {
#pragma unroll
                        for (int h = 0; h < BN / 128; ++h)
                            tma_load(sb + p * C::kB + h * 8192, &map_b, full + 8 * s, col + 64 * h, kb * kBK, p, b);
                    } else {
                        tma_load(sb + p * C::kB, &map_b, full + 8 * s, kb * kBK, col, p, b);
                    }
                }
                if (++s == C::kStages) { s = 0; phase ^= 1; }
            }
        }
        // Every load must have landed before the pair's memory goes: each stage's last use is
        // waited for (through the products that consumed it; a stage never used passes at once).
        for (int i = 0; i < C::kStages; ++i) {
            if (!ok) {
                // the products may have stopped: give the copies in flight their time
                for (int w = 0; w < 4096; ++w) __nanosleep(256);
                break;
            }
            ok = bar_wait(empty + 8 * s, phase ^ 1, &failed);
            if (++s == C::kStages) { s = 0; phase ^= 1; }
        }
    } else if (warp == kMmaWarp && cta == 0 && lane == 0) {
        // ---- products (for the pair) ----
        const uint32_t a_step = a_mn ? 128u : 2u, b_step = b_mn ? 128u : 2u;  // 16 of k, in 16-byte units
        const uint32_t a_lbo = a_mn ? 8192u : 16u, b_lbo = b_mn ? 8192u : 16u;
        int s = 0, buf = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true;
        for (int t = pair; ok && t < grid.total; t += pairs) {
            ok = bar_wait(acc_empty + 8 * buf, acc_phase ^ 1, &failed);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t d = tmem + buf * BN;
            uint32_t accumulate = 0;
            for (int kb = 0; kb < kblocks; ++kb) {
                ok = bar_wait(full + 8 * s, phase, &failed);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t sa = smem_u32(smem) + s * C::kStage, sb = sa + PLANES * C::kA;
                uint64_t da[PLANES], db[PLANES];
#pragma unroll
                for (int p = 0; p < PLANES; ++p) {
                    da[p] = smem_desc(sa + p * C::kA, a_lbo, 1024);
                    db[p] = smem_desc(sb + p * C::kB, b_lbo, 1024);
                }
#pragma unroll
                for (int j = 0; j < kBK / 16; ++j) {
                    mma_f16(d, da[0] + j * a_step, db[0] + j * b_step, idesc, accumulate);
                    accumulate = 1;
                    if (PLANES == 2) {
                        mma_f16(d, da[0] + j * a_step, db[PLANES - 1] + j * b_step, idesc, 1);
                        mma_f16(d, da[PLANES - 1] + j * a_step, db[0] + j * b_step, idesc, 1);
                    }
                }
                mma_commit(empty + 8 * s);
                if (++s == C::kStages) { s = 0; phase ^= 1; }
            }
            mma_commit(acc_full + 8 * buf);
            if (++buf == 2) { buf = 0; acc_phase ^= 1; }
        }
    } else if (warp < kEpiWarps) {
        // ---- epilogue ----
        float *stage = stage_epi + warp * 32 * kStagePad;
        int buf = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        for (int t = pair; t < grid.total; t += pairs) {
            int b, ti, tj;
            tile_of<BN>(grid, t, b, ti, tj);
            const int64_t row0 = static_cast<int64_t>(ti) * 2 * kBM + cta * kBM + (warp & 3) * 32;
            const int64_t col0 = static_cast<int64_t>(tj) * BN;
            if (ok) ok = bar_wait(acc_full + 8 * buf, acc_phase, &failed);
            ok = __all_sync(kFull, ok);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t src = tmem + buf * BN + (static_cast<uint32_t>((warp & 3) * 32) << 16);
            const int half = (warp >> 2) * (BN / 2);
            for (int c = half; c < half + BN / 2; c += 32) {
                float v[32];
                if (ok) {
                    tmem_read32(v, src + c);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __int_as_float(0x7fc00000);
                }
                if (row0 < m && col0 + c < n) epi(v, stage, b, row0, col0 + c, m, n, lane);
                __syncwarp();
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive_cta0(acc_empty + 8 * buf);
            if (++buf == 2) { buf = 0; acc_phase ^= 1; }
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN));
    }
}

typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                             const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                             CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
    static const EncodeFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

// Tensor map of one operand: (contiguous index, line, plane, batch); lines and
// columns past the matrix read 0, so tails need no padding in memory.
int operand_map(CUtensorMap *map, const GemmOperand &o, int64_t lines_mn, int64_t k, int64_t batch, int box_rows,
                int kind) {
    FL_REQUIRE((reinterpret_cast<uintptr_t>(o.ptr) & 15) == 0 && o.ld % 8 == 0 && o.plane % 8 == 0 && o.batch % 8 == 0,
               "gemm: operand alignment");
    EncodeFn fn = encode_fn();
    if (fn == nullptr) {
        set_error("gemm: cuTensorMapEncodeTiled is not available");
        return FL_ECUDA;
    }
    const cuuint64_t inner = static_cast<cuuint64_t>(o.mn_major ? lines_mn : k);
    const cuuint64_t lines = static_cast<cuuint64_t>(o.mn_major ? k : lines_mn);
    cuuint64_t dims[4] = {inner, lines, static_cast<cuuint64_t>(o.planes), static_cast<cuuint64_t>(batch)};
    cuuint64_t ld = static_cast<cuuint64_t>(o.ld) * 2;
    // unused strides still have to be multiples of 16 that are not 0
    cuuint64_t strides[3] = {ld, o.planes > 1 ? static_cast<cuuint64_t>(o.plane) * 2 : ld,
                             batch > 1 ? static_cast<cuuint64_t>(o.batch) * 2 : ld};
    cuuint32_t box[4] = {64, static_cast<cuuint32_t>(o.mn_major ? kBK : box_rows), 1, 1};
    cuuint32_t unit[4] = {1, 1, 1, 1};
    const CUresult r = fn(map, kind == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                          const_cast<void *>(o.ptr), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("gemm: tensor map rejected (%d)", static_cast<int>(r));
        return FL_EINVAL;
    }
    return FL_OK;
}

// Tiles of one matrix of the batch.
int64_t tile_count(const GemmShape &s, int bn) {
    const int64_t tm = (s.m + 2 * kBM - 1) / (2 * kBM), tn = (s.n + bn - 1) / bn;
    if (!s.symmetric) return tm * tn;
    int64_t per = 0;
    for (int64_t i = 0; i < tm; ++i) per += (i + 1) * (2 * kBM / bn) < tn ? (i + 1) * (2 * kBM / bn) : tn;
    return per;
}

template <int BN, int PLANES, typename Epi>
int run(const GemmShape &s, const GemmOperand &a, const GemmOperand &b, const Epi &epi, cudaStream_t st) {
    using C = Config<BN, PLANES>;
    CUtensorMap ma, mb;
    int rc = operand_map(&ma, a, s.m, s.k, s.batch, kBM, s.kind);
    if (rc) return rc;
    rc = operand_map(&mb, b, s.n, s.k, s.batch, BN / 2, s.kind);
    if (rc) return rc;
    TileGrid g;
    g.tiles_m = static_cast<int>((s.m + 2 * kBM - 1) / (2 * kBM));
    g.tiles_n = static_cast<int>((s.n + BN - 1) / BN);
    g.symmetric = s.symmetric;
    g.batch = static_cast<int>(s.batch);
    g.n_fast = g.tiles_n <= g.tiles_m;  // the operand with fewer tiles is the one read again and again, from L2
    const int64_t per = tile_count(s, BN);
    FL_REQUIRE(per * s.batch < (1 << 30), "gemm: too many tiles");
    g.per_batch = static_cast<int>(per);
    g.total = static_cast<int>(per * s.batch);
    const int sms = fl_device_sm_count();
    int pairs = (sms > 1 ? sms : 148) / 2;
    if (pairs > g.total) pairs = g.total;
    // fp32 accumulator, operand type, majors, N, M = 256 (the pair's)
    const uint32_t type = s.kind == kBF16 ? 1u : 0u;
    const uint32_t idesc = (1u << 4) | (type << 7) | (type << 10) | (static_cast<uint32_t>(a.mn_major != 0) << 15) |
                           (static_cast<uint32_t>(b.mn_major != 0) << 16) | (static_cast<uint32_t>(BN >> 3) << 17) |
                           (static_cast<uint32_t>(256 >> 4) << 24);
    auto kernel = gemm_kernel<BN, PLANES, Epi>;
    FL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    note_launch();
    kernel<<<2 * pairs, kThreads, C::kSmem, st>>>(ma, mb, s.m, s.n, s.k, g, a.mn_major, b.mn_major, idesc, epi);
    return check_launch("gemm");
}

// 256-wide or 128-wide tiles: whichever needs less time on the slowest pair of
// SMs, 256 when equal (half the loads of A per product).
template <int PLANES, typename Epi>
int run_any(const GemmShape &s, const GemmOperand &a, const GemmOperand &b, const Epi &epi, cudaStream_t st) {
    FL_REQUIRE(s.m > 0 && s.n > 0 && s.k > 0 && s.batch > 0 && s.m < (1ll << 31) - 512 && s.n < (1ll << 31) - 512 &&
                   s.k < (1ll << 31) - 512 && s.batch < (1ll << 31),
               "gemm: bad shape");
    const int sms = fl_device_sm_count();
    const int64_t pairs = (sms > 1 ? sms : 148) / 2;
    const int64_t wide = (tile_count(s, 256) * s.batch + pairs - 1) / pairs;
    const int64_t narrow = (tile_count(s, 128) * s.batch + pairs - 1) / pairs;
    if (2 * wide <= narrow) return run<256, PLANES, Epi>(s, a, b, epi, st);
    return run<128, PLANES, Epi>(s, a, b, epi, st);
}

template <typename T>
int linear_typed(const GemmShape &s, const GemmOperand &a, const GemmOperand &b, const LinearEpilogue &e,
                 cudaStream_t st) {
    EpiLinear<T> epi{e};
    epi.p.pair = (reinterpret_cast<uintptr_t>(e.out) & 3) == 0 && (e.ld_out & 1) == 0 &&
                 (e.residual == nullptr || ((reinterpret_cast<uintptr_t>(e.residual) & 3) == 0 && (e.ld_res & 1) == 0));
    return run_any<sizeof(T) == 4 ? 2 : 1>(s, a, b, epi, st);
}

}  // namespace

int gemm_linear(const GemmShape &s, const GemmOperand &a, const GemmOperand &b, const LinearEpilogue &e,
                cudaStream_t st) {
    const int planes = e.dtype == kOutF32 ? 2 : 1;
    FL_REQUIRE(a.planes == planes && b.planes == planes && !s.symmetric, "gemm: planes");
    if (e.dtype == kOutF32) return linear_typed<float>(s, a, b, e, st);
    if (e.dtype == kOutF16) return linear_typed<__half>(s, a, b, e, st);
    return linear_typed<__nv_bfloat16>(s, a, b, e, st);
}

int gemm_planes(const GemmShape &s, const GemmOperand &a, const GemmOperand &b, const PlanesEpilogue &e,
                cudaStream_t st) {
    FL_REQUIRE(a.planes == 2 && b.planes == 2 && (!s.symmetric || (s.m == s.n && e.fin.ptr == nullptr)), "gemm: planes");
    if (s.symmetric) return run_any<2>(s, a, b, EpiPlanes<true>{e}, st);
    return run_any<2>(s, a, b, EpiPlanes<false>{e}, st);
}

// Reads and clears the device fault word (synchronizes the device).
int gemm_fault(int *fault) {
    int zero = 0;
    FL_CUDA(cudaMemcpyFromSymbol(fault, g_gemm_fault, sizeof(int)));
    if (*fault) FL_CUDA(cudaMemcpyToSymbol(g_gemm_fault, &zero, sizeof(int)));
    return FL_OK;
}

}  // namespace fl

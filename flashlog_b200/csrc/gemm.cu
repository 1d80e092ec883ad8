// gemm.cu -- the persistent tcgen05 matrix product (declared in gemm.cuh).
//
// A pair of CTAs (a cluster of two, cta_group::2) owns one 256 x BN tile at a
// time: each CTA holds 128 rows of A and half of the tile's columns of B in
// shared memory, and the pair's tensor cores read both halves, so an SM loads
// (128 + BN/2) lines for 128 x BN outputs; with one CTA per tile the L2 -> SM
// traffic would be 1.5 times that, above what the L2 delivers at the full
// matrix rate.  Roles per CTA: two warps load by TMA (128-byte swizzle), one A
// and one B, both planes of an operand at once (issuing a load takes about 130
// cycles: one warp for both would hold up 128-wide tiles); one warp (of the
// pair's first CTA) issues the matrix instructions; eight warps read the
// accumulators back (two TMEM buffers, so a tile's epilogue runs under the next
// tile's products).  Waits are bounded: one that runs out marks the device
// fault word, and the tiles left get NaN.
#include <cuda.h>

#include "gemm.cuh"

namespace fl {

namespace {

constexpr int kBM = 128;        // rows of A per CTA
constexpr int kBK = 64;         // contraction per stage: one 128-byte swizzle line
constexpr int kEpiWarps = 8;    // warp w reads TMEM lanes 32 (w % 4).., columns of half w / 4
constexpr int kLoadA = kEpiWarps, kLoadB = kEpiWarps + 1, kMmaWarp = kEpiWarps + 2;
constexpr int kThreads = 32 * (kEpiWarps + 3);
constexpr int kStageBudget = 192 * 1024;
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
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
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

// bar_wait by a whole warp, with one answer
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *failed) {
    return __all_sync(kFull, bar_wait(bar, parity, failed));
}

// One lane of a converged warp, in a form the compiler knows to be one: the
// load and product instructions take their operands from uniform registers.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
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
// Execution only: the barriers' initialisation has its own fence, and nothing
// else passes from one CTA's threads to the other's.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
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
// A tile's epilogue runs once or a few times per block: its code comes from
// memory, so loops that need no unrolling for their registers stay rolled.
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

// The epilogue's transposing tile, 32 x 32 words: the 16-byte pieces of row r
// are permuted by r % 8, so neither row writes nor column reads meet in a bank.
__device__ __forceinline__ int stage_at(int r, int c) { return r * 32 + ((((c >> 2) ^ r) & 7) << 2) + (c & 3); }

__device__ __forceinline__ void stage_rows(float *stage, const float (&v)[32], int lane) {
#pragma unroll
    for (int q = 0; q < 8; ++q)
        *reinterpret_cast<float4 *>(stage + stage_at(lane, 4 * q)) =
            make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
}

// A 32 x 32 tile of 16-bit values in 64-byte rows, as TMA's 64-byte swizzle
// lays it out: the same freedom from bank conflicts, and loads, stores and
// ldmatrix address whole 16-byte pieces.
__device__ __forceinline__ int piece_at(int r, int q) { return r * 64 + (((q ^ (r >> 1)) & 3) << 4); }

// Global memory takes 16-byte accesses at one cache line per cycle: a lane per
// row would touch 32 lines at a time, so rows are moved with the lanes side by
// side (four or eight to a row), through the staging tile.
template <typename T>
__device__ __forceinline__ void rows_to_stage(unsigned char *stage, const float (&v)[32], int lane) {
    if (sizeof(T) == 4) {
        stage_rows(reinterpret_cast<float *>(stage), v, lane);
        return;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        union { uint4 u; unsigned w[4]; } x;
#pragma unroll
        for (int c = 0; c < 4; ++c) x.w[c] = pack_pair<T>(v[q * 8 + 2 * c], v[q * 8 + 2 * c + 1]);
        *reinterpret_cast<uint4 *>(stage + piece_at(lane, q)) = x.u;
    }
}
template <typename T>
__device__ __forceinline__ void rows_from_stage(const unsigned char *stage, float (&v)[32], int lane) {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int q = 0; q < 32 / kPer; ++q) {
        union { uint4 u; T t[kPer]; } x;
        x.u = *reinterpret_cast<const uint4 *>(
            stage + (sizeof(T) == 4 ? 4 * stage_at(lane, 4 * q) : piece_at(lane, q)));
#pragma unroll
        for (int c = 0; c < kPer; ++c) v[q * kPer + c] = to_f32<T>(x.t[c]);
    }
}
template <typename T, bool STORE>
__device__ __forceinline__ void stage_global(unsigned char *stage, T *p, int64_t ld, int rows, int lane) {
    constexpr int kLanes = 2 * sizeof(T);  // per row of 32 values
    constexpr int kRows = 32 / kLanes;
    const int q = lane % kLanes;
#pragma unroll
    for (int it = 0; it < 32 / kRows; ++it) {
        const int r = it * kRows + lane / kLanes;
        uint4 *s = reinterpret_cast<uint4 *>(stage + (sizeof(T) == 4 ? 4 * stage_at(r, 4 * q) : piece_at(r, q)));
        if (r < rows) {
            uint4 *g = reinterpret_cast<uint4 *>(p + r * ld) + q;
            if (STORE) *g = *s;
            else *s = *g;
        }
    }
}

// Rows that start on 16 bytes: lane = row for the arithmetic.
template <typename T>
__device__ __forceinline__ void linear_rows(const LinearEpilogue &e, float (&v)[32], unsigned char *stage, int64_t row0,
                                            int64_t col0, int rows, int lane, float row_factor) {
    if (e.row_exp != nullptr) {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const int4 x = *reinterpret_cast<const int4 *>(e.col_exp + col0 + 4 * q);
            const int ex[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int c = 0; c < 4; ++c) v[4 * q + c] *= row_factor * __int_as_float((ex[c] + 127) << 23);
        }
    }
    if (e.bias != nullptr) {
        constexpr int kPer = 16 / sizeof(T);
#pragma unroll
        for (int q = 0; q < 32 / kPer; ++q) {
            union { uint4 u; T t[kPer]; } x;
            x.u = reinterpret_cast<const uint4 *>(static_cast<const T *>(e.bias) + col0)[q];
#pragma unroll
            for (int c = 0; c < kPer; ++c) v[q * kPer + c] += to_f32<T>(x.t[c]);
        }
    }
    if (e.z != nullptr) {
        rows_to_stage<float>(stage, v, lane);
        __syncwarp();
        stage_global<float, true>(stage, e.z + row0 * e.ld_z + col0, e.ld_z, rows, lane);
        __syncwarp();
    }
    apply_act(v, e.act);
    if (e.residual != nullptr) {
        // (a residual array may be read-only: the template's pointer type is shared with the stores)
        stage_global<T, false>(stage, const_cast<T *>(static_cast<const T *>(e.residual)) + row0 * e.ld_res + col0,
                               e.ld_res, rows, lane);
        __syncwarp();
        float t[32];
        rows_from_stage<T>(stage, t, lane);
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] += t[c];
    }
    rows_to_stage<T>(stage, v, lane);
    __syncwarp();
    stage_global<T, true>(stage, static_cast<T *>(e.out) + row0 * e.ld_out + col0, e.ld_out, rows, lane);
    __syncwarp();
}

// Any alignment: lane = column, the rows one after another from the staging
// tile, so that a warp's store is a whole 64- or 128-byte piece of a row.
template <typename T>
__device__ __forceinline__ void linear_columns(const LinearEpilogue &e, const float *stage, int64_t row0, int64_t col0,
                                               int rows, int64_t n, int lane, bool exact_scale, int row_exp,
                                               int col_exp) {
    const int64_t col = col0 + lane;
    const bool in = col < n;
    const float bias = in && e.bias != nullptr ? to_f32(static_cast<const T *>(e.bias)[col]) : 0.0f;
    const float factor = exact_scale ? 1.0f : __int_as_float((col_exp + 127) << 23);
    T *out = static_cast<T *>(e.out) + row0 * e.ld_out + col;
    const T *res = static_cast<const T *>(e.residual) + row0 * e.ld_res + col;
    float *pz = e.z + row0 * e.ld_z + col;
    const bool plain = !exact_scale && e.z == nullptr && e.act == kActNone && e.residual == nullptr && rows == 32;
    if (plain) {
#pragma unroll
        for (int r = 0; r < 32; ++r) {
            const T y = from_f32<T>(fmaf(stage[stage_at(r, lane)], factor, bias));
            if (in) *out = y;
            out += e.ld_out;
        }
        return;
    }
#pragma unroll 1
    for (int r0 = 0; r0 < rows; r0 += 8) {
        float z[8], y[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const bool on = in && r0 + k < rows;
            y[k] = e.residual != nullptr && on ? to_f32(res[k * e.ld_res]) : 0.0f;
            z[k] = stage[stage_at(r0 + k, lane)];
            if (exact_scale) z[k] = scale_pow2(z[k], __shfl_sync(kFull, row_exp, r0 + k) + col_exp);
            z[k] = fmaf(z[k], factor, bias);
            if (e.z != nullptr && on) pz[k * e.ld_z] = z[k];
        }
        apply_act(z, e.act);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (in && r0 + k < rows) out[k * e.ld_out] = from_f32<T>(z[k] + y[k]);
        out += 8 * e.ld_out;
        res += 8 * e.ld_res;
        pz += 8 * e.ld_z;
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
    const int rows = static_cast<int>(min(static_cast<int64_t>(32), m - row0));
    if (e.aligned && !exact_scale && col0 + 32 <= n) {
        linear_rows<T>(e, v, reinterpret_cast<unsigned char *>(stage), row0, col0, rows, lane, rf);
        return;
    }
    if (e.row_exp != nullptr) {
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] *= rf;
    }
    stage_rows(stage, v, lane);
    __syncwarp();
    linear_columns<T>(e, stage, row0, col0, rows, n, lane, exact_scale, re, ce);
    __syncwarp();
}

// What an epilogue warp keeps from chunk to chunk.
struct EpiWarp {
    float *stage;          // its staging tile (4 KB)
    uint32_t bar, phase;   // its barrier for loads into the tile
    volatile int *failed;
    int lane;
};

template <typename T>
struct EpiLinear {
    LinearEpilogue p;
    __device__ __forceinline__ void prepare(EpiWarp &, int, int64_t, int64_t) const {}
    __device__ __forceinline__ void operator()(float (&v)[32], EpiWarp &w, int, int64_t row0, int64_t col0, int64_t m,
                                               int64_t n, bool) const {
        linear_store<T>(p, v, w.stage, row0, col0, m, n, w.lane);
    }
    __device__ __forceinline__ void finish(EpiWarp &) const {}
};

// ---- 32 x 32 tiles of two planes: hi at the staging tile's start, lo 2 KB on ----
__device__ __forceinline__ void planes_to_stage(unsigned char *stage, const float (&v)[32], int lane) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        union { __half2 h[4]; uint4 u; } a, b;
#pragma unroll
        for (int c = 0; c < 4; ++c) split_pair(v[q * 8 + 2 * c], v[q * 8 + 2 * c + 1], a.h[c], b.h[c]);
        *reinterpret_cast<uint4 *>(stage + piece_at(lane, q)) = a.u;
        *reinterpret_cast<uint4 *>(stage + 2048 + piece_at(lane, q)) = b.u;
    }
}
// Stores the staged tile (all lanes have written it); lane 0 owns the copy.
__device__ __forceinline__ void stage_store(const CUtensorMap *map, uint32_t stage, int col, int row, int b, int lane) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) {
        asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                         reinterpret_cast<uint64_t>(map)), "r"(stage), "r"(col), "r"(row), "r"(0), "r"(b) : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
}
// The staging tile may be written again.
__device__ __forceinline__ void stage_free(int lane) {
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
}

template <typename T>
__device__ __forceinline__ void final_store(const PlanesEpilogue &e, const float (&v)[32], float *stage, int b,
                                            int64_t row0, int64_t col0, int64_t m, int64_t n, int lane) {
    T *out = static_cast<T *>(e.fin.ptr) + e.fin.at(b, e.nb2);
    const float *base = e.base.ptr != nullptr ? static_cast<const float *>(e.base.ptr) + e.base.at(b, e.nb2) : nullptr;
    const bool by_row = e.fin.i == 1;  // lane = row is the contiguous direction
    if (!by_row) {
        stage_rows(stage, v, lane);
        __syncwarp();
    }
    const int64_t row = by_row ? row0 + lane : row0, col = by_row ? col0 : col0 + lane;
    const int lines = static_cast<int>(min(static_cast<int64_t>(32), by_row ? n - col0 : m - row0));
    const bool in = row < m && col < n;
    T *po = out + row * e.fin.i + col * e.fin.j;
    const float *pb = base != nullptr ? base + row * e.base.i + col * e.base.j : nullptr;
    const int64_t so = by_row ? e.fin.j : e.fin.i, sb = by_row ? e.base.j : e.base.i;
    // eight lines at a time: the base's loads are in flight together, ahead of the stores that may alias it
#pragma unroll
    for (int l0 = 0; l0 < 32; l0 += 8) {
        if (l0 >= lines) break;
        float x[8], b0[8];
        if (base != nullptr) {
#pragma unroll
            for (int k = 0; k < 8; ++k) b0[k] = in && l0 + k < lines ? pb[k * sb] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            x[k] = by_row ? v[l0 + k] : stage[stage_at(l0 + k, lane)];
            if (base != nullptr) x[k] = fmaf(e.keep, b0[k], x[k]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (in && l0 + k < lines) po[k * so] = from_f32<T>(x[k]);
        po += 8 * so;
        pb += 8 * sb;
    }
    __syncwarp();
}

// Planes go to and come from memory by TMA: whole tiles through the warp's
// staging tile, C for a tile's first chunk already under the products.
template <bool SYM>
struct EpiPlanes {
    PlanesEpilogue p;
    CUtensorMap map_c, map_out, map_out2;

    __device__ __forceinline__ void load_c(EpiWarp &w, int b, int64_t row0, int64_t col0) const {
        if (w.lane == 0) {
            bar_expect(w.bar, 4096);
            asm volatile(
                "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
                " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(w.stage)),
                "l"(reinterpret_cast<uint64_t>(&map_c)), "r"(w.bar), "r"(static_cast<int>(col0)),
                "r"(static_cast<int>(row0)), "r"(0), "r"(b) : "memory");
        }
    }
    __device__ __forceinline__ bool wanted(int64_t row0, int64_t col0) const {
        return !SYM || col0 <= row0;  // the rest is written as a mirror image
    }
    // The first chunk's C, before the products are waited for.
    __device__ __forceinline__ void prepare(EpiWarp &w, int b, int64_t row0, int64_t col0) const {
        if (p.c != nullptr && wanted(row0, col0)) load_c(w, b, row0, col0);
    }
    __device__ __forceinline__ void finish(EpiWarp &w) const {
        if (w.lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        __syncwarp();
    }
    // first: whether prepare has loaded C
    __device__ __forceinline__ void operator()(float (&v)[32], EpiWarp &w, int b, int64_t row0, int64_t col0, int64_t m,
                                               int64_t n, bool first) const {
        if (!wanted(row0, col0)) return;
        const int lane = w.lane;
        unsigned char *stage = reinterpret_cast<unsigned char *>(w.stage);
        const uint32_t s32 = smem_u32(stage);
        if (p.c != nullptr) {
            if (!first) load_c(w, b, row0, col0);
            const bool ok = warp_wait(w.bar, w.phase, w.failed);
            w.phase ^= 1;
            if (!ok) return;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                union { uint4 u; __half2 h[4]; } a, z;
                a.u = *reinterpret_cast<const uint4 *>(stage + piece_at(lane, q));
                z.u = *reinterpret_cast<const uint4 *>(stage + 2048 + piece_at(lane, q));
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float2 x = __half22float2(a.h[c]), y = __half22float2(z.h[c]);
                    v[q * 8 + 2 * c] = fmaf(p.alpha, v[q * 8 + 2 * c], p.beta * (x.x + y.x));
                    v[q * 8 + 2 * c + 1] = fmaf(p.alpha, v[q * 8 + 2 * c + 1], p.beta * (x.y + y.y));
                }
            }
            __syncwarp();
        } else {
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] *= p.alpha;
        }
        if (!SYM && p.fin.ptr != nullptr) {
            if (p.dtype == kOutF32) final_store<float>(p, v, w.stage, b, row0, col0, m, n, lane);
            else if (p.dtype == kOutF16) final_store<__half>(p, v, w.stage, b, row0, col0, m, n, lane);
            else final_store<__nv_bfloat16>(p, v, w.stage, b, row0, col0, m, n, lane);
            // the staging tile is next written by a TMA load: order it behind these accesses
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            return;
        }
        const int row = static_cast<int>(row0), col = static_cast<int>(col0);
        if (SYM && col == row) {
            // the tile on the diagonal: its upper half from the lower
            stage_rows(w.stage, v, lane);
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = w.stage[stage_at(max(c, lane), min(c, lane))];
            __syncwarp();
        }
#pragma unroll 1
        for (int o = 0; o < (SYM && p.out2 != nullptr ? 2 : 1); ++o) {
            const CUtensorMap *map = o == 0 ? &map_out : &map_out2;
            if (o == 1) {
#pragma unroll
                for (int c = 0; c < 32; ++c) v[c] = p.alpha2 * v[c] + (col + c == row + lane ? p.diag : 0.0f);
            }
            planes_to_stage(stage, v, lane);
            stage_store(map, s32, col, row, b, lane);
            if (SYM && col != row) {
                // the mirror image: 8 x 8 blocks turned on their way through registers
                uint32_t r[2][4][4];
                const int j = lane >> 3, k = lane & 7;
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                                     : "=r"(r[q][i][0]), "=r"(r[q][i][1]), "=r"(r[q][i][2]), "=r"(r[q][i][3])
                                     : "r"(s32 + 2048 * q + piece_at(8 * i + k, j)) : "memory");
                stage_free(lane);
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(
                                         s32 + 2048 * q + piece_at(8 * j + k, i)),
                                     "r"(r[q][i][0]), "r"(r[q][i][1]), "r"(r[q][i][2]), "r"(r[q][i][3]) : "memory");
                stage_store(map, s32, row, col, b, lane);
            }
            stage_free(lane);
        }
    }
};

template <int BN, int PLANES>
struct Config {
    static constexpr int kA = kBM * kBK * 2;              // bytes of one plane of A per stage
    static constexpr int kB = (BN / 2) * kBK * 2;         // of B (this CTA's half)
    static constexpr int kStage = PLANES * (kA + kB);
    static constexpr int kStages = kStageBudget / kStage > 8 ? 8 : kStageBudget / kStage;
    static constexpr int kSmem = kStages * kStage + kEpiWarps * 32 * 32 * 4 + 1024;
};

template <int BN, int PLANES, typename Epi>
__global__ __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1)
void gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, int64_t m,
                 int64_t n, int64_t k, TileGrid grid, int a_mn, int b_mn, uint32_t idesc, const __grid_constant__ Epi epi) {
    using C = Config<BN, PLANES>;
    extern __shared__ unsigned char raw[];
    // (an offset, not a rounded pointer: the compiler keeps knowing that this is shared memory)
    unsigned char *smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    float *stage_epi = reinterpret_cast<float *>(smem + C::kStages * C::kStage);
    __shared__ uint64_t bars[2 * C::kStages + 4 + kEpiWarps];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int failed;

    const int warp = __shfl_sync(kFull, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    uint32_t cta;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(cta));
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const uint32_t full = smem_u32(bars), empty = full + 8 * C::kStages, acc_full = empty + 8 * C::kStages,
                   acc_empty = acc_full + 16;

    if (threadIdx.x < 2 * C::kStages + 4 + kEpiWarps) {
        const int i = threadIdx.x, k = i - (2 * C::kStages + 2);
        // accumulator buffers free: every epilogue warp of both CTAs arrives
        bar_init(full + 8 * i, k == 0 || k == 1 ? 2 * kEpiWarps : 1);
        if (i == 0) failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(2 * BN) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    if (warp == kLoadA && lane < 2)
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(lane == 0 ? &map_a : &map_b)));
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;
    const int kblocks = static_cast<int>((k + kBK - 1) / kBK);

    if (warp == kLoadA || warp == kLoadB) {
        // ---- loads ----
        const bool is_a = warp == kLoadA;
        const CUtensorMap *map = is_a ? &map_a : &map_b;
        const bool mn = is_a ? a_mn != 0 : b_mn != 0;
        const int pieces = mn ? (is_a ? kBM / 64 : BN / 128) : 1;  // 64 lines of an MN-major operand per load
        const uint32_t offset = is_a ? 0 : PLANES * C::kA, plane = is_a ? C::kA : C::kB;
        const bool expects = is_a && cta == 0;
        int s = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int t = pair; ok && t < grid.total; t += pairs) {
            int b, ti, tj;
            tile_of<BN>(grid, t, b, ti, tj);
            const int line = is_a ? ti * 2 * kBM + static_cast<int>(cta) * kBM : tj * BN + static_cast<int>(cta) * (BN / 2);
            for (int kb = 0; kb < kblocks; ++kb) {
                ok = warp_wait(empty + 8 * s, phase ^ 1, &failed);
                if (!ok) break;
                const uint32_t dst = smem_u32(smem) + s * C::kStage + offset;
                if (elect_one()) {
                    // the other CTA's and the other warp's bytes may arrive before they are expected
                    if (expects) bar_expect(full + 8 * s, 2 * C::kStage);
                    if (mn) {
#pragma unroll
                        for (int p = 0; p < PLANES; ++p)
                            for (int h = 0; h < pieces; ++h)
                                tma_load(dst + p * plane + h * 8192, map, full + 8 * s, line + 64 * h, kb * kBK, p, b);
                    } else {
                        tma_load(dst, map, full + 8 * s, kb * kBK, line, 0, b);  // all planes
                    }
                }
                __syncwarp();
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
            ok = warp_wait(empty + 8 * s, phase ^ 1, &failed);
            if (++s == C::kStages) { s = 0; phase ^= 1; }
        }
    } else if (warp == kMmaWarp && cta == 0) {
        // ---- products (for the pair) ----
        const uint32_t a_step = a_mn ? 128u : 2u, b_step = b_mn ? 128u : 2u;  // 16 of k, in 16-byte units
        const uint32_t a_lbo = a_mn ? 8192u : 16u, b_lbo = b_mn ? 8192u : 16u;
        int s = 0, buf = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true;
        for (int t = pair; ok && t < grid.total; t += pairs) {
            ok = warp_wait(acc_empty + 8 * buf, acc_phase ^ 1, &failed);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t d = tmem + buf * BN;
            for (int kb = 0; kb < kblocks; ++kb) {
                ok = warp_wait(full + 8 * s, phase, &failed);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t sa = smem_u32(smem) + s * C::kStage, sb = sa + PLANES * C::kA;
                if (elect_one()) {
                    uint64_t da[PLANES], db[PLANES];
#pragma unroll
                    for (int p = 0; p < PLANES; ++p) {
                        da[p] = smem_desc(sa + p * C::kA, a_lbo, 1024);
                        db[p] = smem_desc(sb + p * C::kB, b_lbo, 1024);
                    }
#pragma unroll
                    for (int j = 0; j < kBK / 16; ++j) {
                        mma_f16(d, da[0] + j * a_step, db[0] + j * b_step, idesc, (kb | j) != 0);
                        if (PLANES == 2) {
                            mma_f16(d, da[0] + j * a_step, db[PLANES - 1] + j * b_step, idesc, 1);
                            mma_f16(d, da[PLANES - 1] + j * a_step, db[0] + j * b_step, idesc, 1);
                        }
                    }
                    mma_commit(empty + 8 * s);
                }
                __syncwarp();
                if (++s == C::kStages) { s = 0; phase ^= 1; }
            }
            if (elect_one()) mma_commit(acc_full + 8 * buf);
            __syncwarp();
            if (++buf == 2) { buf = 0; acc_phase ^= 1; }
        }
    } else if (warp < kEpiWarps) {
        // ---- epilogue ----
        EpiWarp w{stage_epi + warp * 32 * 32, acc_empty + 16 + 8 * warp, 0, &failed, lane};
        int buf = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        for (int t = pair; t < grid.total; t += pairs) {
            int b, ti, tj;
            tile_of<BN>(grid, t, b, ti, tj);
            const int64_t row0 = static_cast<int64_t>(ti) * 2 * kBM + cta * kBM + (warp & 3) * 32;
            const int64_t col0 = static_cast<int64_t>(tj) * BN;
            const int half = (warp >> 2) * (BN / 2);
            if (ok && row0 < m && col0 + half < n) epi.prepare(w, b, row0, col0 + half);
            if (ok) ok = warp_wait(acc_full + 8 * buf, acc_phase, &failed);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t src = tmem + buf * BN + (static_cast<uint32_t>((warp & 3) * 32) << 16);
#pragma unroll 1
            for (int c = half; c < half + BN / 2; c += 32) {
                float v[32];
                if (ok) {
                    tmem_read32(v, src + c);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __int_as_float(0x7fc00000);
                }
                if (row0 < m && col0 + c < n) epi(v, w, b, row0, col0 + c, m, n, c == half);
                __syncwarp();
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive_cta0(acc_empty + 8 * buf);
            if (++buf == 2) { buf = 0; acc_phase ^= 1; }
        }
        epi.finish(w);
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
    cuuint32_t box[4] = {64, static_cast<cuuint32_t>(o.mn_major ? kBK : box_rows),
                         static_cast<cuuint32_t>(o.mn_major ? 1 : o.planes), 1};
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

// Tensor map of 32 x 32 tiles of a two-plane array [rows, cols].
int planes_map(CUtensorMap *map, const __half *ptr, int64_t ld, int64_t plane, int64_t batch_stride, int64_t rows,
               int64_t cols, int64_t batch) {
    FL_REQUIRE((reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && ld % 8 == 0 && plane % 8 == 0 && batch_stride % 8 == 0,
               "gemm: planes alignment");
    EncodeFn fn = encode_fn();
    if (fn == nullptr) {
        set_error("gemm: cuTensorMapEncodeTiled is not available");
        return FL_ECUDA;
    }
    cuuint64_t dims[4] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), 2, static_cast<cuuint64_t>(batch)};
    cuuint64_t strides[3] = {static_cast<cuuint64_t>(ld) * 2, static_cast<cuuint64_t>(plane) * 2,
                             static_cast<cuuint64_t>(batch_stride) * 2};
    cuuint32_t box[4] = {32, 32, 2, 1}, unit[4] = {1, 1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<__half *>(ptr), dims, strides, box, unit,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
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
    const int per = 16 / static_cast<int>(sizeof(T));
    auto rows_ready = [&](const void *p, int64_t ld, int64_t unit) {
        return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % unit == 0);
    };
    epi.p.aligned = rows_ready(e.out, e.ld_out, per) && rows_ready(e.residual, e.ld_res, per) && rows_ready(e.bias, 0, 1) &&
                    rows_ready(e.z, e.ld_z, 4);
    return run_any<sizeof(T) == 4 ? 2 : 1>(s, a, b, epi, st);
}

template <bool SYM>
int planes_typed(const GemmShape &s, const GemmOperand &a, const GemmOperand &b, const PlanesEpilogue &e,
                 cudaStream_t st) {
    EpiPlanes<SYM> epi{};
    epi.p = e;
    int rc = FL_OK;
    if (e.c != nullptr) rc = planes_map(&epi.map_c, e.c, e.c_ld, e.c_plane, e.c_batch, s.m, s.n, s.batch);
    if (!rc && e.out != nullptr) rc = planes_map(&epi.map_out, e.out, e.ld, e.plane, e.batch, s.m, s.n, s.batch);
    if (!rc && e.out2 != nullptr) rc = planes_map(&epi.map_out2, e.out2, e.ld2, e.plane2, e.batch2, s.m, s.n, s.batch);
    return rc ? rc : run_any<2>(s, a, b, epi, st);
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
    FL_REQUIRE(e.out != nullptr || e.fin.ptr != nullptr, "gemm: no output");
    return s.symmetric ? planes_typed<true>(s, a, b, e, st) : planes_typed<false>(s, a, b, e, st);
}

// Reads and clears the device fault word (synchronizes the device).
int gemm_fault(int *fault) {
    int zero = 0;
    FL_CUDA(cudaMemcpyFromSymbol(fault, g_gemm_fault, sizeof(int)));
    if (*fault) FL_CUDA(cudaMemcpyToSymbol(g_gemm_fault, &zero, sizeof(int)));
    return FL_OK;
}

}  // namespace fl

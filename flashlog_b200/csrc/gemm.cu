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
// accumulators back (two or three in TMEM take turns, so an epilogue runs under
// the next products).  Waits are bounded: one that runs out marks the device
// fault word, and the tiles that the block has left get NaN, as does what is
// computed from them.
//
// Measured (1.66 PFLOP/s is what one large bf16 product reaches): 4608 x 1024 ->
// 29649 in bf16 225 us (1.24 PFLOP/s: rows of odd length leave through the
// staging tile), 357 us with SiLU, 670 us with GELU and a residual; its two
// gradients 156 us and 171 us (1.8 and 1.64 PFLOP/s in bursts), of an activation
// on two planes of dz 1295 us with the pass that makes them; 4608 x 1024 -> 1645
// on two planes 45 us (1.0 PFLOP/s of matrix instructions; its 234 tiles take the
// place of 296), 4608 x 4096 -> 4736 with its packing 453 us (1.19 PFLOP/s).
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

__device__ int g_gemm_fault;    // set when a bounded wait ran out
// Limits in ns: of a role for another of its pair, and of a phase's tiles for the phase before.  Four seconds are
// far above any wait between healthy roles.
__device__ uint64_t g_wait_limit = 4000000000ull, g_phase_limit = 4000000000ull;

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
    } while (now - start < *const_cast<volatile uint64_t *>(&g_wait_limit));
    *failed = 1;
    atomicExch(&g_gemm_fault, 1);
    return false;
}

// A copy that was started lands, whatever happens to the roles: nobody writes to its place before.
__device__ __forceinline__ bool landed(uint32_t bar, uint32_t parity) {
    if (bar_try(bar, parity)) return true;
    uint64_t start, now;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(start));
    for (;;) {
        for (int i = 0; i < 64; ++i)
            if (bar_try(bar, parity)) return true;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
        if (now - start >= 4000000000ull) break;
    }
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
    if constexpr (sizeof(T) == 4) {
        stage_rows(reinterpret_cast<float *>(stage), v, lane);
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            union { uint4 u; unsigned w[4]; } x;
#pragma unroll
            for (int c = 0; c < 4; ++c) x.w[c] = pack_pair<T>(v[q * 8 + 2 * c], v[q * 8 + 2 * c + 1]);
            *reinterpret_cast<uint4 *>(stage + piece_at(lane, q)) = x.u;
        }
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

// What an epilogue warp keeps from chunk to chunk.
struct EpiWarp {
    float *stage;          // its staging tiles (4 KB each)
    uint32_t bar, phase;   // their barriers for loads, 8 bytes apart, and a phase bit of each
    uint32_t asked;        // a bit of each into which a load is under way
    volatile int *failed;
    int lane;
    uint4 bias[4], res[4]; // of a linear head's next chunk in 16 bits: asked for a chunk ahead
};

// In 16 bits without z, a chunk's bias and residual are loaded while the chunk
// before it (or the products) are under way.
template <typename T>
__device__ __forceinline__ bool chunk_ahead(const LinearEpilogue &e, int64_t col0, int64_t n) {
    return sizeof(T) == 2 && e.aligned && e.z == nullptr && e.out_batch == 0 && col0 + 32 <= n;
}
template <typename T>
__device__ __forceinline__ void ask_ahead(const LinearEpilogue &e, EpiWarp &w, int64_t row0, int64_t col0, int64_t m) {
    if (e.bias != nullptr) {
#pragma unroll
        for (int q = 0; q < 4; ++q) w.bias[q] = reinterpret_cast<const uint4 *>(static_cast<const T *>(e.bias) + col0)[q];
    }
    if (e.residual != nullptr) {
        const T *p = static_cast<const T *>(e.residual) + (row0 + w.lane / 4) * e.ld_res + col0;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (row0 + w.lane / 4 + 8 * q < m) w.res[q] = reinterpret_cast<const uint4 *>(p + 8 * q * e.ld_res)[w.lane & 3];
    }
}
template <typename T>
__device__ __forceinline__ void linear_ahead(const LinearEpilogue &e, float (&v)[32], EpiWarp &w, int64_t row0,
                                             int64_t col0, int64_t next, int64_t m, int64_t n) {
    const int lane = w.lane;
    unsigned char *stage = reinterpret_cast<unsigned char *>(w.stage), *other = stage + 2048;
    if (e.bias != nullptr) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            union { uint4 u; T t[16 / sizeof(T)]; } x;
            x.u = w.bias[q];
#pragma unroll
            for (int c = 0; c < 8; ++c) v[8 * q + c] += to_f32<T>(x.t[c % (16 / sizeof(T))]);
        }
    }
    if (e.residual != nullptr) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint4 *>(other + piece_at(lane / 4 + 8 * q, lane & 3)) = w.res[q];
    }
    if (next >= 0 && chunk_ahead<T>(e, next, n)) ask_ahead<T>(e, w, row0, next, m);
    apply_act(v, e.act);
    __syncwarp();
    if (e.residual != nullptr) {
        float t[32];
        rows_from_stage<T>(other, t, lane);
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] += t[c];
    }
    rows_to_stage<T>(stage, v, lane);
    __syncwarp();
    stage_global<T, true>(stage, static_cast<T *>(e.out) + row0 * e.ld_out + col0, e.ld_out,
                          static_cast<int>(min(static_cast<int64_t>(32), m - row0)), lane);
    __syncwarp();
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
// tile, so that a warp's store is a whole 64- or 128-byte piece of a row.  (16-bit
// rows of odd length, 4608 x 29649: 248 us, where aligned ones take 208; their
// aligned 16-byte pieces turned into place, with the values around them apart,
// took 318.)
template <typename T>
__device__ __forceinline__ void columns_store(T *p, int64_t ld, const float *stage, int rows, bool in, int lane) {
#pragma unroll 8
    for (int r = 0; r < rows; ++r)
        if (in) p[r * ld] = from_f32<T>(stage[stage_at(r, lane)]);
}
template <typename T>
__device__ __forceinline__ void linear_columns(const LinearEpilogue &e, float (&v)[32], float *stage, int64_t row0,
                                               int64_t col0, int rows, int64_t n, int lane, bool exact_scale,
                                               int row_exp, int col_exp) {
    const int64_t col = col0 + lane;
    const bool in = col < n;
    const float bias = in && e.bias != nullptr ? to_f32(static_cast<const T *>(e.bias)[col]) : 0.0f;
    const float factor = exact_scale ? 1.0f : __int_as_float((col_exp + 127) << 23);
    const float row_factor = exact_scale ? 1.0f : __int_as_float((row_exp + 127) << 23);
    T *out = static_cast<T *>(e.out) + row0 * e.ld_out + col;
    if (!exact_scale) {
        if (e.row_exp != nullptr) {
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] *= row_factor;
        }
        if (e.z == nullptr && e.act == kActNone && e.residual == nullptr && rows == 32) {
            stage_rows(stage, v, lane);
            __syncwarp();
#pragma unroll
            for (int r = 0; r < 32; ++r) {
                const T y = from_f32<T>(fmaf(stage[stage_at(r, lane)], factor, bias));
                if (in) *out = y;
                out += e.ld_out;
            }
            return;
        }
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] = fmaf(v[c], __shfl_sync(kFull, factor, c), __shfl_sync(kFull, bias, c));
    } else {
#pragma unroll 1
        for (int c0 = 0; c0 < 32; c0 += 8) {
#pragma unroll
            for (int c = 0; c < 32; ++c)
                if (c >= c0 && c < c0 + 8)
                    v[c] = scale_pow2(v[c], row_exp + __shfl_sync(kFull, col_exp, c)) + __shfl_sync(kFull, bias, c);
        }
    }
    if (e.z != nullptr) {
        stage_rows(stage, v, lane);
        __syncwarp();
        columns_store<float>(e.z + row0 * e.ld_z + col, e.ld_z, stage, rows, in, lane);
        __syncwarp();
    }
    apply_act(v, e.act);
    stage_rows(stage, v, lane);
    __syncwarp();
    if (e.residual == nullptr) {
        columns_store<T>(out, e.ld_out, stage, rows, in, lane);
        return;
    }
    const T *res = static_cast<const T *>(e.residual) + row0 * e.ld_res + col;
    T y[32];  // in flight together
#pragma unroll
    for (int r = 0; r < 32; ++r) y[r] = in && r < rows ? res[r * e.ld_res] : from_f32<T>(0.0f);
#pragma unroll
    for (int r = 0; r < 32; ++r)
        if (in && r < rows) out[r * e.ld_out] = from_f32<T>(stage[stage_at(r, lane)] + to_f32(y[r]));
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
    linear_columns<T>(e, v, stage, row0, col0, rows, n, lane, exact_scale, re, ce);
    __syncwarp();
}

template <typename T>
struct EpiLinear {
    LinearEpilogue p;
    __device__ __forceinline__ void ask(EpiWarp &w, int64_t row0, int64_t col0, int64_t m, int64_t n) const {
        if (chunk_ahead<T>(p, col0, n)) ask_ahead<T>(p, w, row0, col0, m);
    }
    // next: the warp's next chunk of the tile, or -1
    __device__ __forceinline__ void operator()(float (&v)[32], EpiWarp &w, int b, int64_t row0, int64_t col0, int64_t next,
                                               int64_t m, int64_t n) const {
        if (chunk_ahead<T>(p, col0, n)) {
            linear_ahead<T>(p, v, w, row0, col0, next, m, n);
        } else if (p.out_batch == 0) {
            linear_store<T>(p, v, w.stage, row0, col0, m, n, w.lane);
        } else {
            LinearEpilogue q = p;
            q.out = static_cast<T *>(p.out) + b * p.out_batch;
            linear_store<T>(q, v, w.stage, row0, col0, m, n, w.lane);
        }
    }
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
__device__ __forceinline__ void final_store(const FinalOutput &e, const float (&v)[32], float *stage, int b,
                                            int64_t row0, int64_t col0, int64_t m, int64_t n, int lane) {
    T *out = static_cast<T *>(e.out.ptr) + e.out.at(b, e.nb2);
    const float *base = e.base.ptr != nullptr ? static_cast<const float *>(e.base.ptr) + e.base.at(b, e.nb2) : nullptr;
    const bool closed = e.gate != nullptr && *e.gate == 0.0f;
    const bool by_row = e.out.i == 1;  // lane = row is the contiguous direction
    if constexpr (sizeof(T) == 2) {
        // whole tiles whose lines start on 16 bytes: side by side through the staging tile
        const int64_t pitch = by_row ? e.out.j : e.out.i;
        if (base == nullptr && row0 + 32 <= m && col0 + 32 <= n && (by_row || e.out.j == 1) && pitch % 8 == 0 &&
            (reinterpret_cast<uintptr_t>(out) & 15) == 0) {
            unsigned char *tile = reinterpret_cast<unsigned char *>(stage);
            if (by_row) {
#pragma unroll
                for (int c = 0; c < 32; ++c)
                    *reinterpret_cast<T *>(tile + piece_at(c, lane >> 3) + 2 * (lane & 7)) = from_f32<T>(v[c]);
            } else {
                rows_to_stage<T>(tile, v, lane);
            }
            __syncwarp();
            stage_global<T, true>(tile, out + (by_row ? row0 + col0 * pitch : row0 * pitch + col0), pitch, 32, lane);
            __syncwarp();
            return;
        }
    }
    if (!by_row) {
        stage_rows(stage, v, lane);
        __syncwarp();
    }
    const int64_t row = by_row ? row0 + lane : row0, col = by_row ? col0 : col0 + lane;
    const int lines = static_cast<int>(min(static_cast<int64_t>(32), by_row ? n - col0 : m - row0));
    const bool in = row < m && col < n;
    T *po = out + row * e.out.i + col * e.out.j;
    const float *pb = base != nullptr ? base + row * e.base.i + col * e.base.j : nullptr;
    const int64_t so = by_row ? e.out.j : e.out.i, sb = by_row ? e.base.j : e.base.i;
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
            if (base != nullptr) x[k] = closed ? b0[k] : fmaf(e.keep, b0[k], x[k]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (in && l0 + k < lines) po[k * so] = from_f32<T>(x[k]);
        po += 8 * so;
        pb += 8 * sb;
    }
    __syncwarp();
}

// The epilogue of a Newton-Schulz product, v = alpha * acc + beta * C.  Planes
// go to and come from memory by TMA, whole 32 x 32 tiles through the warp's
// staging tile; C for a tile's first chunk is loaded under the products.
struct PlanesJob {
    float alpha, beta;
    const CUtensorMap *c, *out, *out2;  // C and out2 may be absent; out is, where the result is final
    float alpha2, diag;                 // out2 = alpha2 * v + diag on the diagonal
    bool symmetric;                     // elements on and below the diagonal, the others as their mirror image
};

__device__ __forceinline__ bool planes_wanted(const PlanesJob &p, int64_t row0, int64_t col0) {
    return !p.symmetric || col0 <= row0;
}
__device__ __forceinline__ void planes_load_c(const PlanesJob &p, EpiWarp &w, int tile, int b, int64_t row0, int64_t col0) {
    w.asked |= 1u << tile;
    if (w.lane == 0) {
        bar_expect(w.bar + 8 * tile, 4096);
        asm volatile(
            "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(w.stage + 1024 * tile)),
            "l"(reinterpret_cast<uint64_t>(p.c)), "r"(w.bar + 8 * tile), "r"(static_cast<int>(col0)),
            "r"(static_cast<int>(row0)), "r"(0), "r"(b) : "memory");
    }
}
// tile: the staging tile, into which C of this chunk has been asked for.  ok: the
// products are there; else the tile becomes NaN.
__device__ __forceinline__ void planes_chunk(const PlanesJob &p, const FinalOutput &f, float (&v)[32], EpiWarp &w, int tile,
                                             int b, int64_t row0, int64_t col0, int64_t m, int64_t n, bool ok) {
    const int lane = w.lane;
    float *tile_f = w.stage + 1024 * tile;
    unsigned char *stage = reinterpret_cast<unsigned char *>(tile_f);
    const uint32_t s32 = smem_u32(stage);
    if ((w.asked >> tile) & 1u) {
        ok = __all_sync(kFull, landed(w.bar + 8 * tile, (w.phase >> tile) & 1u)) && ok;
        w.phase ^= 1u << tile;
        w.asked ^= 1u << tile;
    } else if (p.c != nullptr) {
        ok = false;
    }
    if (!ok) {
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] = __int_as_float(0x7fc00000);
    } else if (p.c != nullptr) {
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
    if (p.out == nullptr) {
        if (f.dtype == kOutF32) final_store<float>(f, v, tile_f, b, row0, col0, m, n, lane);
        else if (f.dtype == kOutF16) final_store<__half>(f, v, tile_f, b, row0, col0, m, n, lane);
        else final_store<__nv_bfloat16>(f, v, tile_f, b, row0, col0, m, n, lane);
        // the staging tile is next written by a TMA load: order it behind these accesses
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        return;
    }
    const int row = static_cast<int>(row0), col = static_cast<int>(col0);
    if (p.symmetric && col == row) {
        // the tile on the diagonal: its upper half from the lower
        stage_rows(tile_f, v, lane);
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] = tile_f[stage_at(max(c, lane), min(c, lane))];
        __syncwarp();
    }
#pragma unroll 1
    for (int o = 0; o < (p.out2 != nullptr ? 2 : 1); ++o) {
        const CUtensorMap *map = o == 0 ? p.out : p.out2;
        if (o == 1) {
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = p.alpha2 * v[c] + (col + c == row + lane ? p.diag : 0.0f);
        }
        planes_to_stage(stage, v, lane);
        stage_store(map, s32, col, row, b, lane);
        if (p.symmetric && col != row) {
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

// ---- what a kernel works through: tiles in one order for all its roles ----------
struct Job {
    const CUtensorMap *a, *b;
    int a_mn, b_mn;
    int row, col, width;   // the pair's tile: 256 rows, `width` columns (a multiple of 32)
    int m, n;              // bounds of the output
    int batch_a, batch_b, batch_out;
    int kb0, kb1;          // contraction, in blocks of kBK
    int wrap;              // from this block on, A's second plane with B once more
    int per_acc;           // blocks per accumulator (planes; 1 << 28: all)
    int phase;
};
struct Cursor {
    int phase, base;       // of the tile looked at last
    int seen;              // the dependency known to be met: phase * batch + matrix, or -1
};

// One product.
template <typename Epi>
struct SingleWork {
    CUtensorMap map_a, map_b;
    int m, n, kblocks, splits;  // splits > 1: the contraction in parts, one output each
    int in_turn;                // A's two planes one after the other
    int a_mn, b_mn, per_acc;
    TileGrid grid;
    uint32_t types;             // of the instruction descriptor
    Epi epi;

    __device__ __forceinline__ int total() const { return grid.total; }
    template <int BN>
    __device__ __forceinline__ Job job(int t, Cursor &) const {
        Job j;
        int b, ti, tj;
        tile_of<BN>(grid, t, b, ti, tj);
        const int mat = b / splits, part = b - mat * splits, per = (kblocks + splits - 1) / splits;
        j.a = &map_a;
        j.b = &map_b;
        j.a_mn = a_mn;
        j.b_mn = b_mn;
        j.row = ti * 2 * kBM;
        j.col = tj * BN;
        j.width = min(BN, (n - j.col + 31) & ~31);
        j.m = m;
        j.n = n;
        j.batch_a = j.batch_b = mat;
        j.batch_out = b;
        j.kb0 = part * per;
        j.kb1 = in_turn ? 2 * kblocks : min(kblocks, j.kb0 + per);
        j.wrap = in_turn ? kblocks : 1 << 28;
        j.per_acc = per_acc;
        j.phase = 0;
        return j;
    }
    __device__ __forceinline__ bool wait(const Job &, Cursor &, volatile int *) const { return true; }
    static constexpr int kTiles = 1;  // staging tiles per epilogue warp
    __device__ __forceinline__ float cross() const { return epi.p.second; }
    __device__ __forceinline__ void ask(const Job &j, EpiWarp &w, int, int64_t row0, int64_t col0) const {
        epi.ask(w, row0, col0, j.m, j.n);
    }
    static constexpr bool kAskNext = false;  // the epilogue asks for its next chunk itself
    // (a tile that failed holds NaN)
    __device__ __forceinline__ void chunk(const Job &j, float (&v)[32], EpiWarp &w, int, int64_t row0, int64_t col0,
                                          int64_t next, bool) const {
        epi(v, w, j.batch_out, row0, col0, next, j.m, j.n);
    }
    __device__ __forceinline__ void done(const Job &, EpiWarp &) const {}
};

// All products of a Newton-Schulz run.  A phase is one product (or two that do
// not depend on each other) of every matrix of the batch; a matrix' tiles of a
// phase start once its tiles of the phase before are complete, whatever the
// other matrices do, so that the next phase's tiles fill the SMs that the last
// tiles of this one leave idle.  The tiles are dealt out in phase order and all
// blocks are resident (a cooperative launch), so the tile that a wait is for is
// always being worked on or done.  Against a launch per product: 9 matrices of
// 1644 x 1645 2371 -> 2189 us, one of 29649 x 1024 (five steps in one segment) 750
// -> 599 us.  Nine matrices
// of 474 x 475 take 210 us, 14 us for each of 15 phases: the matrix instructions
// of a tile are 3 us of it, the rest is its way through loads, epilogue, stores
// and the next phase's wait.
struct NsWork {
    static constexpr int kTiles = 2;
    __device__ __forceinline__ float cross() const { return 1.0f; }
    CUtensorMap ka[kNsBuffers], kb[kNsBuffers], pl[kNsBuffers], mn[2];
    NsProgram p;
    TileGrid sym, full;
    int *done_count;            // [phases, batch], zero at the start
    int phases, first, stop;    // all phases; this launch runs those from first to stop - 1
    uint32_t types;

    __device__ __forceinline__ int last() const { return p.steps - 1; }
    // Gram form, phase 1 + 3 k + j: j = 0 B_k; j = 1 Q_k and T_k; j = 2 A_{k+1}, or the result
    __device__ __forceinline__ int parts(int phase) const {
        if (!p.gram || phase == 0 || (phase - 1) % 3 != 1) return 1;
        const int k = (phase - 1) / 3;
        return (k > 0 ? 1 : 0) + (k < last() ? 1 : 0);
    }
    __device__ __forceinline__ bool is_full(int phase) const {
        return phase == phases - 1 || (!p.gram && phase % 3 == 2);
    }
    __device__ __forceinline__ int tiles(int phase) const {  // of one matrix
        return is_full(phase) ? full.per_batch : sym.per_batch * parts(phase);
    }
    __device__ __forceinline__ int total() const {
        int t = 0;
        for (int q = first; q < stop; ++q) t += tiles(q) * p.batch;
        return t;
    }
    // which product of the phase a tile of it belongs to: its position in its matrix' tiles
    __device__ __forceinline__ int part_of(int phase, int r) const {
        const int one = sym.per_batch;
        const int which = parts(phase) == 2 ? r / one : 0;
        return parts(phase) == 1 && p.gram && phase > 0 && (phase - 1) % 3 == 1 && (phase - 1) / 3 == 0 ? 1 : which;
    }
    struct Product {
        int a, b, b_mn, k, n, c, out, out2;  // buffers (-1: none)
        float alpha, beta, alpha2, diag;
    };
    __device__ __forceinline__ Product product(int phase, int part) const {
        Product q;
        q.b_mn = 0;
        q.k = p.lo;
        q.n = p.lo;
        q.out2 = -1;
        q.alpha2 = q.diag = 0.0f;
        int kind, k;  // 0: A = X X^T, 1: B, 2: X' (direct) or the result, 3: Q, 4: T, 5: A' = P A P
        if (!p.gram) {
            k = phase / 3;
            kind = phase % 3;
        } else if (phase == 0) {
            k = 0;
            kind = 0;
        } else if (phase == phases - 1) {
            k = last();
            kind = 2;
        } else {
            k = (phase - 1) / 3;
            const int j = (phase - 1) % 3;
            kind = j == 0 ? 1 : j == 2 ? 5 : part == 0 ? 3 : 4;
        }
        const int x = p.gram ? 0 : k & 1;
        if (kind == 0) {
            q.a = q.b = x;
            q.k = p.hi;
            q.c = -1;
            q.alpha = p.scale_a / (p.scale_x * p.scale_x);
            q.beta = 0.0f;
            q.out = kNsA;
        } else if (kind == 1) {
            q.a = q.b = q.c = kNsA;
            q.alpha = p.c / p.scale_a;
            q.beta = p.b;
            q.out = kNsB;
            if (p.gram && k == 0) {
                q.out2 = kNsQ;
                q.alpha2 = p.scale_q / p.scale_a;
                q.diag = p.a * p.scale_q;
            }
        } else if (kind == 2) {
            q.n = p.hi;
            q.b = x;
            q.b_mn = 1;
            q.out = phase == phases - 1 && p.last ? -1 : x ^ 1;
            if (p.gram) {
                q.a = kNsQ + (last() & 1);
                q.c = -1;
                q.alpha = q.out < 0 ? p.factor / (p.scale_q * p.scale_x) : 1.0f / p.scale_q;
                q.beta = 0.0f;
            } else {
                const float f = q.out < 0 ? p.factor / p.scale_x : 1.0f;
                q.a = kNsB;
                q.c = x;
                q.alpha = f / p.scale_a;
                q.beta = f * p.a;
            }
        } else {
            // Q <- a Q + B Q;  T = a A + B A;  A <- a T + T B
            q.a = kind == 5 ? kNsT : kNsB;
            q.b = kind == 3 ? kNsQ + ((k - 1) & 1) : kind == 4 ? kNsA : kNsB;
            q.c = kind == 5 ? kNsT : q.b;
            q.out = kind == 3 ? kNsQ + (k & 1) : kind == 4 ? kNsT : kNsA;
            q.alpha = 1.0f / p.scale_a;
            q.beta = p.a;
        }
        return q;
    }
    // phase and matrix of tile t, and its position r among the matrix' tiles
    __device__ __forceinline__ void locate(int t, Cursor &cur, int &b, int &r) const {
        for (;;) {
            const int per = tiles(cur.phase), count = per * p.batch;
            if (t - cur.base < count) {
                b = (t - cur.base) / per;
                r = t - cur.base - b * per;
                return;
            }
            cur.base += count;
            ++cur.phase;
        }
    }
    template <int BN>
    __device__ __forceinline__ Job job(int t, Cursor &cur) const {
        Job j;
        int b, r;
        locate(t, cur, b, r);
        const bool f = is_full(cur.phase);
        const int part = f ? 0 : part_of(cur.phase, r);
        const Product q = product(cur.phase, part);
        const TileGrid &g = f ? full : sym;
        int zero, ti, tj;
        tile_of<BN>(g, f ? r : r % sym.per_batch, zero, ti, tj);
        j.a = ka + q.a;
        j.b = q.b_mn ? mn + q.b : kb + q.b;
        j.a_mn = 0;
        j.b_mn = q.b_mn;
        j.row = ti * 2 * kBM;
        j.col = tj * BN;
        j.m = p.lo;
        j.n = q.n;
        j.width = min(BN, (q.n - j.col + 31) & ~31);
        j.batch_a = j.batch_b = j.batch_out = b;
        j.kb0 = 0;
        j.kb1 = (q.k + kBK - 1) / kBK;
        j.wrap = 1 << 28;
        j.per_acc = p.gram ? 3 : 6;
        j.phase = cur.phase | (part << 16);
        return j;
    }
    __device__ __forceinline__ PlanesJob planes(const Job &j) const {
        const int phase = j.phase & 65535;
        const Product q = product(phase, j.phase >> 16);
        PlanesJob e;
        e.alpha = q.alpha;
        e.beta = q.beta;
        const int shift = p.shift[j.batch_out];
        if (shift != 0 && (phase == 0 || (!p.gram && phase % 3 == 0))) {
            e.alpha *= exp2f(-2.0f * static_cast<float>(shift));  // A = X X^T
        } else if (shift != 0 && phase == phases - 1 && p.last) {
            e.alpha *= exp2f(-static_cast<float>(shift));
            e.beta *= exp2f(-static_cast<float>(shift));
        }
        e.c = q.c < 0 ? nullptr : pl + q.c;
        e.out = q.out < 0 ? nullptr : pl + q.out;
        e.out2 = q.out2 < 0 ? nullptr : pl + q.out2;
        e.alpha2 = q.alpha2;
        e.diag = q.diag;
        e.symmetric = !is_full(phase);
        return e;
    }
    // Until the matrix' tiles of the phase before are complete (both CTAs count
    // each).  All lanes call it.
    __device__ __forceinline__ bool wait(const Job &j, Cursor &cur, volatile int *failed) const {
        const int phase = j.phase & 65535;
        if (phase == first) return true;
        const int at = (phase - 1) * p.batch + j.batch_out;
        if (cur.seen == at) return true;
        const int want = tiles(phase - 1) * 2;
        uint64_t start = 0, now = 0;
        for (int i = 0;; ++i) {
            int have;
            asm volatile("ld.acquire.gpu.global.b32 %0, [%1];" : "=r"(have) : "l"(done_count + at) : "memory");
            if (__all_sync(kFull, have >= want)) break;
            if ((i & 63) == 0) {
                asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
                if (start == 0) start = now;
                const bool over = now - start >= *const_cast<volatile uint64_t *>(&g_phase_limit);
                if (__any_sync(kFull, over)) {
                    atomicExch(&g_gemm_fault, 1);
                    *failed = 1;
                }
                if (__any_sync(kFull, *failed != 0)) return false;
            }
        }
        asm volatile("fence.proxy.async.global;" ::: "memory");  // the loads that follow go through the other proxy
        cur.seen = at;
        return true;
    }
    // C of a chunk into a staging tile that is free
    __device__ __forceinline__ void ask(const Job &j, EpiWarp &w, int tile, int64_t row0, int64_t col0) const {
        const PlanesJob e = planes(j);
        if (e.c != nullptr && planes_wanted(e, row0, col0)) planes_load_c(e, w, tile, j.batch_out, row0, col0);
    }
    static constexpr bool kAskNext = true;
    __device__ __forceinline__ void chunk(const Job &j, float (&v)[32], EpiWarp &w, int tile, int64_t row0, int64_t col0,
                                          int64_t, bool ok) const {
        const PlanesJob e = planes(j);
        if (planes_wanted(e, row0, col0))
            planes_chunk(e, p.final, v, w, tile, j.batch_out, row0, col0, j.m, j.n, ok);
    }
    // The tile's part of this CTA is in memory: one count for all its epilogue warps.
    __device__ __forceinline__ void done(const Job &j, EpiWarp &w) const {
        const int phase = j.phase & 65535;
        if (phase == stop - 1) return;
        // a complete copy is visible to the thread that waited for it; the barrier and the release hand that on
        if (w.lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
        if (threadIdx.x == 0)
            asm volatile("red.release.gpu.global.add.s32 [%0], 1;" ::"l"(done_count + phase * p.batch + j.batch_out)
                         : "memory");
    }
};

template <typename W> __device__ __forceinline__ int work_first(const W &) { return 0; }
__device__ __forceinline__ int work_first(const NsWork &w) { return w.first; }

// The tensor cores truncate where they add to an accumulator, which loses 2e-8
// of the sum per addition: 4e-6 at k = 1024 with the 12 additions that two
// planes take per block of k.  So the two cross products (hi lo, lo hi), 2^-11
// of the whole, have an accumulator of their own, and hi hi is cut into chunks of
// six blocks of k (24 additions, 0.5e-6 whatever k; three blocks where the Gram
// form squares singular values), each into the next of three accumulators; the
// epilogue warps add the chunks in registers, rounding to nearest.  64 sums a
// thread: 128-wide tiles.  (Chunks of two blocks with the
// cross products inside reached the same accuracy 25% slower: three times the
// accumulator reads.  256-wide tiles, 128 sums a thread and one accumulator whose
// reads the cross products covered, took 2950 us instead of 2430 for 9 matrices
// of 1644 x 1645 and 475 instead of 453 for 4608 x 4096 -> 4736.)  16-bit results keep one accumulator per tile.
template <int BN, int PLANES, int TILES>
struct Config {
    static constexpr int kAccs = PLANES == 2 ? 3 : 2;
    static constexpr int kCross = kAccs * BN;                 // the cross products' columns of TMEM
    static constexpr int kColumns = PLANES == 2 ? 4 * BN : 2 * BN;
    static_assert(PLANES == 1 || BN <= 128, "the chunks' sums have to fit the epilogue's registers");
    static constexpr int kA = kBM * kBK * 2;              // bytes of one plane of A per stage
    static constexpr int kB = (BN / 2) * kBK * 2;         // of B (this CTA's half)
    static constexpr int kStage = PLANES * (kA + kB);
    // a second staging tile per epilogue warp, where it has two chunks of 32 columns
    static constexpr int kTiles = TILES < BN / 64 ? TILES : BN / 64;
    static constexpr int kFit = (kStageBudget - (kTiles - 1) * kEpiWarps * 4096) / kStage;
    static constexpr int kStages = kFit > 8 ? 8 : kFit;
    static constexpr int kSmem = kStages * kStage + kTiles * kEpiWarps * 4096 + 1024;
};

template <int BN, int PLANES, typename Work>
__global__ __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1)
void gemm_kernel(const __grid_constant__ Work work) {
    using C = Config<BN, PLANES, Work::kTiles>;
    extern __shared__ unsigned char raw[];
    // (an offset, not a rounded pointer: the compiler keeps knowing that this is shared memory)
    unsigned char *smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    float *stage_epi = reinterpret_cast<float *>(smem + C::kStages * C::kStage);
    __shared__ uint64_t bars[2 * C::kStages + 2 * C::kAccs + 1 + C::kTiles * kEpiWarps];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int failed;

    const int warp = __shfl_sync(kFull, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    uint32_t cta;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(cta));
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const uint32_t full = smem_u32(bars), empty = full + 8 * C::kStages, acc_full = empty + 8 * C::kStages,
                   acc_empty = acc_full + 8 * C::kAccs, cross_empty = acc_empty + 8 * C::kAccs;

    if (threadIdx.x < 2 * C::kStages + 2 * C::kAccs + 1 + C::kTiles * kEpiWarps) {
        const int i = threadIdx.x, k = i - (2 * C::kStages + C::kAccs);
        // accumulators free: every epilogue warp of both CTAs arrives
        bar_init(full + 8 * i, k >= 0 && k <= C::kAccs ? 2 * kEpiWarps : 1);
        if (i == 0) failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(C::kColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;
    const int total = work.total();
    Cursor cur{work_first(work), 0, -1};

    if (warp == kLoadA || warp == kLoadB) {
        // ---- loads ----
        const bool is_a = warp == kLoadA;
        const uint32_t offset = is_a ? 0 : PLANES * C::kA, plane = is_a ? C::kA : C::kB;
        const bool expects = is_a && cta == 0;
        int s = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int t = pair; ok && t < total; t += pairs) {
            const Job j = work.template job<BN>(t, cur);
            ok = work.wait(j, cur, &failed);
            if (!ok) break;
            const CUtensorMap *map = is_a ? j.a : j.b;
            const bool mn = is_a ? j.a_mn != 0 : j.b_mn != 0;
            const int pieces = mn ? (is_a ? kBM / 64 : BN / 128) : 1;  // 64 lines of an MN-major operand per load
            const int line = is_a ? j.row + static_cast<int>(cta) * kBM : j.col + static_cast<int>(cta) * (j.width >> 1);
            const int b = is_a ? j.batch_a : j.batch_b;
            for (int kb = j.kb0; kb < j.kb1; ++kb) {
                ok = warp_wait(empty + 8 * s, phase ^ 1, &failed);
                if (!ok) break;
                const uint32_t dst = smem_u32(smem) + s * C::kStage + offset;
                const int k = (kb >= j.wrap ? kb - j.wrap : kb) * kBK, turn = is_a && kb >= j.wrap ? 1 : 0;
                if (elect_one()) {
                    // the other CTA's and the other warp's bytes may arrive before they are expected
                    if (expects) bar_expect(full + 8 * s, 2 * C::kStage);
                    if (mn) {
                        for (int p = 0; p < PLANES; ++p)
                            for (int h = 0; h < pieces; ++h)
                                tma_load(dst + p * plane + h * 8192, map, full + 8 * s, line + 64 * h, k, p + turn, b);
                    } else {
                        tma_load(dst, map, full + 8 * s, k, line, turn, b);  // all planes
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
        int s = 0, buf = 0;
        uint32_t phase = 0, acc_phase = 0, cross_phase = 0;
        bool ok = true;
        for (int t = pair; ok && t < total; t += pairs) {
            const Job j = work.template job<BN>(t, cur);
            if (PLANES == 2) {
                ok = warp_wait(cross_empty, cross_phase ^ 1, &failed);
                cross_phase ^= 1;
                if (!ok) break;
            }
            const uint32_t a_step = j.a_mn ? 128u : 2u, b_step = j.b_mn ? 128u : 2u;  // 16 of k, in 16-byte units
            const uint32_t a_lbo = j.a_mn ? 8192u : 16u, b_lbo = j.b_mn ? 8192u : 16u;
            const uint32_t idesc = work.types | (static_cast<uint32_t>(j.a_mn) << 15) | (static_cast<uint32_t>(j.b_mn) << 16) |
                                   (static_cast<uint32_t>(j.width >> 3) << 17);
            for (int k0 = j.kb0; ok && k0 < j.kb1; k0 = k0 + j.per_acc < j.kb1 ? k0 + j.per_acc : j.kb1) {
                const int k1 = min(j.kb1, k0 + j.per_acc);
                ok = warp_wait(acc_empty + 8 * buf, acc_phase ^ 1, &failed);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t d = tmem + buf * BN;
                for (int kb = k0; kb < k1; ++kb) {
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
                        for (int i = 0; i < kBK / 16; ++i) {
                            mma_f16(d, da[0] + i * a_step, db[0] + i * b_step, idesc, kb != k0 || i != 0);
                            if (PLANES == 2) {
                                mma_f16(tmem + C::kCross, da[0] + i * a_step, db[PLANES - 1] + i * b_step, idesc,
                                        kb != j.kb0 || i != 0);
                                mma_f16(tmem + C::kCross, da[PLANES - 1] + i * a_step, db[0] + i * b_step, idesc, 1);
                            }
                        }
                        mma_commit(empty + 8 * s);
                    }
                    __syncwarp();
                    if (++s == C::kStages) { s = 0; phase ^= 1; }
                }
                if (elect_one()) mma_commit(acc_full + 8 * buf);
                __syncwarp();
                if (++buf == C::kAccs) { buf = 0; acc_phase ^= 1; }
            }
        }
    } else if (warp < kEpiWarps) {
        // ---- epilogue ----
        EpiWarp w;
        w.stage = stage_epi + warp * C::kTiles * 1024;
        w.bar = cross_empty + 8 + 8 * warp * C::kTiles;
        w.phase = w.asked = 0;
        w.failed = &failed;
        w.lane = lane;
        int buf = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        for (int t = pair; t < total; t += pairs) {
            const Job j = work.template job<BN>(t, cur);
            const int64_t row0 = j.row + static_cast<int>(cta) * kBM + (warp & 3) * 32;
            const int half = (warp >> 2) * (BN / 2);
            const bool any = row0 < j.m && j.col + half < j.n;
            if (ok && any) {
                ok = work.wait(j, cur, &failed);  // (long met: the loads waited for it; here for this warp's own loads)
#pragma unroll
                for (int q = 0; q < C::kTiles; ++q)
                    if (ok && j.col + half + 32 * q < j.n) work.ask(j, w, q, row0, j.col + half + 32 * q);
            }
            const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
            auto next_acc = [&] {
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) bar_arrive_cta0(acc_empty + 8 * buf);
                if (++buf == C::kAccs) { buf = 0; acc_phase ^= 1; }
            };
            auto finish = [&](float (&v)[32], int c) {
                const int tile = ((c - half) >> 5) % C::kTiles, next = c + 32 * C::kTiles;
                const bool more = next < half + BN / 2 && j.col + next < j.n;
                work.chunk(j, v, w, tile, row0, j.col + c, more ? j.col + next : -1, ok);
                __syncwarp();
                if (Work::kAskNext && ok && more) work.ask(j, w, tile, row0, j.col + next);
            };
            if constexpr (PLANES == 2) {
                constexpr int kChunks = BN / 64;
                float sum[kChunks][32];
#pragma unroll
                for (int q = 0; q < kChunks; ++q)
#pragma unroll
                    for (int i = 0; i < 32; ++i) sum[q][i] = 0.0f;
                auto add = [&](uint32_t columns, float factor) {
#pragma unroll
                    for (int q = 0; q < kChunks; ++q) {
                        float v[32];
                        tmem_read32(v, tmem + columns + lanes + half + 32 * q);
#pragma unroll
                        for (int i = 0; i < 32; ++i) sum[q][i] = fmaf(v[i], factor, sum[q][i]);
                    }
                };
                for (int k0 = j.kb0; k0 < j.kb1; k0 += j.per_acc) {
                    if (ok) ok = warp_wait(acc_full + 8 * buf, acc_phase, &failed);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (ok && any) add(buf * BN, 1.0f);
                    next_acc();
                }
                // the last chunk's barrier covers the cross products too
                if (ok && any) add(C::kCross, work.cross());
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) bar_arrive_cta0(cross_empty);
#pragma unroll
                for (int q = 0; q < kChunks; ++q) {
                    const int c = half + 32 * q;
                    if (!any || j.col + c >= j.n) continue;
                    if (!ok) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) sum[q][i] = __int_as_float(0x7fc00000);
                    }
                    finish(sum[q], c);
                }
            } else {
                const bool two = j.kb1 - j.kb0 > j.per_acc;  // A's planes in turn: both accumulators
                if (ok) ok = warp_wait(acc_full + 8 * buf, acc_phase, &failed);
                if (two && ok) ok = warp_wait(acc_full + 8 * (buf ^ 1), acc_phase ^ static_cast<uint32_t>(buf), &failed);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                for (int c = half; c < half + BN / 2; c += 32) {
                    if (!any || j.col + c >= j.n) break;
                    float v[32];
                    if (ok) {
                        tmem_read32(v, tmem + buf * BN + lanes + c);
                        if (two) {
                            float lo[32];
                            tmem_read32(lo, tmem + (buf ^ 1) * BN + lanes + c);
                            const float f0 = work.epi.p.first, f1 = work.epi.p.second;
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = fmaf(f1, lo[i], f0 * v[i]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = __int_as_float(0x7fc00000);
                    }
                    finish(v, c);
                }
                next_acc();
                if (two) next_acc();
            }
            work.done(j, w);
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        __syncwarp();
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kColumns));
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
                         static_cast<cuuint32_t>(o.mn_major || o.in_turn ? 1 : o.planes), 1};
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

TileGrid tile_grid(const GemmShape &s, int bn, int64_t copies) {
    TileGrid g;
    g.tiles_m = static_cast<int>((s.m + 2 * kBM - 1) / (2 * kBM));
    g.tiles_n = static_cast<int>((s.n + bn - 1) / bn);
    g.symmetric = s.symmetric;
    g.batch = static_cast<int>(copies);
    g.n_fast = g.tiles_n <= g.tiles_m;  // the operand with fewer tiles is the one read again and again, from L2
    g.per_batch = static_cast<int>(tile_count(s, bn));
    g.total = static_cast<int>(g.per_batch * copies);
    return g;
}

int sm_pairs() {
    const int sms = fl_device_sm_count();
    return (sms > 1 ? sms : 148) / 2;
}

// fp32 accumulator, operand type, M = 256 (the pair's)
uint32_t instruction_types(int kind) {
    const uint32_t type = kind == kBF16 ? 1u : 0u;
    return (1u << 4) | (type << 7) | (type << 10) | (static_cast<uint32_t>(256 >> 4) << 24);
}

template <int BN, int PLANES, typename Epi>
int run(const GemmShape &s, const GemmOperand &a, const GemmOperand &b, const Epi &epi, int splits, cudaStream_t st) {
    using W = SingleWork<Epi>;
    using C = Config<BN, PLANES, W::kTiles>;
    W w;
    int rc = operand_map(&w.map_a, a, s.m, s.k, s.batch, kBM, s.kind);
    if (rc) return rc;
    rc = operand_map(&w.map_b, b, s.n, s.k, s.batch, BN / 2, s.kind);
    if (rc) return rc;
    FL_REQUIRE(tile_count(s, BN) * s.batch * splits < (1 << 30), "gemm: too many tiles");
    w.m = static_cast<int>(s.m);
    w.n = static_cast<int>(s.n);
    w.kblocks = static_cast<int>((s.k + kBK - 1) / kBK);
    w.splits = splits;
    w.a_mn = a.mn_major;
    w.b_mn = b.mn_major;
    w.in_turn = a.in_turn;
    w.per_acc = PLANES == 1 ? (a.in_turn ? w.kblocks : 1 << 28) : splits > 1 ? 3 : 6;  // (split: the Gram form's first product)
    w.grid = tile_grid(s, BN, s.batch * splits);
    w.types = instruction_types(s.kind);
    w.epi = epi;
    int pairs = sm_pairs();
    if (pairs > w.grid.total) pairs = w.grid.total;
    auto kernel = gemm_kernel<BN, PLANES, W>;
    FL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    note_launch();
    kernel<<<2 * pairs, kThreads, C::kSmem, st>>>(w);
    return check_launch("gemm");
}

int check_shape(const GemmShape &s) {
    FL_REQUIRE(s.m > 0 && s.n > 0 && s.k > 0 && s.batch > 0 && s.m < (1ll << 31) - 512 && s.n < (1ll << 31) - 512 &&
                   s.k < (1ll << 31) - 512 && s.batch < (1ll << 31),
               "gemm: bad shape");
    return FL_OK;
}

// 256-wide or 128-wide tiles: whichever needs less time on the slowest pair of
// SMs.  A 256-wide tile takes 1.6 times a 128-wide one, whose loads (62 bytes per
// clock and SM instead of 43) the L2 does not deliver at the full matrix rate:
// 29649 x 1024 x 4608 took 360 us in 128-wide tiles, 13 rounds of them, and
// 200 us in 256-wide ones, 7 rounds.
bool wide_tiles(const GemmShape &s) {
    const int64_t pairs = sm_pairs();
    const int64_t wide = (tile_count(s, 256) * s.batch + pairs - 1) / pairs;
    const int64_t narrow = (tile_count(s, 128) * s.batch + pairs - 1) / pairs;
    return 8 * wide <= 5 * narrow;
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
    constexpr int kPlanes = sizeof(T) == 4 ? 2 : 1;
    if constexpr (kPlanes == 1)
        if (wide_tiles(s)) return run<256, 1>(s, a, b, epi, 1, st);
    return run<128, kPlanes>(s, a, b, epi, 1, st);
}

template <int BN>
int launch_ns(const NsProgram &p, const NsBuffer *buf, int phases, int first, int stop, int *done_count, cudaStream_t st) {
    using C = Config<BN, 2, NsWork::kTiles>;
    NsWork w{};
    w.p = p;
    w.phases = phases;
    w.first = first;
    w.stop = stop;
    w.done_count = done_count;
    w.types = instruction_types(kF16);
    GemmShape square{p.lo, p.lo, p.lo, p.batch, 1, kF16}, full{p.lo, p.hi, p.lo, p.batch, 0, kF16};
    w.sym = tile_grid(square, BN, 1);
    w.full = tile_grid(full, BN, 1);
    FL_REQUIRE(static_cast<double>(w.full.per_batch) * p.batch * phases * 2 < 1e9, "newton-schulz: too many tiles");
    for (int i = 0; i < kNsBuffers; ++i) {
        if (buf[i].p == nullptr) continue;
        const int cols = i < 2 ? p.hi : p.lo;
        GemmOperand o{buf[i].p, buf[i].ld, buf[i].plane, 2 * buf[i].plane, 2, 0};
        int rc = operand_map(&w.ka[i], o, p.lo, cols, p.batch, kBM, kF16);
        if (!rc) rc = operand_map(&w.kb[i], o, p.lo, cols, p.batch, BN / 2, kF16);
        if (!rc) rc = planes_map(&w.pl[i], buf[i].p, o.ld, o.plane, o.batch, p.lo, cols, p.batch);
        o.mn_major = 1;
        if (!rc && i < 2 && BN >= 128) rc = operand_map(&w.mn[i], o, p.hi, p.lo, p.batch, BN / 2, kF16);
        if (rc) return rc;
    }
    auto kernel = gemm_kernel<BN, 2, NsWork>;
    FL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeCooperative;  // the blocks wait for one another: all resident, or no launch
    attr[0].val.cooperative = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int64_t most = static_cast<int64_t>(w.full.per_batch > 2 * w.sym.per_batch ? w.full.per_batch : 2 * w.sym.per_batch) * p.batch;
    int pairs = sm_pairs();
    if (pairs > most) pairs = static_cast<int>(most);
    cfg.gridDim = dim3(2 * pairs);
    // pairs of SMs that can be resident at once, asked once per device
    static thread_local int known_device = -1, known_pairs = 0;
    int device = 0;
    FL_CUDA(cudaGetDevice(&device));
    if (known_device != device) {
        cudaLaunchConfig_t q = cfg;
        cudaLaunchAttribute qa[1];
        qa[0].id = cudaLaunchAttributeClusterDimension;
        qa[0].val.clusterDim.x = 2;
        qa[0].val.clusterDim.y = qa[0].val.clusterDim.z = 1;
        q.attrs = qa;
        q.numAttrs = 1;
        q.gridDim = dim3(2 * sm_pairs());
        FL_CUDA(cudaOccupancyMaxActiveClusters(&known_pairs, kernel, &q));
        known_device = device;
    }
    FL_REQUIRE(known_pairs > 0, "newton-schulz: no pair of SMs can hold the kernel");
    if (pairs > known_pairs) cfg.gridDim = dim3(2 * known_pairs);
    note_launch();
    FL_CUDA(cudaLaunchKernelEx(&cfg, kernel, w));
    return check_launch("newton-schulz products");
}

// Sums the parts of A = X X^T into planes, both halves from the lower one: 32 x 32
// tiles, grid (tiles, tiles, batch).
__global__ void __launch_bounds__(256) combine_kernel(const float *parts, int splits, int lo, int64_t ldp, float scale,
                                                      const int *shift, __half *out, int64_t ld, int64_t plane) {
    __shared__ float tile[32][33];
    if (blockIdx.x > blockIdx.y) return;
    const int64_t b = blockIdx.z;
    const float alpha = scale * exp2f(-2.0f * static_cast<float>(shift[b]));
    const int i0 = blockIdx.y * 32, j0 = blockIdx.x * 32;
    const int64_t size = static_cast<int64_t>(lo) * ldp;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int i = i0 + threadIdx.y + 8 * q, j = j0 + threadIdx.x;
        float s = 0.0f;
        if (i < lo && j < lo)
            for (int k = 0; k < splits; ++k) s += parts[(b * splits + k) * size + i * ldp + j];
        tile[threadIdx.y + 8 * q][threadIdx.x] = s * alpha;
    }
    __syncthreads();
    __half *hi = out + b * 2 * plane;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int r = threadIdx.y + 8 * q, c = threadIdx.x;
        for (int turned = 0; turned < 2; ++turned) {
            if (turned && blockIdx.x == blockIdx.y) continue;
            const int i = (turned ? j0 : i0) + r, j = (turned ? i0 : j0) + c;
            if (i >= lo || j >= lo) continue;
            const float v = turned ? tile[c][r] : blockIdx.x == blockIdx.y && c > r ? tile[c][r] : tile[r][c];
            const __half h = __float2half_rn(v);
            hi[i * ld + j] = h;
            hi[plane + i * ld + j] = __float2half_rn(v - __half2float(h));
        }
    }
}

// How A = X X^T is split along the long side: enough parts to fill the pairs of
// SMs, each at least 8 blocks of k long; 1 when its tiles fill half of them.
int outer_splits(int64_t lo, int64_t hi, int64_t batch) {
    GemmShape s{lo, lo, hi, batch, 1, kF16};
    const int64_t tiles = tile_count(s, 128) * batch, kblocks = (hi + kBK - 1) / kBK;
    int64_t n = sm_pairs() / tiles;
    if (n > kblocks / 8) n = kblocks / 8;
    if (n < 2) return 1;
    const int64_t per = (kblocks + n - 1) / n;
    return static_cast<int>((kblocks + per - 1) / per);  // every part has blocks
}

}  // namespace

int gemm_linear(const GemmShape &s, const GemmOperand &a, const GemmOperand &b, const LinearEpilogue &e,
                cudaStream_t st) {
    const int planes = e.dtype == kOutF32 ? 2 : 1;
    FL_REQUIRE(a.planes == (a.in_turn ? 2 : planes) && b.planes == planes && !b.in_turn && !s.symmetric &&
                   (!a.in_turn || planes == 1),
               "gemm: planes");
    const int rc = check_shape(s);
    if (rc) return rc;
    FL_REQUIRE(!a.in_turn || s.k < (1ll << 30), "gemm: bad shape");
    if (e.dtype == kOutF32) return linear_typed<float>(s, a, b, e, st);
    if (e.dtype == kOutF16) return linear_typed<__half>(s, a, b, e, st);
    return linear_typed<__nv_bfloat16>(s, a, b, e, st);
}

// At most three steps on squared singular values, then X is formed and squared
// again (see muon.cu).
int ns_segments(int steps, int gram) { return gram ? (steps + 2) / 3 : 1; }

namespace {
int segment_phases(int steps, int gram) { return gram ? (steps == 1 ? 3 : 1 + 3 * steps) : 3 * steps; }
}  // namespace

int ns_phases(int steps, int gram) {
    const int segments = ns_segments(steps, gram);
    int phases = 0;
    for (int i = 0; i < segments; ++i) phases += segment_phases(ns_segment_steps(steps, segments, i), gram);
    return phases;
}

size_t ns_parts_bytes(int64_t lo, int64_t hi, int64_t batch) {
    const int64_t n = outer_splits(lo, hi, batch);
    return n > 1 ? static_cast<size_t>(n * batch * lo * ((lo + 7) & ~int64_t(7))) * sizeof(float) : 0;
}

static int ns_segment(const NsProgram &p, const NsBuffer *buf, int *done_count, float *parts, cudaStream_t st) {
    const int phases = segment_phases(p.steps, p.gram);
    GemmShape outer{p.lo, p.lo, p.hi, p.batch, 1, kF16};
    int rc = check_shape(outer);
    if (rc) return rc;
    FL_REQUIRE(phases < 65536, "newton-schulz: too many steps");
    const int splits = p.gram ? outer_splits(p.lo, p.hi, p.batch) : 1;
    if (splits > 1) {
        const GemmOperand x{buf[kNsX].p, buf[kNsX].ld, buf[kNsX].plane, 2 * buf[kNsX].plane, 2, 0};
        EpiLinear<float> e{};
        e.p.out = parts;
        e.p.ld_out = (p.lo + 7) & ~7;
        e.p.out_batch = p.lo * e.p.ld_out;
        e.p.second = 1.0f;
        e.p.dtype = kOutF32;
        e.p.aligned = 1;
        rc = run<128, 2>(outer, x, x, e, splits, st);
        if (rc) return rc;
        const unsigned tiles = static_cast<unsigned>((p.lo + 31) / 32);
        launch(combine_kernel, dim3(tiles, tiles, static_cast<unsigned>(p.batch)), dim3(32, 8), 0, st, parts, splits, p.lo,
               e.p.ld_out, p.scale_a / (p.scale_x * p.scale_x), p.shift, buf[kNsA].p, buf[kNsA].ld, buf[kNsA].plane);
        rc = check_launch("newton-schulz combine");
        if (rc) return rc;
    }
    const int first = splits > 1 ? 1 : 0;
    // Few matrices: 64-wide tiles put the short products on twice the SMs and leave each half the products and
    // half the epilogue, which is most of a phase's time; the last product, with X, has tiles enough.
    const GemmShape square{p.lo, p.lo, p.lo, p.batch, 1, kF16};
    if (p.gram && tile_count(square, 64) * p.batch <= sm_pairs()) {
        rc = launch_ns<64>(p, buf, phases, first, phases - 1, done_count, st);
        return rc ? rc : launch_ns<128>(p, buf, phases, phases - 1, phases, done_count, st);
    }
    return launch_ns<128>(p, buf, phases, first, phases, done_count, st);
}

int ns_products(const NsProgram &program, const NsBuffer *buffers, int *done_count, float *parts, cudaStream_t st) {
    const int segments = ns_segments(program.steps, program.gram);
    NsBuffer buf[kNsBuffers];
    for (int i = 0; i < kNsBuffers; ++i) buf[i] = buffers[i];
    for (int i = 0; i < segments; ++i) {
        NsProgram p = program;
        p.steps = ns_segment_steps(program.steps, segments, i);
        p.last = i == segments - 1;
        const int rc = ns_segment(p, buf, done_count, parts, st);
        if (rc) return rc;
        done_count += segment_phases(p.steps, p.gram) * p.batch;
        const NsBuffer x = buf[kNsX];  // the next segment starts from what this one has written
        buf[kNsX] = buf[kNsX2];
        buf[kNsX2] = x;
    }
    return FL_OK;
}

// Reads and clears the device fault word (synchronizes the device).
int gemm_fault(int *fault) {
    int zero = 0;
    FL_REQUIRE(fault != nullptr, "gemm_fault: null result");
    FL_CUDA(cudaDeviceSynchronize());  // (a copy waits for streams that block the legacy one only)
    FL_CUDA(cudaMemcpyFromSymbol(fault, g_gemm_fault, sizeof(int)));
    if (*fault) FL_CUDA(cudaMemcpyToSymbol(g_gemm_fault, &zero, sizeof(int)));
    return FL_OK;
}

int gemm_wait_limits(int64_t wait_ns, int64_t phase_ns) {
    FL_REQUIRE(wait_ns >= 0 && phase_ns >= 0, "gemm_wait_limits: limits must be at least 0");
    const uint64_t wait = static_cast<uint64_t>(wait_ns), phase = static_cast<uint64_t>(phase_ns);
    FL_CUDA(cudaDeviceSynchronize());
    FL_CUDA(cudaMemcpyToSymbol(g_wait_limit, &wait, sizeof(wait)));
    FL_CUDA(cudaMemcpyToSymbol(g_phase_limit, &phase, sizeof(phase)));
    return FL_OK;
}

}  // namespace fl

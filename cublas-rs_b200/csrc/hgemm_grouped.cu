// hgemm_grouped.cu -- matrix products of ragged row groups: the products of
// an expert layer whose tokens are sorted by expert.  No counterpart in
// cublas-rs, whose batched family (crates/cublas-l3/src/batched.rs) takes one
// size for every matrix of a batch.
//
//   forward   C[r] = alpha * A[r] op(B_g) + beta * C[r],  r in group g
//   wgrad     C_g = alpha * A[rows of g]^T B[rows of g] + beta * C_g
//
// 16-bit operands (f16 or bf16), f32 sums.
#include <cuda.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <mutex>

#include "half_types.cuh"
#include "internal.h"
#include "sm100.cuh"

namespace {

constexpr int kMaxGroups = 1024;

// Tiles of `bm` rows that groups 0..g-1 hold, for g = 0..groups, in
// start[0..groups], and the offsets themselves in off[0..groups]; false when
// the offsets do not ascend within [0, rows].
// One warp; every lane returns the verdict.
__device__ bool scan_groups(const int32_t *offsets, int groups, int64_t rows, int bm, int *start, int *off) {
    const int lane = threadIdx.x & 31;
    bool ok = true;
    int carry = 0;
    for (int g0 = 0; g0 < groups; g0 += 32) {
        const int g = g0 + lane;
        int tiles = 0;
        if (g < groups) {
            const int64_t lo = offsets[g], hi = offsets[g + 1];
            off[g] = static_cast<int>(lo);
            if (g == groups - 1) off[groups] = static_cast<int>(hi);
            if (lo < 0 || hi < lo || hi > rows)
                ok = false;
            else
                tiles = static_cast<int>((hi - lo + bm - 1) / bm);
        }
        int sum = tiles;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += up;
        }
        if (g < groups) start[g + 1] = carry + sum;
        carry += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) start[0] = 0;
    return __all_sync(0xffffffffu, ok);
}

// ---------------------------------------------------------------------------
// Tensor-core kernel: tcgen05.mma on 128 x BN tiles of one CTA, or 256 x 256
// tiles of a CTA pair, persistent over the tiles of all groups.
//
// What bounds it, and what it reaches on a B200 (warm; calls in turn with pauses
// between them, at 1950 MHz, and without, where the power limit sets the clock):
//   many rows a group    the tensor pipe: 8 groups of 2048 rows, 4096 x 4096, 405 us
//                        = 1.36 PFLOP/s (470 at 1335 MHz), where the dense HGEMM of
//                        as many rows, in tiles twice as wide, takes 374 (429).
//                        Ragged groups: 68 to 70 tile rows of 256 for 64 make 15 or
//                        16 turns of 14, 444 to 463 us (515 to 553)
//   few rows a group     HBM, for the matrices: 16 groups of 2 rows, 4096 x 2048,
//                        46 us = 5.8 TB/s; 64 of 128, 2048 x 1024, 59 us = 5.4 TB/s
//   wgrad, short groups  writing C: 32 groups of 128 rows, 1024 x 1024, 29.5 us for
//                        67 MB (pure writes reach 3.9 TB/s)
//   wgrad, long groups   the tensor pipe: 8 groups of 2048 rows, 2048 x 4096, 202 us
//                        = 1.36 PFLOP/s in 16 bits (234 at 1480 MHz); f32 231 us
//                        (273), for its pieces (below) and twice the bytes of C;
//                        ragged groups 219 and 247 (252 and 300)
//
//   kNN  C[r] = A[r] B_g     A K-major, B (k x n rows) MN-major
//   kNT  C[r] = A[r] B_g^T   A K-major, B (n x k rows) K-major
//   kTN  C_g = A_g^T B_g     both MN-major; the ragged rows are the k axis
//
// The accumulators' f32 additions cut low bits, always toward zero: measured
// 2.4 f32 steps of the running sum for each 16 deep step.  A sum of one sign
// loses 2.4e-6 of itself over 512 terms, 2.5e-5 over 4096, 1.5e-3 over 2^18.
// So no accumulator sums up more than a piece; the epilogue adds the pieces,
// rounded, while the MMAs fill the other accumulator:
//   f32 C_g    pieces of 512, added up in registers (random terms, 2048 rows:
//              2.9e-6 off in one piece, 0.5e-6 in four)
//   16-bit C   pieces of 4096, whose loss is a twentieth of the rounding to f16,
//              added up in local memory, which only longer sums touch: 16384 rows
//              of each of 4 groups, 1024 x 2048: 267 us in one piece, 285 in four
//
// No operand is transposed or copied: the three products differ in the shared
// memory layouts that the MMA descriptors name.  B of kNN / kNT is a 3-D
// tensor map (columns, rows, group), so a box never reads across a matrix and
// ragged edges arrive as zeros.  Boxes of A start at any row: those past a
// group's end belong to the next group and, rows being independent, only
// reach accumulator rows that are not stored.  In kTN they would reach every
// sum, so the last k block of a group is wiped: a warp of its own zeroes the
// rows past the end, in A and B both (0 times a neighbour's NaN is a NaN),
// up to the next multiple of 16, and the MMA issues only those k steps.
//
// Operands that TMA cannot describe (rows of a length or at a base that is not
// a multiple of 16 bytes) are loaded by the HAND form: 16 warps in fours, two
// for A and two for B of a k block, four blocks at a time, write the same
// swizzled layouts with plain loads and fill ragged edges with zeros
// themselves.  Their loads keep L1 busy two thirds of the time and wait for it
// in the rest; a pair, whose CTAs load half of what a result needs, is
// 1.6 times as fast where its tiles fill the machine.
//
// SPLIT: where there are fewer tiles than SMs, a cluster of 2, 4 or 8 CTAs shares
// each tile's k blocks.  Their f32 sums meet in shared memory, where the stages
// were, and every CTA adds up some of the rows, always in the order of the k
// blocks.  One row of 4 groups, 512 x 4096: 25 -> 11 us; 7 rows of 4 groups, 1052 x
// 3770: 50 -> 30; the gradient of 16000 rows of 2 groups, 65 x 129: 124 -> 24.
//
// Warps: 0 TMA producer, 1 TMEM allocator and MMA issuer, 2..9 epilogue, 10
// (kTN) the wiper; HAND: 10.. load.  Two accumulators: the epilogue of a tile
// runs under the MMAs of the next.  The epilogue goes through shared memory to
// 64-byte row segments: in kNN and kNT a TMA store would write past a group's
// last row.  In kTN every C_g has M rows and a 3-D map would clip there; its
// results take the same way.  The epilogue is a chain of short latencies, so two
// warps share each quarter of the TMEM lanes.
enum Mode { kNN = 0, kNT = 1, kTN = 2 };

template <int MODE, bool PAIR, int BN_, bool F32_, bool HAND_>
struct Cfg {
    static constexpr bool HAND = HAND_;                // loads by warps
    static constexpr bool F32 = F32_;                  // C is f32 (kTN)
    static constexpr int PIECE = F32 ? 8 : 64;         // k blocks that an accumulator sums up
    static constexpr int BN = BN_;                     // columns of a tile
    static constexpr int BM = PAIR ? 256 : 128;        // rows of a tile, 128 to a CTA
    static constexpr int BN_CTA = PAIR ? BN / 2 : BN;  // columns of B that a CTA loads
    static constexpr int A_BYTES = 128 * 64 * 2;
    static constexpr int B_BYTES = BN_CTA * 64 * 2;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int STAGES = 196608 / STAGE_BYTES;
    static constexpr int EPI_BYTES = 8 * 2048;  // 32 rows of 64 bytes for each epilogue warp
    static constexpr int TMEM_COLS = 2 * BN;
    static constexpr int LOADERS = F32 ? 12 : 16;  // HAND: loading warps, in fours; F32 needs the registers
    static constexpr int THREADS = 320 + (HAND ? 32 * LOADERS : MODE == kTN ? 32 : 0);
    static constexpr int TABLE_BYTES = 2 * 4224;  // tile starts and offsets: kMaxGroups + 1 ints each, rounded up
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_BYTES + TABLE_BYTES + 1024 + 512;
    static_assert(SMEM_BYTES <= 232448 && TABLE_BYTES / 2 >= 4 * (kMaxGroups + 1), "shared memory per CTA");
};
constexpr int kBoxBytes = 64 * 64 * 2;  // 64 columns x 64 rows of an MN-major operand
constexpr int kSumPitch = 132;          // SPLIT: floats of a row of sums, 128 of them in use
constexpr int kGroupM = 16;             // raster: tile rows that sweep a group's columns together

struct TcArgs {
    const uint16_t *A, *B;  // HAND
    void *C;
    const int32_t *offsets;
    int *status;
    uint64_t wait_ns;
    int groups, rows, M, N, K;  // M: kTN only; K: kNN and kNT
    float alpha, beta;
    uint32_t idesc;
    int bf16;       // element type of the operands, and of C unless that is f32
    int vec;        // rows of C start on 16-byte boundaries
};

struct Tile {
    int g;
    int row0;       // first row of A (kTN: of A and B)
    int m0, n0;     // first row (kTN) and column within the group's C
    int valid;      // rows of the tile that exist
    int depth;           // of the sum
    int kblocks, klast;  // k blocks of 64, and what the last one holds
    int kfirst, kend;    // the k blocks of this CTA: all but where SPLIT
};

// The t-th tile, t ascending from call to call (g is kept between them).
template <int MODE, typename Cf>
__device__ __forceinline__ Tile tile_at(const TcArgs &p, const int *start, const int *off, uint32_t t, int &g) {
    const uint32_t nt = static_cast<uint32_t>(p.N + Cf::BN - 1) / Cf::BN;
    uint32_t mt, local;
    Tile o;
    if constexpr (MODE == kTN) {
        mt = static_cast<uint32_t>(p.M + Cf::BM - 1) / Cf::BM;
        g = static_cast<int>(t / (mt * nt));
        local = t % (mt * nt);
    } else {
        while (t >= static_cast<uint32_t>(start[g + 1]) * nt) ++g;
        mt = start[g + 1] - start[g];
        local = t - static_cast<uint32_t>(start[g]) * nt;
    }
    const uint32_t span = kGroupM * nt;
    const uint32_t first = local / span * kGroupM;
    const uint32_t gm = min(mt - first, static_cast<uint32_t>(kGroupM));
    const uint32_t r = local % span;
    o.g = g;
    o.n0 = static_cast<int>(r / gm) * Cf::BN;
    o.m0 = static_cast<int>(first + r % gm) * Cf::BM;
    const int lo = off[g], hi = off[g + 1];
    const int depth = o.depth = MODE == kTN ? hi - lo : p.K;
    o.row0 = MODE == kTN ? lo : lo + o.m0;
    o.valid = min(Cf::BM, (MODE == kTN ? p.M : hi - lo) - o.m0);
    o.kblocks = static_cast<int>(static_cast<uint32_t>(depth + 63) / 64);
    o.klast = depth - (o.kblocks - 1) * 64;
    o.kfirst = 0;
    o.kend = o.kblocks;
    return o;
}

// The limit of a wait for tiles of `kblocks` k blocks in all: the bound of any
// wait, and 2 us for each block (they take up to 1.1), so that no sum is too long.
__device__ __forceinline__ uint64_t tile_wait_ns(const TcArgs &p, int64_t kblocks) {
    return p.wait_ns + 2000ull * static_cast<uint64_t>(kblocks);
}

// Rows of A that CTA `rank` of a kNN / kNT tile loads: all 128 in one box, or
// boxes of 16 when half of them or fewer exist (a decoding step has a few
// rows an expert: 16 of 128 loaded rows leave the L2 to the weights).
__device__ __forceinline__ int a_boxes16(int valid, int rank) {
    const int v = valid - 128 * rank;
    return v > 64 ? 8 : v > 0 ? (v + 15) / 16 : 0;
}

// Where 16-byte chunk j (0..3) of row i sits in an epilogue warp's 32 x 64
// byte buffer: rows i and i + 1 share 128 bytes, chunks turn with i / 2, so
// that writes by row and reads by segment both meet every bank once.
__device__ __forceinline__ int seg_chunk(int i, int j) { return i * 64 + ((j ^ ((i >> 1) & 3)) << 4); }

// The buffer's rows to C: `ncols` columns (at most a segment's) of `rows` rows.
template <typename T>
__device__ __forceinline__ void store_segment(uint8_t *c, int64_t pitch, const uint8_t *buf, int rows, int ncols,
                                              int vec, int lane) {
    constexpr int per16 = 16 / sizeof(T);
    if (vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = i * 8 + (lane >> 2), j = lane & 3;
            if (row < rows && j * per16 < ncols)
                *reinterpret_cast<uint4 *>(c + row * pitch + j * 16) =
                    *reinterpret_cast<const uint4 *>(buf + seg_chunk(row, j));
        }
    } else {
        const int col = lane % (4 * per16);
        if (col < ncols)
            for (int row = lane / (4 * per16); row < rows; row += 32 / (4 * per16))
                *reinterpret_cast<T *>(c + row * pitch + col * sizeof(T)) =
                    *reinterpret_cast<const T *>(buf + seg_chunk(row, col / per16) + col % per16 * sizeof(T));
    }
}

// x += beta * (the row's old 16-bit values).
__device__ __forceinline__ void add_old(float (&x)[32], const uint8_t *row, int ncols, const TcArgs &p) {
    const uint16_t *c = reinterpret_cast<const uint16_t *>(row);
#pragma unroll
    for (int e = 0; e < 32; e += 8) {
        uint4 v = make_uint4(0, 0, 0, 0);
        uint32_t *w = reinterpret_cast<uint32_t *>(&v);
        if (p.vec) {
            if (e < ncols) v = *reinterpret_cast<const uint4 *>(c + e);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (e + i < ncols) w[i / 2] |= static_cast<uint32_t>(c[e + i]) << (i % 2 * 16);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = p.bf16 ? b2b::Half16<true>::get2(w[i]) : b2b::Half16<false>::get2(w[i]);
            x[e + 2 * i] = fmaf(p.beta, f.x, x[e + 2 * i]);
            x[e + 2 * i + 1] = fmaf(p.beta, f.y, x[e + 2 * i + 1]);
        }
    }
}

// The word (or the 16-bit value) at `a`, or 0 unless `take`: without a branch,
// so that many are in flight.
__device__ __forceinline__ uint32_t ldg16_if(uint64_t a, bool take) {
    uint32_t v;
    asm volatile("{\n\t.reg .pred p;\n\t.reg .u16 h;\n\tsetp.ne.u32 p, %2, 0;\n\tmov.u16 h, 0;\n\t"
                 "@p ld.global.nc.u16 h, [%1];\n\tcvt.u32.u16 %0, h;\n\t}"
                 : "=r"(v) : "l"(a), "r"(static_cast<uint32_t>(take)));
    return v;
}
__device__ __forceinline__ uint32_t ldg32_if(uint64_t a, bool take) {
    uint32_t v;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\tmov.u32 %0, 0;\n\t@p ld.global.nc.u32 %0, [%1];\n\t}"
                 : "=r"(v) : "l"(a), "r"(static_cast<uint32_t>(take)));
    return v;
}

// One warp writes a box of an operand, 64 rows of 64 values in the 128-byte
// swizzle: rows of A or B and their k values (K-major), or k rows and columns.
// `slow` rows and `fast` values exist; zeros take the others' places up to the
// next 16 rows, and what lies behind meets no result.  A lane takes pieces of 8
// values, by the aligned words that hold them: four, or five where the row
// starts between two words.  Those reach a value beyond the box on either side,
// so where that may lie outside the operand, [lo, hi), values are read one by
// one.  8 pieces of a lane are in flight at once.
__device__ __forceinline__ void fill_by_hand(uint8_t *to, const uint16_t *from, int ld, int slow, int fast,
                                             const uint16_t *lo, const uint16_t *hi, int lane) {
    constexpr int kPieces = 8;
    slow = min(slow, 64);
    fast = min(fast, 64);
    if (slow <= 0 || fast <= 0) return;
    const int rows = (slow + 15) & ~15;
    if (from == lo || from + static_cast<int64_t>(slow - 1) * ld + (fast + 7) / 8 * 8 + 1 > hi) {
        // a row a turn, two values to a lane, 16 rows in flight
        uint8_t *out = to + (lane & 3) * 4;
        const int left = fast - 2 * lane;
#pragma unroll 1
        for (int i0 = 0; i0 < rows; i0 += 16) {
            const uint64_t p0 = reinterpret_cast<uint64_t>(from + static_cast<int64_t>(i0) * ld + 2 * lane);
            uint32_t a[16], b[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const uint64_t p = p0 + static_cast<uint64_t>(ld) * 2u * j;
                a[j] = ldg16_if(p, i0 + j < slow && left > 0);
                b[j] = ldg16_if(p + 2, i0 + j < slow && left > 1);
            }
#pragma unroll
            for (int j = 0; j < 16; ++j)
                *reinterpret_cast<uint32_t *>(out + (i0 + j) * 128 + (((lane >> 2) ^ (j & 7)) << 4)) = a[j] | b[j] << 16;
        }
        return;
    }
    // piece j of a turn: chunk lane % 8 of the turn's row lane / 8 + 4 j
    const int c = lane & 7, r = lane >> 3;
    const int left = fast - c * 8;                         // values that exist
    const uint64_t step = static_cast<uint64_t>(ld) * 8u;  // bytes of four rows
#pragma unroll 1
    for (int i0 = 0; i0 < rows; i0 += 4 * kPieces) {
        const int row0 = i0 + r;
        const uint64_t p0 = reinterpret_cast<uint64_t>(from + static_cast<int64_t>(row0) * ld + c * 8);
        uint32_t w[kPieces][5];
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            const uint64_t p = p0 + step * j;
            const bool have = row0 + 4 * j < slow && left > 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[j][i] = ldg32_if((p & ~3ull) + 4 * i, have);
            w[j][4] = ldg32_if((p & ~3ull) + 16, have && (p & 2));
        }
        uint8_t *out = to + row0 * 128;
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            const uint32_t shift = (static_cast<uint32_t>(p0 + step * j) & 2u) << 3;
            uint32_t v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = __funnelshift_r(w[j][i], w[j][i + 1], shift);
                if (left < 8 && left < 2 * i + 2) v[i] = left < 2 * i + 1 ? 0u : v[i] & 0xffffu;
            }
            *reinterpret_cast<uint4 *>(out + j * 512 + ((c ^ ((row0 + 4 * j) & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
        }
    }
}

template <int MODE, bool PAIR, int BN, bool F32, bool HAND, bool SPLIT>  // SPLIT: a tile at most to each cluster
__global__ void __launch_bounds__((Cfg<MODE, PAIR, BN, F32, HAND>::THREADS), 1)
    grouped_tc_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmA16,
                      const __grid_constant__ CUtensorMap tmB, TcArgs p) {
    using namespace sm100;
    using Cf = Cfg<MODE, PAIR, BN, F32, HAND>;
    constexpr int S = Cf::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t *sA = smem;
    uint8_t *sB = smem + S * Cf::A_BYTES;
    uint8_t *epi = smem + S * Cf::STAGE_BYTES;
    int *start = reinterpret_cast<int *>(epi + Cf::EPI_BYTES);
    int *off = start + Cf::TABLE_BYTES / 8;
    uint64_t *bars = reinterpret_cast<uint64_t *>(epi + Cf::EPI_BYTES + Cf::TABLE_BYTES);
    uint64_t *full = bars, *empty = bars + S, *landed = bars + 2 * S;  // landed: kTN, last k block of a group
    uint64_t *tfull = bars + 3 * S, *tempty = bars + 3 * S + 2, *drain = bars + 3 * S + 4;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 3 * S + 5);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *valid_flag = reinterpret_cast<int *>(tmem_slot + 2);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = PAIR ? static_cast<int>(cluster_ctarank()) : 0;
    const bool leader = rank == 0;
    // SPLIT: the CTAs of a cluster share one tile's k blocks
    const int part = SPLIT ? static_cast<int>(cluster_ctarank()) : 0, parts = SPLIT ? static_cast<int>(cluster_nctarank()) : 1;
    const uint32_t first = PAIR ? blockIdx.x >> 1 : SPLIT ? blockIdx.x / parts : blockIdx.x;
    const uint32_t step = PAIR ? gridDim.x >> 1 : SPLIT ? gridDim.x / parts : gridDim.x;
    auto tile_of = [&](uint32_t t, int &g) {
        Tile o = tile_at<MODE, Cf>(p, start, off, t, g);
        if constexpr (SPLIT) {
            o.kfirst = static_cast<int>(static_cast<int64_t>(o.kblocks) * part / parts);
            o.kend = static_cast<int>(static_cast<int64_t>(o.kblocks) * (part + 1) / parts);
        }
        return o;
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            // a pair's kTN stage is full when both CTAs say so: their
            // producers, or for a group's last k block their wipers; HAND:
            // when both its warps do
            mbar_init(&full[s], HAND ? (PAIR ? 8 : 4) : PAIR && MODE == kTN ? 2 : 1);
            mbar_init(&empty[s], 1);
            mbar_init(&landed[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&tfull[a], 1);
            mbar_init(&tempty[a], PAIR ? 16 : 8);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_barrier_init();
        if constexpr (!HAND) {
            prefetch_tensormap(&tmA);
            prefetch_tensormap(&tmB);
        }
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            tmem_alloc_pair(tmem_slot, Cf::TMEM_COLS);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(tmem_slot, Cf::TMEM_COLS);
            tmem_relinquish();
        }
    }
    if (warp == 2) {
        const bool ok = scan_groups(p.offsets, p.groups, p.rows, Cf::BM, start, off);
        if (lane == 0) {
            *valid_flag = ok;
            if (!ok) atomicCAS(p.status, 0, B2B_DEVSTAT_OFFSETS);
        }
    }
    tc_fence_before();
    if constexpr (PAIR)
        cluster_sync();
    else
        __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    uint32_t tiles = 0;  // the launcher has seen to it that they stay below 2^31
    if (*valid_flag)
        tiles = static_cast<uint32_t>(MODE == kTN ? p.groups * (static_cast<uint32_t>(p.M + Cf::BM - 1) / Cf::BM)
                                                  : start[p.groups]) *
                (static_cast<uint32_t>(p.N + BN - 1) / BN);

    if (warp == 0) {
        // ------------------------------------------------ TMA producer
        if (!HAND && lane == 0) {
            int stage = 0, g = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (uint32_t t = first; t < tiles && ok; t += step) {
                const Tile o = tile_of(t, g);
                const int mine = MODE == kTN ? 8 : a_boxes16(o.valid, rank);
                const int both = !PAIR ? mine : MODE == kTN ? 16 : a_boxes16(o.valid, 0) + a_boxes16(o.valid, 1);
                for (int kb = o.kfirst; kb < o.kend; ++kb) {
                    if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, p.status, B2B_DEVSTAT_TIMEOUT | 0x21,
                                   p.wait_ns)) {
                        ok = false;
                        break;
                    }
                    uint8_t *a_dst = sA + stage * Cf::A_BYTES, *b_dst = sB + stage * Cf::B_BYTES;
                    const int bn0 = o.n0 + rank * Cf::BN_CTA;
                    const bool tail = MODE == kTN && kb == o.kblocks - 1 && o.klast < 64;
                    if (tail) {
                        // both operands land on this CTA's own barrier, for its wiper
                        mbar_arrive_expect_tx(&landed[stage], Cf::STAGE_BYTES);
                        for (int j = 0; j < 2; ++j)
                            tma_load_2d(a_dst + j * kBoxBytes, &tmA, &landed[stage], o.m0 + rank * 128 + 64 * j,
                                        o.row0 + kb * 64);
                        for (int j = 0; j < Cf::BN_CTA / 64; ++j)
                            tma_load_2d(b_dst + j * kBoxBytes, &tmB, &landed[stage], bn0 + 64 * j, o.row0 + kb * 64);
                    } else if constexpr (PAIR) {
                        const uint32_t bar = mapa_shared(smem_u32(&full[stage]), 0);
                        if (leader)
                            mbar_arrive_expect_tx(&full[stage], both * 2048 + 2 * Cf::B_BYTES);
                        else if (MODE == kTN)
                            mbar_arrive_cluster_relaxed(bar);
                        if constexpr (MODE == kTN) {
                            for (int j = 0; j < 2; ++j)
                                tma_load_2d_pair(a_dst + j * kBoxBytes, &tmA, bar, o.m0 + rank * 128 + 64 * j,
                                                 o.row0 + kb * 64);
                            for (int j = 0; j < Cf::BN_CTA / 64; ++j)
                                tma_load_2d_pair(b_dst + j * kBoxBytes, &tmB, bar, bn0 + 64 * j, o.row0 + kb * 64);
                        } else {
                            const int r0 = o.row0 + rank * 128;
                            if (mine == 8)
                                tma_load_2d_pair(a_dst, &tmA, bar, kb * 64, r0);
                            else
                                for (int j = 0; j < mine; ++j)
                                    tma_load_2d_pair(a_dst + j * 2048, &tmA16, bar, kb * 64, r0 + 16 * j);
                            if constexpr (MODE == kNN)
                                for (int j = 0; j < Cf::BN_CTA / 64; ++j)
                                    tma_load_3d_pair(b_dst + j * kBoxBytes, &tmB, bar, bn0 + 64 * j, kb * 64, o.g);
                            else
                                tma_load_3d_pair(b_dst, &tmB, bar, kb * 64, bn0, o.g);
                        }
                    } else {
                        uint64_t *bar = &full[stage];
                        mbar_arrive_expect_tx(bar, mine * 2048 + Cf::B_BYTES);
                        if constexpr (MODE == kTN) {
                            for (int j = 0; j < 2; ++j)
                                tma_load_2d(a_dst + j * kBoxBytes, &tmA, bar, o.m0 + 64 * j, o.row0 + kb * 64);
                            for (int j = 0; j < Cf::BN_CTA / 64; ++j)
                                tma_load_2d(b_dst + j * kBoxBytes, &tmB, bar, bn0 + 64 * j, o.row0 + kb * 64);
                        } else {
                            if (mine == 8)
                                tma_load_2d(a_dst, &tmA, bar, kb * 64, o.row0);
                            else
                                for (int j = 0; j < mine; ++j)
                                    tma_load_2d(a_dst + j * 2048, &tmA16, bar, kb * 64, o.row0 + 16 * j);
                            if constexpr (MODE == kNN)
                                for (int j = 0; j < Cf::BN_CTA / 64; ++j)
                                    tma_load_3d(b_dst + j * kBoxBytes, &tmB, bar, bn0 + 64 * j, kb * 64, o.g);
                            else
                                tma_load_3d(b_dst, &tmB, bar, kb * 64, bn0, o.g);
                        }
                    }
                    if (++stage == S) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (!ok) {
                // loads in flight complete on barriers of three kinds, a
                // partner's among them: give them a bounded grace period
                const uint64_t t0 = globaltimer_ns();
                while (globaltimer_ns() - t0 < 2000000ull) {
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issuer (a pair's leader)
        if (leader && lane == 0) {
            int stage = 0, acc = 0, g = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true, issued = false;
            for (uint32_t t = first; t < tiles && ok; t += step) {
                int depth = p.K, kfirst = 0, kend = static_cast<int>(static_cast<uint32_t>(depth + 63) / 64);
                if constexpr (MODE == kTN || SPLIT) {
                    const Tile o = tile_of(t, g);
                    depth = o.depth;
                    kfirst = o.kfirst;
                    kend = o.kend;
                }
                for (int kb0 = kfirst; ok && (kb0 == kfirst || kb0 < kend); kb0 += Cf::PIECE) {
                    if (!mbar_wait(&tempty[acc], acc_phase ^ 1u, abort_flag, p.status, B2B_DEVSTAT_TIMEOUT | 0x22,
                                   p.wait_ns)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t d = tmem_base + static_cast<uint32_t>(acc * BN);
                    const int kb_end = kend - kb0 < Cf::PIECE ? kend : kb0 + Cf::PIECE;
                    for (int kb = kb0; kb < kb_end; ++kb) {
                        // the other CTA's loading warps or its wiper may have written its half
                        if (PAIR && (HAND || (MODE == kTN && depth - kb * 64 < 64)))
                            ok = mbar_wait<true>(&full[stage], phase, abort_flag, p.status, B2B_DEVSTAT_TIMEOUT | 0x23,
                                                 p.wait_ns);
                        else
                            ok = mbar_wait(&full[stage], phase, abort_flag, p.status, B2B_DEVSTAT_TIMEOUT | 0x23, p.wait_ns);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t a = smem_u32(sA + stage * Cf::A_BYTES), b = smem_u32(sB + stage * Cf::B_BYTES);
                        // K-major: 8-row atoms 1024 bytes apart, a k step of 16
                        // moves 32 bytes inside the swizzled row.  MN-major:
                        // 64-wide boxes, 8-row k groups 1024 bytes apart, a k
                        // step moves 16 rows.
                        auto k_step = [&](int kk) {
                            const uint64_t ad = MODE == kTN ? sdesc_sw128(a + kk * 2048, kBoxBytes, 1024)
                                                            : sdesc_sw128(a + kk * 32, 16, 1024);
                            const uint64_t bd = MODE == kNT ? sdesc_sw128(b + kk * 32, 16, 1024)
                                                            : sdesc_sw128(b + kk * 2048, kBoxBytes, 1024);
                            if constexpr (PAIR)
                                umma_f16_pair(d, ad, bd, p.idesc, ((kb - kb0) | kk) != 0 ? 1u : 0u);
                            else
                                umma_f16(d, ad, bd, p.idesc, ((kb - kb0) | kk) != 0 ? 1u : 0u);
                        };
                        const int left = depth - kb * 64;
                        if (left >= 64) {
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk) k_step(kk);
                        } else {
                            for (int kk = 0; kk * 16 < left; ++kk) k_step(kk);
                        }
                        if constexpr (PAIR)
                            umma_commit_pair(&empty[stage], 0x3);
                        else
                            umma_commit(&empty[stage]);
                        issued = true;
                        if (++stage == S) {
                            stage = 0;
                            phase ^= 1u;
                        }
                    }
                    if (!ok) break;
                    if constexpr (PAIR)
                        umma_commit_pair(&tfull[acc], 0x3);
                    else
                        umma_commit(&tfull[acc]);
                    if (++acc == 2) {
                        acc = 0;
                        acc_phase ^= 1u;
                    }
                }
            }
            if (!ok && issued) {
                if constexpr (PAIR)
                    umma_commit_pair(drain, 0x1);
                else
                    umma_commit(drain);
                mbar_wait_drain(drain, 0, 1000000000ull);
            }
        }
        __syncwarp();
    } else if (HAND && warp >= 10) {
        // ------------------------------------------------ loading warps (HAND)
        const int turn = (warp - 10) >> 2;  // of the k blocks that are in flight
        const int h = (warp - 10) & 1;      // box of the operand
        const bool is_b = (warp - 10) & 2;
        const uint16_t *a_end = p.A + static_cast<int64_t>(p.rows) * (MODE == kTN ? p.M : p.K);
        const uint16_t *b_end = p.B + (MODE == kTN ? static_cast<int64_t>(p.rows) * p.N
                                                   : static_cast<int64_t>(p.groups) * p.N * p.K);
        int g = 0;
        uint32_t it = 0;  // k blocks of all tiles so far
        bool ok = true;
        for (uint32_t t = first; t < tiles && ok; t += step) {
            const Tile o = tile_of(t, g);
            const int am = rank * 128 + 64 * h, bn = o.n0 + rank * Cf::BN_CTA + 64 * h;
            for (int kb = o.kfirst; kb < o.kend; ++kb, ++it) {
                if (static_cast<int>(it % (Cf::LOADERS / 4u)) != turn) continue;
                const int s = static_cast<int>(it % S);
                const uint32_t phase = it / S & 1u;
                ok = mbar_wait(&empty[s], phase ^ 1u, abort_flag, p.status, B2B_DEVSTAT_TIMEOUT | 0x21, p.wait_ns);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const int k0 = kb * 64, k_left = o.depth - k0;
                if (!is_b) {
                    uint8_t *to = sA + s * Cf::A_BYTES + h * kBoxBytes;
                    if constexpr (MODE == kTN)
                        fill_by_hand(to, p.A + static_cast<int64_t>(o.row0 + k0) * p.M + o.m0 + am, p.M, k_left,
                                     p.M - o.m0 - am, p.A, a_end, lane);
                    else
                        fill_by_hand(to, p.A + static_cast<int64_t>(o.row0 + am) * p.K + k0, p.K, o.valid - am, k_left, p.A,
                                     a_end, lane);
                } else {
                    uint8_t *to = sB + s * Cf::B_BYTES + h * kBoxBytes;
                    const uint16_t *matrix = p.B + (MODE == kTN ? static_cast<int64_t>(o.row0) * p.N
                                                                : static_cast<int64_t>(o.g) * p.N * p.K);
                    if constexpr (MODE == kNT)
                        fill_by_hand(to, matrix + static_cast<int64_t>(bn) * p.K + k0, p.K, p.N - bn, k_left, p.B, b_end, lane);
                    else
                        fill_by_hand(to, matrix + static_cast<int64_t>(k0) * p.N + bn, p.N, k_left, p.N - bn, p.B, b_end, lane);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    if (leader)
                        mbar_arrive(&full[s]);
                    else
                        mbar_arrive_cluster(mapa_shared(smem_u32(&full[s]), 0));
                }
            }
        }
    } else if (!HAND && MODE == kTN && warp == 10) {
        // ------------------------------------------------ wiper (kTN)
        int stage = 0, g = 0;
        uint32_t phases = 0;  // bit s: parity of landed[s]
        int64_t behind = 0;   // k blocks since the last wait, and 16 for each tile's epilogue: all come before this one
        for (uint32_t t = first; t < tiles; t += step) {
            const Tile o = tile_of(t, g);
            const int count = o.kend - o.kfirst;
            behind += count + 16;
            if (count == 0) continue;
            const int s = (stage + count - 1) % S;
            stage = (stage + count) % S;
            if (o.klast == 64 || o.kend < o.kblocks) continue;
            const bool ok = mbar_wait_sleepy(&landed[s], phases >> s & 1u, abort_flag, p.status,
                                             B2B_DEVSTAT_TIMEOUT | 0x25, tile_wait_ns(p, behind));
            behind = 0;
            if (!__all_sync(0xffffffffu, ok)) break;
            phases ^= 1u << s;
            // row r of a box is its 128 bytes at r * 128, whatever the swizzle
            const int chunks = ((o.klast + 15) / 16 * 16 - o.klast) * 8;
            for (int box = 0; box < 2 + Cf::BN_CTA / 64; ++box) {
                uint8_t *at = (box < 2 ? sA + s * Cf::A_BYTES + box * kBoxBytes
                                       : sB + s * Cf::B_BYTES + (box - 2) * kBoxBytes) + o.klast * 128;
                for (int i = lane; i < chunks; i += 32) *reinterpret_cast<uint4 *>(at + i * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (leader)
                    mbar_arrive(&full[s]);
                else
                    mbar_arrive_cluster(mapa_shared(smem_u32(&full[s]), 0));
            }
        }
    } else {
        // ------------------------------------------------ epilogue
        const int q = warp & 3;  // TMEM lanes 32q .. 32q + 31
        const int c_first = (warp - 2) / 4 * (BN / 2), c_end = c_first + BN / 2;  // the warp's columns
        uint8_t *buf = epi + (warp - 2) * 2048;
        constexpr int csize = F32 ? 4 : 2;
        const int64_t pitch = static_cast<int64_t>(p.N) * csize;
        float *sums = reinterpret_cast<float *>(smem) + (q * 32 + lane) * kSumPitch;  // SPLIT: this thread's row
        int acc = 0, g = 0;
        uint32_t acc_phase = 0;
        // the warp has read its share of the accumulator
        auto release = [&] {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (leader)
                    mbar_arrive(&tempty[acc]);
                else
                    mbar_arrive_cluster(mapa_shared(smem_u32(&tempty[acc]), 0));
            }
        };
        auto turn = [&] {  // to the other accumulator
            if (++acc == 2) {
                acc = 0;
                acc_phase ^= 1u;
            }
        };
        auto wait_full = [&](const Tile &o) {
            const bool ok = mbar_wait_sleepy(&tfull[acc], acc_phase, abort_flag, p.status, B2B_DEVSTAT_TIMEOUT | 0x24,
                                             tile_wait_ns(p, o.kblocks));
            const bool all = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            return all;
        };
        const uint32_t tmem_warp = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
        bool ok = true;
        for (uint32_t t = first; t < tiles && ok; t += step) {
            const Tile o = tile_of(t, g);
            const int r0 = rank * 128 + q * 32;  // the warp's first row in the tile
            const int rows = min(32, o.valid - r0);
            uint8_t *C = static_cast<uint8_t *>(p.C) +
                         ((MODE == kTN ? static_cast<int64_t>(o.g) * p.M + o.m0 : static_cast<int64_t>(o.row0)) + r0) *
                             pitch;
            // the warp's columns that exist, in steps of 32; none where no row does
            const int left = p.N - o.n0 - c_first;
            const int c_stop = rows > 0 && left > 0 ? min(c_end, c_first + (left + 31) / 32 * 32) : c_first;
            if constexpr (F32) {
                float x[BN / 2];
#pragma unroll
                for (int e = 0; e < BN / 2; ++e) x[e] = 0.0f;
                for (int kb0 = o.kfirst; kb0 < o.kend || kb0 == o.kfirst; kb0 += Cf::PIECE) {
                    ok = wait_full(o);
                    if (!ok) break;
                    if (o.kend > o.kfirst) {
#pragma unroll
                        for (int c = 0; c < BN / 2; c += 16) {
                            uint32_t r[16];
                            tmem_ld_32x32b_x16(tmem_warp + static_cast<uint32_t>(acc * BN + c_first + c), r);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 16; ++e) x[c + e] += __uint_as_float(r[e]);
                        }
                    }
                    release();
                    turn();
                }
                if (!ok) break;
                if constexpr (SPLIT) {
#pragma unroll
                    for (int c = 0; c < BN / 2; c += 4)
                        *reinterpret_cast<float4 *>(sums + c_first + c) = make_float4(x[c], x[c + 1], x[c + 2], x[c + 3]);
                    continue;
                }
                // segments of 16 columns
#pragma unroll
                for (int c = 0; c < BN / 2; c += 16) {
                    if (c_first + c >= c_stop) break;
                    const int col0 = o.n0 + c_first + c, ncols = min(16, p.N - col0);
                    if (ncols <= 0) break;
                    uint8_t *cbase = C + static_cast<int64_t>(col0) * 4;
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[c + e] = o.kblocks ? p.alpha * x[c + e] : 0.0f;
                    if (p.beta != 0.0f && lane < rows) {
                        const float *old = reinterpret_cast<const float *>(cbase + lane * pitch);
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (e < ncols) x[c + e] = fmaf(p.beta, old[e], x[c + e]);
                    }
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        *reinterpret_cast<float4 *>(buf + seg_chunk(lane, j)) =
                            make_float4(x[c + 4 * j], x[c + 4 * j + 1], x[c + 4 * j + 2], x[c + 4 * j + 3]);
                    __syncwarp();
                    store_segment<float>(cbase, pitch, buf, rows, ncols, p.vec, lane);
                }
            } else {
                // A sum of several pieces: the warp's columns of all but the last are added up
                // here (in local memory: the columns are a loop), and then into the accumulator
                // of the last, from where all sums go on.
                float held[BN / 2];
                for (int kb0 = o.kfirst;; kb0 += Cf::PIECE) {
                    ok = wait_full(o);
                    const bool last = o.kend - kb0 <= Cf::PIECE;
                    if (!ok || (last && kb0 == o.kfirst)) break;
#pragma unroll 1
                    for (int c = 0; c < c_stop - c_first; c += 16) {
                        const uint32_t at = tmem_warp + static_cast<uint32_t>(acc * BN + c_first + c);
                        uint32_t r[16];
                        __syncwarp();
                        tmem_ld_32x32b_x16(at, r);
                        tmem_ld_wait();
                        if (kb0 != o.kfirst) {
#pragma unroll
                            for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(held[c + e] + __uint_as_float(r[e]));
                        }
                        if (last) {
                            tmem_st_32x32b_x16(at, r);
                        } else {
#pragma unroll
                            for (int e = 0; e < 16; ++e) held[c + e] = __uint_as_float(r[e]);
                        }
                    }
                    if (last) {
                        tmem_st_wait();
                        break;
                    }
                    release();
                    turn();
                }
                if (!ok) break;
                if (c_stop == c_first) release();
#pragma unroll 1
                for (int c = c_first; c < c_stop; c += 32) {
                    uint32_t r[32];
                    __syncwarp();
                    tmem_ld_32x32b_x32(tmem_warp + static_cast<uint32_t>(acc * BN + c), r);
                    tmem_ld_wait();
                    if (c + 32 == c_stop) release();
                    if constexpr (SPLIT) {
                        // no k block: nothing was summed
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            *reinterpret_cast<float4 *>(sums + c + e) =
                                o.kend > o.kfirst ? make_float4(__uint_as_float(r[e]), __uint_as_float(r[e + 1]),
                                                                __uint_as_float(r[e + 2]), __uint_as_float(r[e + 3]))
                                                  : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        continue;
                    }
                    const int col0 = o.n0 + c;
                    const int ncols = min(32, p.N - col0);
                    uint8_t *cbase = C + static_cast<int64_t>(col0) * csize;
                    float x[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) x[e] = p.alpha * __uint_as_float(r[e]);
                    if (MODE == kTN && o.kblocks == 0) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) x[e] = 0.0f;
                    }
                    if (p.beta != 0.0f && lane < rows) add_old(x, cbase + lane * pitch, ncols, p);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint4 v;
                        uint32_t *w = reinterpret_cast<uint32_t *>(&v);
                        if (p.bf16) {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                w[e] = b2b::Half16<true>::put2(x[8 * j + 2 * e], x[8 * j + 2 * e + 1]);
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                w[e] = b2b::Half16<false>::put2(x[8 * j + 2 * e], x[8 * j + 2 * e + 1]);
                        }
                        *reinterpret_cast<uint4 *>(buf + seg_chunk(lane, j)) = v;
                    }
                    __syncwarp();
                    store_segment<uint16_t>(cbase, pitch, buf, rows, ncols, p.vec, lane);
                }
                turn();
            }
        }
    }

    tc_fence_before();
    if constexpr (SPLIT) {
        // the tile's sums are in the CTAs of the cluster: each adds up its
        // share of the rows, in the order of their k blocks
        __syncwarp();
        cluster_sync();
        if (first < tiles) {
            int g = 0;
            const Tile o = tile_of(first, g);
            const int col = lane * 4, ncols = min(4, p.N - o.n0 - col);
            for (int row = warp * parts + part; row < o.valid; row += Cf::THREADS / 32 * parts) {
                if (ncols <= 0) continue;
                const uint32_t at = smem_u32(smem) + (row * kSumPitch + col) * 4;
                float4 of[8];
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < parts) of[r] = ld_shared_cluster_v4(mapa_shared(at, r));
                float x[4] = {};
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < parts) x[0] += of[r].x, x[1] += of[r].y, x[2] += of[r].z, x[3] += of[r].w;
                const int64_t i = ((MODE == kTN ? static_cast<int64_t>(o.g) * p.M + o.m0 : static_cast<int64_t>(o.row0)) + row) * p.N +
                                  o.n0 + col;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = o.kblocks ? p.alpha * x[e] : 0.0f;
                if constexpr (F32) {
                    float *c = static_cast<float *>(p.C) + i;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e < ncols) c[e] = p.beta != 0.0f ? fmaf(p.beta, c[e], x[e]) : x[e];
                } else {
                    uint16_t *c = static_cast<uint16_t *>(p.C) + i;
                    using B = b2b::Half16<true>;
                    using H = b2b::Half16<false>;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (e >= ncols) continue;
                        if (p.beta != 0.0f) x[e] = fmaf(p.beta, p.bf16 ? B::get(c[e]) : H::get(c[e]), x[e]);
                        c[e] = p.bf16 ? B::put(x[e]) : H::put(x[e]);
                    }
                }
            }
        }
        __syncwarp();
        cluster_sync();  // no CTA leaves while another reads its sums
    } else if constexpr (PAIR) {
        cluster_sync();
    } else {
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        if constexpr (PAIR)
            tmem_dealloc_pair(tmem_base, Cf::TMEM_COLS);
        else
            tmem_dealloc(tmem_base, Cf::TMEM_COLS);
    }
}

// Launch state of one kernel instance on each device: the shared-memory
// attribute is set, and how many CTAs (or pairs) are resident at once.
struct Launch {
    int ready[64] = {};
    int resident[64] = {};
};
std::mutex g_mu;

template <int MODE, bool PAIR, int BN, bool F32 = false, bool HAND = false, bool SPLIT = false>
int launch_tc(b2b_handle *h, const CUtensorMap &tmA, const CUtensorMap &tmA16, const CUtensorMap &tmB,
              const TcArgs &p, int64_t most_tiles, int parts = 1) {
    using Cf = Cfg<MODE, PAIR, BN, F32, HAND>;
    static_assert(!SPLIT || (!PAIR && BN == 128 && 128 * kSumPitch * 4 <= Cf::STAGES * Cf::STAGE_BYTES), "SPLIT");
    static Launch state;
    auto kernel = grouped_tc_kernel<MODE, PAIR, BN, F32, HAND, SPLIT>;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = PAIR ? 2 : parts;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(Cf::THREADS);
    cfg.dynamicSmemBytes = Cf::SMEM_BYTES;
    cfg.stream = h->stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const int dev = h->device & 63;
    int resident;
    {
        std::lock_guard<std::mutex> lock(g_mu);
        if (!state.ready[dev]) {
            cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cf::SMEM_BYTES);
            if (e != cudaSuccess) return b2b::fail_cuda(e, "grouped HGEMM shared memory");
            int clusters = h->sm_count;
            if (PAIR) {
                cfg.gridDim = dim3(2 * (h->sm_count / 2));
                e = cudaOccupancyMaxActiveClusters(&clusters, reinterpret_cast<const void *>(kernel), &cfg);
                if (e != cudaSuccess) return b2b::fail_cuda(e, "cudaOccupancyMaxActiveClusters");
                if (clusters < 1) clusters = h->sm_count / 2;
            }
            state.resident[dev] = clusters;
            state.ready[dev] = 1;
        }
        resident = state.resident[dev];
    }
    // SPLIT: a cluster to every tile
    const int units = static_cast<int>(SPLIT || most_tiles < resident ? most_tiles : resident);
    cfg.gridDim = dim3((PAIR ? 2 : parts) * units);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tmA, tmA16, tmB, p);
    return e == cudaSuccess ? B2B_OK : b2b::fail_cuda(e, "grouped HGEMM tcgen05 launch");
}

template <bool F32>
int launch_wgrad(b2b_handle *h, bool pair, int bn, const CUtensorMap &tmA, const CUtensorMap &tmB, const TcArgs &p,
                 int64_t most) {
    if (pair) return launch_tc<kTN, true, 256, F32>(h, tmA, tmA, tmB, p, most);
    if (bn == 256) return launch_tc<kTN, false, 256, F32>(h, tmA, tmA, tmB, p, most);
    if (bn == 128) return launch_tc<kTN, false, 128, F32>(h, tmA, tmA, tmB, p, most);
    return launch_tc<kTN, false, 64, F32>(h, tmA, tmA, tmB, p, most);
}

// Tensor maps describe rows of a multiple of 16 bytes at 16-byte aligned
// bases, and matrices less than 2^40 bytes apart.
bool tma_can(const void *A, const void *B, int64_t ld_a, int64_t rows_b, int64_t ld_b) {
    return b2b::aligned16(A) && b2b::aligned16(B) && ld_a % 8 == 0 && ld_b % 8 == 0 && rows_b * ld_b < (1ll << 39);
}

// SPLIT: into how many parts to cut the k blocks of each of `tiles` 128 x 128
// tiles, 1 where the machine has no SMs left for more (7 of 8 where clusters of
// 4 leave some out, 3 of 4 with 8) or `us` that it takes otherwise is less: a k
// block takes a CTA `per` us, and the parts' joining about 2.5.
int k_parts(const b2b_handle *h, int64_t tiles, int64_t kblocks, double per, double us) {
    int best = 1;
    for (int parts = 2, eighths = 8; parts <= 8; parts *= 2, --eighths) {
        const double t = 2.5 + per * static_cast<double>((kblocks + parts - 1) / parts);
        if (tiles * parts * 8 > static_cast<int64_t>(h->sm_count) * eighths || t > 0.95 * us) continue;
        best = parts;
        us = t;
    }
    return best;
}

// HAND: whether pairs' turns, over that many tile rows of 128 and of 256, take
// less.  A k block costs a pair 1.1 us and a CTA 0.92 us for half the rows and
// columns (16384 x 2049 x 2047: 283 and 442 us), but pairs have half as many turns
// to fill (1000 x 515 x 1001: 27 and 21 us).
bool by_hand_in_pairs(const b2b_handle *h, double rows128, double rows256, int64_t N) {
    const double one = ceil(rows128 * static_cast<double>((N + 127) / 128) / h->sm_count);
    const double two = ceil(rows256 * static_cast<double>((N + 255) / 256) / (h->sm_count / 2));
    return 1.2 * two < one;
}

}  // namespace

namespace b2b {

int launch_hgemm_grouped(b2b_handle *h, int type, int trans_b, size_t groups, size_t rows, size_t n, size_t k,
                         float alpha, const uint16_t *A, const uint16_t *B, float beta, uint16_t *C,
                         const int32_t *offsets) {
    const int64_t N = static_cast<int64_t>(n), K = static_cast<int64_t>(k), R = static_cast<int64_t>(rows);
    const int G = static_cast<int>(groups);
    const bool bf16 = type == B2B_TYPE_BF16;
    const bool tma = tma_can(A, B, K, trans_b ? N : K, trans_b ? K : N);
    if ((R / 128 + (R < G ? R : G)) * (N / 64 + 1) >= 1ll << 31)
        return fail(B2B_ERR_NOT_SUPPORTED, "grouped HGEMM: 2^31 tiles or more");
    TcArgs p{A, B, C, offsets, h->d_status, h->wait_limit_ns, G, static_cast<int>(rows), 0, static_cast<int>(n),
             static_cast<int>(k), alpha, beta, 0, bf16, n % 8 == 0 && aligned16(C)};
    // pairs where groups are long enough on average to fill their 256 rows
    bool pair = R >= 192 * static_cast<int64_t>(G) && N > 128;
    const int64_t kb = (K + 63) / 64, tiles128 = (R / 128 + (R < G ? R : G)) * ((N + 127) / 128);
    if (!tma) {
        pair = pair && by_hand_in_pairs(h, static_cast<double>(R) / 128 + 0.5 * G, static_cast<double>(R) / 256 + 0.5 * G, N);
        const int parts = pair ? 1 : k_parts(h, tiles128, kb, 1.1, 1.1 * static_cast<double>(kb));
        if (parts > 1) {
            p.idesc = sm100::idesc_f32acc(bf16, 0, trans_b ? 0 : 1, 128, 128);
            const CUtensorMap none{};
            return trans_b ? launch_tc<kNT, false, 128, false, true, true>(h, none, none, none, p, tiles128, parts)
                           : launch_tc<kNN, false, 128, false, true, true>(h, none, none, none, p, tiles128, parts);
        }
        const int bm = pair ? 256 : 128;
        p.idesc = sm100::idesc_f32acc(bf16, 0, trans_b ? 0 : 1, bm, bm);
        const int64_t most = (R / bm + (R < G ? R : G)) * ((N + bm - 1) / bm);
        const CUtensorMap none{};
        if (pair)
            return trans_b ? launch_tc<kNT, true, 256, false, true>(h, none, none, none, p, most)
                           : launch_tc<kNN, true, 256, false, true>(h, none, none, none, p, most);
        return trans_b ? launch_tc<kNT, false, 128, false, true>(h, none, none, none, p, most)
                       : launch_tc<kNN, false, 128, false, true>(h, none, none, none, p, most);
    }
    int bn = 256, parts = 1;
    if (pair) {  // a pair's k block takes 0.4 us; two CTAs a tile leave none idle where there are few
        if (tiles128 < h->sm_count / 2) parts = k_parts(h, tiles128, kb, 0.375, 0.4 * static_cast<double>(kb));
        if (parts > 1) pair = false, bn = 128;
    } else {
        // The width whose turns of CTAs take least.  A k block of 64 costs a
        // CTA about 340 ns at 64 columns, 375 at 128 and 680 at 256 (its MMAs
        // take as long at any width, its share of HBM does not).
        const int64_t tiles_m = R / 128 + (R < G ? R : G);
        auto turns = [&](int w) { return (tiles_m * ((N + w - 1) / w) + h->sm_count - 1) / h->sm_count; };
        const double t256 = 2.0 * turns(256), t128 = 1.1 * turns(128), t64 = 1.0 * turns(64);
        if (t128 < t256 || N <= 128) bn = 128;
        if (t64 < (bn == 128 ? t128 : t256) || N <= 64) bn = 64;
        parts = k_parts(h, tiles128, kb, 0.375, 0.34 * static_cast<double>(kb) * (bn == 64 ? t64 : bn == 128 ? t128 : t256));
        if (parts > 1) bn = 128;
    }
    const CUtensorMapDataType dt = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    CUtensorMap tmA, tmA16, tmB;
    if (int rc = encode_tma_2d(&tmA, dt, 2, A, rows, k, 64, 128)) return rc;
    if (int rc = encode_tma_2d(&tmA16, dt, 2, A, rows, k, 64, 16)) return rc;
    const uint32_t ncta = pair ? 128 : bn;
    const uint64_t cols = trans_b ? k : n, brows = trans_b ? n : k;
    if (int rc = encode_tma_3d(&tmB, dt, 2, B, cols, brows, groups, cols * 2, cols * brows * 2, 64, trans_b ? ncta : 64,
                               CU_TENSOR_MAP_SWIZZLE_128B))
        return rc;
    p.idesc = sm100::idesc_f32acc(bf16, 0, trans_b ? 0 : 1, pair ? 256 : 128, pair ? 256 : bn);
    const int bm = pair ? 256 : 128;
    const int64_t most = (R / bm + (R < G ? R : G)) * ((N + bn - 1) / bn);
    if (parts > 1)
        return trans_b ? launch_tc<kNT, false, 128, false, false, true>(h, tmA, tmA16, tmB, p, tiles128, parts)
                       : launch_tc<kNN, false, 128, false, false, true>(h, tmA, tmA16, tmB, p, tiles128, parts);
    if (trans_b) {
        if (pair) return launch_tc<kNT, true, 256>(h, tmA, tmA16, tmB, p, most);
        if (bn == 256) return launch_tc<kNT, false, 256>(h, tmA, tmA16, tmB, p, most);
        if (bn == 128) return launch_tc<kNT, false, 128>(h, tmA, tmA16, tmB, p, most);
        return launch_tc<kNT, false, 64>(h, tmA, tmA16, tmB, p, most);
    }
    if (pair) return launch_tc<kNN, true, 256>(h, tmA, tmA16, tmB, p, most);
    if (bn == 256) return launch_tc<kNN, false, 256>(h, tmA, tmA16, tmB, p, most);
    if (bn == 128) return launch_tc<kNN, false, 128>(h, tmA, tmA16, tmB, p, most);
    return launch_tc<kNN, false, 64>(h, tmA, tmA16, tmB, p, most);
}

int launch_hgemm_grouped_wgrad(b2b_handle *h, int type, int c_type, size_t groups, size_t rows, size_t m, size_t n,
                               float alpha, const uint16_t *A, const uint16_t *B, float beta, void *C,
                               const int32_t *offsets) {
    const int64_t M = static_cast<int64_t>(m), N = static_cast<int64_t>(n);
    const int G = static_cast<int>(groups);
    const bool bf16 = type == B2B_TYPE_BF16, f32 = c_type == B2B_TYPE_F32;
    if (G * (M / 128 + 1) * (N / 64 + 1) >= 1ll << 31)
        return fail(B2B_ERR_NOT_SUPPORTED, "grouped HGEMM: 2^31 tiles or more");
    TcArgs p{A, B, C, offsets, h->d_status, h->wait_limit_ns, G, static_cast<int>(rows), static_cast<int>(m),
             static_cast<int>(n), 0, alpha, beta, 0, bf16, n % (f32 ? 4 : 8) == 0 && aligned16(C)};
    bool pair = M > 128 && N > 128;
    // k blocks of a group as long as the average
    const int64_t kb = (static_cast<int64_t>(rows) + 64 * G - 1) / (64 * G), tiles128 = G * ((M + 127) / 128) * ((N + 127) / 128);
    if (rows == 0 || !tma_can(A, B, M, 1, N)) {  // without rows nothing is loaded
        const bool two = pair && !f32 && by_hand_in_pairs(h, G * ((M + 127) / 128), G * ((M + 255) / 256), N);
        const int parts = two ? 1 : k_parts(h, tiles128, kb, 1.1, 1.1 * static_cast<double>(kb));
        const int bm = two ? 256 : 128;
        p.idesc = sm100::idesc_f32acc(bf16, 1, 1, bm, bm);
        const int64_t most = G * ((M + bm - 1) / bm) * ((N + bm - 1) / bm);
        const CUtensorMap none{};
        if (parts > 1)
            return f32 ? launch_tc<kTN, false, 128, true, true, true>(h, none, none, none, p, most, parts)
                       : launch_tc<kTN, false, 128, false, true, true>(h, none, none, none, p, most, parts);
        if (f32) return launch_tc<kTN, false, 128, true, true>(h, none, none, none, p, most);
        return two ? launch_tc<kTN, true, 256, false, true>(h, none, none, none, p, most)
                    : launch_tc<kTN, false, 128, false, true>(h, none, none, none, p, most);
    }
    int bn = 256;
    const int parts = tiles128 < h->sm_count / 2 ? k_parts(h, tiles128, kb, 0.375, (pair ? 0.4 : 0.34) * static_cast<double>(kb)) : 1;
    if (parts > 1) pair = false, bn = 128;
    while (!pair && parts == 1 && bn > 64 && (G * ((M + 127) / 128) * ((N + bn - 1) / bn) < h->sm_count || N <= bn / 2)) bn /= 2;
    const CUtensorMapDataType dt = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    CUtensorMap tmA, tmB;
    if (int rc = encode_tma_2d(&tmA, dt, 2, A, rows, m, 64, 64)) return rc;
    if (int rc = encode_tma_2d(&tmB, dt, 2, B, rows, n, 64, 64)) return rc;
    p.idesc = sm100::idesc_f32acc(bf16, 1, 1, pair ? 256 : 128, pair ? 256 : bn);
    const int bm = pair ? 256 : 128;
    const int64_t most = G * ((M + bm - 1) / bm) * ((N + bn - 1) / bn);
    if (parts > 1)
        return f32 ? launch_tc<kTN, false, 128, true, false, true>(h, tmA, tmA, tmB, p, most, parts)
                   : launch_tc<kTN, false, 128, false, false, true>(h, tmA, tmA, tmB, p, most, parts);
    return f32 ? launch_wgrad<true>(h, pair, bn, tmA, tmB, p, most) : launch_wgrad<false>(h, pair, bn, tmA, tmB, p, most);
}

}  // namespace b2b

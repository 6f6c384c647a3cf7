// w4.cu -- matrices held in 4 bits with a scale (and a zero point) for each
// group of a row's columns: quantisation, the way back to 16 bits, and
// products with vectors.  No counterpart in cublas-rs, whose GEMVs
// (crates/cublas-l2/src/gemv.rs) read 16-, 32- and 64-bit matrices.
//
//   W[i][j] = scale[i][j / group] * (q[i][j] - zero[i][j / group])
//   y_i = alpha * W x_i + beta * y_i
#include <cuda.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <mutex>
#include <type_traits>

#include "half_types.cuh"
#include "internal.h"
#include "sm100.cuh"

namespace {

struct W4Args {
    const uint8_t *packed;
    const uint16_t *scales;
    const uint8_t *zeros;  // nullptr: 8 everywhere
    int64_t m, n, group, pitch, gs;  // pitch = bytes of a packed row, gs = groups of a row
};

// ---------------------------------------------------------------------------
// Quantisation.  All arithmetic that decides a value is f32 on the scale
// rounded to 16 bits.  The quotient w / s that rounds to a value is of two
// numbers with at most 11 significant bits: unless it lies exactly on the
// border between two values it is at least 2^-12 away from it.  So w times the
// reciprocal, at most 2^-18 off, decides as the quotient would, and where it is
// that near to a border the quotient is on the border: the even value it is.

// The scale of a group from its extremes (0 among them); NaN unless all its
// values are finite.
template <bool BF16>
__device__ __forceinline__ uint16_t w4_scale(float lo, float hi, bool finite, bool zeros) {
    // halves, so that hi - lo of bf16 extremes stays finite
    const float s = zeros ? __fdiv_rn(0.5f * hi - 0.5f * lo, 7.5f) : __fdiv_rn(fmaxf(hi, -lo), 7.0f);
    return b2b::Half16<BF16>::put(finite ? s : __int_as_float(0x7fffffff));
}

// Values of a group whose scale is s.
struct Quantizer {
    static constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: adding it rounds to a whole number, ties to even
    float s, inverse, zero;
    static constexpr float kBorder = 0.499996185302734375f;  // 1/2 - 2^-18
    bool live;    // s > 0: false for a zero and a NaN scale, whose groups hold their zero point
    bool divide;  // the reciprocal overflows
    bool clamps;  // values may pass 0..15: with zero points, or where the scale was rounded by more than 1 / 100
    // `normal`: the least normal number of the scale's type
    __device__ __forceinline__ Quantizer(float scale, float lo, bool zeros, float normal) : s(scale) {
        live = s > 0.0f;
        inverse = __fdividef(1.0f, s);
        divide = !(inverse < 1e38f);
        clamps = zeros || !(s >= normal);
        zero = 8.0f;
        if (zeros) zero = live ? fminf(rintf(__fdiv_rn(-lo, s)), 15.0f) : 0.0f;
    }
    __device__ __forceinline__ float clamp(float r) const { return fminf(fmaxf(r + zero, 0.0f), 15.0f); }
    __device__ __forceinline__ float exact(float w) const { return live ? clamp(rintf(__fdiv_rn(w, s))) : zero; }
    // N values 0..15, as floats, less `zero` where that is returned; else 0.
    template <int N>
    __device__ __forceinline__ float operator()(const float (&w)[N], float (&out)[N]) const {
        if (divide) {
#pragma unroll
            for (int i = 0; i < N; ++i) out[i] = exact(w[i]);
            return 0.0f;
        }
        float far = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            out[i] = fmaf(w[i], inverse, kRound) - kRound;
            far = fmaxf(far, fabsf(fmaf(w[i], inverse, -out[i])));
        }
        if (far > kBorder) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float off = fmaf(w[i], inverse, -out[i]);
                const bool odd = __float_as_uint(out[i] + kRound) & 1u;
                if (fabsf(off) > kBorder && odd) out[i] += copysignf(1.0f, off);
            }
        }
        if (!clamps) return zero;
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = clamp(out[i]);
        return 0.0f;
    }
};

// Eight values, `less` added to each, to a word: the nibbles of two halves are
// added up in f32, where they are exact.
__device__ __forceinline__ uint32_t pack8(const float *q, float less) {
    const float all = 4369.0f * less;  // 0x1111
    const float low = fmaf(4096.0f, q[3], fmaf(256.0f, q[2], fmaf(16.0f, q[1], q[0] + all)));
    const float high = fmaf(4096.0f, q[7], fmaf(256.0f, q[6], fmaf(16.0f, q[5], q[4] + all)));
    return static_cast<uint32_t>(low) | static_cast<uint32_t>(high) << 16;
}

// Least and largest of 0 and 16 values, two at a time; false where one of them
// is an infinity or a NaN.
template <bool BF16>
__device__ __forceinline__ bool extremes(const uint32_t (&words)[8], float &lo, float &hi) {
    using T = typename std::conditional<BF16, __nv_bfloat162, __half2>::type;
    const T *v = reinterpret_cast<const T *>(words);
    uint32_t none = 0;
    const T zero = *reinterpret_cast<const T *>(&none);
    T a = zero, b = zero, nan = zero;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        a = __hmin2(a, v[i]);
        b = __hmax2(b, v[i]);
        nan = __hfma2(v[i], zero, nan);  // 0, or a NaN once an infinity or a NaN is met
    }
    const float2 fa = b2b::Half16<BF16>::get2(*reinterpret_cast<const uint32_t *>(&a));
    const float2 fb = b2b::Half16<BF16>::get2(*reinterpret_cast<const uint32_t *>(&b));
    const float2 fn = b2b::Half16<BF16>::get2(*reinterpret_cast<const uint32_t *>(&nan));
    lo = fminf(fa.x, fa.y);
    hi = fmaxf(fb.x, fb.y);
    return fn.x == 0.0f && fn.y == 0.0f;
}

// Groups of 16 LANES columns, 16 of them to a lane, which reads them once.
// WHOLE: n is a multiple of 8 and W and packed allow 16-byte loads and 4-byte
// stores; else values and bytes one at a time.  Bound by its instructions where
// WHOLE: about 250 for the 40 bytes that a lane moves, most of them the rounding
// and clamping of its values: 4096 x 4096 takes 14.3 us (2.9 TB/s), 8192 x 8192
// 50 to 55 us (3.1 to 3.4 TB/s) with its schedulers 72 % busy.
template <bool BF16, int LANES, bool WHOLE>
__global__ void __launch_bounds__(256) w4_quantize_kernel(const uint16_t *W, uint8_t *packed, uint16_t *scales,
                                                          uint8_t *zeros, int64_t m, int64_t n, int64_t pitch, int64_t gs) {
    using H = b2b::Half16<BF16>;
    const int lane = threadIdx.x & 31;
    const int64_t per = (gs * LANES + 31) / 32;  // tasks of a row: a warp's 512 columns
    const int64_t step = static_cast<int64_t>(gridDim.x) * 8;
    for (int64_t task = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); task < m * per; task += step) {
        const int64_t row = task / per;
        const int64_t unit = task % per * 32 + lane, j0 = unit * 16;
        const uint16_t *w = W + row * n + j0;
        uint32_t words[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if constexpr (WHOLE) {
                uint4 in = make_uint4(0, 0, 0, 0);
                if (j0 + 8 * h < n) in = __ldg(reinterpret_cast<const uint4 *>(w) + h);
                words[4 * h] = in.x, words[4 * h + 1] = in.y, words[4 * h + 2] = in.z, words[4 * h + 3] = in.w;
            } else {
#pragma unroll
                for (int i = 4 * h; i < 4 * h + 4; ++i) {
                    words[i] = j0 + 2 * i < n ? __ldg(w + 2 * i) : 0u;
                    if (j0 + 2 * i + 1 < n) words[i] |= static_cast<uint32_t>(__ldg(w + 2 * i + 1)) << 16;
                }
            }
        }
        float v[16], lo, hi;
        if (!extremes<BF16>(words, lo, hi)) hi = __int_as_float(0x7f800000);  // reaches the group's other lanes as an infinity
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 f = H::get2(words[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
#pragma unroll
        for (int d = LANES / 2; d; d >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
        }
        const uint16_t s16 = w4_scale<BF16>(lo, hi, hi < __int_as_float(0x7f800000), zeros != nullptr);
        const Quantizer q(H::get(s16), lo, zeros != nullptr, H::kNormal);
        float out[16];
        const float less = q(v, out);
        const uint32_t word0 = pack8(out, less), word1 = pack8(out + 8, less);
        uint8_t *to = packed + row * pitch + unit * 8;
        if constexpr (WHOLE) {
            if (j0 + 8 < n) {
                if ((reinterpret_cast<uintptr_t>(to) & 7) == 0) {
                    *reinterpret_cast<uint2 *>(to) = make_uint2(word0, word1);
                } else {
                    reinterpret_cast<uint32_t *>(to)[0] = word0;
                    reinterpret_cast<uint32_t *>(to)[1] = word1;
                }
            } else if (j0 < n) {
                *reinterpret_cast<uint32_t *>(to) = word0;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (j0 + 2 * i < n) {
                    uint32_t byte = (i < 4 ? word0 : word1) >> (i % 4 * 8) & 0xffu;
                    if (j0 + 2 * i + 1 == n) byte &= 15u;
                    to[i] = static_cast<uint8_t>(byte);
                }
        }
        if (lane % LANES == 0 && j0 < n) {
            const int64_t at = row * gs + unit / LANES;
            scales[at] = s16;
            if (zeros) zeros[at] = static_cast<uint8_t>(q.zero);
        }
    }
}

// Other groups: one warp a group, which it reads twice, the second time out of
// L1 or L2 unless it is very long.  WHOLE as above: 8 neighbouring values a
// lane, else two.
template <bool BF16, bool WHOLE>
__global__ void __launch_bounds__(256) w4_quantize_any_kernel(const uint16_t *W, uint8_t *packed, uint16_t *scales,
                                                              uint8_t *zeros, int64_t m, int64_t n, int64_t group,
                                                              int64_t pitch, int64_t gs) {
    using H = b2b::Half16<BF16>;
    const int lane = threadIdx.x & 31;
    const int64_t step = static_cast<int64_t>(gridDim.x) * 8;
    for (int64_t at = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); at < m * gs; at += step) {
        const int64_t row = at / gs, j0 = at % gs * group;
        const int64_t j1 = j0 + group < n ? j0 + group : n;
        const uint16_t *w = W + row * n;
        float lo = 0.0f, hi = 0.0f, nan = 0.0f;
        auto take = [&](float v) {
            nan = fmaf(v, 0.0f, nan);
            lo = fminf(lo, v);
            hi = fmaxf(hi, v);
        };
        auto eight = [&](int64_t j, float (&v)[8]) {
            const uint4 in = __ldg(reinterpret_cast<const uint4 *>(w + j));
            const uint32_t words[4] = {in.x, in.y, in.z, in.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = H::get2(words[i]);
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        };
        if constexpr (WHOLE) {
#pragma unroll 2
            for (int64_t j = j0 + 8 * lane; j < j1; j += 256) {
                float v[8];
                eight(j, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) take(v[i]);
            }
        } else {
            for (int64_t j = j0 + lane; j < j1; j += 32) take(H::get(w[j]));
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
        }
        const bool finite = __all_sync(0xffffffffu, nan == 0.0f);
        const uint16_t s16 = w4_scale<BF16>(lo, hi, finite, zeros != nullptr);
        const Quantizer q(H::get(s16), lo, zeros != nullptr, H::kNormal);
        if (lane == 0) {
            scales[at] = s16;
            if (zeros) zeros[at] = static_cast<uint8_t>(q.zero);
        }
        if constexpr (WHOLE) {
#pragma unroll 2
            for (int64_t j = j0 + 8 * lane; j < j1; j += 256) {
                float v[8], out[8];
                eight(j, v);
                const float less = q(v, out);
                *reinterpret_cast<uint32_t *>(packed + row * pitch + j / 2) = pack8(out, less);
            }
            continue;
        }
        for (int64_t j = j0 + 2 * lane; j < j1; j += 64) {
            uint32_t byte = static_cast<uint32_t>(q.exact(H::get(w[j])));
            if (j + 1 < j1) byte |= static_cast<uint32_t>(q.exact(H::get(w[j + 1]))) << 4;
            packed[row * pitch + j / 2] = static_cast<uint8_t>(byte);
        }
    }
}

// ---------------------------------------------------------------------------
// Products with vectors: y_i = alpha W x_i + beta y_i for up to 8 vectors that
// share W.  The packed values are read once, and to be bound by HBM the work for
// each must stay well under the ~2.5 instructions that 148 SMs can issue in the
// time a value takes to arrive.  Multiplying on the tensor cores with the 8
// columns of mma.m16n8k16 does that for 1 vector as for 8: a word of 8 values
// becomes four register pairs of exact (q - zero) in 9 instructions (f16: or
// the bits into 1024 + q or 1024 + 16 q, then one packed subtraction or fma),
// and 16 words of a warp are one MMA operand.  Sums are f32; a group's sum is
// scaled in f32 and added to the row's.  No product or sum is rounded to 16
// bits.
//
//   * A tile is 32 rows of W for one set of vectors; its n columns are cut
//     into boxes of 256, which the CTAs of a cluster and some of a CTA's 16
//     warps take in turn.  A cluster has an equal share of all tiles, next to
//     each other, and takes them in rounds: of 16 tiles, a warp to each, while
//     it has as many, then of 8, 4, 2 and 1 with 2, 4, 8 and 16 warps to a
//     tile, so that no warp idles while another has two; what is left in one
//     round as soon as there are warps for all its boxes.
//   * Each warp holds one box (32 rows x 128 bytes, 128-byte swizzle), copies
//     it to registers, and TMA refills it, across rounds, so nothing drains at
//     a round's end: 64 KiB of an SM in flight.  Two boxes to a warp took 38 us
//     where one takes 36 (18944 x 16384), and the room is the vectors'.
//   * The vectors are staged once for each set, each 8 columns reordered to
//     the pairs (0,4) (1,5) (2,6) (3,7) that the words unpack to.  Only where
//     they do not fit one SM, or where there are fewer tiles than SMs, is a
//     tile shared by a cluster: its joining costs most of what it saves.
//   * The last of a tile's warps to arrive adds their sums up while the others
//     go on; the CTAs of a cluster join the sums of up to 8 rounds at once,
//     when those of the next ones are ready (18944 x 16384 by 8 vectors: 104
//     us where all waited for all after each batch, 47 now).  Both in a fixed
//     order, whoever adds.
// f16 by one vector, no zero points: 7.6 us, and 7.1 for each tile of an SM where
// rows have 16384 columns (5.6 TB/s of packed bytes), 6.5 and 7.9 for 8 tiles of
// 2048 (5.1).  Tiles are whole: 16384 rows, 3.46 tiles for each of 148 SMs, take
// 35.7 us, 18944, 4 for each, 36.3 (by 8 vectors both 47).  Unpacking bfloat16 with
// zero points adds a tenth.  What a tile lacks to HBM's 6.4 is instructions, 20
// for each word of a warp, half a cycle each on the pipes that most of them need.
// Rows that TMA cannot describe (n not a multiple of 32, packed not 16-byte
// aligned) come by cp.async (HAND): the aligned words that hold a box's rows, 33
// of each, which are shifted into place on their way to registers: 16384 x
// 16388 takes 61 us, 16384 x 16376, whose rows begin at words, 53.  Groups
// that do not fit a box evenly (SPG = 0) read their scales when they begin.
constexpr int kWarps = 16;
constexpr int kThreads = kWarps * 32;
constexpr int kTileRows = 32;
constexpr int kBoxCols = 256;                     // 128 bytes of a row
constexpr int kBoxSteps = kBoxCols / 32;          // of 32 columns
constexpr int kBoxBytes = kTileRows * kBoxCols / 2;
constexpr int kHandPitch = 144;                   // HAND: bytes of a row's 33 words, so that 8 rows meet every bank once
constexpr int kHandBytes = kTileRows * kHandPitch;
constexpr int kMaxBatch = 8;                      // rounds that the CTAs of a cluster join at once
constexpr int kMaxIndexed = 256;                  // products of one launch that choose their matrix

struct GemvArgs {
    W4Args w;
    const uint16_t *x;
    const int32_t *index;  // nullptr: every product uses matrix 0
    uint16_t *y;
    int *status;
    uint64_t wait_ns;
    int matrices, count, fan, first;  // first: number of this launch's first product
    int width;    // vectors of a set: 8, or fewer where longer rows leave room for fewer
    int parts;    // most tiles of a round, a power of two
    int batch;    // rounds that the CTAs of a cluster join at once, a power of two
    int x_bytes;  // of the staged vectors
    int vec;      // a box's scales and zero points of a row are one aligned word each
    float alpha, beta;
    int64_t total;  // bytes of packed
};

// Products that share a matrix, at most 8; counted from the launch's first.
struct Item {
    int matrix;  // -1: none
    int count;
    uint8_t member[8];
};
// What a launch that chooses matrices keeps of its products.
struct Table {
    Item item[kMaxIndexed];
    int4 index[kMaxIndexed / 4];      // the matrix that each product names, -1 where none
    uint32_t leads[kMaxIndexed / 32];  // the products that are their sets' first, a bit each
};

// `bytes` of the aligned word at `src` to shared memory, and zeros for the rest.
__device__ __forceinline__ void copy_word(uint32_t to, const uint8_t *src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(src), "r"(bytes) : "memory");
}

// c += a b, or c = a b where FRESH.
template <bool BF16, bool FRESH>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    const float c0 = FRESH ? 0.0f : c[0], c1 = FRESH ? 0.0f : c[1], c2 = FRESH ? 0.0f : c[2], c3 = FRESH ? 0.0f : c[3];
    if constexpr (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%10, %11, %12, %13};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%10, %11, %12, %13};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// (v & mask) | bits
__device__ __forceinline__ uint32_t and_or(uint32_t v, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(v), "r"(mask), "r"(bits));
    return r;
}

__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}

__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<const __half2 *>(&v); }
__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t v) { return *reinterpret_cast<const __nv_bfloat162 *>(&v); }
template <typename T>
__device__ __forceinline__ uint32_t as_word(T v) { return *reinterpret_cast<const uint32_t *>(&v); }

// The pairs (0,4) (1,5) (2,6) (3,7) of a word's values, less `zero` (0..15),
// exact in 16 bits.
template <bool BF16>
struct Unpack;
template <>
struct Unpack<false> {
    uint32_t low, high;  // pairs of 1024 + zero and of -(64 + zero)
    __device__ __forceinline__ explicit Unpack(uint32_t zero) {
        low = (0x6400u + zero) * 0x10001u;
        high = (0xd400u + (zero << 4)) * 0x10001u;
    }
    __device__ __forceinline__ void operator()(uint32_t w, uint32_t (&v)[4]) const {
#pragma unroll
        for (int i = 0; i < 2; ++i, w >>= 8) {
            v[2 * i] = as_word(__hsub2(as_half2(and_or(w, 0x000f000fu, 0x64006400u)), as_half2(low)));
            v[2 * i + 1] = as_word(__hfma2(as_half2(and_or(w, 0x00f000f0u, 0x64006400u)), as_half2(0x2c002c00u),
                                           as_half2(high)));
        }
    }
};
template <>
struct Unpack<true> {
    uint32_t low;  // pair of 128 + zero
    __device__ __forceinline__ explicit Unpack(uint32_t zero) { low = (0x4300u + zero) * 0x10001u; }
    __device__ __forceinline__ void operator()(uint32_t w, uint32_t (&v)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i, w >>= 4)
            v[i] = as_word(__hsub2(as_bf162(and_or(w, 0x000f000fu, 0x43004300u)), as_bf162(low)));
    }
};

// Two tiles of 16 rows times 32 columns: words of rows g, g + 8, g + 16, g + 24.
template <bool BF16, bool FRESH>
__device__ __forceinline__ void step32(float (&sum)[2][4], const uint32_t (&words)[4], const Unpack<BF16> (&un)[4],
                                       const uint4 &x) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t a[4], b[4];
        un[2 * h](words[2 * h], a);
        un[2 * h + 1](words[2 * h + 1], b);
        mma16816<BF16, FRESH>(sum[h], a[0], b[0], a[1], b[1], x.x, x.y);
        mma16816<BF16, false>(sum[h], a[2], b[2], a[3], b[3], x.z, x.w);
    }
}

__device__ __forceinline__ void add_scaled(float (&total)[2][4], const float (&sum)[2][4], const float (&scale)[4]) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
        total[i >> 2][i & 3] = fmaf(scale[i >> 1], sum[i >> 2][i & 3], total[i >> 2][i & 3]);
}

// Scales and zero points of one row's groups in a box (at most 8).
template <int SPG, bool ZEROS>
struct RowScales {
    static constexpr int N = SPG ? kBoxSteps / SPG : 1;
    uint32_t s[(N + 1) / 2];
    uint32_t z[(N + 3) / 4];
    template <int WORDS>
    __device__ __forceinline__ static void words(uint32_t *to, const void *from) {
        if constexpr (WORDS >= 4) {
#pragma unroll
            for (int i = 0; i < WORDS / 4; ++i) {
                const uint4 v = __ldg(static_cast<const uint4 *>(from) + i);
                to[4 * i] = v.x, to[4 * i + 1] = v.y, to[4 * i + 2] = v.z, to[4 * i + 3] = v.w;
            }
        } else if constexpr (WORDS == 2) {
            const uint2 v = __ldg(static_cast<const uint2 *>(from));
            to[0] = v.x, to[1] = v.y;
        } else {
            to[0] = __ldg(static_cast<const uint32_t *>(from));
        }
    }
    // `left`: groups that the row has from here on
    __device__ __forceinline__ void load(const uint16_t *scales, const uint8_t *zeros, int left, int vec) {
        if (N == 1) {
            s[0] = __ldg(scales);
            if constexpr (ZEROS) z[0] = __ldg(zeros);
        } else if (vec) {
            words<(N + 1) / 2>(s, scales);
            if constexpr (ZEROS && N >= 4) words<(N + 3) / 4>(z, zeros);
            if constexpr (ZEROS && N == 2) z[0] = __ldg(reinterpret_cast<const uint16_t *>(zeros));
        } else {
#pragma unroll
            for (int i = 0; i < (N + 1) / 2; ++i) s[i] = 0;
#pragma unroll
            for (int i = 0; i < (N + 3) / 4; ++i) z[i] = 0;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < left) {
                    s[i / 2] |= static_cast<uint32_t>(__ldg(scales + i)) << (16 * (i & 1));
                    if constexpr (ZEROS) z[i / 4] |= static_cast<uint32_t>(__ldg(zeros + i)) << (8 * (i & 3));
                }
        }
    }
    __device__ __forceinline__ uint16_t scale(int i) const { return static_cast<uint16_t>(s[i / 2] >> (16 * (i & 1))); }
    __device__ __forceinline__ uint32_t zero(int i) const { return ZEROS ? z[i / 4] >> (8 * (i & 3)) & 15u : 8u; }
};

// Where row g + 8 i's word of step st is, from that of g's first step: 16-byte
// piece st of row r sits at piece st ^ (r % 8), or in order (HAND).
template <bool HAND>
__device__ __forceinline__ uint32_t word_of(uint32_t w, int st, int i) {
    return HAND ? w + st * 16 + i * 8 * kHandPitch : (w ^ (st << 4)) + i * 1024;
}

// A box's products: this lane's words of its steps, in registers (EARLY) or at
// shared address w, the vectors' pieces of its first step at shared address x.
// FULL: it has all its steps.
template <bool BF16, bool ZEROS, int SPG, bool EARLY, bool HAND, bool FULL>
__device__ __forceinline__ void box_products(float (&total)[2][4], const uint32_t (&words)[EARLY ? kBoxSteps : 1][4],
                                             uint32_t w, const uint32_t (&shift)[HAND ? 4 : 1], bool shifts, uint32_t x,
                                             int xstep, const RowScales<SPG, ZEROS> &row, int g, int steps) {
    using H = b2b::Half16<BF16>;
    uint32_t sw[4], zw[4];  // of rows g, g + 8, g + 16, g + 24: two groups' scales, four groups' zero points
#pragma unroll
    for (int gi = 0; gi < kBoxSteps / SPG; ++gi) {
        if (!FULL && gi * SPG >= steps) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (gi % 2 == 0) sw[i] = __shfl_sync(0xffffffffu, row.s[gi / 2], g + 8 * i);
            if (ZEROS && gi % 4 == 0) zw[i] = __shfl_sync(0xffffffffu, row.z[gi / 4], g + 8 * i);
        }
        auto scale_of = [&](int i) { return H::get(static_cast<uint16_t>(gi % 2 ? sw[i] >> 16 : sw[i])); };
        auto zero_of = [&](int i) { return ZEROS ? zw[i] >> (8 * (gi % 4)) & 15u : 8u; };
        const Unpack<BF16> un[4] = {Unpack<BF16>(zero_of(0)), Unpack<BF16>(zero_of(1)), Unpack<BF16>(zero_of(2)),
                                    Unpack<BF16>(zero_of(3))};
        const float scale[4] = {scale_of(0), scale_of(1), scale_of(2), scale_of(3)};
        float sum[2][4];
#pragma unroll
        for (int si = 0; si < SPG; ++si) {
            const int st = gi * SPG + si;
            if (!FULL && si > 0 && st >= steps) break;
            const uint4 xv = lds128(x);
            x += xstep;
            uint32_t own[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) own[i] = EARLY ? words[EARLY ? st : 0][i] : lds32(word_of<HAND>(w, st, i));
            if constexpr (HAND && !EARLY) {
                if (shifts) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) own[i] = __funnelshift_r(own[i], lds32(word_of<HAND>(w, st, i) + 4), shift[i]);
                }
            }
            if (si == 0)
                step32<BF16, true>(sum, own, un, xv);
            else
                step32<BF16, false>(sum, own, un, xv);
        }
        add_scaled(total, sum, scale);
    }
}

// Waits until *count reaches `want`; bounded like every wait (the warps that
// raise it wait for their own loads, each at most wait_ns).
__device__ __forceinline__ bool wait_finished(const volatile int *count, int want, volatile int *abort, const GemvArgs &p,
                                              int lane) {
    int ok = 1;
    if (lane == 0 && *count < want) {
        const uint64_t t0 = sm100::globaltimer_ns();
        while (*count < want) {
            if (*abort || sm100::globaltimer_ns() - t0 > 2 * p.wait_ns) {
                *abort = 1;
                atomicCAS(p.status, 0, B2B_DEVSTAT_TIMEOUT | 0x32);
                ok = 0;
                break;
            }
        }
    }
    return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

// A round: `count` tiles with 2^lk warps to each; the warps left over idle.
struct Round {
    int count, lk;
};
// A place in a cluster's sequence of rounds.
struct Place {
    uint32_t set, tile, left;  // next tile, and how many are left
    // Takes the next round, from `tile` on: all tiles that are left if there
    // are warps for their boxes (2^lbox of them), else 2^i tiles.
    __device__ __forceinline__ Round take(uint32_t tiles, uint32_t most, int lbox) {
        const uint32_t have = min(left, tiles - tile);
        Round r{static_cast<int>(have), lbox};
        if (have > min(most, 16u >> lbox)) {
            const int lp = 31 - __clz(static_cast<int>(min(have, most)));
            r = Round{1 << lp, min(4 - lp, lbox)};
        }
        left -= r.count;
        tile += r.count;
        return r;
    }
    // ... after which a set may be done.
    __device__ __forceinline__ void settle(uint32_t tiles) {
        if (tile == tiles) {
            tile = 0;
            ++set;
        }
    }
};

// SPG: steps of 32 columns in a group, 8 standing for its multiples; 0: any
// group (HAND).
template <bool BF16, bool ZEROS, int SPG, bool HAND>
__global__ void __launch_bounds__(kThreads, 1)
    w4_gemv_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ GemvArgs p) {
    using namespace sm100;
    using H = b2b::Half16<BF16>;
    static_assert(HAND || SPG != 0, "any group: HAND");
    constexpr bool TMA = !HAND;
    extern __shared__ uint8_t smem_raw[];
    __shared__ int abort_flag;
    __shared__ int arrived[2][5][kWarps];         // warps of a tile (by log2 of their number) whose sums are in `part`
    __shared__ volatile int finished[2][kWarps];  // rounds whose sums of this warp are joined
    __shared__ Place begin[2][kWarps];            // KS > 1: where the last two batches of rounds began, for each warp
    uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, q = lane & 3;
    const int KS = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
    uint8_t *box = smem + warp * (TMA ? kBoxBytes : kHandBytes);
    uint8_t *sx = smem + kWarps * (TMA ? kBoxBytes : kHandBytes);
    const int sums = kTileRows * p.width;                     // of a tile
    float *part = reinterpret_cast<float *>(sx + p.x_bytes);  // [2][kWarps][32 rows][width]
    float *slots = part + 2 * kWarps * sums;                  // KS > 1: [2][p.batch][p.parts][32 rows][width]
    uint64_t *bars = reinterpret_cast<uint64_t *>(slots + (KS > 1 ? 2 * p.batch * p.parts * sums : 0));
    uint64_t *full = bars + warp;
    uint8_t *nothing = reinterpret_cast<uint8_t *>(bars + kWarps);  // 16 bytes of 0
    Table *table = reinterpret_cast<Table *>(nothing + 16);
    const Item *items = table->item;

    // ---- the sets of products
    const int named = p.index && tid < p.count ? __ldg(p.index + p.first + tid) : 0;
    if (TMA && tid == 0) prefetch_tensormap(&tmW);
    if (tid == 0) abort_flag = 0;
    if (tid < 4) reinterpret_cast<uint32_t *>(nothing)[tid] = 0;
    if (tid < 2 * 5 * kWarps) (&arrived[0][0][0])[tid] = 0;
    if (tid < 2 * kWarps) finished[tid / kWarps][tid % kWarps] = 0;
    if (TMA && lane == 0) {
        mbar_init(full, 1);
        fence_barrier_init();
    }
    int sets_named = 0;
    if (p.index) {
        const int e = named >= 0 && named < p.matrices ? named : -1;
        if (tid < kMaxIndexed) reinterpret_cast<int *>(table->index)[tid] = tid < p.count ? e : -2;
        __syncthreads();
        int place = 0, lead = tid;  // in the set; the set's first product
        if (tid < kMaxIndexed) {
            for (int i = 0; i < tid && tid < p.count; i += 4) {  // products before this one of its matrix
                const int4 four = table->index[i >> 2];
                const int other[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (other[k] == e && i + k < tid) {
                        if (place == 0) lead = i + k;
                        if (++place == p.width) place = 0;
                    }
            }
            if (place == 0) lead = tid;
            const uint32_t leads = __ballot_sync(0xffffffffu, tid < p.count && lead == tid);
            if (lane == 0) table->leads[warp] = leads;
        }
        __syncthreads();
        int number = 0;  // of this product's set
        for (int w = 0; w < kMaxIndexed / 32; ++w) {
            const uint32_t leads = table->leads[w];
            sets_named += __popc(leads);
            if (w < lead >> 5) number += __popc(leads);
            if (w == lead >> 5) number += __popc(leads & ((1u << (lead & 31)) - 1));
        }
        if (tid < p.count && lead == tid) {
            table->item[number].matrix = e;
            table->item[number].count = 0;
        }
        __syncthreads();
        if (tid < p.count) {
            table->item[number].member[place] = static_cast<uint8_t>(tid);
            atomicMax(&table->item[number].count, place + 1);
        }
    }
    __syncthreads();
    const uint32_t tiles = static_cast<uint32_t>((p.w.m + kTileRows - 1) / kTileRows);
    const uint32_t sets = p.index ? sets_named : (static_cast<uint32_t>(p.count) + p.width - 1) / p.width;
    const int boxes = static_cast<int>((p.w.n + kBoxCols - 1) / kBoxCols);
    const int local = boxes > rank ? (boxes - rank + KS - 1) / KS : 0;  // this CTA's boxes of a tile
    const int lbox = min(4, 32 - __clz((boxes + KS - 1) / KS - 1));  // log2 of the warps that a tile can use
    const uint32_t clusters = gridDim.x / KS, cluster = blockIdx.x / KS;
    // next to each other, so that a cluster changes its vectors rarely
    const uint64_t all = static_cast<uint64_t>(sets) * tiles;
    const uint64_t t_begin = all * cluster / clusters, t_end = all * (cluster + 1) / clusters;

    Place here{static_cast<uint32_t>(t_begin / tiles), static_cast<uint32_t>(t_begin % tiles),
               static_cast<uint32_t>(t_end - t_begin)};
    auto matrix_of = [&](uint32_t set) { return p.index ? items[set].matrix : 0; };

    bool dead = false;
    auto vectors_of = [&](uint32_t set) {
        return p.index ? items[set].count
                       : static_cast<int>(min(static_cast<int64_t>(p.width), p.count - static_cast<int64_t>(set) * p.width));
    };
    // The sum of a tile's row r and its set's vector v leaves.
    auto put = [&](uint32_t set, int e, uint32_t tile, int r, int v, float sum) {
        const int64_t row = static_cast<int64_t>(tile) * kTileRows + r;
        if (row >= p.w.m) return;
        const int64_t i = p.index ? p.first + items[set].member[v] : static_cast<int64_t>(set) * p.width + v;
        uint16_t *y = p.y + i * p.w.m + row;
        float res = e >= 0 ? p.alpha * sum : 0.0f;
        if (p.beta != 0.0f) res = fmaf(p.beta, H::get(*y), res);
        *y = H::put(res);
    };

    const int spg = static_cast<int>(p.w.group / 32);
    const int nsteps = static_cast<int>((p.w.n + 31) / 32);
    int nb = 0;
    uint32_t phase = 0;

    // The warp's next box, of this round or a later one: it takes the present
    // one's place as soon as that is used up, and the scales and zero points
    // that belong to it are read, row `lane`'s by each lane (the tile's last
    // one by lanes whose row is not there).
    RowScales<SPG, ZEROS> scales;
    Place ahead = here;
    bool more = true;  // there is a next box
    int nc = 0, nstep = 0, nbox = 0;  // boxes left of its tile, and how far apart they are
    int64_t nrow = 0, nleft = 0;      // the tile's first row, and how many are behind it
    const uint16_t *nscales = nullptr;
    const uint8_t *nzeros = nullptr;
    auto seek = [&] {
        while (ahead.left) {
            const int e = matrix_of(ahead.set);
            const uint32_t first = ahead.tile;
            const Round round = ahead.take(tiles, p.parts, lbox);
            const int lk = round.lk, kwarp = warp & ((1 << lk) - 1);
            ahead.settle(tiles);
            if (e < 0 || kwarp >= local || warp >> lk >= round.count) continue;
            const int64_t tile = first + (warp >> lk), row = e * p.w.m + tile * kTileRows;
            const int64_t left = p.w.m - 1 - tile * kTileRows;  // rows behind the tile's first
            const int64_t at = (row + min(left, static_cast<int64_t>(lane))) * p.w.gs;
            nrow = row;
            nleft = left;
            nscales = p.w.scales + at;
            if (ZEROS) nzeros = p.w.zeros + at;
            nbox = kwarp * KS + rank;
            nstep = KS << lk;
            nc = (local - kwarp + (1 << lk) - 1) >> lk;
            return;
        }
        more = false;
    };
    auto load = [&] {
        if (!more || dead) return;
        if constexpr (TMA) {
            if (lane == 0) {
                mbar_arrive_expect_tx(full, kBoxBytes);
                tma_load_2d(box, &tmW, full, nbox * (kBoxCols / 2), static_cast<int>(nrow));
            }
        } else {
            // a lane copies word `lane` of each row, and the last one of row `lane`;
            // words behind a row's end stay what they are (they meet zeros of x)
            const int64_t at = nrow * p.w.pitch + static_cast<int64_t>(nbox) * (kBoxCols / 2);
            const uint8_t *src = p.w.packed + at;
            const uint32_t to = smem_u32(box) + lane * 4, last = smem_u32(box) + lane * kHandPitch + 128;
            auto word = [](const uint8_t *q) { return reinterpret_cast<const uint8_t *>(reinterpret_cast<uintptr_t>(q) & ~uintptr_t(3)); };
            const int have = static_cast<int>(min(static_cast<int64_t>(33), (p.w.n - static_cast<int64_t>(nbox) * kBoxCols + 7) / 8 + 1));
            // rows that do not exist repeat the last one
            const int behind = static_cast<int>(min(nleft, static_cast<int64_t>(kTileRows - 1)));
            if ((at >= 4 || (reinterpret_cast<uintptr_t>(p.w.packed) & 3) == 0) && at + behind * p.w.pitch + 136 <= p.total) {
                if (have == 33) copy_word(last, word(src + min(lane, behind) * p.w.pitch) + 128, 4);
                if (lane < have && behind == kTileRows - 1) {
#pragma unroll 8
                    for (int r = 0; r < kTileRows; ++r, src += p.w.pitch) copy_word(to + r * kHandPitch, word(src) + lane * 4, 4);
                } else if (lane < have) {
#pragma unroll 4
                    for (int r = 0; r < kTileRows; ++r) {
                        copy_word(to + r * kHandPitch, word(src) + lane * 4, 4);
                        if (r < behind) src += p.w.pitch;
                    }
                }
            } else {
                // bytes outside `packed` are 0
                auto careful = [&](uint32_t dst, const uint8_t *q) {
                    const int64_t have = p.w.packed + p.total - q;
                    if (q >= p.w.packed) {
                        copy_word(dst, have > 0 ? q : word(p.w.packed + 3), have > 4 ? 4 : have > 0 ? static_cast<int>(have) : 0);
                        return;
                    }
                    uint32_t v = 0;  // the word that `packed` begins in
                    for (int i = 0; i < 4; ++i)
                        if (q + i >= p.w.packed && i < have) v |= static_cast<uint32_t>(q[i]) << (8 * i);
                    asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst), "r"(v) : "memory");
                };
                careful(last, word(src + min(lane, behind) * p.w.pitch) + 128);
#pragma unroll 1
                for (int r = 0; r < kTileRows; ++r)
                    careful(to + r * kHandPitch, word(src + min(r, behind) * p.w.pitch) + lane * 4);
            }
        }
        if constexpr (SPG != 0) {
            const int step = nbox * kBoxSteps, grp = SPG == kBoxSteps ? step / spg : step / SPG;
            scales.load(nscales + grp, nzeros + grp, static_cast<int>(p.w.gs) - grp, p.vec);
        }
        nbox += nstep;
        if (--nc == 0) seek();
    };
    seek();
    load();

    int e = -1;          // the set's matrix
    uint32_t over = 0;   // 2^16 / nb, rounded up: o * over >> 16 is o / nb for the sums of a tile
    uint32_t staged = 0xffffffffu;  // the set whose vectors are staged
    // KS > 1: the CTAs' sums of a batch of rounds are joined when those of the
    // next one are ready, so that no warp waits for the others' last boxes.  A
    // CTA adds up its share; a batch's slots are free again when all have
    // arrived with the next batch's sums.
    auto slots_of = [&](int v) { return slots + (v & p.batch ? p.batch : 0) * p.parts * sums; };  // of round v's batch
    auto join_cluster = [&](int v) {  // v: the batch's last round
        __syncwarp();
        cluster_wait();
        const float *joins = slots_of(v);
        const int rounds = (v & (p.batch - 1)) + 1;
        Place at = begin[v & p.batch ? 1 : 0][warp];
        int share = 0;  // 512 sums each
        for (int i = 0; i < rounds; ++i) {
            const uint32_t set = at.set, first = at.tile;
            const int count = at.take(tiles, p.parts, lbox).count;
            at.settle(tiles);
            const int nb = vectors_of(set), e = matrix_of(set);
            for (int k = tid; k - tid < 256 * count; k += kThreads) {
                if ((share++ & (KS - 1)) != rank) continue;
                const int t = k >> 8, o = k & 255;
                if (t >= count || o >= kTileRows * nb) continue;
                const uint32_t from = smem_u32(joins + (i * p.parts + t) * sums + o);
                float of[8];
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < KS) of[r] = ld_shared_cluster(mapa_shared(from, r));
                float sum = 0.0f;
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < KS) sum += of[r];
                put(set, e, first + t, o / nb, o % nb, sum);
            }
        }
    };
    bool single = true;  // the cluster has one round: nothing to go on with at its end
    int v = 0;
    for (; here.left; ++v) {
        const uint32_t set = here.set, first = here.tile;
        if (KS > 1 && (v & (p.batch - 1)) == 0 && lane == 0) begin[v & p.batch ? 1 : 0][warp] = here;
        const Round round = here.take(tiles, p.parts, lbox);
        const int lk = round.lk, kw = 1 << lk;
        here.settle(tiles);
        single = single && here.left == 0;
        const int part_no = warp >> lk, kwarp = warp & (kw - 1);
        const bool idle = part_no >= round.count;
        const int own = local > kwarp && !idle ? (local - kwarp + kw - 1) >> lk : 0;
        const uint32_t tile = first + part_no;
        if (set != staged) {
            staged = set;
            e = matrix_of(set);
            nb = vectors_of(set);
            over = (65536u + nb - 1) / nb;
            __syncthreads();  // everyone is done with the old vectors
            if (e >= 0) {
                // 8 columns of a vector a piece, four pieces of a thread at
                // once; local box l is box l * KS + rank
                constexpr int kOcts = kBoxCols / 8;
                const int pieces = local * kOcts;
                int i = tid, b = 0;  // the next piece, of vector b
                auto settle = [&] {
                    while (i >= pieces && b < nb) {
                        i -= pieces;
                        ++b;
                    }
                };
                settle();
                while (b < nb) {
                    uint4 in[4];
                    int to[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        to[k] = -1;
                        if (b >= nb) continue;
                        // step i / 4 of the vectors' steps, vector, quarter i % 4
                        to[k] = ((i >> 2) * nb + b) * 64 + (i & 3) * 16;
                        const int64_t j = (static_cast<int64_t>(i / kOcts) * KS + rank) * kBoxCols + i % kOcts * 8;
                        const int64_t v = p.index ? p.first + items[set].member[b] : static_cast<int64_t>(set) * p.width + b;
                        const uint16_t *src = p.x + (p.fan == 1 ? v : static_cast<uint32_t>(v) / static_cast<uint32_t>(p.fan)) * p.w.n + j;
                        if (j + 8 <= p.w.n && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
                            in[k] = __ldg(reinterpret_cast<const uint4 *>(src));
                        } else {
                            uint16_t h[8];
#pragma unroll
                            for (int t = 0; t < 8; ++t) h[t] = j + t < p.w.n ? src[t] : uint16_t(0);
                            in[k] = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
                        }
                        i += kThreads;
                        settle();
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (to[k] < 0) continue;
                        *reinterpret_cast<uint4 *>(sx + to[k]) =
                            make_uint4(__byte_perm(in[k].x, in[k].z, 0x5410), __byte_perm(in[k].x, in[k].z, 0x7632),
                                       __byte_perm(in[k].y, in[k].w, 0x5410), __byte_perm(in[k].y, in[k].w, 0x7632));
                    }
                }
            }
            __syncthreads();
        }
        float total[2][4] = {};
        if (e >= 0 && !idle) {
            const int64_t row0 = e * p.w.m + static_cast<int64_t>(tile) * kTileRows + g;
            const int rows = static_cast<int>(p.w.m - static_cast<int64_t>(tile) * kTileRows) - g;  // > 8 i: row g + 8 i exists
            // lanes of vectors that the set does not have read zeros
            const int xstep = g < nb ? nb * 64 : 0;
            // SPG = 0: the rows whose scales this lane reads, its own or the last
            // one for those that are not there, and the group that they are of
            int64_t row[SPG ? 1 : 4];
            int held = -1;
            float scale[4];
            Unpack<BF16> un[4] = {Unpack<BF16>(8), Unpack<BF16>(8), Unpack<BF16>(8), Unpack<BF16>(8)};
            if constexpr (SPG == 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i) row[i] = row0 + min(8 * i, rows - 1);
            }
            uint32_t shift[HAND ? 4 : 1];  // bits that rows g + 8 i begin behind a word
            if constexpr (HAND) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    shift[i] = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p.w.packed) + (row0 + min(8 * i, rows - 1)) * p.w.pitch & 3) * 8;
            }
            const bool shifts = HAND && ((reinterpret_cast<uintptr_t>(p.w.packed) | static_cast<uint64_t>(p.w.pitch)) & 3) != 0;
            for (int c = 0; c < own; ++c) {
                const int l = kwarp + (c << lk), step0 = (l * KS + rank) * kBoxSteps, steps = nsteps - step0;
                if constexpr (TMA) {
                    if (!dead) {
                        const bool ok = mbar_wait(full, phase, &abort_flag, p.status, B2B_DEVSTAT_TIMEOUT | 0x31, p.wait_ns);
                        dead = !__all_sync(0xffffffffu, ok);
                    }
                    phase ^= 1u;
                } else {
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    __syncwarp();
                }
                const uint32_t w = smem_u32(box) + (TMA ? g * 128 + (g << 4) : g * kHandPitch) + q * 4;
                const uint32_t xs = g < nb ? smem_u32(sx) + l * kBoxSteps * nb * 64 + lane * 16 : smem_u32(nothing);
                // EARLY: the words go to registers at once, so that the box is in
                // flight again while they are multiplied.  Groups of 32 columns,
                // and of 64 with zero points, need the registers for their scales
                // and leave the words where they are (4096 x 4096 by 8 vectors,
                // groups of 32: 8.7 us, early 9.4; 18944 x 16384 by 8, groups of
                // 64: 67 and 69 us, without zero points 52 and 50), and so do rows
                // that are copied by words (16384 x 16388: early is 5 % slower).
                constexpr bool EARLY = SPG == 0 || (TMA && (SPG >= 4 || (SPG == 2 && !ZEROS)));
                uint32_t words[EARLY ? kBoxSteps : 1][4];
                const RowScales<SPG, ZEROS> mine = scales;
                auto refill = [&] {
                    // every lane's reads come before the box's next contents
                    if constexpr (TMA) fence_proxy_async_smem();
                    __syncwarp();
                    load();
                };
                if constexpr (EARLY) {
#pragma unroll
                    for (int st = 0; st < kBoxSteps; ++st)
#pragma unroll
                        for (int i = 0; i < 4; ++i) words[st][i] = lds32(word_of<HAND>(w, st, i));
                    if constexpr (HAND) {
                        if (shifts) {
#pragma unroll
                            for (int st = 0; st < kBoxSteps; ++st)
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    words[st][i] = __funnelshift_r(words[st][i], lds32(word_of<HAND>(w, st, i) + 4), shift[i]);
                        }
                    }
                    refill();
                }
                if constexpr (SPG != 0) {
                    if (steps >= kBoxSteps)
                        box_products<BF16, ZEROS, SPG, EARLY, HAND, true>(total, words, w, shift, shifts, xs, xstep, mine, g, steps);
                    else
                        box_products<BF16, ZEROS, SPG, EARLY, HAND, false>(total, words, w, shift, shifts, xs, xstep, mine, g,
                                                                            steps);
                } else {
#pragma unroll
                    for (int st = 0; st < kBoxSteps; ++st) {
                        if (st >= steps) break;
                        const int grp = (step0 + st) / spg;
                        if (grp != held) {
                            held = grp;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                scale[i] = H::get(__ldg(p.w.scales + row[i] * p.w.gs + grp));
                                if (ZEROS) un[i] = Unpack<BF16>(__ldg(p.w.zeros + row[i] * p.w.gs + grp) & 15u);
                            }
                        }
                        float sum[2][4];
                        step32<BF16, true>(sum, words[st], un, lds128(xs + st * xstep));
                        add_scaled(total, sum, scale);
                    }
                }
                if constexpr (!EARLY) refill();
            }
        }

        // ---- join.  A warp that has its tile to itself puts it out.  Else the
        // last of a tile's warps to get here adds their sums up; none waits,
        // but to reuse a buffer that is not joined yet.  A CTA of one round has
        // nothing to go on with: all its threads add up and put out.
        const int flip = v & 1, turn = v & (p.batch - 1);
        if (KS > 1 && turn == 0 && v > 0) join_cluster(v - 1);
        // A warp that had nothing to hand over may be here before its sums of two
        // rounds ago are joined: the larger number stays.  It writes sums again
        // in another set, after the barriers of its vectors.
        auto joined = [&](int w) { atomicMax(const_cast<int *>(&finished[flip][w]), (v >> 1) + 1); };
        if (idle && !single) {
            if (lane == 0) joined(warp);
        } else if (kw == 1 && !(single && round.count <= 4)) {
#pragma unroll
            for (int i = 0; i < 8 && !idle; ++i) {
                const int r = g + 8 * (i >> 1), b = 2 * q + (i & 1);
                if (b >= nb) continue;
                if (KS == 1)
                    put(set, e, tile, r, b, total[i >> 2][i & 3]);
                else
                    slots_of(v)[(turn * p.parts + part_no) * sums + r * nb + b] = total[i >> 2][i & 3];
            }
            if (lane == 0) joined(warp);
        } else {
            if (v >= 2 && !idle && !wait_finished(&finished[flip][warp], v >> 1, &abort_flag, p, lane)) dead = true;
            float *mine = part + (flip * kWarps + warp) * sums;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int col = 2 * q + (i & 1);
                if (col < nb && !idle) mine[(g + 8 * (i >> 1)) * nb + col] = total[i >> 2][i & 3];
            }
            auto add_up = [&](int t, int o) {  // sum o of the round's tile t
                const float *from = part + (flip * kWarps + (t << lk)) * sums + o;
                float sum = 0.0f;
#pragma unroll 4
                for (int w = 0; w < kw; ++w) sum += from[w * sums];
                const int r = static_cast<int>(o * over >> 16);
                if (KS == 1)
                    put(set, e, first + t, r, o - r * nb, sum);
                else
                    slots_of(v)[(turn * p.parts + t) * sums + o] = sum;
            };
            if (single) {
                __syncthreads();
                for (int i = tid; i < 256 * round.count; i += kThreads)
                    if ((i & 255) < kTileRows * nb) add_up(i >> 8, i & 255);
            } else {
                __threadfence_block();
                __syncwarp();
                int last = 0;
                if (lane == 0) last = atomicAdd(&arrived[flip][lk][part_no], 1) == kw - 1;
                if (__shfl_sync(0xffffffffu, last, 0)) {
                    __threadfence_block();
                    if (lane == 0) arrived[flip][lk][part_no] = 0;
                    for (int o = lane; o < kTileRows * nb; o += 32) add_up(part_no, o);
                    __threadfence_block();
                    __syncwarp();
                    if (lane < kw) joined((part_no << lk) + lane);
                }
            }
        }
        if (KS > 1 && (turn == p.batch - 1 || here.left == 0)) {
            __syncwarp();
            cluster_arrive();
        }
    }
    if (KS > 1) {
        if (v > 0) join_cluster(v - 1);
        __syncwarp();  // no CTA leaves while another reads its sums
        cluster_sync();
    }
    if (TMA && dead && lane == 0) {  // loads in flight land before the CTA leaves
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 2000000ull) {
        }
    }
}

// ---------------------------------------------------------------------------
// Back to 16 bits.  scale * (q - zero) is 11 bits times 5: its product in 16
// bits is the exact one rounded once.

// Whether a finite scale may take values beyond the type, where they become its
// largest finite one; infinities and NaN show in every value.
template <bool BF16>
__device__ __forceinline__ bool w4_clamps(float scale) {
    using H = b2b::Half16<BF16>;
    return fabsf(scale) > H::kMax / 16.0f && fabsf(scale) <= H::kMax;
}
template <bool BF16>
__device__ __forceinline__ uint16_t w4_back(float scale, bool clamps, int q) {
    using H = b2b::Half16<BF16>;
    const float v = scale * static_cast<float>(q);
    return H::put(clamps ? fminf(fmaxf(v, -H::kMax), H::kMax) : v);
}

__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b, __half) { return as_word(__hmul2(as_half2(a), as_half2(b))); }
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b, __nv_bfloat16) {
    return as_word(__hmul2(as_bf162(a), as_bf162(b)));
}

// Whole words and 16-byte stores: n a multiple of 8.  About 25 instructions for the
// 20 bytes and more that a lane moves: 4096 x 4096 takes 9.4 us, 8192 x 8192 35 to
// 39 (4.3 to 4.8 TB/s, of which four fifths are writes).
template <bool BF16>
__global__ void __launch_bounds__(256) w4_dequantize_kernel(W4Args p, uint16_t *W) {
    using H = b2b::Half16<BF16>;
    using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    const int lane = threadIdx.x & 31;
    const int64_t octs = p.n / 8, per = (octs + 63) / 64;
    const uint32_t og = static_cast<uint32_t>(p.group / 8);
    const int64_t step = static_cast<int64_t>(gridDim.x) * 8;
    for (int64_t task = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); task < p.m * per; task += step) {
        const int64_t row = task / per;
        const uint32_t oct0 = static_cast<uint32_t>(task % per) * 64 + lane;
        uint32_t word[2], zero[2];
        uint16_t scale[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // all loads before their use
            const uint32_t oct = min(oct0 + 32 * h, static_cast<uint32_t>(octs - 1));
            const int64_t at = row * p.gs + oct / og;
            word[h] = __ldg(reinterpret_cast<const uint32_t *>(p.packed) + row * octs + oct);
            scale[h] = __ldg(p.scales + at);
            zero[h] = p.zeros ? __ldg(p.zeros + at) & 15u : 8u;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (oct0 + 32 * h >= octs) continue;
            const float s = H::get(scale[h]);
            uint32_t o[4];
            if (fabsf(s) <= H::kMax / 16.0f) {
                uint32_t v[4];
                Unpack<BF16>{zero[h]}(word[h], v);
                const uint32_t ss = scale[h] * 0x10001u;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = mul2(v[i], ss, T{});
                // pairs (0,4) (1,5) (2,6) (3,7) to (0,1) (2,3) (4,5) (6,7)
                o[0] = __byte_perm(v[0], v[1], 0x5410);
                o[1] = __byte_perm(v[2], v[3], 0x5410);
                o[2] = __byte_perm(v[0], v[1], 0x7632);
                o[3] = __byte_perm(v[2], v[3], 0x7632);
            } else {  // a product may pass the largest value, or the scale is not finite
                const bool clamps = w4_clamps<BF16>(s);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int a = static_cast<int>(word[h] >> (8 * i) & 15u), b = static_cast<int>(word[h] >> (8 * i + 4) & 15u);
                    const int z = static_cast<int>(zero[h]);
                    o[i] = w4_back<BF16>(s, clamps, a - z) | static_cast<uint32_t>(w4_back<BF16>(s, clamps, b - z)) << 16;
                }
            }
            *(reinterpret_cast<uint4 *>(W + row * p.n) + oct0 + 32 * h) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
}

// Any n and alignment: bytes 32 apart to a lane, four of them in flight.
template <bool BF16>
__global__ void __launch_bounds__(256) w4_dequantize_any_kernel(W4Args p, uint16_t *W) {
    using H = b2b::Half16<BF16>;
    const int lane = threadIdx.x & 31;
    const int64_t per = (p.pitch + 127) / 128;
    const int64_t step = static_cast<int64_t>(gridDim.x) * 8;
    const uint32_t half_group = static_cast<uint32_t>(p.group / 2);
    for (int64_t task = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); task < p.m * per; task += step) {
        const int64_t row = task / per;
        const uint32_t at0 = static_cast<uint32_t>(task % per) * 128 + lane;  // byte of the row
        int byte[4], zero[4];
        float s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t at = min(at0 + 32 * i, static_cast<uint32_t>(p.pitch - 1));
            const int64_t grp = row * p.gs + at / half_group;
            byte[i] = __ldg(p.packed + row * p.pitch + at);
            zero[i] = p.zeros ? __ldg(p.zeros + grp) & 15 : 8;
            s[i] = H::get(__ldg(p.scales + grp));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t at = at0 + 32 * i;
            uint16_t *w = W + row * p.n + 2 * at;
            const bool clamps = w4_clamps<BF16>(s[i]);
            if (2 * at < p.n) w[0] = w4_back<BF16>(s[i], clamps, (byte[i] & 15) - zero[i]);
            if (2 * at + 1 < p.n) w[1] = w4_back<BF16>(s[i], clamps, (byte[i] >> 4) - zero[i]);
        }
    }
}

W4Args w4_args(size_t m, size_t n, size_t group, const uint8_t *packed, const uint16_t *scales, const uint8_t *zeros) {
    const int64_t N = static_cast<int64_t>(n), G = static_cast<int64_t>(group);
    return W4Args{packed, scales, zeros, static_cast<int64_t>(m), N, G, (N + 1) / 2, (N + G - 1) / G};
}

unsigned ctas_for(b2b_handle *h, const void *kernel, int64_t blocks) {
    const int64_t most = b2b::resident_ctas(h, kernel, 256, 0);
    return static_cast<unsigned>(blocks < most ? blocks : most);
}

int launched(const char *what) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? B2B_OK : b2b::fail_cuda(e, what);
}

constexpr int kMaxSmem = 227 * 1024 - 1536;  // dynamic shared memory of the GEMV kernel, static beside it
constexpr int64_t kMaxXBytes = 80 * 1024;    // of its staged vectors where 8 CTAs share a tile; fewer may have more

// Its shared memory for KS CTAs a tile; sets the vectors' bytes.
size_t gemv_smem(GemvArgs &p, bool tma, int KS, int64_t local) {
    p.x_bytes = static_cast<int>(local * kBoxCols * p.width * 2);
    return p.x_bytes + 2 * (kWarps + (KS > 1 ? p.batch * p.parts : 0)) * kTileRows * p.width * 4 +
           kWarps * ((tma ? kBoxBytes : kHandBytes) + 8) + 16 + (p.index ? sizeof(Table) : 0) + 1024;
}

// Clusters of KS CTAs (1, 2, 4 or 8) of the GEMV kernel that are resident at
// once, asked once for each device: a CTA has an SM to itself by its registers,
// so neither its type nor its shared memory matters.
int resident_clusters(b2b_handle *h, const void *kernel, int KS) {
    static std::mutex mu;
    static int known[64][9];
    std::lock_guard<std::mutex> lock(mu);
    int &clusters = known[h->device & 63][KS];
    if (clusters == 0) {
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = KS;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(KS);
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = kMaxSmem;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess || clusters < 1) {
            cudaGetLastError();
            clusters = h->sm_count / KS;
        }
    }
    return clusters;
}

using QuantizeKernel = void (*)(const uint16_t *, uint8_t *, uint16_t *, uint8_t *, int64_t, int64_t, int64_t, int64_t);

template <bool BF16, bool WHOLE>
QuantizeKernel quantize_kernel(size_t group) {
    switch (group) {
        case 32: return w4_quantize_kernel<BF16, 2, WHOLE>;
        case 64: return w4_quantize_kernel<BF16, 4, WHOLE>;
        case 128: return w4_quantize_kernel<BF16, 8, WHOLE>;
        default: return w4_quantize_kernel<BF16, 16, WHOLE>;
    }
}

using GemvKernel = void (*)(CUtensorMap, GemvArgs);

template <bool BF16, bool ZEROS, bool HAND>
GemvKernel gemv_kernel(int spg) {
    switch (spg) {
        case 1: return w4_gemv_kernel<BF16, ZEROS, 1, HAND>;
        case 2: return w4_gemv_kernel<BF16, ZEROS, 2, HAND>;
        case 4: return w4_gemv_kernel<BF16, ZEROS, 4, HAND>;
        case 8: return w4_gemv_kernel<BF16, ZEROS, 8, HAND>;
        default: return w4_gemv_kernel<BF16, ZEROS, 0, true>;
    }
}

int launch_gemv(b2b_handle *h, bool bf16, int spg, bool tma, const CUtensorMap &tmW, GemvArgs &p) {
    const bool zeros = p.w.zeros != nullptr;
    auto pick = [&](auto hand) {
        constexpr bool HAND = decltype(hand)::value;
        return bf16 ? (zeros ? gemv_kernel<true, true, HAND>(spg) : gemv_kernel<true, false, HAND>(spg))
                    : (zeros ? gemv_kernel<false, true, HAND>(spg) : gemv_kernel<false, false, HAND>(spg));
    };
    const GemvKernel kernel = tma ? pick(std::false_type{}) : pick(std::true_type{});
    const void *fn = reinterpret_cast<const void *>(kernel);
    const int64_t cols = (p.w.n + kBoxCols - 1) / kBoxCols, tiles = (p.w.m + kTileRows - 1) / kTileRows;
    p.width = p.count < 8 ? p.count : 8;
    while (p.width > 1 && (cols + 7) / 8 * kBoxCols * p.width * 2 > kMaxXBytes) --p.width;
    if ((cols + 7) / 8 * kBoxCols * p.width * 2 > kMaxXBytes)
        return b2b::fail(B2B_ERR_NOT_SUPPORTED, "4-bit GEMV: rows longer than 327680 columns");
    // with an index: the matrices that it names, if it names them at random,
    // and their sets
    const int64_t count = p.count, full = (count + p.width - 1) / p.width;  // sets without an index
    double sets = static_cast<double>(full);
    if (p.index) {
        const double named = p.matrices * (1.0 - pow(1.0 - 1.0 / p.matrices, p.count));
        sets = named * ceil(p.count / named / p.width);
    }
    const int64_t all = static_cast<int64_t>(ceil(sets * static_cast<double>(tiles)));
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kThreads);
    cfg.stream = h->stream;
    cfg.attrs = attr;
    {
        static std::mutex mu;
        static bool ready[2][2][2][9][64];
        std::lock_guard<std::mutex> lock(mu);
        bool &done = ready[tma][bf16][zeros][spg][h->device & 63];
        if (!done) {
            const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
            if (e != cudaSuccess) return b2b::fail_cuda(e, "4-bit GEMV shared memory");
            done = true;
        }
    }
    // Share a tile's columns among KS CTAs of a cluster so that it takes least, in
    // boxes that a warp computes one after another (1.5 to 2 us): with its share of
    // the vectors to stage, a fifth of a box for 16 KB, and where KS > 1 a quarter
    // of one for the cluster and a fifth for each tile's joining.  It picks the
    // fastest KS of 1, 2, 4 and 8 or comes within 1 % of it for 12 measured
    // shapes: 16384 x 1024 takes 12.5 us by 1 and 22 by 4, 300 x 16384 13 and 7.7.
    GemvArgs best = p;
    int best_ks = 0;
    double best_time = 0;
    for (int KS = 1; KS <= 8 && (KS == 1 || KS < 2 * cols); KS *= 2) {
        const int64_t local = (cols + KS - 1) / KS, clusters = resident_clusters(h, fn, KS);
        auto fits = [&] { return gemv_smem(p, tma, KS, local) <= static_cast<size_t>(kMaxSmem); };
        p.parts = kWarps;
        p.batch = KS > 1 ? kMaxBatch : 1;
        while (p.batch > 1 && !fits()) p.batch /= 2;
        while (p.parts > 1 && !fits()) p.parts /= 2;
        if (!fits()) continue;
        int64_t left = (all + clusters - 1) / clusters;  // tiles of a cluster
        double time = 0.2 * static_cast<double>(local * p.width) / 32.0;
        if (KS > 1) time += 0.25 + 0.2 * static_cast<double>(left);
        for (int parts = p.parts; parts >= 1; parts /= 2) {  // rounds of as many tiles
            const int64_t kw = kWarps / parts;
            time += static_cast<double>(left / parts * ((local + kw - 1) / kw));
            left %= parts;
            if (left * local <= kWarps && left <= p.parts) {  // one round of what is left
                time += left > 0;
                break;
            }
        }
        if (!best_ks || time < best_time) {
            best = p;
            best_ks = KS;
            best_time = time;
        }
    }
    p = best;
    const int64_t local = (cols + best_ks - 1) / best_ks, clusters = resident_clusters(h, fn, best_ks);
    // an index may name more matrices than expected, but not more tiles than this
    const int64_t most = (p.index ? count : full) * tiles;
    attr[0].val.clusterDim.x = best_ks;
    cfg.dynamicSmemBytes = gemv_smem(p, tma, best_ks, local);
    cfg.numAttrs = best_ks > 1;
    cfg.gridDim = dim3(static_cast<unsigned>(best_ks * (most < clusters ? most : clusters)));
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tmW, p);
    return e == cudaSuccess ? B2B_OK : b2b::fail_cuda(e, "4-bit GEMV launch");
}

}  // namespace

namespace b2b {

int launch_quantize_w4(b2b_handle *h, int type, size_t m, size_t n, size_t group, const uint16_t *W, uint8_t *packed,
                       uint16_t *scales, uint8_t *zeros) {
    const W4Args p = w4_args(m, n, group, packed, scales, zeros);
    const bool bf16 = type == B2B_TYPE_BF16;
    const bool whole = n % 8 == 0 && aligned16(W) && (reinterpret_cast<uintptr_t>(packed) & 3) == 0;
    if (group == 32 || group == 64 || group == 128 || group == 256) {
        const QuantizeKernel kernel = bf16 ? (whole ? quantize_kernel<true, true>(group) : quantize_kernel<true, false>(group))
                                           : (whole ? quantize_kernel<false, true>(group) : quantize_kernel<false, false>(group));
        const int64_t tasks = p.m * ((p.gs * static_cast<int64_t>(group / 16) + 31) / 32);
        const unsigned ctas = ctas_for(h, reinterpret_cast<const void *>(kernel), (tasks + 7) / 8);
        kernel<<<ctas, 256, 0, h->stream>>>(W, packed, scales, zeros, p.m, p.n, p.pitch, p.gs);
    } else {
        auto kernel = whole ? (bf16 ? w4_quantize_any_kernel<true, true> : w4_quantize_any_kernel<false, true>)
                            : (bf16 ? w4_quantize_any_kernel<true, false> : w4_quantize_any_kernel<false, false>);
        const unsigned ctas = ctas_for(h, reinterpret_cast<const void *>(kernel), (p.m * p.gs + 7) / 8);
        kernel<<<ctas, 256, 0, h->stream>>>(W, packed, scales, zeros, p.m, p.n, p.group, p.pitch, p.gs);
    }
    return launched("4-bit quantisation launch");
}

int launch_dequantize_w4(b2b_handle *h, int type, size_t m, size_t n, size_t group, const uint8_t *packed,
                         const uint16_t *scales, const uint8_t *zeros, uint16_t *W) {
    const W4Args p = w4_args(m, n, group, packed, scales, zeros);
    const bool bf16 = type == B2B_TYPE_BF16;
    const bool whole = n % 8 == 0 && aligned16(W) && (reinterpret_cast<uintptr_t>(packed) & 3) == 0;
    auto kernel = whole ? (bf16 ? w4_dequantize_kernel<true> : w4_dequantize_kernel<false>)
                        : (bf16 ? w4_dequantize_any_kernel<true> : w4_dequantize_any_kernel<false>);
    const int64_t tasks = p.m * (whole ? (p.n / 8 + 63) / 64 : (p.pitch + 127) / 128);
    kernel<<<ctas_for(h, reinterpret_cast<const void *>(kernel), (tasks + 7) / 8), 256, 0, h->stream>>>(p, W);
    return launched("4-bit dequantisation launch");
}

int launch_hgemv_w4(b2b_handle *h, int type, size_t groups, size_t m, size_t n, size_t group, float alpha,
                    const uint8_t *packed, const uint16_t *scales, const uint8_t *zeros, const uint16_t *x,
                    size_t count, size_t fan, const int32_t *index, float beta, uint16_t *y) {
    GemvArgs p{};
    p.w = w4_args(m, n, group, packed, scales, zeros);
    p.x = x;
    p.index = index;
    p.y = y;
    p.status = h->d_status;
    p.wait_ns = h->wait_limit_ns;
    p.matrices = static_cast<int>(groups);
    p.fan = static_cast<int>(fan);
    p.alpha = alpha;
    p.beta = beta;
    const int64_t rows = static_cast<int64_t>(groups) * p.w.m;
    p.total = rows * p.w.pitch;
    const bool bf16 = type == B2B_TYPE_BF16;
    // steps of a group that divide a box's
    int spg = static_cast<int>(group / 32);
    if (spg % kBoxSteps == 0) spg = kBoxSteps;
    if (kBoxSteps % spg != 0) spg = 0;
    const bool tma = n % 32 == 0 && aligned16(packed) && rows < (1ll << 31) && spg != 0;
    CUtensorMap tmW{};
    if (tma) {
        if (int rc = encode_tma_2d(&tmW, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, packed, rows, p.w.pitch, kBoxCols / 2,
                                   kTileRows))
            return rc;
    }
    if (spg != 0) {
        const int64_t per = kBoxSteps / spg;  // groups of a box
        p.vec = p.w.gs % per == 0 && aligned16(scales) && aligned16(zeros);
    }
    const int64_t all = static_cast<int64_t>(count);
    for (int64_t first = 0; first < all; first += index ? kMaxIndexed : all) {
        p.first = static_cast<int>(first);
        p.count = static_cast<int>(index && all - first > kMaxIndexed ? kMaxIndexed : all - first);
        if (int rc = launch_gemv(h, bf16, spg, tma, tmW, p)) return rc;
    }
    return B2B_OK;
}

}  // namespace b2b

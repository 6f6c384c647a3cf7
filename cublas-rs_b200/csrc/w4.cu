// w4.cu -- matrices held in 4 bits with a scale (and a zero point) for each
// group of a row's columns: quantisation, the way back to 16 bits, and
// products with vectors.  No counterpart in cublas-rs, whose GEMVs
// (crates/cublas-l2/src/gemv.rs) read 16-, 32- and 64-bit matrices.
//
//   W[i][j] = scale[i][j / group] * (q[i][j] - zero[i][j / group])
//   y_i = alpha * W x_i + beta * y_i
#include <cuda_runtime.h>
#include <stdint.h>

#include "half_types.cuh"
#include "internal.h"

namespace {

struct W4Args {
    const uint8_t *packed;
    const uint16_t *scales;
    const uint8_t *zeros;  // nullptr: 8 everywhere
    int64_t m, n, group, pitch, gs;  // pitch = bytes of a packed row, gs = groups of a row
};

__device__ __forceinline__ int w4_value(const W4Args &p, int64_t row, int64_t j) {
    const int byte = p.packed[row * p.pitch + j / 2];
    const int zero = p.zeros ? p.zeros[row * p.gs + j / p.group] & 15 : 8;
    return ((j & 1) ? byte >> 4 : byte & 15) - zero;
}

// One warp a group of a row.  All arithmetic that decides a value is f32 on
// the scale rounded to 16 bits.  The quotient w / s that rounds to a value is
// of two numbers with at most 11 significant bits: unless it lies exactly on
// the border between two values it is at least 2^-12 away from it, so f32's
// rounding decides as exact arithmetic would.
template <bool BF16>
__global__ void __launch_bounds__(256) w4_quantize_kernel(const uint16_t *W, uint8_t *packed, uint16_t *scales,
                                                          uint8_t *zeros, int64_t m, int64_t n, int64_t group,
                                                          int64_t pitch, int64_t gs) {
    using H = b2b::Half16<BF16>;
    const int lane = threadIdx.x & 31;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * 8;
    for (int64_t at = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); at < m * gs; at += warps) {
        const int64_t row = at / gs, j0 = at % gs * group;
        const int64_t j1 = j0 + group < n ? j0 + group : n;
        float lo = 0.0f, hi = 0.0f;
        bool finite = true;
        for (int64_t j = j0 + lane; j < j1; j += 32) {
            const float w = H::get(W[row * n + j]);
            finite = finite && isfinite(w);
            lo = fminf(lo, w);
            hi = fmaxf(hi, w);
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
        }
        finite = __all_sync(0xffffffffu, finite);
        // halves, so that hi - lo of bf16 extremes stays finite
        float s = zeros ? __fdiv_rn(0.5f * hi - 0.5f * lo, 7.5f) : __fdiv_rn(fmaxf(hi, -lo), 7.0f);
        const uint16_t s16 = H::put(finite ? s : __int_as_float(0x7fffffff));
        s = H::get(s16);
        const bool live = s > 0.0f;  // false for a NaN scale too
        float zero = 8.0f;
        if (zeros) zero = live ? fminf(rintf(__fdiv_rn(-lo, s)), 15.0f) : 0.0f;
        if (lane == 0) {
            scales[at] = s16;
            if (zeros) zeros[at] = static_cast<uint8_t>(zero);
        }
        for (int64_t j = j0 + 2 * lane; j < j1; j += 64) {
            uint32_t byte = 0;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (j + e >= j1) continue;
                float q = zero;
                if (live) q = fminf(fmaxf(rintf(__fdiv_rn(H::get(W[row * n + j + e]), s)) + zero, 0.0f), 15.0f);
                byte |= static_cast<uint32_t>(q) << (4 * e);
            }
            packed[row * pitch + j / 2] = static_cast<uint8_t>(byte);
        }
    }
}

template <bool BF16>
__global__ void __launch_bounds__(256) w4_dequantize_kernel(W4Args p, uint16_t *W) {
    using H = b2b::Half16<BF16>;
    const int64_t total = p.m * p.n, step = static_cast<int64_t>(gridDim.x) * 256;
    for (int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; at < total; at += step) {
        const int64_t row = at / p.n, j = at % p.n;
        // 11 bits times 5: exact in f32, rounded once
        const float v = H::get(p.scales[row * p.gs + j / p.group]) * static_cast<float>(w4_value(p, row, j));
        W[at] = H::put(v > H::kMax ? H::kMax : v < -H::kMax ? -H::kMax : v);
    }
}

// One warp a row and product.
template <bool BF16>
__global__ void __launch_bounds__(256)
    w4_gemv_kernel(W4Args p, int64_t matrices, const uint16_t *x, int64_t count, int64_t fan, const int32_t *index,
                   float alpha, float beta, uint16_t *y) {
    using H = b2b::Half16<BF16>;
    const int lane = threadIdx.x & 31;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * 8;
    for (int64_t at = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); at < count * p.m; at += warps) {
        const int64_t i = at / p.m, e = index ? index[i] : 0;
        float sum = 0.0f;
        if (e >= 0 && e < matrices) {
            const int64_t row = e * p.m + at % p.m;
            for (int64_t j = lane; j < p.n; j += 32)
                sum = fmaf(H::get(p.scales[row * p.gs + j / p.group]) * static_cast<float>(w4_value(p, row, j)),
                           H::get(x[i / fan * p.n + j]), sum);
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == 0) {
            float v = e >= 0 && e < matrices ? alpha * sum : 0.0f;
            if (beta != 0.0f) v = fmaf(beta, H::get(y[at]), v);
            y[at] = H::put(v);
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

}  // namespace

namespace b2b {

int launch_quantize_w4(b2b_handle *h, int type, size_t m, size_t n, size_t group, const uint16_t *W, uint8_t *packed,
                       uint16_t *scales, uint8_t *zeros) {
    const W4Args p = w4_args(m, n, group, packed, scales, zeros);
    auto kernel = type == B2B_TYPE_BF16 ? w4_quantize_kernel<true> : w4_quantize_kernel<false>;
    const unsigned ctas = ctas_for(h, reinterpret_cast<const void *>(kernel), (p.m * p.gs + 7) / 8);
    kernel<<<ctas, 256, 0, h->stream>>>(W, packed, scales, zeros, p.m, p.n, p.group, p.pitch, p.gs);
    return launched("4-bit quantisation launch");
}

int launch_dequantize_w4(b2b_handle *h, int type, size_t m, size_t n, size_t group, const uint8_t *packed,
                         const uint16_t *scales, const uint8_t *zeros, uint16_t *W) {
    const W4Args p = w4_args(m, n, group, packed, scales, zeros);
    auto kernel = type == B2B_TYPE_BF16 ? w4_dequantize_kernel<true> : w4_dequantize_kernel<false>;
    kernel<<<ctas_for(h, reinterpret_cast<const void *>(kernel), (p.m * p.n + 255) / 256), 256, 0, h->stream>>>(p, W);
    return launched("4-bit dequantisation launch");
}

int launch_hgemv_w4(b2b_handle *h, int type, size_t groups, size_t m, size_t n, size_t group, float alpha,
                    const uint8_t *packed, const uint16_t *scales, const uint8_t *zeros, const uint16_t *x,
                    size_t count, size_t fan, const int32_t *index, float beta, uint16_t *y) {
    const W4Args p = w4_args(m, n, group, packed, scales, zeros);
    const int64_t products = static_cast<int64_t>(count);
    auto kernel = type == B2B_TYPE_BF16 ? w4_gemv_kernel<true> : w4_gemv_kernel<false>;
    const unsigned ctas = ctas_for(h, reinterpret_cast<const void *>(kernel), (p.m * products + 7) / 8);
    kernel<<<ctas, 256, 0, h->stream>>>(p, static_cast<int64_t>(groups), x, products, static_cast<int64_t>(fan),
                                        index, alpha, beta, y);
    return launched("4-bit GEMV launch");
}

}  // namespace b2b

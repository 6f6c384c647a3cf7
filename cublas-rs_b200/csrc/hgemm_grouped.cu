// hgemm_grouped.cu -- matrix products of ragged row groups: the products of
// an expert layer whose tokens are sorted by expert.  No counterpart in
// cublas-rs, whose batched family (crates/cublas-l3/src/batched.rs) takes one
// size for every matrix of a batch.
//
//   forward   C[r] = alpha * A[r] op(B_g) + beta * C[r],  r in group g
//   wgrad     C_g = alpha * A[rows of g]^T B[rows of g] + beta * C_g
//
// 16-bit operands (f16 or bf16), f32 sums.
#include <cuda_runtime.h>
#include <stdint.h>

#include "half_types.cuh"
#include "internal.h"

namespace {

constexpr int kMaxGroups = 1024;

// One product of every group, addressed by strides: within group g, sum over
// kk of A(i, kk) * B(kk, j) for M x N outputs.
struct GroupedArgs {
    const uint16_t *A, *B;
    void *C;
    const int32_t *offsets;
    int *status;
    int groups;
    int64_t rows;    // rows of A (and of C, or of B in wgrad)
    int64_t M, N, K; // M is the group's row count in forward, K in wgrad
    int64_t a_i, a_k, b_k, b_j;
    float alpha, beta;
};

// Tiles of `bm` rows that groups 0..g-1 hold, for g = 0..groups, in
// start[0..groups]; false when the offsets do not ascend within [0, rows].
// One warp; every lane returns the verdict.
__device__ bool scan_groups(const int32_t *offsets, int groups, int64_t rows, int bm, int *start) {
    const int lane = threadIdx.x & 31;
    bool ok = true;
    int carry = 0;
    for (int g0 = 0; g0 < groups; g0 += 32) {
        const int g = g0 + lane;
        int tiles = 0;
        if (g < groups) {
            const int64_t lo = offsets[g], hi = offsets[g + 1];
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

// 64 x 64 tiles, 4 x 4 outputs a thread, f32 sums: right for every size,
// stride and alignment.
template <bool BF16, bool WGRAD, bool F32>
__global__ void __launch_bounds__(256) grouped_simt_kernel(GroupedArgs p) {
    using H = b2b::Half16<BF16>;
    __shared__ float As[16][64 + 4];
    __shared__ float Bs[16][64 + 4];
    __shared__ int start[kMaxGroups + 1];
    __shared__ int valid;
    const int tid = threadIdx.x;
    if (tid < 32) {
        const bool ok = scan_groups(p.offsets, p.groups, p.rows, 64, start);
        if (tid == 0) {
            valid = ok;
            if (!ok) atomicCAS(p.status, 0, B2B_DEVSTAT_OFFSETS);
        }
    }
    __syncthreads();
    if (!valid) return;
    const int tx = tid & 15, ty = tid >> 4;
    const int64_t tiles_n = (p.N + 63) / 64;
    const int64_t tiles_m = (p.M + 63) / 64;  // wgrad
    const int64_t tiles = WGRAD ? p.groups * tiles_m * tiles_n : start[p.groups] * tiles_n;
    int g = 0;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        int64_t m0;
        const int64_t n0 = t % tiles_n * 64;
        if (WGRAD) {
            g = static_cast<int>(t / (tiles_m * tiles_n));
            m0 = t / tiles_n % tiles_m * 64;
        } else {
            while (t / tiles_n >= start[g + 1]) ++g;
            m0 = (t / tiles_n - start[g]) * 64;
        }
        const int64_t row0 = p.offsets[g], count = p.offsets[g + 1] - row0;
        const int64_t M = WGRAD ? p.M : count, K = WGRAD ? count : p.K;
        const uint16_t *A = p.A + (WGRAD ? row0 * p.a_k : row0 * p.a_i);
        const uint16_t *B = p.B + (WGRAD ? row0 * p.b_k : g * p.N * p.K);
        const int64_t c0 = WGRAD ? g * p.M * p.N : row0 * p.N;
        float acc[4][4] = {};
        for (int64_t k0 = 0; k0 < K; k0 += 16) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int idx = tid + i * 256;
                const int r = idx & 63, kc = idx >> 6;
                const int64_t kk = k0 + kc;
                As[kc][r] = m0 + r < M && kk < K ? H::get(A[(m0 + r) * p.a_i + kk * p.a_k]) : 0.0f;
                Bs[kc][r] = n0 + r < p.N && kk < K ? H::get(B[(n0 + r) * p.b_j + kk * p.b_k]) : 0.0f;
            }
            __syncthreads();
#pragma unroll
            for (int kk = 0; kk < 16; ++kk)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        acc[i][j] = fmaf(As[kk][ty * 4 + i], Bs[kk][tx * 4 + j], acc[i][j]);
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (m0 + ty * 4 + i >= M) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (n0 + tx * 4 + j >= p.N) continue;
                const int64_t at = c0 + (m0 + ty * 4 + i) * p.N + n0 + tx * 4 + j;
                float v = K ? p.alpha * acc[i][j] : 0.0f;
                if constexpr (F32) {
                    float *C = static_cast<float *>(p.C);
                    C[at] = p.beta != 0.0f ? fmaf(p.beta, C[at], v) : v;
                } else {
                    uint16_t *C = static_cast<uint16_t *>(p.C);
                    if (p.beta != 0.0f) v = fmaf(p.beta, H::get(C[at]), v);
                    C[at] = H::put(v);
                }
            }
        }
    }
}

template <bool WGRAD, bool F32>
int launch_simt(b2b_handle *h, int type, const GroupedArgs &p) {
    auto kernel = type == B2B_TYPE_BF16 ? grouped_simt_kernel<true, WGRAD, F32> : grouped_simt_kernel<false, WGRAD, F32>;
    const int ctas = b2b::resident_ctas(h, reinterpret_cast<const void *>(kernel), 256, 0);
    kernel<<<ctas, 256, 0, h->stream>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? B2B_OK : b2b::fail_cuda(e, "grouped HGEMM launch");
}

}  // namespace

namespace b2b {

int launch_hgemm_grouped(b2b_handle *h, int type, int trans_b, size_t groups, size_t rows, size_t n, size_t k,
                         float alpha, const uint16_t *A, const uint16_t *B, float beta, uint16_t *C,
                         const int32_t *offsets) {
    const int64_t N = static_cast<int64_t>(n), K = static_cast<int64_t>(k);
    const GroupedArgs p{A, B, C, offsets, h->d_status, static_cast<int>(groups), static_cast<int64_t>(rows), 0, N, K,
                        K, 1, trans_b ? 1 : N, trans_b ? K : 1, alpha, beta};
    return launch_simt<false, false>(h, type, p);
}

int launch_hgemm_grouped_wgrad(b2b_handle *h, int type, int c_type, size_t groups, size_t rows, size_t m, size_t n,
                               float alpha, const uint16_t *A, const uint16_t *B, float beta, void *C,
                               const int32_t *offsets) {
    const int64_t M = static_cast<int64_t>(m), N = static_cast<int64_t>(n);
    const GroupedArgs p{A, B, C, offsets, h->d_status, static_cast<int>(groups), static_cast<int64_t>(rows), M, N, 0,
                        1, M, N, 1, alpha, beta};
    return c_type == B2B_TYPE_F32 ? launch_simt<true, true>(h, type, p) : launch_simt<true, false>(h, type, p);
}

}  // namespace b2b

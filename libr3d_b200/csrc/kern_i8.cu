/* kern_i8.cu -- gemm_nt_q @ i8a8, any shape and any alignment: y[m, n] = (sum_k a[m, k] b[n, k] * sa[m]) * sb[n].
 *
 * The sum is exact in 32-bit integers (K <= 131071), so its order is free and every arm of this band gives the same
 * bits. 64 tokens x 64 channels a block, 64 of K at a time in shared memory as four-byte words, dp4a; a thread owns
 * 4 x 4 outputs. Serves operands that TMA cannot take (rows off the 16-byte grid). Bound by its own instructions, far
 * below the tensor-core arms: with K = 5121 instead of 5120, 16 x 27648 takes 369 us for 24, 128 x 5120 321 for 11.4, 2048 x
 * 5120 1830 for 39; 1 x 4096, K = 4097, 204 for 6.6. Rows padded to 16 bytes keep a caller off it.
 */
#include "r3d_kernels.h"
#include "r3d_numerics.cuh"

namespace r3d {

namespace {

constexpr int kT = 64;                 /* tokens, channels and K bytes of a step */

__device__ __forceinline__ uint32_t load4(const int8_t* row, int k, int K, bool words) {
    if (words && k + 4 <= K) return *(const uint32_t*)(row + k);
    uint32_t v = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) if (k + j < K) v |= (uint32_t)(uint8_t)row[k + j] << (8 * j);
    return v;
}

__global__ void __launch_bounds__(256) k_i8_tile(const R3dGemmI8 P, const int a_words, const int b_words) {
    __shared__ uint32_t sa[kT][kT / 4 + 1], sb[kT][kT / 4 + 1];
    const int n0 = blockIdx.x * kT, m0 = blockIdx.y * kT;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < P.k; k0 += kT) {
        for (int i = threadIdx.x; i < kT * kT / 4; i += 256) {
            const int r = i >> 4, c = i & 15;
            sa[r][c] = m0 + r < P.m ? load4((const int8_t*)P.a + (int64_t)(m0 + r) * P.a_pitch, k0 + 4 * c, P.k, a_words) : 0u;
            sb[r][c] = n0 + r < P.n ? load4((const int8_t*)P.b + (int64_t)(n0 + r) * P.b_pitch, k0 + 4 * c, P.k, b_words) : 0u;
        }
        __syncthreads();
#pragma unroll 4
        for (int c = 0; c < kT / 4; ++c) {
            int av[4], bv[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) { av[j] = (int)sa[ty + 16 * j][c]; bv[j] = (int)sb[tx + 16 * j][c]; }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(av[i], bv[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = m0 + ty + 16 * i;
        if (m >= P.m) continue;
        const float s = P.a_scale[(int64_t)m * P.as_pitch];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + tx + 16 * j;
            if (n >= P.n) continue;
            const int64_t at = (int64_t)n * P.bs_pitch;
            const float t = P.bs_dtype == RAD_F32 ? ((const float*)P.b_scale)[at] : bf16_to_f32(((const uint16_t*)P.b_scale)[at]);
            if (P.y_dtype == RAD_F32) ((float*)P.y)[(int64_t)m * P.y_pitch + n] = scaled_once(acc[i][j], s, t);
            else ((uint16_t*)P.y)[(int64_t)m * P.y_pitch + n] = f32_to_bf16(__fmul_rn(__fmul_rn((float)acc[i][j], s), t));
        }
    }
}

bool words_ok(const void* p, int64_t pitch) { return (((uintptr_t)p | (uintptr_t)pitch) & 3) == 0; }

} /* namespace */

int i8_tile(const R3dGemmI8& p, cudaStream_t st) {
    /* blockIdx.y ends at 65535: longer batches in parts */
    const int part = 65535 * kT;
    for (int m0 = 0; m0 < p.m; m0 += part) {
        R3dGemmI8 c = p;
        c.m = p.m - m0 < part ? p.m - m0 : part;
        c.a = (const int8_t*)p.a + (int64_t)m0 * p.a_pitch;
        c.a_scale = p.a_scale + (int64_t)m0 * p.as_pitch;
        c.y = (char*)p.y + (int64_t)m0 * p.y_pitch * (p.y_dtype == RAD_F32 ? 4 : 2);
        count_launch();
        k_i8_tile<<<dim3((unsigned)((c.n + kT - 1) / kT), (unsigned)((c.m + kT - 1) / kT)), 256, 0, st>>>(
            c, words_ok(c.a, c.a_pitch), words_ok(c.b, c.b_pitch));
    }
    return cudaGetLastError() == cudaSuccess ? RAD_OK : RAD_E_DEVICE;
}

} /* namespace r3d */

/* kern_token_i8.cu -- the activation producers of the int8 band: one scale per token, int8 codes.
 *
 *   quant     h = x
 *   gated     h = silu(gate) * up, or sigmoid(gate) * up
 *   rmsnorm   r = x (+ residual, narrowed to the residual's type and stored back);
 *             h = (r * 1/sqrt(mean(r^2) + eps)) * (w + wadd)
 *   all       amax = max |h|; scale = amax / 127; code = rint(h * (127 / amax)).
 *
 * h stays in f32 from the operands to the code: it is rounded once, to eight bits. A row of zeros (amax below
 * 2^-100, where 127 / amax would overflow) has scale 1 and codes 0; a NaN or an infinity in a row makes its scale
 * NaN or infinite, so it reaches the product's output, and the codes of what cannot be scaled are 0.
 *
 * Bound by memory: x is read once (rmsnorm also reads and writes the residual), one byte a value is written. So a
 * block owns a row and keeps it in registers between the reduction and the codes.
 */
#include <cmath>
#include "r3d_kernels.h"
#include "r3d_numerics.cuh"

namespace r3d {

namespace {

enum { kQuant = 0, kSilu = 1, kSigmoid = 2, kRms = 3 };

struct TokenI8 {
    const void* x; int64_t x_pitch;
    void* res; int64_t r_pitch;
    const void* w; int w_f32;
    int8_t* q; int64_t q_pitch;
    float* scale; int64_t s_pitch;
    void* ob; int ob_f32; int64_t ob_pitch;
    int n;
    float eps, wadd;
};

__device__ __forceinline__ float ld1(const float* p) { return *p; }
__device__ __forceinline__ float ld1(const uint16_t* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ float narrow(float v, const float*) { return v; }
__device__ __forceinline__ float narrow(float v, const uint16_t*) { return bf16_to_f32(f32_to_bf16(v)); }
__device__ __forceinline__ void st1(float* p, float v) { *p = v; }
__device__ __forceinline__ void st1(uint16_t* p, float v) { *p = f32_to_bf16(v); }

/* max that keeps a NaN: the larger bit pattern of two non-negative floats is the larger value, NaN above all */
__device__ __forceinline__ float max_nan(float a, float b) {
    return __uint_as_float(max(__float_as_uint(a) & 0x7fffffffu, __float_as_uint(b) & 0x7fffffffu));
}

template <typename F>
__device__ __forceinline__ float block_reduce(float v, float* part, F f) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[0];
    for (int i = 1; i < warps; ++i) v = f(v, part[i]);
    __syncthreads();
    return v;
}

template <int KIND, typename T>
__device__ __forceinline__ float value_of(const TokenI8& P, int64_t row, int i, float rs) {
    const T* x = (const T*)P.x + row * P.x_pitch;
    if (KIND == kQuant) return ld1(x + i);
    if (KIND == kRms) {
        const float v = P.res ? ld1((const T*)P.res + row * P.r_pitch + i) : ld1(x + i);
        const float w = P.w_f32 ? ((const float*)P.w)[i] : bf16_to_f32(((const uint16_t*)P.w)[i]);
        return v * rs * (w + P.wadd);
    }
    const float g = ld1(x + i), u = ld1(x + P.n + i);
    const float s = __fdividef(1.0f, 1.0f + __expf(-g));
    return (KIND == kSilu ? g * s : s) * u;
}

/* any width, any alignment: the row is read again for each of the passes (it stays in the caches) */
template <int KIND, typename T>
__global__ void __launch_bounds__(512) k_token_i8(const TokenI8 P) {
    __shared__ float part[16];
    const int64_t row = blockIdx.x;
    float rs = 0.0f;
    if (KIND == kRms) {
        const T* x = (const T*)P.x + row * P.x_pitch;
        T* r = P.res ? (T*)P.res + row * P.r_pitch : nullptr;
        float ss = 0.0f;
        for (int i = threadIdx.x; i < P.n; i += blockDim.x) {
            float v = ld1(x + i);
            if (r) { v = narrow(v + ld1(r + i), r); st1(r + i, v); }
            ss = fmaf(v, v, ss);
        }
        ss = block_reduce(ss, part, [](float a, float b) { return a + b; });
        rs = 1.0f / sqrtf(ss / (float)P.n + P.eps);
    }
    float amax = 0.0f;
    for (int i = threadIdx.x; i < P.n; i += blockDim.x) amax = max_nan(amax, value_of<KIND, T>(P, row, i, rs));
    amax = block_reduce(amax, part, max_nan);
    const bool zero = amax < 0x1p-100f;
    const float step = zero ? 0.0f : 127.0f / amax;
    if (threadIdx.x == 0) P.scale[row * P.s_pitch] = zero ? 1.0f : amax / 127.0f;
    for (int i = threadIdx.x; i < P.n; i += blockDim.x) {
        const float h = value_of<KIND, T>(P, row, i, rs);
        P.q[row * P.q_pitch + i] = (int8_t)max(-127, min(127, __float2int_rn(h * step)));
        if (P.ob) {
            if (P.ob_f32) ((float*)P.ob)[row * P.ob_pitch + i] = h;
            else ((uint16_t*)P.ob)[row * P.ob_pitch + i] = f32_to_bf16(h);
        }
    }
}

template <int KIND>
int launch_kind(const TokenI8& P, int x_f32, int rows, cudaStream_t st) {
    const int t = P.n >= 512 ? 512 : (P.n + 31) / 32 * 32;
    count_launch();
    if (x_f32) k_token_i8<KIND, float><<<(unsigned)rows, t, 0, st>>>(P);
    else k_token_i8<KIND, uint16_t><<<(unsigned)rows, t, 0, st>>>(P);
    return cudaGetLastError() == cudaSuccess ? RAD_OK : RAD_E_DEVICE;
}

} /* namespace */

int launch_token_i8(const R3dTokenI8& p, cudaStream_t st) {
    TokenI8 P{};
    P.x = p.x; P.x_pitch = p.x_pitch; P.res = p.residual; P.r_pitch = p.r_pitch;
    P.w = p.w; P.w_f32 = p.w_dtype == RAD_F32;
    P.q = (int8_t*)p.q; P.q_pitch = p.q_pitch; P.scale = p.scale; P.s_pitch = p.s_pitch;
    P.ob = p.out; P.ob_f32 = p.out_dtype == RAD_F32; P.ob_pitch = p.out_pitch;
    P.n = p.n; P.eps = p.eps; P.wadd = p.wadd;
    const int f32 = p.x_dtype == RAD_F32;
    switch (p.kind) {
        case R3D_TOKEN_QUANT:   return launch_kind<kQuant>(P, f32, p.rows, st);
        case R3D_TOKEN_SILU:    return launch_kind<kSilu>(P, f32, p.rows, st);
        case R3D_TOKEN_SIGMOID: return launch_kind<kSigmoid>(P, f32, p.rows, st);
        case R3D_TOKEN_RMSNORM: return launch_kind<kRms>(P, f32, p.rows, st);
    }
    return RAD_E_INVAL;
}

} /* namespace r3d */

/* kern_token_i8.cu -- the activation producers of the int8 band: one scale per token, int8 codes.
 *
 *   quant     h = x
 *   gated     h = silu(gate) * up, or sigmoid(gate) * up
 *   rmsnorm   r = x (+ residual, narrowed to the residual's type and stored back);
 *             h = (r * 1/sqrt(mean(r^2) + eps)) * (w + wadd)
 *   all       amax = max |h|; scale = amax / 127; code = rint(h * 127 / amax), halves to even.
 *
 * h stays in f32 from the operands to the code: it is rounded once, to eight bits. A row of zeros (amax below
 * 2^-100, before 127 / amax comes near the end of f32) has scale 1 and codes 0; a NaN or an infinity in a row makes its scale
 * NaN or infinite, so it reaches the product's output, and the codes of what cannot be scaled are 0.
 *
 * Bound by memory: x is read once (rmsnorm also reads and writes the residual), one byte a value is written. So a
 * block walks rows and keeps a row's h in registers between the reduction and the codes: k_token_i8_regs, chunks of eight
 * values on the codes' 8-byte grid. Each operand whose chunks lie on the 16-byte grid is copied ahead by cp.async, whatever
 * the others do; gated halves off it, and a norm's w off it beside f32 rows, are read by the 16-byte words around them, a
 * row's ends (and the other operands off the grid) one value at a time. The sum of a norm's squares follows the chunks and
 * the threads, so its last bit depends on how many rows a call has and on where they begin. Rows of more than 32760 values,
 * or of f32 values and two streams beyond 27648, which the shared memory does not hold, are read again for each step.
 */
#include <atomic>
#include <cmath>
#include "r3d_kernels.h"
#include "r3d_numerics.cuh"

namespace r3d {

bool tc_pdl_on();                     /* kern_tc.cu: false under R3D_NO_PDL */
int tc_sm_count();

namespace {

/* the next kernel may begin to launch (`early`: a row a block; among many rows its blocks only took room, 8192 x 5120 norm 53.5
 * instead of 51.3 us, while 3 x 6144 codes go from 2.2 to 1.8); the previous one's results are there, and all reads and writes
 * come behind this */
__device__ __forceinline__ void in_turn(bool early) {
    if (early) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
template <typename... P, typename... A>
cudaError_t launch_in_turn(void (*kernel)(P...), unsigned grid, unsigned threads, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid); cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at; cfg.numAttrs = tc_pdl_on() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

enum { kQuant = 0, kSilu = 1, kSigmoid = 2, kRms = 3 };

struct TokenI8 {
    const void* x; int64_t x_pitch;
    void* res; int64_t r_pitch;
    const void* w; int w_f32;
    int8_t* q; int64_t q_pitch;
    float* scale; int64_t s_pitch;
    void* ob; int ob_f32; int64_t ob_pitch;
    int n, rows;
    float eps, wadd;
};

__device__ __forceinline__ float ld1(const float* p) { return *p; }
__device__ __forceinline__ float ld1(const uint16_t* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ float narrow(float v, const float*) { return v; }
__device__ __forceinline__ float narrow(float v, const uint16_t*) { return bf16_to_f32(f32_to_bf16(v)); }
__device__ __forceinline__ void st1(float* p, float v) { *p = v; }
__device__ __forceinline__ void st1(uint16_t* p, float v) { *p = f32_to_bf16(v); }

__device__ __forceinline__ float max_nan(float a, float b) {          /* keeps a NaN */
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_size_nan(float a, float b, float c) {      /* of their sizes */
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
/* two values an instruction */
using f2 = unsigned long long;
__device__ __forceinline__ f2 two_of(float a, float b) { f2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void parts_of(f2 v, float* f) { asm("mov.b64 {%0, %1}, %2;" : "=f"(f[0]), "=f"(f[1]) : "l"(v)); }
__device__ __forceinline__ f2 add2(f2 a, f2 b) { f2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) { f2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) { f2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }

/* over the block, the same in every thread; every warp finishes it by itself (one warp doing so for all, the quotients
 * behind it included, saves a tenth of the instructions and waits longer: 54.5 instead of 51.2 us for 8192 x 5120) */
template <typename F>
__device__ __forceinline__ float block_reduce(float v, float* part, F f) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < warps ? part[lane] : 0.0f;                          /* 0 is neutral for both: a sum, a largest size */
#pragma unroll
    for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

/* The code of h is the low byte of h * step + kCode, kCode = 1.5 * 2^23: the whole number next to it, halves to even.
 * A row of zeros, and one so small that 127 / amax is not a number of this type, has step 0: codes 0. So has a row with a NaN
 * or an infinity in it.
 * h of eight bits (bf16 rows as they are): step is 127 / amax rounded up, and the sum rounds once. h * step is never below the
 * quotient it stands for, so that h = amax / 2, where that is 63.5 exactly, goes to the even 64 whatever amax is (rounded to
 * nearest, the step of 66 of the 128 significands that amax has in bf16 is low, and their halves went to 63). Among quotients
 * of two bf16 numbers there is no other half, save where the step is exact (amax = 127 2^n), and what is not a half lies
 * further from one than the step's error: the codes are the quotients' own.
 * Other h: quotients lie anywhere, so the step goes on with what its rounding left, and h * step is off by its own rounding
 * alone, a quarter of what the step rounded up leaves on average; halves stay halves. (8192 x 5120 norm: 14 codes of a
 * million are not the 64-bit quotient's, with the step rounded up 25, 16 by plain f32 operations.) Not for the gated
 * product, whose own roundings are ten times the step's (8192 x 13824 101 us instead of 97). */
constexpr float kCode = 12582912.0f;

__device__ __forceinline__ bool has_step(float amax) { return amax >= 0x1p-100f && amax < INFINITY; }
template <int KIND, typename T> constexpr bool kShortStep = KIND != kRms && (KIND != kQuant || sizeof(T) == 2);
template <bool SHORT> struct Step;
template <> struct Step<true> {
    float s;
    __device__ __forceinline__ explicit Step(float amax) : s(0.0f) {
        if (!has_step(amax)) return;
        s = 127.0f / amax;
        if (fmaf(s, amax, -127.0f) < 0.0f) s = __uint_as_float(__float_as_uint(s) + 1u);      /* the residual's sign is exact */
    }
    __device__ __forceinline__ f2 codes(f2 h) const { return fma2(h, two_of(s, s), two_of(kCode, kCode)); }
};
template <> struct Step<false> {
    float s, rest;
    __device__ __forceinline__ explicit Step(float amax) : s(0.0f), rest(0.0f) {
        if (!has_step(amax)) return;
        s = 127.0f / amax;
        rest = fmaf(-s, amax, 127.0f) * (s * (1.0f / 127.0f));
    }
    __device__ __forceinline__ f2 codes(f2 h) const {
        return add2(fma2(h, two_of(s, s), mul2(h, two_of(rest, rest))), two_of(kCode, kCode));
    }
};
__device__ __forceinline__ float scale_of(float amax) { return amax < 0x1p-100f ? 1.0f : amax / 127.0f; }

/* silu(g) * u or sigmoid(g) * u; the exponential and the quotient by the special-function unit (2^-22 and 2^-23 of their
 * results). An argument -g log2 e rounded to f32 would be off by up to 2^-25 of itself, and the exponential by 1.2 |g| units
 * in the last place for it. So the exponential is of an argument that is known exactly, and what it lacks follows as a factor
 * 1 + d. SHORT, g of eight bits: its product with the first 16 bits of log2 e is exact, d = -g ln 2 times the other bits
 * (at most 5e-4 before the sigmoid is 0; d^2 / 2 is left out). Else the product's rounding error is found by a multiply-add
 * (for g of eight bits, too, that took 5 % more for 8192 x 13824). Where d is infinite or not a number the exponential is 0
 * or infinite and has to stay so: the factor is held on the side of 1 that it leaves there. */
template <int KIND, bool SHORT>
__device__ __forceinline__ f2 gate2(f2 g, f2 u) {
    const f2 one = two_of(1.0f, 1.0f);
    const float log2e = SHORT ? 1.442687988f : 1.44269502f;       /* 47274 / 2^15; the nearest f32 */
    const f2 t = mul2(g, two_of(-log2e, -log2e));
    float e[2], f[2];
    parts_of(t, e);
#pragma unroll
    for (int i = 0; i < 2; ++i) asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e[i]));
    if (SHORT) parts_of(fma2(g, two_of(-4.88849515e-6f, -4.88849515e-6f), one), f);
    else {
        const f2 d = fma2(g, two_of(1.92596299e-8f, 1.92596299e-8f), fma2(g, two_of(log2e, log2e), t));
        parts_of(fma2(d, two_of(-0.693147182f, -0.693147182f), one), f);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) f[i] = SHORT ? fmaxf(f[i], 0.5f) : fminf(f[i], 2.0f);
    parts_of(fma2(two_of(e[0], e[1]), two_of(f[0], f[1]), one), e);
#pragma unroll
    for (int i = 0; i < 2; ++i) asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e[i]));
    const f2 s = two_of(e[0], e[1]);
    return mul2(KIND == kSilu ? mul2(g, s) : s, u);
}
template <int KIND, bool SHORT>
__device__ __forceinline__ float gate(float g, float u) {
    float f[2];
    parts_of(gate2<KIND, SHORT>(two_of(g, 0.0f), two_of(u, 0.0f)), f);
    return f[0];
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
    return gate<KIND, sizeof(T) == 2>(ld1(x + i), ld1(x + P.n + i));
}

/* Eight neighbouring values as they lie in memory. */
template <typename T> struct Raw;
template <> struct Raw<uint16_t> {
    uint32_t w[4];
    __device__ __forceinline__ void get(const uint16_t* p) { const uint4 v = *(const uint4*)p; w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
    /* from any element on: the 16-byte words that hold some of the eight, moved down by the elements in front */
    __device__ __forceinline__ void get_off(const uint16_t* p) {
        const uint4* const q = (const uint4*)((uintptr_t)p & ~(uintptr_t)15);
        const uint4 a = q[0], b = q[1];
        const int d = (int)((uintptr_t)p & 15) >> 1;
        uint32_t v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 6; ++i) v[i] = d & 4 ? v[i + 2] : v[i];
#pragma unroll
        for (int i = 0; i < 5; ++i) v[i] = d & 2 ? v[i + 1] : v[i];
        const uint32_t take = d & 1 ? 0x5432 : 0x3210;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __byte_perm(v[i], v[i + 1], take);
    }
    __device__ __forceinline__ void put(uint16_t* p) const { *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]); }
    __device__ __forceinline__ f2 pair(int j) const { return two_of(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u)); }
    __device__ __forceinline__ void set(int j, f2 v) {
        float f[2];
        parts_of(v, f);
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[j]) : "f"(f[1]), "f"(f[0]));
    }
    /* the sum of two bf16 numbers rounded once: what its f32 sum, narrowed, is (that one is exact up to 2^16 between
     * them, and beyond that both round to the larger) */
    __device__ __forceinline__ void add(const Raw& o) {
#pragma unroll
        for (int j = 0; j < 4; ++j) asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(w[j]) : "r"(w[j]), "r"(o.w[j]));
    }
    __device__ __forceinline__ void scalars(const uint16_t* p, int at, int n) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t lo = (unsigned)(at + 2 * j) < (unsigned)n ? p[at + 2 * j] : 0, hi = (unsigned)(at + 2 * j + 1) < (unsigned)n ? p[at + 2 * j + 1] : 0;
            w[j] = lo | hi << 16;
        }
    }
    __device__ __forceinline__ void put_scalars(uint16_t* p, int at, int n) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) if ((unsigned)(at + j) < (unsigned)n) p[at + j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
    }
};
template <> struct Raw<float> {
    f2 v[4];
    __device__ __forceinline__ void get(const float* p) {
        const ulonglong2 a = *(const ulonglong2*)p, b = *(const ulonglong2*)(p + 4);
        v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
    }
    __device__ __forceinline__ void get_off(const float* p) {
        const uint4* const q = (const uint4*)((uintptr_t)p & ~(uintptr_t)15);
        const uint4 a = q[0], b = q[1], c = q[2];
        const int d = (int)((uintptr_t)p & 15) >> 2;
        uint32_t w[12] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, c.x, c.y, c.z, c.w};
#pragma unroll
        for (int i = 0; i < 10; ++i) w[i] = d & 2 ? w[i + 2] : w[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = d & 1 ? w[i + 1] : w[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = two_of(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
    }
    __device__ __forceinline__ void put(float* p) const { *(ulonglong2*)p = make_ulonglong2(v[0], v[1]); *(ulonglong2*)(p + 4) = make_ulonglong2(v[2], v[3]); }
    __device__ __forceinline__ f2 pair(int j) const { return v[j]; }
    __device__ __forceinline__ void set(int j, f2 x) { v[j] = x; }
    __device__ __forceinline__ void add(const Raw& o) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = add2(v[j], o.v[j]);
    }
    __device__ __forceinline__ void scalars(const float* p, int at, int n) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            v[j] = two_of((unsigned)(at + 2 * j) < (unsigned)n ? p[at + 2 * j] : 0.0f, (unsigned)(at + 2 * j + 1) < (unsigned)n ? p[at + 2 * j + 1] : 0.0f);
    }
    __device__ __forceinline__ void put_scalars(float* p, int at, int n) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float f[2];
            parts_of(v[j], f);
            if ((unsigned)(at + 2 * j) < (unsigned)n) p[at + 2 * j] = f[0];
            if ((unsigned)(at + 2 * j + 1) < (unsigned)n) p[at + 2 * j + 1] = f[1];
        }
    }
};
__device__ __forceinline__ bool on16(const void* p) { return ((uintptr_t)p & 15) == 0; }
/* the chunk at value `at` of a row, which may reach over either end of it unless `in`: by 16 bytes where it lies on their grid,
 * else (OFF) by those around it, or one value at a time */
template <bool OFF, typename T>
__device__ __forceinline__ Raw<T> load_chunk(const T* row, int at, int n, bool in, bool grid) {
    Raw<T> r;
    if (in && grid) r.get(row + at); else if (OFF && in) r.get_off(row + at); else r.scalars(row, at, n);
    return r;
}
template <typename T>
__device__ __forceinline__ void store_chunk(T* row, int at, int n, bool fast, const f2* h) {
    Raw<T> r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r.set(j, h[j]);
    if (fast) r.put(row + at); else r.put_scalars(row, at, n);
}

/* The block walks rows gridDim apart. A row is cut into chunks of eight values on the codes' 8-byte grid, wherever the row
 * begins, C chunks a thread; what else lies on that grid is copied by 16 bytes, and the gated form's halves that do not (an
 * odd width) are read by the 16-byte words around them: one value at a time took 100 instead of 67 us for 8191 x 5125, 25
 * instead of 17 for 6043 x 1291. GRID: every row of every operand begins on its grid and ends a chunk. While a row is
 * reduced, the next one is on its way into shared memory by cp.async, each thread's chunks to places of its own: no barrier,
 * no registers. Instructions, not bytes, bound the bf16 forms at first (46 a value): hence two values an instruction wherever
 * there is one, and the residual's sum in bf16 pairs. */
template <int KIND, typename T, int C, bool GRID>
__global__ void __launch_bounds__(1024, C == 4 ? 1 : 2) k_token_i8_regs(const TokenI8 P) {
    constexpr bool kTwo = KIND != kQuant;                         /* the residual, or the up half */
    constexpr int kPer = 8 * (int)sizeof(T);                      /* bytes of a chunk */
    constexpr bool kOff = KIND == kSilu || KIND == kSigmoid;      /* the others' operands lie on one grid if their rows follow each other */
    extern __shared__ __align__(16) uint8_t slots[];
    __shared__ float part[2][32];
    in_turn(P.rows <= (int)gridDim.x);
    const int n = P.n, threads = blockDim.x;
    const bool two = kTwo && (KIND != kRms || P.res);
    const int64_t rows = P.rows;
    int64_t row = blockIdx.x;
    const T* x = (const T*)P.x + row * P.x_pitch;                 /* the row's operands: y is the residual or the up half */
    T* y = KIND == kRms ? (T*)P.res + (P.res ? row * P.r_pitch : 0) : const_cast<T*>(x) + n;
    const int64_t x_step = P.x_pitch * gridDim.x, y_step = KIND == kRms ? P.r_pitch * gridDim.x : x_step;
    uint8_t* const slot = slots + threadIdx.x * kPer;             /* chunk c of x: c * threads on; of y: C + c */
    const auto lead = [&](int64_t r) { return GRID ? 0 : -(int)((uintptr_t)(P.q + r * P.q_pitch) & 7); };
    const auto whole = [&](int at) { return GRID ? at < n : at >= 0 && at + 8 <= n; };
    const auto copy = [&](int place, const T* from) {
#pragma unroll
        for (int b = 0; b < kPer; b += 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                         ::"r"((uint32_t)__cvta_generic_to_shared(slot + place * threads * kPer) + b), "l"((const char*)from + b) : "memory");
    };
    const auto fetch = [&](int first) {
        const bool x_grid = GRID || on16(x + first), y_grid = two && (GRID || on16(y + first));
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int at = first + c * threads * 8;
            if (!whole(at)) continue;
            if (x_grid) copy(c, x + at);
            if (kTwo && y_grid) copy(C + c, y + at);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int first = lead(row) + (int)threadIdx.x * 8;
    fetch(first);
    /* a norm's two reductions lie a barrier apart each; the other kinds have one barrier a row, so that a warp may be a row
     * ahead of another that still reads: their rows take the two places by turns */
    int turn = 1;
    for (; row < rows; row += gridDim.x) {
        f2 h[C][4];
        f2 ss = 0;
        float amax = 0.0f;
        const int here = first;                                   /* this row's; `first` moves on to the next below */
        const bool x_grid = GRID || on16(x + here), y_grid = two && (GRID || on16(y + here));
        asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int at = here + c * threads * 8;
#pragma unroll
            for (int j = 0; j < 4; ++j) h[c][j] = 0;
            if (GRID && at >= n) continue;
            const bool in = whole(at);
            Raw<T> r, s;
            if (in && x_grid) r.get((const T*)(slot + c * threads * kPer)); else r = load_chunk<kOff, T>(x, at, n, in, false);
            if (two) {
                if (in && y_grid) s.get((const T*)(slot + (C + c) * threads * kPer)); else s = load_chunk<kOff, T>(y, at, n, in, false);
                if (KIND == kRms) {
                    r.add(s);
                    if (in && y_grid) r.put(y + at); else r.put_scalars(y, at, n);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                h[c][j] = r.pair(j);
                if (KIND == kRms) ss = fma2(h[c][j], h[c][j], ss);
                else if (KIND != kQuant) h[c][j] = gate2<KIND, sizeof(T) == 2>(h[c][j], s.pair(j));
            }
        }
        /* the slots have been read once their values are in use */
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) asm volatile("" : "+l"(h[c][j]));
        if (row + gridDim.x < rows) {
            x += x_step; y += y_step;
            first = lead(row + gridDim.x) + (int)threadIdx.x * 8;
            fetch(first);
        }
        if (KIND == kRms) {
            float half[2];
            parts_of(ss, half);
            const float sum = block_reduce(half[0] + half[1], part[0], [](float a, float b) { return a + b; });
            const float rs = 1.0f / sqrtf(sum / (float)n + P.eps);
            const f2 rs2 = two_of(rs, rs), wadd2 = two_of(P.wadd, P.wadd);
            const bool w_grid = GRID || (P.w_f32 ? on16((const float*)P.w + here) : on16((const uint16_t*)P.w + here));
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int at = here + c * threads * 8;
                if (GRID && at >= n) continue;
                const bool in = whole(at);
                if (P.w_f32) {
                    const Raw<float> w = load_chunk<sizeof(T) == 4>((const float*)P.w, at, n, in, w_grid);
#pragma unroll
                    for (int j = 0; j < 4; ++j) h[c][j] = mul2(mul2(h[c][j], rs2), add2(w.pair(j), wadd2));
                } else {
                    const Raw<uint16_t> w = load_chunk<sizeof(T) == 4>((const uint16_t*)P.w, at, n, in, w_grid);
#pragma unroll
                    for (int j = 0; j < 4; ++j) h[c][j] = mul2(mul2(h[c][j], rs2), add2(w.pair(j), wadd2));
                }
            }
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float f[2];
                parts_of(h[c][j], f);
                amax = max_size_nan(amax, f[0], f[1]);
            }
        amax = block_reduce(amax, part[turn], max_nan);
        if (KIND != kRms) turn ^= 1;
        const Step<kShortStep<KIND, T>> step(amax);
        if (threadIdx.x == 0) P.scale[row * P.s_pitch] = scale_of(amax);
        int8_t* const q = P.q + row * P.q_pitch;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int at = here + c * threads * 8;
            if (GRID && at >= n) continue;
            const bool in = whole(at);
            uint32_t w[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float f[4];
                parts_of(step.codes(h[c][2 * j]), f);
                parts_of(step.codes(h[c][2 * j + 1]), f + 2);
                w[j] = __byte_perm(__byte_perm(__float_as_uint(f[0]), __float_as_uint(f[1]), 0x0040),
                                   __byte_perm(__float_as_uint(f[2]), __float_as_uint(f[3]), 0x0040), 0x5410);
                if (step.s == 0.0f) w[j] = 0u;
            }
            if (in) *(uint2*)(q + at) = make_uint2(w[0], w[1]);
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) if ((unsigned)(at + j) < (unsigned)n) q[at + j] = (int8_t)(w[j >> 2] >> (8 * (j & 3)));
            if (P.ob) {
                if (P.ob_f32) { float* const o = (float*)P.ob + row * P.ob_pitch; store_chunk(o, at, n, in && on16(o + at), h[c]); }
                else { uint16_t* const o = (uint16_t*)P.ob + row * P.ob_pitch; store_chunk(o, at, n, in && on16(o + at), h[c]); }
            }
        }
    }
}

/* rows too long for that, any alignment: read again for each of the steps (they stay in the caches) */
template <int KIND, typename T>
__global__ void __launch_bounds__(512) k_token_i8(const TokenI8 P) {
    __shared__ float part[2][32];
    in_turn(false);
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
        ss = block_reduce(ss, part[0], [](float a, float b) { return a + b; });
        rs = 1.0f / sqrtf(ss / (float)P.n + P.eps);
    }
    float amax = 0.0f;
    for (int i = threadIdx.x; i < P.n; i += blockDim.x) amax = max_nan(amax, fabsf(value_of<KIND, T>(P, row, i, rs)));
    amax = block_reduce(amax, part[1], max_nan);
    const Step<kShortStep<KIND, T>> step(amax);
    if (threadIdx.x == 0) P.scale[row * P.s_pitch] = scale_of(amax);
    for (int i = threadIdx.x; i < P.n; i += blockDim.x) {
        const float h = value_of<KIND, T>(P, row, i, rs);
        float f[2];
        parts_of(step.codes(two_of(h, 0.0f)), f);
        P.q[row * P.q_pitch + i] = step.s == 0.0f ? (int8_t)0 : (int8_t)(__float_as_uint(f[0]) & 0xffu);
        if (P.ob) {
            if (P.ob_f32) ((float*)P.ob)[row * P.ob_pitch + i] = h;
            else ((uint16_t*)P.ob)[row * P.ob_pitch + i] = f32_to_bf16(h);
        }
    }
}

constexpr int kSlotBytes = 224 * 1024;
/* a row's values as they are fetched; the threads' places are at most a warp's of 32 values each more (8 KiB of f32 pairs) */
template <int KIND, typename T>
bool fits_slots(const TokenI8& P) {
    const int streams = KIND == kQuant || (KIND == kRms && !P.res) ? 1 : 2;
    return P.n <= 32760 && (int64_t)P.n * streams * (int)sizeof(T) <= kSlotBytes - 8 * 1024;
}

template <int KIND, typename T, int C, bool GRID>
int launch_rows(const TokenI8& P, int rows, int threads, cudaStream_t st) {
    const int one = KIND == kQuant || (KIND == kRms && !P.res), smem = threads * C * 8 * (int)sizeof(T) * (one ? 1 : 2);
    const auto kernel = k_token_i8_regs<KIND, T, C, GRID>;
    static std::atomic<int> fits[64][33][2];                      /* resident blocks, by device, warps a block and streams */
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return RAD_E_DEVICE;
    std::atomic<int>& known = fits[dev][threads / 32][one];
    int grid = known.load(std::memory_order_relaxed);
    if (!grid) {
        int per = 0, sms = 0;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSlotBytes) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, threads, smem) != cudaSuccess ||
            cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
            return RAD_E_DEVICE;
        grid = (per > 0 ? per : 1) * sms;
        known.store(grid, std::memory_order_relaxed);
    }
    return launch_in_turn(kernel, (unsigned)(rows < grid ? rows : grid), (unsigned)threads, (size_t)smem, st, P) == cudaSuccess ? RAD_OK : RAD_E_DEVICE;
}

bool rows_on(const void* p, int64_t pitch, int esz, int grid) { return !p || (((uintptr_t)p | (uintptr_t)(pitch * esz)) & (uintptr_t)(grid - 1)) == 0; }

template <int KIND, typename T, bool GRID>
int launch_regs(const TokenI8& P, int rows, cudaStream_t st) {
    const int most = P.n + (GRID ? 0 : 7);                        /* a row may begin anywhere inside its first chunk */
    /* Chunks a thread. Few rows: as many threads as the row has chunks (4 x 5120 norm: 2.6 us with one chunk a thread,
     * 3.0 with two, 3.7 with four). Many rows: fewer threads, whose barriers cost less (8192 x 5120 norm: 62 / 51 / 53 us;
     * 4099 x 5120 codes alone: 17.8 / 13.7 / 12.5 us; 8192 x 13824 gated: two 101, four 96 us, but off the grid, 8191 x 5125, 67 and 88; 16384 x 512 codes:
     * 8.7 / 7.3 / 8.2 us). */
    int c = most <= 8192 ? 1 : most <= 16384 ? 2 : 4;
    if (rows > 2 * tc_sm_count() && c < 4) c = KIND != kRms && most > 4096 && (GRID || KIND == kQuant) ? 4 : most > 256 ? 2 : 1;
    const int t = ((most + 8 * c - 1) / (8 * c) + 31) / 32 * 32;
    return c == 1 ? launch_rows<KIND, T, 1, GRID>(P, rows, t, st) : c == 2 ? launch_rows<KIND, T, 2, GRID>(P, rows, t, st)
                                                                             : launch_rows<KIND, T, 4, GRID>(P, rows, t, st);
}

template <int KIND, typename T>
int launch_type(const TokenI8& P, int rows, cudaStream_t st) {
    count_launch();
    const int esz = (int)sizeof(T);
    const bool grid = P.n % 8 == 0 && rows_on(P.x, P.x_pitch, esz, 16) && rows_on(P.res, P.r_pitch, esz, 16) && rows_on(P.w, 0, 1, 16) &&
                      rows_on(P.q, P.q_pitch, 1, 8);
    int rc = RAD_OK;
    if (!fits_slots<KIND, T>(P)) rc = launch_in_turn(k_token_i8<KIND, T>, (unsigned)rows, 512u, 0, st, P) == cudaSuccess ? RAD_OK : RAD_E_DEVICE;
    else rc = grid ? launch_regs<KIND, T, true>(P, rows, st) : launch_regs<KIND, T, false>(P, rows, st);
    return rc != RAD_OK ? rc : cudaGetLastError() == cudaSuccess ? RAD_OK : RAD_E_DEVICE;
}
template <int KIND>
int launch_kind(const TokenI8& P, int x_f32, int rows, cudaStream_t st) {
    return x_f32 ? launch_type<KIND, float>(P, rows, st) : launch_type<KIND, uint16_t>(P, rows, st);
}

} /* namespace */

int launch_token_i8(const R3dTokenI8& p, cudaStream_t st) {
    TokenI8 P{};
    P.x = p.x; P.x_pitch = p.x_pitch; P.res = p.residual; P.r_pitch = p.r_pitch;
    P.w = p.w; P.w_f32 = p.w_dtype == RAD_F32;
    P.q = (int8_t*)p.q; P.q_pitch = p.q_pitch; P.scale = p.scale; P.s_pitch = p.s_pitch;
    P.ob = p.out; P.ob_f32 = p.out_dtype == RAD_F32; P.ob_pitch = p.out_pitch;
    P.n = p.n; P.rows = p.rows; P.eps = p.eps; P.wadd = p.wadd;
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

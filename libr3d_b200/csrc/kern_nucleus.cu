/* kern_nucleus.cu -- sample_nucleus: temperature, top-k, top-p, min-p and a given random number, one token a row.
 *
 * With mx the row's largest logit and T its temperature, token i has the weight w_i = 2^((x_i - mx) log2(e) / T) in
 * (0, 1]. The tokens are ordered by value, descending, ties to the lower id (the order of row_topk and
 * sample_argmax); each filter keeps a first part of that order: top-k its first k, top-p the shortest part whose
 * weight reaches p times the weight that top-k left, min-p those with w_i >= min_p; the first token always stays.
 * The answer is the first kept token, by ascending id, whose running weight exceeds u times the kept weight.
 *
 * Weights are whole numbers of 2^-S (S the largest for which a row's sum fits 62 bits; 44 at 151936 tokens), made
 * from 64-bit floating point. Their sums are exact in any order, so the answer depends neither on the order of
 * threads nor on how a row is split, and it agrees with a 64-bit computation except where a running sum is
 * within about sqrt(V) 2^-S of a border.
 *
 * -inf and NaN logits are masked: never kept. A row with nothing left reports token -1, kept 0, logprob -inf.
 */
#include <cmath>
#include "r3d_kernels.h"
#include "r3d_numerics.cuh"

namespace r3d {

namespace {

using u64 = unsigned long long;

/* monotone map of a float onto unsigned integers, -0 folded onto +0; 0 is "masked" */
__device__ __forceinline__ uint32_t key_of(float v) {
    uint32_t u = __float_as_uint(v);
    if (u == 0x80000000u) u = 0u;
    if ((u & 0x7fffffffu) > 0x7f800000u || u == 0xff800000u) return 0u;      /* NaN, -inf */
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float val_of(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

struct Row {
    double c;             /* log2(e) / T */
    double mx;
    bool inf;             /* the largest logit is +inf: it has all the weight */
    int S;
};
__device__ __forceinline__ double exponent_of(const Row& R, uint32_t key) {
    const double x = (double)val_of(key);
    if (R.inf) return isinf(x) ? 0.0 : -HUGE_VAL;
    return (x - R.mx) * R.c;
}
__device__ __forceinline__ u64 weight_of(const Row& R, uint32_t key) {
    if (!key) return 0;
    return (u64)__double2ull_rn(exp2(exponent_of(R, key) + R.S));
}

struct Sum { int n; u64 w; };

__device__ Sum block_sum(Sum v, Sum* part) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        v.n += __shfl_xor_sync(0xffffffffu, v.n, o);
        v.w += __shfl_xor_sync(0xffffffffu, v.w, o);
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    Sum s{0, 0};
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) { s.n += part[i].n; s.w += part[i].w; }
    return s;
}

/* one block a row, the row read again for each step of the searches */
__global__ void __launch_bounds__(1024) k_nucleus(const R3dNucleus P) {
    __shared__ Sum part[32];
    const int64_t m = blockIdx.x;
    const int V = P.n_vocab;
    const auto key_at = [&](int i) {
        return key_of(P.x_dtype == RAD_F32 ? ((const float*)P.logits)[m * P.x_pitch + i]
                                           : bf16_to_f32(((const uint16_t*)P.logits)[m * P.x_pitch + i]));
    };
    const auto sum_if = [&](auto f) {
        Sum s{0, 0};
        for (int i = threadIdx.x; i < V; i += blockDim.x) f(s, key_at(i), i);
        return block_sum(s, part);
    };

    uint32_t best = 0;
    for (int i = threadIdx.x; i < V; i += blockDim.x) best = max(best, key_at(i));
    for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5].n = (int)best;
    __syncthreads();
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) best = max(best, (uint32_t)part[i].n);
    if (!best) {
        if (threadIdx.x == 0) {
            P.token[m * P.token_pitch] = -1;
            if (P.logprob) P.logprob[m * P.lp_pitch] = -INFINITY;
            if (P.kept) P.kept[m * P.kept_pitch] = 0;
        }
        return;
    }
    const float t = P.temperature ? P.temperature[m * P.t_pitch] : 1.0f;
    const bool greedy = !(t > 0.0f);
    Row R;
    R.mx = (double)val_of(best);
    R.inf = isinf(val_of(best));
    R.c = greedy ? 0.0 : 1.4426950408889634 / (double)t;
    R.S = P.shift;

    const int live = sum_if([&](Sum& s, uint32_t k, int) { s.n += k != 0; }).n;
    int k = P.top_k ? P.top_k[m * P.k_pitch] : 0;
    if (k <= 0 || k > live) k = live;
    const float low = P.min_p ? P.min_p[m * P.mp_pitch] : 0.0f;
    if (greedy || low > 1.0f) k = 1;                   /* nothing but the first is more than as likely as it */
    /* cut: keys above `cut` are kept, of those equal to it the first `ties` */
    uint32_t cut = 1;
    int ties = live;
    const auto search = [&](auto enough) {      /* the largest key c with enough(sums over keys >= c) */
        uint32_t lo = 1, hi = best;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2 + 1;
            if (enough(mid)) lo = mid; else hi = mid - 1;
        }
        return lo;
    };
    if (k < live) {
        cut = search([&](uint32_t c) { return sum_if([&](Sum& s, uint32_t key, int) { s.n += key >= c; }).n >= k; });
        ties = k - sum_if([&](Sum& s, uint32_t key, int) { s.n += key > cut; }).n;
    }
    const float p = P.top_p ? P.top_p[m * P.p_pitch] : 1.0f;
    if (!greedy && p < 1.0f) {
        const u64 over = sum_if([&](Sum& s, uint32_t key, int) { if (key > cut) s.w += weight_of(R, key); }).w;
        const u64 total = over + (cut > 1 ? (u64)ties * weight_of(R, cut) : sum_if([&](Sum& s, uint32_t key, int) { if (key == cut) s.w += weight_of(R, key); }).w);
        const u64 want = p > 0.0f ? max(1ull, (u64)__double2ull_ru((double)p * (double)total)) : 1ull;
        if (over >= want) {
            cut = search([&](uint32_t c) { return sum_if([&](Sum& s, uint32_t key, int) { if (key >= c) s.w += weight_of(R, key); }).w >= want; });
            ties = V;
        }
        const u64 above = sum_if([&](Sum& s, uint32_t key, int) { if (key > cut) s.w += weight_of(R, key); }).w;
        const u64 one = weight_of(R, cut);
        if (one && want > above) ties = (int)min((u64)ties, (want - above + one - 1) / one);
    }
    /* the cut's last kept id */
    int last = V - 1;
    if (sum_if([&](Sum& s, uint32_t key, int) { s.n += key == cut; }).n > ties) {
        int lo = 0, hi = V - 1;
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (sum_if([&](Sum& s, uint32_t key, int i) { s.n += key == cut && i <= mid; }).n >= ties) hi = mid; else lo = mid + 1;
        }
        last = lo;
    }
    /* half a step of a 64-bit weight below min_p rounds up to it */
    const double floor_y = low > 0.0f ? fmin(log2((double)low), 0.0) - 8e-17 : -HUGE_VAL;
    const auto keep = [&](uint32_t key, int i) {
        return key && (key > cut || (key == cut && i <= last)) && (greedy || exponent_of(R, key) >= floor_y);
    };
    const Sum all = sum_if([&](Sum& s, uint32_t key, int i) { if (keep(key, i)) { ++s.n; s.w += weight_of(R, key); } });
    const float u = P.u[m * P.u_pitch];
    const u64 at = u > 0.0f ? (u < 1.0f ? min(all.w - 1, (u64)__double2ull_rd((double)u * (double)all.w)) : all.w - 1) : 0ull;
    int lo = 0, hi = V - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (sum_if([&](Sum& s, uint32_t key, int i) { if (i <= mid && keep(key, i)) s.w += weight_of(R, key); }).w > at) hi = mid; else lo = mid + 1;
    }
    if (threadIdx.x == 0) {
        P.token[m * P.token_pitch] = lo;
        if (P.kept) P.kept[m * P.kept_pitch] = all.n;
        if (P.logprob) P.logprob[m * P.lp_pitch] = (float)(0.6931471805599453 * (exponent_of(R, key_at(lo)) + R.S) - log((double)all.w));
    }
}

} /* namespace */

int launch_nucleus(const R3dNucleus& p, cudaStream_t st) {
    R3dNucleus P = p;
    int bits = 0;
    while ((1ll << bits) < (long long)p.n_vocab) ++bits;
    P.shift = 62 - bits < 50 ? 62 - bits : 50;
    count_launch();
    k_nucleus<<<(unsigned)p.rows, 1024, 0, st>>>(P);
    return cudaGetLastError() == cudaSuccess ? RAD_OK : RAD_E_DEVICE;
}

} /* namespace r3d */

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
#include <atomic>
#include <cmath>
#include <cstdlib>
#include "r3d_kernels.h"
#include "r3d_numerics.cuh"

namespace r3d {

namespace {

using u64 = unsigned long long;

__device__ __forceinline__ void answer(const R3dNucleus& P, int64_t m, int token, int kept, float logprob) {
    P.token[m * P.token_pitch] = token;
    if (P.kept) P.kept[m * P.kept_pitch] = kept;
    if (P.logprob) P.logprob[m * P.lp_pitch] = logprob;
}

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

__device__ __forceinline__ float load_x(const R3dNucleus& P, int64_t m, int i) {
    return P.x_dtype == RAD_F32 ? ((const float*)P.logits)[m * P.x_pitch + i] : bf16_to_f32(((const uint16_t*)P.logits)[m * P.x_pitch + i]);
}

struct Row {
    double c;             /* log2(e) / T */
    double mx;
    bool inf;             /* the largest logit is +inf: it has all the weight */
    int S;
};
__device__ __forceinline__ Row row_of(uint32_t best, float t, int shift) {
    Row R;
    R.mx = (double)val_of(best);
    R.inf = isinf(val_of(best));
    R.c = t > 0.0f ? 1.4426950408889634 / (double)t : 0.0;
    R.S = shift;
    return R;
}
/* min-p as a bound on the exponent; half a step of a 64-bit weight below it rounds up to it */
__device__ __forceinline__ double floor_of(float low) { return low > 0.0f ? fmin(log2((double)low), 0.0) - 8e-17 : -HUGE_VAL; }
/* the weight before which the first part that holds p of `total` ends */
__device__ __forceinline__ u64 want_of(float p, u64 total) { return max(1ull, (u64)__double2ull_ru((double)p * (double)total)); }
/* the running weight that the answer is the first to exceed */
__device__ __forceinline__ u64 point_of(float u, u64 total) {
    return u > 0.0f ? (u < 1.0f ? min(total - 1, (u64)__double2ull_rd((double)u * (double)total)) : total - 1) : 0ull;
}
__device__ __forceinline__ double exponent_of(const Row& R, uint32_t key) {
    const double x = (double)val_of(key);
    if (R.inf) return isinf(x) ? 0.0 : -HUGE_VAL;
    return (x - R.mx) * R.c;
}
__device__ __forceinline__ u64 weight_of(const Row& R, uint32_t key) {
    if (!key) return 0;
    return (u64)__double2ull_rn(exp2(exponent_of(R, key) + R.S));
}

__device__ __forceinline__ float logprob_of(const Row& R, uint32_t key, u64 total) {
    return (float)(0.6931471805599453 * (exponent_of(R, key) + R.S) - log((double)total));
}

struct Sum { int n; u64 w; };
struct Sum3 { u64 w[3]; int n[3]; };

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

/* rows too long for a cluster's shared memory: one block a row, read again for each step of the searches */
__global__ void __launch_bounds__(1024) k_nucleus_long(const R3dNucleus P) {
    __shared__ Sum part[32];
    const int64_t m = blockIdx.x;
    const int V = P.n_vocab;
    const auto key_at = [&](int i) { return key_of(load_x(P, m, i)); };
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
        if (threadIdx.x == 0) answer(P, m, -1, 0, -INFINITY);
        return;
    }
    const float t = P.temperature ? P.temperature[m * P.t_pitch] : 1.0f;
    const bool greedy = !(t > 0.0f);
    const Row R = row_of(best, t, P.shift);

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
        const u64 want = want_of(p, total);
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
    const double floor_y = floor_of(low);
    const auto keep = [&](uint32_t key, int i) {
        return key && (key > cut || (key == cut && i <= last)) && (greedy || exponent_of(R, key) >= floor_y);
    };
    const Sum all = sum_if([&](Sum& s, uint32_t key, int i) { if (keep(key, i)) { ++s.n; s.w += weight_of(R, key); } });
    const float u = P.u[m * P.u_pitch];
    const u64 at = point_of(u, all.w);
    int lo = 0, hi = V - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (sum_if([&](Sum& s, uint32_t key, int i) { if (i <= mid && keep(key, i)) s.w += weight_of(R, key); }).w > at) hi = mid; else lo = mid + 1;
    }
    if (threadIdx.x == 0) answer(P, m, lo, all.n, logprob_of(R, key_at(lo), all.w));
}

/* ------------------------------------------------------------------ a cluster a row
 * The row is read once, as ordered keys into the shared memory of the cluster's CTAs; a thread owns `e` neighbouring ids
 * (an odd number: its reads fall into banks of their own), so id order is the order of threads. What the CTAs find out
 * goes to all of them through distributed shared memory: the largest key; a histogram of the distance to it in
 * kBins steps over the range of distances that have any weight; sums.
 *   - Filters that leave few: the steps of the histogram that hold k tokens, or surely p of the weight, are gathered
 *     in the first CTA, up to kCap tokens, sorted there, cut and summed.
 *   - Filters that leave many: the last kept key is searched, three probes of exact sums a round.
 *   - None: the running weight alone.
 * Latency bounds it (a round through the cluster is about a microsecond), and for rows without top-k the 64-bit
 * exponential of every token. */
constexpr int kT = 512;
constexpr int kBins = 4096;
constexpr int kCap = 2048;
constexpr int kMaxCluster = 16;
constexpr double kRange = 44.0 * 0.6931471805599453;              /* distances with a weight, in temperatures: 2^-44 and up */

struct Part { u64 w[3]; u64 key; int n[3]; int pad; };

struct Shared {
    Part parts[2][kMaxCluster];                                   /* what each CTA says, by turns */
    Part mine;
    u64 warp_w[kT / 32];
    int warp_n[kT / 32];
    Sum3 sums[kT / 32];
    u64 list[kCap];
    uint32_t hist[kBins], merged[kBins];
    int gathered, pick[2];
    float edge[2];
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t peer_addr(const void* p, int rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ void peer_put(uint32_t at, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory"); }
__device__ __forceinline__ void peer_put(uint32_t at, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ uint32_t peer_get(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void meet() {                          /* of the cluster; orders what was put before it */
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

/* one row's state, the same in every thread of the cluster */
struct Cluster {
    Shared* s;
    int size, rank, turn;

    /* every CTA's `mine` to every CTA; parts() is valid until the turn after next */
    __device__ __forceinline__ const Part* exchange() {
        __syncthreads();
        constexpr int kWords = sizeof(Part) / 8;
        for (int i = threadIdx.x; i < size * kWords; i += kT)
            peer_put(peer_addr((u64*)&s->parts[turn][rank] + i % kWords, i / kWords), ((const u64*)&s->mine)[i % kWords]);
        meet();
        const Part* p = s->parts[turn];
        turn ^= 1;
        return p;
    }
    /* sums over the cluster */
    __device__ __forceinline__ Sum3 sum(Sum3 v) {
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            v.n[j] = __reduce_add_sync(0xffffffffu, v.n[j]);
#pragma unroll
            for (int o = 16; o; o >>= 1) v.w[j] += __shfl_xor_sync(0xffffffffu, v.w[j], o);
        }
        if ((threadIdx.x & 31) == 0) s->sums[threadIdx.x >> 5] = v;
        __syncthreads();
        if (threadIdx.x < 6) {
            const int j = threadIdx.x % 3;
            u64 w = 0; int n = 0;
            for (int i = 0; i < kT / 32; ++i) { w += s->sums[i].w[j]; n += s->sums[i].n[j]; }
            if (threadIdx.x < 3) s->mine.w[j] = w; else s->mine.n[j] = n;
        }
        const Part* p = exchange();
        Sum3 all{};
        for (int r = 0; r < size; ++r)
#pragma unroll
            for (int j = 0; j < 3; ++j) { all.n[j] += p[r].n[j]; all.w[j] += p[r].w[j]; }
        return all;
    }
};

/* exclusive over the block's threads, in their order; *total over all of them */
__device__ __forceinline__ u64 scan_w(Shared* s, u64 v, u64* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const u64 y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
    __syncthreads();
    if (lane == 31) s->warp_w[warp] = x;
    __syncthreads();
    u64 before = 0, all = 0;
    for (int i = 0; i < kT / 32; ++i) { if (i < warp) before += s->warp_w[i]; all += s->warp_w[i]; }
    *total = all;
    return before + x - v;
}
__device__ __forceinline__ int scan_n(Shared* s, int v, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
    __syncthreads();
    if (lane == 31) s->warp_n[warp] = x;
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < kT / 32; ++i) { if (i < warp) before += s->warp_n[i]; all += s->warp_n[i]; }
    *total = all;
    return before + x - v;
}

/* n2 (a power of two) words, largest first */
__device__ __forceinline__ void sort_desc(u64* a, int n2) {
    for (int k = 2; k <= n2; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < n2 / 2; i += kT) {
                const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
                const u64 x = a[lo], y = a[hi];
                if ((x < y) == ((lo & k) == 0)) { a[lo] = y; a[hi] = x; }
            }
        }
    __syncthreads();
}

__global__ void __launch_bounds__(kT) k_nucleus_row(const R3dNucleus P, const int e) {
    extern __shared__ __align__(16) uint8_t raw[];
    Shared* const s = (Shared*)raw;
    uint32_t* const keys = (uint32_t*)(raw + sizeof(Shared));
    Cluster cl;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(cl.size));
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(cl.rank));
    cl.s = s; cl.turn = 0;
    const int64_t m = blockIdx.x / cl.size;
    const int V = P.n_vocab, base = cl.rank * kT * e, tid = threadIdx.x;
    uint32_t* const own = keys + tid * e;                         /* ids base + tid * e ... */
    const int own_id = base + tid * e;

    const float t = P.temperature ? P.temperature[m * P.t_pitch] : 1.0f, p = P.top_p ? P.top_p[m * P.p_pitch] : 1.0f;
    const float low = P.min_p ? P.min_p[m * P.mp_pitch] : 0.0f, u = P.u[m * P.u_pitch];
    int k = P.top_k ? P.top_k[m * P.k_pitch] : 0;

    /* the peers' shared memory may be written once they have all begun: waited for below */
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

    /* ---- read the row; its largest key, the lowest id that has it, and how many are not masked */
    u64 best_id = 0;
    int live = 0;
#pragma unroll 8
    for (int j = 0; j < e; ++j) {
        const int i = j * kT + tid, id = base + i;
        const uint32_t key = id < V ? key_of(load_x(P, m, id)) : 0u;
        keys[i] = key;
        live += key != 0;
        if (key) best_id = max(best_id, (u64)key << 32 | (0xffffffffu - (uint32_t)id));
    }
    for (int i = tid; i < kBins; i += kT) s->hist[i] = 0;
    if (tid == 0) s->gathered = 0;
    live = __reduce_add_sync(0xffffffffu, live);
#pragma unroll
    for (int o = 16; o; o >>= 1) best_id = max(best_id, (u64)__shfl_xor_sync(0xffffffffu, best_id, o));
    if ((tid & 31) == 0) { s->warp_w[tid >> 5] = best_id; s->warp_n[tid >> 5] = live; }
    __syncthreads();
    if (tid == 0) {
        u64 b = 0; int n = 0;
        for (int i = 0; i < kT / 32; ++i) { b = max(b, s->warp_w[i]); n += s->warp_n[i]; }
        s->mine.key = b; s->mine.n[0] = n;
    }
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    {
        const Part* parts = cl.exchange();
        best_id = 0; live = 0;
        for (int r = 0; r < cl.size; ++r) { best_id = max(best_id, parts[r].key); live += parts[r].n[0]; }
    }
    const uint32_t best = (uint32_t)(best_id >> 32);
    const bool first_cta = cl.rank == 0;
    if (!best) {
        if (first_cta && tid == 0) answer(P, m, -1, 0, -INFINITY);
        return;
    }
    if (k <= 0 || k > live) k = live;
    if (!(t > 0.0f) || low > 1.0f || k == 1 || p <= 0.0f) {       /* the first alone */
        if (first_cta && tid == 0) answer(P, m, (int)(0xffffffffu - (uint32_t)best_id), 1, 0.0f);
        return;
    }
    const Row R = row_of(best, t, P.shift);
    const double floor_y = floor_of(low);
    const bool by_k = k < live, by_p = p < 1.0f;

    uint32_t cut = 1;                                             /* kept: keys above cut, and the first `ties` equal to it */
    int ties = V;
    if (by_k || by_p) {
        /* ---- histogram of the distance to the largest logit (key order and step order agree) */
        const float mx = val_of(best), inv = (float)((kBins - 1) / kRange) / t;
        const auto bin_of = [&](uint32_t key) {
            if (R.inf) return key == best ? 0 : kBins - 1;
            const float d = __fsub_rn(mx, val_of(key)) * inv;
            return d < (float)(kBins - 1) ? (int)d : d >= (float)(kBins - 1) ? kBins - 1 : 0;     /* not a number: 0 * inf, every weight is 1 */
        };
        u64 mass = 0;
        for (int j = 0; j < e; ++j) {
            const uint32_t key = own[j];
            if (!key) continue;
            atomicAdd(&s->hist[bin_of(key)], 1u);
            if (!by_k) mass += weight_of(R, key);
        }
        /* the total, which top-p alone is a share of, goes along */
        Sum3 v{};
        v.w[0] = mass;
        const u64 total = cl.sum(v).w[0];                         /* also: every CTA's histogram is complete */
        const int seg = kBins / cl.size;
        for (int i = tid; i < seg; i += kT) {
            const int b = cl.rank * seg + i;
            uint32_t n = 0;
            for (int r = 0; r < cl.size; ++r) n += peer_get(peer_addr(&s->hist[b], r));
            for (int r = 0; r < cl.size; ++r) peer_put(peer_addr(&s->merged[b], r), n);
        }
        meet();
        /* ---- the steps that hold the first k tokens, or surely p of the weight: a token of step b weighs at least what
         * the end of its step does (less a little for the rounding of b) */
        constexpr int kEach = kBins / kT;
        int n_own = 0; float low_own = 0.0f;
        uint32_t cnt[kEach];
        const float per_bin = (float)(kRange / (kBins - 1) * 1.4426950408889634);    /* halvings a step */
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            cnt[j] = s->merged[tid * kEach + j];
            n_own += (int)cnt[j];
            low_own += (float)cnt[j] * exp2f(-per_bin * (float)(tid * kEach + j + 1)) * 0.999f;
        }
        int all_n; u64 all_w;
        int n_before = scan_n(s, n_own, &all_n);
        const u64 low_before = scan_w(s, (u64)(low_own * 0x1p24f), &all_w);     /* rounded down, and again below */
        const u64 need_low = by_k ? 0 : (u64)((double)want_of(p, total) * exp2((double)(24 - R.S))) + 1;
        if (tid == 0) { s->pick[0] = kBins; s->pick[1] = 0; }
        __syncthreads();
        u64 low_run = low_before;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int b = tid * kEach + j;
            const int n_after = n_before + (int)cnt[j];
            if (by_k) { if (n_before < k && n_after >= k) { s->pick[0] = b; s->pick[1] = n_after; } }
            else if (cnt[j]) {
                const u64 after = low_run + (u64)((float)cnt[j] * exp2f(-per_bin * (float)(b + 1)) * 0.999f * 0x1p24f);
                if (after >= need_low && b < kBins - 1) atomicMin(&s->pick[0], b);
                low_run = after;
            }
            n_before = n_after;
        }
        __syncthreads();
        const int top = s->pick[0];
        int n_top = by_k ? s->pick[1] : 0;
        if (!by_k && top < kBins) {                               /* how many the chosen steps hold */
            int n = 0;
#pragma unroll
            for (int j = 0; j < kEach; ++j) if (tid * kEach + j <= top) n += (int)cnt[j];
            scan_n(s, n, &n_top);
        }
        if (top < kBins && n_top <= kCap) {
            /* ---- few: to the first CTA, in any order */
            int n = 0, n_cta;
            for (int j = 0; j < e; ++j) n += own[j] && bin_of(own[j]) <= top;
            int at = scan_n(s, n, &n_cta);
            if (tid == 0) {
                uint32_t from;
                asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(from) : "r"(peer_addr(&s->gathered, 0)), "r"(n_cta) : "memory");
                s->pick[0] = (int)from;
            }
            __syncthreads();
            at += s->pick[0];
            for (int j = 0; j < e && n; ++j)
                if (own[j] && bin_of(own[j]) <= top)
                    peer_put(peer_addr(&s->list[at++], 0), (u64)own[j] << 32 | (0xffffffffu - (uint32_t)(own_id + j)));
            meet();
            if (!first_cta) return;
            int n2 = 32;
            while (n2 < n_top) n2 <<= 1;
            for (int i = n_top + tid; i < n2; i += kT) s->list[i] = 0;
            sort_desc(s->list, n2);
            const int each = (n2 + kT - 1) / kT, i0 = tid * each;
            const auto weight_at = [&](int i) { return i < n2 ? weight_of(R, (uint32_t)(s->list[i] >> 32)) : 0ull; };
            u64 w = 0, sum, dummy;
            for (int i = i0; i < i0 + each; ++i) if (i < k) w += weight_at(i);
            u64 before = scan_w(s, w, &sum);
            const u64 want = by_p ? want_of(p, by_k ? sum : total) : ~0ull;
            int kept = 0;
            w = 0;
            for (int i = i0; i < i0 + each && i < k && i < n_top; ++i) {
                const u64 x = weight_at(i);
                if (i && (before >= want || exponent_of(R, (uint32_t)(s->list[i] >> 32)) < floor_y)) break;
                before += x; w += x; ++kept;
            }
            int n_kept;
            scan_n(s, kept, &n_kept);
            scan_w(s, w, &sum);
            /* by id, ascending: the low words are 0xffffffff - id; the key moves below */
            n2 = 32;
            while (n2 < n_kept) n2 <<= 1;
            for (int i = tid; i < n2; i += kT) { const u64 v2 = s->list[i]; s->list[i] = i < n_kept ? v2 << 32 | v2 >> 32 : 0ull; }
            sort_desc(s->list, n2);
            w = 0;
            const int each2 = (n2 + kT - 1) / kT, j0 = tid * each2;
            for (int i = j0; i < j0 + each2 && i < n_kept; ++i) w += weight_of(R, (uint32_t)s->list[i]);
            before = scan_w(s, w, &dummy);
            const u64 point = point_of(u, sum);
            for (int i = j0; i < j0 + each2 && i < n_kept; ++i) {
                const uint32_t key = (uint32_t)s->list[i];
                const u64 x = weight_of(R, key);
                if (before <= point && point < before + x)
                    answer(P, m, (int)(0xffffffffu - (uint32_t)(s->list[i] >> 32)), n_kept, logprob_of(R, key, sum));
                before += x;
            }
            return;
        }
        /* ---- many: the largest key c with enough tokens (weight) from c on. enough(sum over keys in [c, hi)) */
        const auto search = [&](uint32_t lo, uint32_t hi, u64 need, u64* above, auto value) {
            while (hi - lo > 1) {
                const uint32_t step = max(1u, (hi - lo) / 4);
                uint32_t c[3];
#pragma unroll
                for (int j = 0; j < 3; ++j) c[j] = min(lo + (j + 1) * step, hi);
                Sum3 v3{};
                for (int j = 0; j < e; ++j) {
                    const uint32_t key = own[j];
                    if (key < c[0] || key >= hi) continue;
                    const u64 x = value(key);
                    v3.w[0] += x;
                    if (key >= c[1]) v3.w[1] += x;
                    if (key >= c[2]) v3.w[2] += x;
                }
                v3 = cl.sum(v3);
                int j = -1;
                for (int i = 0; i < 3; ++i) if (c[i] < hi && *above + v3.w[i] >= need) j = i;
                const uint32_t nhi = j < 2 ? c[j + 1] : hi;
                if (j < 2 && nhi < hi) *above += v3.w[j + 1];
                if (j >= 0) lo = c[j];
                hi = nhi;
            }
            return lo;
        };
        u64 above = 0;
        if (by_k) {
            cut = search(1u, best + 1, (u64)k, &above, [](uint32_t) { return 1ull; });
            ties = (int)((u64)k - above);
        }
        if (by_p) {
            Sum3 v3{};
            for (int j = 0; j < e; ++j) if (own[j] > cut) v3.w[0] += weight_of(R, own[j]);
            const u64 over = by_k ? cl.sum(v3).w[0] : total;
            const u64 one = weight_of(R, cut), want = want_of(p, by_k ? over + (u64)ties * one : total);
            above = 0;
            if (!by_k || over >= want) {
                cut = search(by_k ? cut : 1u, best + 1, want, &above, [&](uint32_t key) { return weight_of(R, key); });
                ties = V;
            } else above = over;
            const u64 one_cut = weight_of(R, cut);
            if (one_cut && want > above) ties = (int)min((u64)ties, (want - above + one_cut - 1) / one_cut);
        }
    }

    /* ---- the kept ones by id */
    int tie_rank = 0;
    if (ties < V) {
        int n = 0, n_cta;
        for (int j = 0; j < e; ++j) n += own[j] == cut;
        tie_rank = scan_n(s, n, &n_cta);
        if (tid == 0) s->mine.n[0] = n_cta;
        const Part* parts = cl.exchange();
        for (int r = 0; r < cl.rank; ++r) tie_rank += parts[r].n[0];
    }
    const auto each_kept = [&](auto f) {
        int rank = tie_rank;
        for (int j = 0; j < e; ++j) {
            const uint32_t key = own[j];
            if (key < cut || !key || (key == cut && rank++ >= ties) || exponent_of(R, key) < floor_y) continue;
            if (!f(j, key)) return;
        }
    };
    u64 w = 0, w_cta;
    int n = 0, n_cta;
    each_kept([&](int, uint32_t key) { w += weight_of(R, key); ++n; return true; });
    u64 before = scan_w(s, w, &w_cta);
    scan_n(s, n, &n_cta);
    if (tid == 0) { s->mine.w[0] = w_cta; s->mine.n[0] = n_cta; }
    const Part* parts = cl.exchange();
    u64 sum = 0; int kept = 0;
    for (int r = 0; r < cl.size; ++r) {
        if (r < cl.rank) before += parts[r].w[0];
        sum += parts[r].w[0]; kept += parts[r].n[0];
    }
    const u64 point = point_of(u, sum);
    if (before <= point && point < before + w)
        each_kept([&](int j, uint32_t key) {
            before += weight_of(R, key);
            if (before <= point) return true;
            answer(P, m, own_id + j, kept, logprob_of(R, key, sum));
            return false;
        });
}

} /* namespace */

int launch_nucleus(const R3dNucleus& p, cudaStream_t st) {
    R3dNucleus P = p;
    int bits = 0;
    while ((1ll << bits) < (long long)p.n_vocab) ++bits;
    P.shift = 62 - bits < 50 ? 62 - bits : 50;
    count_launch();
    int size = getenv("DEV_CL") ? atoi(getenv("DEV_CL")) : 8;
    int e = (p.n_vocab + kT * size - 1) / (kT * size);
    e |= 1;
    const size_t smem = sizeof(Shared) + (size_t)kT * e * 4;
    if (smem > 220 * 1024) {
        k_nucleus_long<<<(unsigned)p.rows, 1024, 0, st>>>(P);
        return cudaGetLastError() == cudaSuccess ? RAD_OK : RAD_E_DEVICE;
    }
    static std::atomic<bool> set[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return RAD_E_DEVICE;
    if (!set[dev].load(std::memory_order_relaxed)) {
        if (cudaFuncSetAttribute(k_nucleus_row, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024) != cudaSuccess ||
            cudaFuncSetAttribute(k_nucleus_row, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return RAD_E_DEVICE;
        set[dev].store(true, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)p.rows * (unsigned)size); cfg.blockDim = dim3(kT); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)size; at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_nucleus_row, P, e) == cudaSuccess && cudaGetLastError() == cudaSuccess ? RAD_OK : RAD_E_DEVICE;
}

} /* namespace r3d */

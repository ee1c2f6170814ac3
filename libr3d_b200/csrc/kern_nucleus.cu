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
/* 2^(exponent + S), rounded to a whole number: 2^n times the Taylor series of 2^r, |r| <= 1/2, to the eleventh power
 * (its remainder is below 2^-47; 2^0 is 1 exactly), rounded by adding 2^52. */
__device__ __forceinline__ u64 weight_of(const Row& R, uint32_t key) {
    const double z = exponent_of(R, key) + R.S;
    if (!key || !(z > -1.5)) return 0;
    const double whole = z + 6755399441055744.0;                  /* 1.5 * 2^52: the nearest whole number in the low word */
    const double r = z - (whole - 6755399441055744.0);
    double p = 4.445538271870811e-10;                             /* ln(2)^i / i!, i = 11 .. 0 */
    p = fma(p, r, 7.054911620801122e-09);
    p = fma(p, r, 1.0178086009239699e-07);
    p = fma(p, r, 1.3215486790144307e-06);
    p = fma(p, r, 1.5252733804059841e-05);
    p = fma(p, r, 1.5403530393381608e-04);
    p = fma(p, r, 1.3333558146428443e-03);
    p = fma(p, r, 9.618129107628477e-03);
    p = fma(p, r, 5.5504108664821576e-02);
    p = fma(p, r, 0.2402265069591007);
    p = fma(p, r, 0.6931471805599453);
    p = fma(p, r, 1.0);
    const double scaled = __hiloint2double(__double2hiint(p) + (__double2loint(whole) << 20), __double2loint(p));
    return (u64)__double_as_longlong(scaled + 4503599627370496.0) - 0x4330000000000000ull;
}

__device__ __forceinline__ float logprob_of(const Row& R, uint32_t key, u64 total) {
    return (float)(0.6931471805599453 * (exponent_of(R, key) + R.S) - log((double)total));
}

struct Sum { int n; u64 w; };
struct Sum3 { u64 w[3]; };

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
 * (an odd number of words: its reads fall into banks of their own), so id order is the order of threads. What the CTAs
 * find out goes to all of them through distributed shared memory.
 *   - Top-k of a few: every quarter of a warp knows the largest key it read. The k-th largest of these is a bound that
 *     at least k tokens reach, and hardly more: they are gathered in the first CTA, sorted, cut and summed there.
 *     Two rounds through the cluster, and no work on the other tokens but reading them.
 *   - Top-p alone, or a k beyond that: a histogram of the distance to the largest logit, with counts and exact
 *     weights, tells the step in which the last kept token lies; the tokens of that step are gathered and sorted, and
 *     the key and the number of ties at which it ends goes back to all.
 *   - More tokens in one step than can be gathered (a flat row): the key is searched by exact sums, three probes a round.
 * The answer among the kept ones follows from running weights by id. Latency bounds single rows (a round through the
 * cluster is about a microsecond); rows without top-k need the 64-bit exponential of every token. */
constexpr int kT = 1024, kWarps = kT / 32;
constexpr int kBins = 2048;
constexpr int kCap = 2048;
constexpr int kMaxCluster = 16;
constexpr int kGroups = 4 * kWarps;                               /* of eight threads */
constexpr int kSel = 1024;                                        /* groups that are ranked, at most */
constexpr double kRange = 44.0 * 0.6931471805599453;              /* distances with a weight, in temperatures: 2^-44 and up */

struct Part { u64 w[3]; u64 key; int n[3]; int pad; };

struct Shared {
    Part parts[2][kMaxCluster];                                   /* what each CTA says, by turns */
    Part mine;
    u64 warp_w[kWarps];
    int warp_n[kWarps];
    Sum3 sums[kWarps];
    uint32_t my_tops[kGroups], sel[kSel];
    int gathered, pick;
    u64 found;
    union { u64 list[kCap]; u64 hist_w[kBins]; };                 /* gathered tokens; this CTA's histogram */
    union { uint32_t tops[kMaxCluster][kGroups]; uint32_t hist_n[kBins]; };   /* the groups' largest keys */
    u64 all_w[kBins];                                             /* the cluster's histogram */
    uint32_t all_n[kBins];
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t peer_addr(const void* p, int rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ void peer_put(uint32_t at, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory"); }
__device__ __forceinline__ void peer_put(uint32_t at, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ uint32_t peer_get32(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}
__device__ __forceinline__ u64 peer_get64(uint32_t at) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at));
    return v;
}
__device__ __forceinline__ void meet() {                          /* of the cluster; orders what was put before it */
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

/* the cluster, the same in every thread of it */
struct Cluster {
    Shared* s;
    int size, rank, turn;

    /* every CTA's `mine` to every CTA, and with it what the threads put before; parts are valid until the turn after next */
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
        for (int j = 0; j < 3; ++j)
#pragma unroll
            for (int o = 16; o; o >>= 1) v.w[j] += __shfl_xor_sync(0xffffffffu, v.w[j], o);
        if ((threadIdx.x & 31) == 0) s->sums[threadIdx.x >> 5] = v;
        __syncthreads();
        if (threadIdx.x < 32) {
            v = s->sums[threadIdx.x];
#pragma unroll
            for (int j = 0; j < 3; ++j)
#pragma unroll
                for (int o = 16; o; o >>= 1) v.w[j] += __shfl_xor_sync(0xffffffffu, v.w[j], o);
            if (threadIdx.x < 3) s->mine.w[threadIdx.x] = v.w[threadIdx.x];
        }
        const Part* p = exchange();
        Sum3 all{};
        for (int r = 0; r < size; ++r)
#pragma unroll
            for (int j = 0; j < 3; ++j) all.w[j] += p[r].w[j];
        return all;
    }
};

/* exclusive over the block's threads, in their order; *total over all of them */
template <typename V>
__device__ __forceinline__ V scan(V* warps, V v, V* total) {
    static_assert(kWarps == 32, "one lane a warp");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    V x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const V y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
    __syncthreads();
    if (lane == 31) warps[warp] = x;
    __syncthreads();
    V all = warps[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const V y = __shfl_up_sync(0xffffffffu, all, o); if (lane >= o) all += y; }
    *total = __shfl_sync(0xffffffffu, all, 31);
    const V before = __shfl_sync(0xffffffffu, all, max(warp - 1, 0));
    return (warp ? before : 0) + x - v;
}

/* n2 (a power of two, 32 at least) words, largest first: the first warp alone where it can keep two a lane */
__device__ __forceinline__ void sort_desc(u64* a, int n2) {
    const bool one_warp = n2 <= 64;
    __syncthreads();
    if (one_warp && threadIdx.x >= 32) { __syncthreads(); return; }
    for (int k = 2; k <= n2; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            if (one_warp) __syncwarp(); else __syncthreads();
            for (int i = threadIdx.x; i < n2 / 2; i += kT) {
                const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
                const u64 x = a[lo], y = a[hi];
                if ((x < y) == ((lo & k) == 0)) { a[lo] = y; a[hi] = x; }
            }
        }
    __syncthreads();
}

/* a token's key as it is kept: a bf16 key is the upper half of its f32 one */
template <typename K> __device__ __forceinline__ uint32_t wide(K k);
template <> __device__ __forceinline__ uint32_t wide<uint32_t>(uint32_t k) { return k; }
template <> __device__ __forceinline__ uint32_t wide<uint16_t>(uint16_t k) { return k & 0x8000u ? (uint32_t)k << 16 : k ? (uint32_t)k << 16 | 0xffffu : 0u; }

template <typename K>
__global__ void __launch_bounds__(kT) k_nucleus_row(const R3dNucleus P, const int e) {
    extern __shared__ __align__(16) uint8_t raw[];
    Shared* const s = (Shared*)raw;
    K* const keys = (K*)(raw + sizeof(Shared));
    Cluster cl;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(cl.size));
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(cl.rank));
    cl.s = s; cl.turn = 0;
    const int64_t m = blockIdx.x / cl.size;
    const int V = P.n_vocab, base = cl.rank * kT * e, tid = threadIdx.x;
    const K* const own = keys + tid * e;                          /* ids own_id ... own_id + e - 1 */
    const int own_id = base + tid * e;
    /* the peers' shared memory may be written once they have all begun: waited for below */
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

    const float t = P.temperature ? P.temperature[m * P.t_pitch] : 1.0f, p = P.top_p ? P.top_p[m * P.p_pitch] : 1.0f;
    const float low = P.min_p ? P.min_p[m * P.mp_pitch] : 0.0f, u = P.u[m * P.u_pitch];
    int k = P.top_k ? P.top_k[m * P.k_pitch] : 0;

    /* ---- read the row; its largest key, the lowest id that has it, and how many are not masked */
    u64 best_id = 0;
    uint32_t top = 0;                                             /* the largest key this thread read */
    int live = 0;
    {
        int at = -1;
        const int here = min(e, (V - base - tid + kT - 1) / kT);  /* negative: none */
#pragma unroll 8
        for (int j = 0; j < here; ++j) {
            const uint32_t key = key_of(load_x(P, m, base + j * kT + tid));
            keys[j * kT + tid] = (K)(sizeof(K) == 2 ? key >> 16 : key);
            live += key != 0;
            if (key > top) { top = key; at = j; }
        }
        for (int j = max(here, 0); j < e; ++j) keys[j * kT + tid] = 0;
        if (top) best_id = (u64)top << 32 | (0xffffffffu - (uint32_t)(base + at * kT + tid));
    }
    {
        uint32_t g = top;
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
        if ((tid & 7) == 0) s->my_tops[tid >> 3] = g;
    }
    if (tid == 0) s->gathered = 0;
    live = __reduce_add_sync(0xffffffffu, live);
#pragma unroll
    for (int o = 16; o; o >>= 1) best_id = max(best_id, (u64)__shfl_xor_sync(0xffffffffu, best_id, o));
    if ((tid & 31) == 0) { s->warp_w[tid >> 5] = best_id; s->warp_n[tid >> 5] = live; }
    __syncthreads();
    if (tid < 32) {
        best_id = s->warp_w[tid];
        live = __reduce_add_sync(0xffffffffu, s->warp_n[tid]);
#pragma unroll
        for (int o = 16; o; o >>= 1) best_id = max(best_id, (u64)__shfl_xor_sync(0xffffffffu, best_id, o));
        if (tid == 0) { s->mine.key = best_id; s->mine.n[0] = live; }
    }
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    for (int i = tid; i < kGroups * cl.size; i += kT) peer_put(peer_addr(&s->tops[cl.rank][i % kGroups], i / kGroups), s->my_tops[i % kGroups]);
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
    /* `n` tokens of this thread that `pick` says, to the list of the first CTA, in any order */
    const auto gather = [&](auto pick) {
        int n = 0, n_cta;
        for (int j = 0; j < e; ++j) { const uint32_t key = wide(own[j]); n += key && pick(key); }
        int at = scan(s->warp_n, n, &n_cta);
        if (tid == 0) {
            uint32_t from;
            asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(from) : "r"(peer_addr(&s->gathered, 0)), "r"(n_cta) : "memory");
            s->pick = (int)from;
        }
        __syncthreads();
        at += s->pick;
        for (int j = 0; j < e && n; ++j) {
            const uint32_t key = wide(own[j]);
            if (!key || !pick(key)) continue;
            if (at < kCap) peer_put(peer_addr(&s->list[at], 0), (u64)key << 32 | (0xffffffffu - (uint32_t)(own_id + j)));
            ++at; --n;
        }
    };

    /* ---- top-k of a few */
    int sel = 128;                                                /* groups to rank: at least four times k */
    while (sel < 4 * k && sel <= kSel) sel *= 2;
    if (by_k && sel <= min(kSel, kGroups * cl.size)) {
        /* the k-th largest of the groups' keys, neighbours taken together down to `sel` groups */
        const int of = kGroups * cl.size / sel, share = kT / sel;     /* threads a group */
        const uint32_t* const tops = &s->tops[0][0];
        if (tid < sel) {
            uint32_t g = 0;
            for (int j = 0; j < of; ++j) g = max(g, tops[tid * of + j]);
            s->sel[tid] = g;
        }
        __syncthreads();
        const uint32_t mine = s->sel[tid / share];
        int larger = 0;
        for (int j = tid % share * 4; j < sel; j += share * 4) {
            const uint4 o = *(const uint4*)&s->sel[j];
            larger += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
        }
        for (int o = 1; o < share; o <<= 1) larger += __shfl_xor_sync(0xffffffffu, larger, o);
        /* fewer than k groups lie above it: the least such key is the k-th largest */
        uint32_t bound = __reduce_min_sync(0xffffffffu, larger < k ? mine : 0xffffffffu);
        if ((tid & 31) == 0) s->warp_n[tid >> 5] = (int)bound;
        __syncthreads();
        bound = __reduce_min_sync(0xffffffffu, (uint32_t)s->warp_n[tid & 31]);
        gather([&](uint32_t key) { return key >= bound; });
        meet();
        const int n_top = (int)peer_get32(peer_addr(&s->gathered, 0));
        if (bound && n_top <= kCap) {
            if (!first_cta) { meet(); return; }                   /* the first CTA's memory outlives the reads of it, too */
            meet();
            int n2 = 32;
            while (n2 < n_top) n2 <<= 1;
            for (int i = n_top + tid; i < n2; i += kT) s->list[i] = 0;
            sort_desc(s->list, n2);
            const int each = (n2 + kT - 1) / kT, i0 = tid * each;
            u64 w = 0, sum, dummy;
            for (int i = i0; i < i0 + each && i < k; ++i) w += i < n_top ? weight_of(R, (uint32_t)(s->list[i] >> 32)) : 0ull;
            u64 before = scan(s->warp_w, w, &sum);
            const u64 want = by_p ? want_of(p, sum) : ~0ull;
            int kept = 0;
            w = 0;
            for (int i = i0; i < i0 + each && i < k && i < n_top; ++i) {
                const uint32_t key = (uint32_t)(s->list[i] >> 32);
                if (i && (before >= want || exponent_of(R, key) < floor_y)) break;
                const u64 x = weight_of(R, key);
                before += x; w += x; ++kept;
            }
            int n_kept;
            scan(s->warp_n, kept, &n_kept);
            scan(s->warp_w, w, &sum);
            /* by id, ascending: the low words are 0xffffffff - id; the key moves below */
            n2 = 32;
            while (n2 < n_kept) n2 <<= 1;
            for (int i = tid; i < n2; i += kT) { const u64 v2 = s->list[i]; s->list[i] = i < n_kept ? v2 << 32 | v2 >> 32 : 0ull; }
            sort_desc(s->list, n2);
            w = 0;
            const int each2 = (n2 + kT - 1) / kT, j0 = tid * each2;
            for (int i = j0; i < j0 + each2 && i < n_kept; ++i) w += weight_of(R, (uint32_t)s->list[i]);
            before = scan(s->warp_w, w, &dummy);
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
    }

    uint32_t cut = 1;                                             /* kept: keys above cut, and the first `ties` equal to it */
    int ties = V;
    if (by_k || by_p) {
        /* ---- histogram of the distance to the largest logit (key order and step order agree) */
        __syncthreads();
        for (int i = tid; i < kBins; i += kT) { s->hist_n[i] = 0; s->hist_w[i] = 0; }
        __syncthreads();
        const float mx = val_of(best), inv = (float)((kBins - 1) / kRange) / t;
        const auto bin_of = [&](uint32_t key) {
            if (R.inf) return key == best ? 0 : kBins - 1;
            const float d = __fsub_rn(mx, val_of(key)) * inv;
            return d < (float)(kBins - 1) ? (int)d : d >= (float)(kBins - 1) ? kBins - 1 : 0;     /* not a number: 0 * inf, every weight is 1 */
        };
#pragma unroll 2
        for (int j = 0; j < e; ++j) {
            const uint32_t key = wide(own[j]);
            if (!key) continue;
            const int b = bin_of(key);
            atomicAdd(&s->hist_n[b], 1u);
            if (by_p) {
                const u64 x = weight_of(R, key);
                if (x) atomicAdd(&s->hist_w[b], x);
            }
        }
        __syncthreads();
        meet();
        const int seg = kBins / cl.size;
        for (int i = tid; i < seg; i += kT) {
            const int b = cl.rank * seg + i;
            uint32_t ns[kMaxCluster], n = 0;
            u64 ws[kMaxCluster], w = 0;
#pragma unroll
            for (int r = 0; r < kMaxCluster; ++r) if (r < cl.size) { ns[r] = peer_get32(peer_addr(&s->hist_n[b], r)); ws[r] = peer_get64(peer_addr(&s->hist_w[b], r)); }
#pragma unroll
            for (int r = 0; r < kMaxCluster; ++r) if (r < cl.size) { n += ns[r]; w += ws[r]; }
            for (int r = 0; r < cl.size; ++r) { peer_put(peer_addr(&s->all_n[b], r), n); peer_put(peer_addr(&s->all_w[b], r), w); }
        }
        meet();
        static_assert(kBins == 2 * kT, "two steps a thread");
        const uint32_t n0 = s->all_n[2 * tid], n1 = s->all_n[2 * tid + 1];
        const u64 w0 = s->all_w[2 * tid], w1 = s->all_w[2 * tid + 1];
        int live2; u64 total;
        const int n_before = scan(s->warp_n, (int)(n0 + n1), &live2);
        const u64 w_before = scan(s->warp_w, w0 + w1, &total);
        /* the step whose running count (weight) first reaches `need`, and what lies before it */
        const auto step_at = [&](u64 before, u64 a, u64 b, u64 need, u64* above) {
            __syncthreads();
            if (before < need && before + a + b >= need) {
                const bool second = before + a < need;
                s->pick = 2 * tid + second;
                s->found = second ? before + a : before;
            }
            __syncthreads();
            *above = s->found;
            return s->pick;
        };
        /* the largest key c of a step such that above + the value of the step's keys from c on reaches `need`; *above
         * moves on to what lies over c. The step's tokens are gathered and sorted, or the key is searched */
        const auto key_at = [&](int step, uint32_t least, u64 need, u64* above, auto value) {
            meet();
            if (first_cta && tid == 0) s->gathered = 0;
            meet();
            gather([&](uint32_t key) { return key >= least && bin_of(key) == step; });
            meet();
            const int n = (int)peer_get32(peer_addr(&s->gathered, 0));
            if (n <= kCap) {
                if (first_cta) {
                    int n2 = 32;
                    while (n2 < n) n2 <<= 1;
                    for (int i = n + tid; i < n2; i += kT) s->list[i] = 0;
                    sort_desc(s->list, n2);
                    const int each = (n2 + kT - 1) / kT, i0 = tid * each;
                    u64 v = 0, all;
                    for (int i = i0; i < i0 + each && i < n; ++i) v += value((uint32_t)(s->list[i] >> 32));
                    u64 run = *above + scan(s->warp_w, v, &all);
                    for (int i = i0; i < i0 + each && i < n; ++i) {
                        const uint32_t key = (uint32_t)(s->list[i] >> 32);
                        const u64 x = value(key);
                        if (run < need && run + x >= need) {
                            int over = i;                          /* ties of it may stand before it */
                            u64 then = run;
                            while (over > 0 && (uint32_t)(s->list[over - 1] >> 32) == key) { --over; then -= x; }
                            s->mine.key = key; s->mine.w[0] = then;
                        }
                        run += x;
                    }
                }
                const Part* parts = cl.exchange();
                *above = parts[0].w[0];
                return (uint32_t)parts[0].key;
            }
            uint32_t lo = least, hi = best + 1;
            u64 over = 0;                                         /* of the step's keys from hi on */
            while (hi - lo > 1) {
                const uint32_t d = max(1u, (hi - lo) / 4);
                uint32_t c[3];
#pragma unroll
                for (int j = 0; j < 3; ++j) c[j] = min(lo + (j + 1) * d, hi);
                Sum3 v3{};
                for (int j = 0; j < e; ++j) {
                    const uint32_t key = wide(own[j]);
                    if (key < c[0] || key >= hi || bin_of(key) != step) continue;
                    const u64 x = value(key);
                    v3.w[0] += x;
                    if (key >= c[1]) v3.w[1] += x;
                    if (key >= c[2]) v3.w[2] += x;
                }
                v3 = cl.sum(v3);
                int j = -1;
                for (int i = 0; i < 3; ++i) if (c[i] < hi && *above + over + v3.w[i] >= need) j = i;
                if (j < 2 && c[j + 1] < hi) { over += v3.w[j + 1]; hi = c[j + 1]; }
                if (j >= 0) lo = c[j];
            }
            *above += over;
            return lo;
        };
        u64 above;
        if (by_k) {
            const int step = step_at((u64)n_before, n0, n1, (u64)k, &above);
            cut = key_at(step, 1u, (u64)k, &above, [](uint32_t) { return 1ull; });
            ties = (int)((u64)k - above);
        }
        if (by_p) {
            u64 over = total;
            if (by_k) {                                           /* the weight over the cut: whole steps, and the cut's own */
                Sum3 v3{};
                for (int j = 0; j < e; ++j) { const uint32_t key = wide(own[j]); if (key > cut) v3.w[0] += weight_of(R, key); }
                over = cl.sum(v3).w[0];
            }
            const u64 want = want_of(p, by_k ? over + (u64)ties * weight_of(R, cut) : total);
            above = over;
            if (!by_k || over >= want) {
                const int step = step_at(w_before, w0, w1, want, &above);
                cut = key_at(step, by_k ? cut : 1u, want, &above, [&](uint32_t key) { return weight_of(R, key); });
                ties = V;
            }
            const u64 one = weight_of(R, cut);
            if (one && want > above) ties = (int)min((u64)ties, (want - above + one - 1) / one);
        }
    }

    /* ---- the kept ones by id */
    int tie_rank = 0;
    if (ties < V) {
        int n = 0, n_cta;
        for (int j = 0; j < e; ++j) n += wide(own[j]) == cut;
        tie_rank = scan(s->warp_n, n, &n_cta);
        if (tid == 0) s->mine.n[0] = n_cta;
        const Part* parts = cl.exchange();
        for (int r = 0; r < cl.rank; ++r) tie_rank += parts[r].n[0];
    }
    int rank = tie_rank;
    const bool by_low = low > 0.0f;
    const auto kept = [&](uint32_t key) { return key >= cut && (key > cut || rank++ < ties) && (!by_low || exponent_of(R, key) >= floor_y); };
    u64 w = 0, w_cta;
    int n = 0, n_cta;
#pragma unroll 2
    for (int j = 0; j < e; ++j) {
        const uint32_t key = wide(own[j]);
        if (!kept(key)) continue;
        w += weight_of(R, key);
        ++n;
    }
    u64 before = scan(s->warp_w, w, &w_cta);
    scan(s->warp_n, n, &n_cta);
    if (tid == 0) { s->mine.w[0] = w_cta; s->mine.n[0] = n_cta; }
    const Part* parts = cl.exchange();
    u64 sum = 0;
    int n_kept = 0;
    for (int r = 0; r < cl.size; ++r) {
        if (r < cl.rank) before += parts[r].w[0];
        sum += parts[r].w[0]; n_kept += parts[r].n[0];
    }
    const u64 point = point_of(u, sum);
    if (before <= point && point < before + w) {
        rank = tie_rank;
        for (int j = 0; j < e; ++j) {
            const uint32_t key = wide(own[j]);
            if (!kept(key)) continue;
            before += weight_of(R, key);
            if (before <= point) continue;
            answer(P, m, own_id + j, n_kept, logprob_of(R, key, sum));
            break;
        }
    }
}

template <typename K>
int launch_row(const R3dNucleus& P, int size, int e, size_t smem, cudaStream_t st) {
    static std::atomic<bool> set[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return RAD_E_DEVICE;
    if (!set[dev].load(std::memory_order_relaxed)) {
        if (cudaFuncSetAttribute(k_nucleus_row<K>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess ||
            cudaFuncSetAttribute(k_nucleus_row<K>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return RAD_E_DEVICE;
        set[dev].store(true, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)P.rows * (unsigned)size); cfg.blockDim = dim3(kT); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)size; at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_nucleus_row<K>, P, e) == cudaSuccess && cudaGetLastError() == cudaSuccess ? RAD_OK : RAD_E_DEVICE;
}

} /* namespace */

int launch_nucleus(const R3dNucleus& p, cudaStream_t st) {
    R3dNucleus P = p;
    int bits = 0;
    while ((1ll << bits) < (long long)p.n_vocab) ++bits;
    P.shift = 62 - bits < 50 ? 62 - bits : 50;
    count_launch();
    const int ksz = p.x_dtype == RAD_F32 ? 4 : 2;
    int size = 1, e = 0;
    size_t smem = 0;
    for (;; size *= 2) {
        e = ((p.n_vocab + kT * size - 1) / (kT * size)) | 1;
        smem = sizeof(Shared) + (size_t)kT * e * ksz;
        if (size == kMaxCluster) break;
        if (smem <= 220 * 1024 && ((long long)p.rows * size >= 148 || kT * e <= 4096)) break;
    }
    if (getenv("DEV_CL")) { size = atoi(getenv("DEV_CL")); e = ((p.n_vocab + kT * size - 1) / (kT * size)) | 1; smem = sizeof(Shared) + (size_t)kT * e * ksz; }
    if (smem > 220 * 1024) {
        k_nucleus_long<<<(unsigned)p.rows, 1024, 0, st>>>(P);
        return cudaGetLastError() == cudaSuccess ? RAD_OK : RAD_E_DEVICE;
    }
    return ksz == 4 ? launch_row<uint32_t>(P, size, e, smem, st) : launch_row<uint16_t>(P, size, e, smem, st);
}

} /* namespace r3d */

/* kern_nucleus.cu -- sample_nucleus: temperature, top-k, top-p, min-p and a given random number, one token a row.
 *
 * With mx the row's largest logit and T its temperature, token i has the weight w_i = 2^((x_i - mx) log2(e) / T) in
 * (0, 1]. The tokens are ordered by value, descending, ties to the lower id (the order of row_topk and
 * sample_argmax); each filter keeps a first part of that order: top-k its first k, top-p the shortest part whose
 * weight reaches p times the weight that top-k left, min-p those with w_i >= min_p; the first token always stays.
 * The answer is the first kept token, by ascending id, whose running weight exceeds u times the kept weight.
 *
 * Weights are whole numbers of 2^-S (S the largest for which a row's sum fits 62 bits; 44 at 151936 tokens). Their
 * sums are exact in any order, so the answer depends neither on the order of threads nor on how a row is split. A weight
 * is off by at most 2.3 2^-39 of itself and half a unit (mostly by a fifth of that), so the answer is a 64-bit
 * computation's except where that one's running sum lies within about 2^-39 of the kept weight of a border.
 *
 * -inf and NaN logits are masked: never kept. A row with nothing left reports token -1, kept 0, logprob -inf.
 */
#include <atomic>
#include <cmath>
#include <cstddef>
#include "r3d_kernels.h"
#include "r3d_numerics.cuh"

namespace r3d {

bool tc_pdl_on();                     /* kern_tc.cu: false under R3D_NO_PDL */
int tc_sm_count();

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
/* 2^y as a whole number of 2^-S, y = (x - mx) log2(e) / T. One 64-bit multiply-add makes 128 y in fixed point: the high
 * word its whole part, the low word the fraction r. 2^y is then 2^(whole / 128), by table and exponent, times
 * 1 + r (C1 + r (C2 + r C3)), the polynomial that meets (2^(r / 128) - 1) / r at the three Chebyshev points of [0, 1], in
 * 32-bit products of units of 2^-39; one more 64-bit multiply-add rounds by adding 2^52. A row's largest logit weighs 2^S
 * exactly. No case is tested for: NaN (what is masked) and what lies far below give a high word out of range, which is
 * held at a weight of a quarter. 22 cycles of a scheduler for a warp's 32; with twelve operations in 64 bits, or with
 * whole numbers alone (64-bit shifts, half as fast as products), 60. */
struct Powers { double of[128]; };                                /* 2^(-i / 128) */
constexpr Powers make_powers() {
    Powers t{};
    for (int i = 0; i < 128; ++i) {
        const double x = -0.6931471805599453 * i / 128.0;
        double sum = 1.0, term = 1.0;
        for (int j = 1; j < 30; ++j) { term *= x / j; sum += term; }
        t.of[i] = sum;
    }
    return t;
}
__device__ const Powers kPowers = make_powers();

struct Weigh {
    double mx, c;                                                 /* the largest logit; 128 log2(e) / T */
    float top;                                                    /* the largest again */
    int S;
    bool inf;
    __device__ __forceinline__ u64 of(const double* powers, float x) const {
        if (inf) return x == top ? 1ull << S : 0ull;
        const double z = fma((double)x - mx, c, 1572864.0);       /* 1.5 * 2^20: the fraction is the low word */
        const uint32_t down = min(0x41380000u - (uint32_t)__double2hiint(z), (uint32_t)(S + 2) << 7);
        const uint32_t r = (uint32_t)__double2loint(z);
        const uint32_t q = __umulhi(r, 2977044473u + __umulhi(r, 8060653u + __umulhi(r, 14580u)));
        const double a = powers[down & 127];
        const double power = __hiloint2double(__double2hiint(a) + (S << 20) - (int)((down & ~127u) << 13), __double2loint(a));
        const double more = __longlong_as_double((long long)((u64)q * 8192u + 0x3ff0000000000000ull));
        return (u64)__double_as_longlong(fma(more, power, 4503599627370496.0)) - 0x4330000000000000ull;
    }
};

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

/* rows too long for a cluster's shared memory (16 CTAs hold 778 thousand f32 or 1.55 million bf16 tokens): one block a row,
 * read again for each step of the searches, some hundred times: 3 x 900001 f32, top-k 50 and top-p, take 22 ms (1 x 1300000
 * bf16, in a cluster, 27 us). */
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
    const Weigh weigh{R.mx, R.c * 128.0, val_of(best), R.S, R.inf};
    const auto weight_of = [&](uint32_t key) { return weigh.of(kPowers.of, val_of(key)); };

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
        const u64 over = sum_if([&](Sum& s, uint32_t key, int) { if (key > cut) s.w += weight_of(key); }).w;
        const u64 total = over + (cut > 1 ? (u64)ties * weight_of(cut) : sum_if([&](Sum& s, uint32_t key, int) { if (key == cut) s.w += weight_of(key); }).w);
        const u64 want = want_of(p, total);
        if (over >= want) {
            cut = search([&](uint32_t c) { return sum_if([&](Sum& s, uint32_t key, int) { if (key >= c) s.w += weight_of(key); }).w >= want; });
            ties = V;
        }
        const u64 above = sum_if([&](Sum& s, uint32_t key, int) { if (key > cut) s.w += weight_of(key); }).w;
        const u64 one = weight_of(cut);
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
    const Sum all = sum_if([&](Sum& s, uint32_t key, int i) { if (keep(key, i)) { ++s.n; s.w += weight_of(key); } });
    const float u = P.u[m * P.u_pitch];
    const u64 at = point_of(u, all.w);
    int lo = 0, hi = V - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (sum_if([&](Sum& s, uint32_t key, int i) { if (i <= mid && keep(key, i)) s.w += weight_of(key); }).w > at) hi = mid; else lo = mid + 1;
    }
    if (threadIdx.x == 0) answer(P, m, lo, all.n, logprob_of(R, key_at(lo), all.w));
}

/* ------------------------------------------------------------------ a cluster a row
 * The row is read once, by 16 bytes, as ordered keys into the shared memory of the cluster's CTAs; for what goes by id a
 * thread owns neighbouring words of keys, so id order is the order of threads. What the CTAs find out goes to all of them
 * through distributed shared memory.
 *   - Top-k of a few: every one to eight threads know the largest key they read. A bound that k of these reach, and hardly
 *     more, is one that at least k tokens reach: these are gathered in the first CTA, which orders them, cuts and sums. Two
 *     rounds through the cluster, and no work on the other tokens but reading them.
 *   - Top-p alone, or a k beyond that: a histogram of the distance to the largest logit gives the exact step of the k-th
 *     token, and for top-p a window of steps in which its end lies by the steps' middle weights; one pass of exact sums
 *     proves the window (or moves it). If it and what lies over it are a few tokens, they end like a top-k of as many; else
 *     the tokens of the window are gathered and ranked, and the key and the number of ties at which the kept ones end go
 *     back to all.
 *   - More tokens in a window than can be gathered (a flat row): the key is searched by exact sums, three probes a round.
 * The answer among the kept ones follows from running weights by id.
 * Latency bounds single rows (1 x 151936: top-k 50 13.5 us, top-p 28.6): a round through the cluster is about a
 * microsecond, and so is the first run through a few hundred instructions, which is why what is used more than once is a
 * call here. Batches are bound by instructions, half of the issue slots (64 x 151936 bf16, settings of their own: 64 us).
 * Rows without top-k need the exponential of every token. (An atomic add of 64 bits in shared memory takes ten times one of
 * 32: a histogram of exact weights cost 12 of 37 us.) */
constexpr int kT = 512, kWarps = kT / 32;
constexpr int kGroups = 1024;                                     /* of threads, in the cluster, at most */
constexpr int kBins = 1024, kBinsEach = kBins / kT;
constexpr int kCap = 1024;                                        /* gathered tokens, at most */
constexpr int kMaxCluster = 16;
constexpr double kRange = 26.0;                                   /* halvings of weight over the steps; the last takes the rest */

struct Part { u64 w[3]; u64 key; };

struct Shared {
    Part parts[2][kMaxCluster];                                   /* what each CTA says, by turns */
    Part mine;
    double c, floor_y, drop;                                      /* log2(e) / T; min-p as an exponent, and in logits */
    Powers powers;
    Weigh weigh;
    u64 warp_w[kWarps];
    int warp_n[kWarps];
    Sum3 sums[kWarps];
    uint32_t my_tops[kT];
    int gathered, pick, from;
    uint32_t edge[2];
    u64 list[kCap], weight[kCap];                                 /* gathered tokens, key << 32 | ~id; their values */
    union { uint32_t tops[kGroups]; uint32_t hist[kBins]; };   /* the groups' largest keys; this CTA's histogram */
    uint32_t upto[kBins];                                         /* the cluster's, summed up to each step */
};

/* the kernel's shared memory: its state, then the keys. The calls name it themselves: a pointer handed on would be read as
 * one to any memory */
extern __shared__ __align__(16) uint8_t raw[];
__device__ __forceinline__ Shared* shared() { return (Shared*)raw; }
__device__ __forceinline__ const uint32_t* key_words() { return (const uint32_t*)(raw + sizeof(Shared)); }

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
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}
__device__ __forceinline__ void meet() {                          /* of the cluster; orders what was put before it */
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll 1
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

static_assert(sizeof(Shared) % 16 == 0, "the keys behind it are written by 16 bytes");
static_assert(offsetof(Shared, parts) % 8 == 0 && offsetof(Shared, mine) % 8 == 0 && sizeof(Part) % 8 == 0, "sent by 8 bytes");
/* the cluster, the same in every thread of it */
struct Cluster {
    int size, rank, turn;

    /* every CTA's `mine` to every CTA, and with it what the threads put before; parts are valid until the turn after next */
    __device__ __forceinline__ const Part* exchange() {
        const Part* p = shared()->parts[turn];
        send(size, rank, turn);
        turn ^= 1;
        return p;
    }
    __device__ static __noinline__ void send(int size, int rank, int turn) {
        Shared* const s = shared();
        __syncthreads();
        constexpr int kWords = sizeof(Part) / 8;
        for (int i = threadIdx.x; i < size * kWords; i += kT)
            peer_put(peer_addr((u64*)&s->parts[turn][rank] + i % kWords, i / kWords), ((const u64*)&s->mine)[i % kWords]);
        meet();
    }
    /* sums over the cluster */
    __device__ __forceinline__ Sum3 sum(Sum3 v) {
        block_sums(v.w[0], v.w[1], v.w[2]);
        const Part* p = exchange();
        Sum3 all{};
#pragma unroll 1
        for (int r = 0; r < size; ++r) { all.w[0] += p[r].w[0]; all.w[1] += p[r].w[1]; all.w[2] += p[r].w[2]; }
        return all;
    }
    __device__ static __noinline__ void block_sums(u64 a, u64 b, u64 c) {
        Shared* const s = shared();
        a = warp_sum(a); b = warp_sum(b); c = warp_sum(c);
        if ((threadIdx.x & 31) == 0) s->sums[threadIdx.x >> 5] = Sum3{{a, b, c}};
        __syncthreads();
        if (threadIdx.x < 3) {
            u64 v = 0;
            for (int i = 0; i < kT / 32; ++i) v += s->sums[i].w[threadIdx.x];
            s->mine.w[threadIdx.x] = v;
        }
    }
};

/* exclusive over the block's threads, in their order; *total over all of them */
template <typename V>
__device__ __noinline__ V scan(V v, V* total) {
    V* const warps = sizeof(V) == 8 ? (V*)shared()->warp_w : (V*)shared()->warp_n;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    V x = v;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) { const V y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
    __syncthreads();
    if (lane == 31) warps[warp] = x;
    __syncthreads();
    V all = lane < kWarps ? warps[lane] : (V)0;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) { const V y = __shfl_up_sync(0xffffffffu, all, o); if (lane >= o) all += y; }
    *total = __shfl_sync(0xffffffffu, all, 31);
    const V before = __shfl_sync(0xffffffffu, all, max(warp - 1, 0));
    return (warp ? before : (V)0) + x - v;
}

/* For the i-th of n gathered tokens (i = the thread's place among groups of `share` threads): how many stand before it in
 * the order, and the sum of their values. */
__device__ __noinline__ int count_before(int n, int i, int share) {
    const u64* const list = shared()->list;
    const u64 a = i < n ? list[i] : ~0ull;
    int r = 0;
#pragma unroll 4
    for (int j = threadIdx.x % share; j < n; j += share) r += list[j] > a;
#pragma unroll 1
    for (int o = 1; o < share; o <<= 1) r += __shfl_xor_sync(0xffffffffu, r, o);
    return r;
}
__device__ __noinline__ u64 sum_before(int n, int i, int share) {
    const u64* const list = shared()->list;
    const u64* const weight = shared()->weight;
    const u64 a = i < n ? list[i] : ~0ull;
    u64 r = 0;
#pragma unroll 4
    for (int j = threadIdx.x % share; j < n; j += share) r += list[j] > a ? weight[j] : 0;
#pragma unroll 1
    for (int o = 1; o < share; o <<= 1) r += __shfl_xor_sync(0xffffffffu, r, o);
    return r;
}
/* threads for each of n tokens, a power of two up to a warp */
__device__ __forceinline__ int share_of(int n) {
    int share = 32;
    while (share > 1 && n * share > kT) share >>= 1;
    return share;
}

/* a token's key as it is kept: a bf16 key is the upper half of its f32 one */
template <typename K> __device__ __forceinline__ uint32_t wide(K k);
template <> __device__ __forceinline__ uint32_t wide<uint32_t>(uint32_t k) { return k; }
template <> __device__ __forceinline__ uint32_t wide<uint16_t>(uint16_t k) { return k & 0x8000u ? (uint32_t)k << 16 : k ? (uint32_t)k << 16 | 0xffffu : 0u; }

/* f(key as it is kept, its value, its id in the CTA) of a word of keys; what is masked, or lies around the row, has key 0
 * and is not a number */
template <typename K, typename F>
__device__ __forceinline__ void word_of(const uint32_t* words, int lead, int i, F f) {
    const uint32_t w = words[i];
    if (sizeof(K) == 2) {
        uint32_t sign;                                            /* of both halves; the keys' map the other way round */
        asm("prmt.b32 %0, %1, 0, 0xbb99;" : "=r"(sign) : "r"(w));
        const uint32_t v = w ^ (~sign | 0x80008000u);
        f((K)w, __uint_as_float(v << 16), 2 * i - lead);
        f((K)(w >> 16), __uint_as_float(v & 0xffff0000u), 2 * i + 1 - lead);
    } else f((K)w, val_of(w), i - lead);
}
template <typename K, typename F>
__device__ __forceinline__ void each_of(const uint32_t* words, int lead, int e, F f) {
    constexpr int kUnroll = sizeof(K) == 2 ? 2 : 4;
#pragma unroll kUnroll
    for (int i = threadIdx.x; i < kT * e; i += kT) word_of<K>(words, lead, i, f);
}
/* a thread's own words, by id: neighbouring ones, an odd number (banks of their own) */
template <typename K, typename F>
__device__ __forceinline__ void own_of(const uint32_t* words, int lead, int e, F f) {
    constexpr int kUnroll = sizeof(K) == 2 ? 2 : 4;
    const uint32_t* const mine = words + threadIdx.x * e;
#pragma unroll kUnroll
    for (int i = 0; i < e; ++i) word_of<K>(mine, lead, i, f);
}
/* The passes that weigh many are calls, for registers of their own: inside the kernel they took twice the time.
 * Over this thread's words: the weights of the keys from `over` on (0: of all), of those from `high` and from `low` on. */
template <typename K>
__device__ __noinline__ Sum3 weigh_all(int e, uint32_t over, uint32_t high, uint32_t low) {
    const Weigh weigh = shared()->weigh;
    Sum3 v{};
    each_of<K>(key_words(), 0, e, [&](K key, float x, int) {
        if (key < over) return;
        const u64 w = weigh.of(shared()->powers.of, x);
        v.w[0] += w;
        if (key >= low) {
            v.w[2] += w;
            if (key >= high) v.w[1] += w;
        }
    });
    return v;
}
/* Of this thread's own words: how many keys are kept, and their weight. `rank`: of its first key `over` - 1 among those. */
template <typename K>
__device__ __noinline__ Sum weigh_kept(int e, uint32_t least, uint32_t over, int rank, int ties) {
    const Weigh weigh = shared()->weigh;
    Sum v{0, 0};
    own_of<K>(key_words(), 0, e, [&](K key, float x, int) {
        if (key < least || (key < over && rank++ >= ties)) return;
        ++v.n;
        v.w += weigh.of(shared()->powers.of, x);
    });
    return v;
}

/* key_of by the integer pipe alone: +0 folds -0; the keys of what is not masked lie next to each other */
__device__ __forceinline__ uint32_t key_fast(uint32_t bits) {
    const int v = __float_as_int(__uint_as_float(bits) + 0.0f);
    const uint32_t k = (uint32_t)v ^ ((uint32_t)(v >> 31) | 0x80000000u);
    return k - 0x00800000u <= 0xff000000u ? k : 0u;               /* from the least number to +inf */
}

/* The row of the q-th cluster, those that need every token's weight (top-p without a small top-k) first: they take three
 * times as long, and begun in the last wave they end it alone. At most kT rows. */
constexpr int kSmallK = 256;
__device__ __forceinline__ int long_rows_first(const R3dNucleus& P, int q) {
    Shared* const s = shared();
    const int i = threadIdx.x, lane = i & 31;
    bool heavy = false;
    if (i < P.rows) {
        const float p = P.top_p[i * P.p_pitch];
        const int k = P.top_k ? P.top_k[i * P.k_pitch] : 0;
        heavy = p < 1.0f && p > 0.0f && (k <= 0 || k > kSmallK) && !(P.temperature && P.temperature[i * P.t_pitch] <= 0.0f);
    }
    const uint32_t in_warp = __ballot_sync(0xffffffffu, heavy);
    if (lane == 0) s->warp_n[i >> 5] = __popc(in_warp);
    const int all = __syncthreads_count(heavy);
    int before = __popc(in_warp & ((1u << lane) - 1u));
    for (int w = 0; w < i >> 5; ++w) before += s->warp_n[w];
    if (i < P.rows && (heavy ? before : all + i - before) == q) s->pick = i;
    __syncthreads();
    return s->pick;
}

/* the least key with exponent_of(key) >= floor_y, the same in every lane: keys and exponents have one order, and `best`
 * is one of them */
__device__ __noinline__ uint32_t least_kept(Row R, uint32_t best, double floor_y) {
    uint32_t lo = 0x00800000u, hi = best;                         /* from the least number on */
#pragma unroll 1
    while (lo < hi) {
        const uint32_t step = (hi - lo + 31) / 32, at = lo + (threadIdx.x & 31) * step;
        const uint32_t yes = __ballot_sync(0xffffffffu, at >= hi || exponent_of(R, at) >= floor_y);
        if (!yes) { lo += 31 * step + 1; continue; }
        const int first = __ffs(yes) - 1;                         /* the lane before says no, this one yes */
        hi = min(hi, lo + first * step);
        if (first) lo += (first - 1) * step + 1;
    }
    return hi;
}

template <typename K>
__global__ void __launch_bounds__(kT, 2) k_nucleus_row(const R3dNucleus P, const int e, const int early, const int reorder) {
    /* the next kernel may begin to launch, unless CTAs of this one still wait for room; the previous one's results are there */
    if (early) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    Shared* const s = shared();
    constexpr int kEach = 16 / (int)sizeof(K), kPer = 4 / (int)sizeof(K);     /* values of 16 bytes and of four, as logits and as keys */
    Cluster cl;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(cl.size));
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(cl.rank));
    cl.turn = 0;
    const int64_t m = reorder ? long_rows_first(P, blockIdx.x / cl.size) : blockIdx.x / cl.size;
    const int V = P.n_vocab, span = kT * e * kPer - kEach, base = cl.rank * span, tid = threadIdx.x;      /* this CTA's ids */
    /* the keys lie to the 16-byte grid as the logits do, which takes up to 16 bytes more than the ids' own */
    const K* const x = (const K*)P.logits + m * P.x_pitch + base;
    const int lead = (int)((uintptr_t)x & 15) / (int)sizeof(K);
    K* const keys = (K*)(raw + sizeof(Shared)) + lead;
    const uint32_t* const words = key_words();
    /* the peers' shared memory may be written once they have all begun: waited for below */
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

    const float t = P.temperature ? P.temperature[m * P.t_pitch] : 1.0f, p = P.top_p ? P.top_p[m * P.p_pitch] : 1.0f;
    const float low = P.min_p ? P.min_p[m * P.mp_pitch] : 0.0f, u = P.u[m * P.u_pitch];
    int k = P.top_k ? P.top_k[m * P.k_pitch] : 0;

    const int mine_groups = min(kT, kGroups / cl.size);           /* 1, 1, 2, 4 or 8 threads each */

    /* ---- read the row; its largest key, the lowest id that has it, and how many are not masked */
    u64 best_id = 0;
    int live = 0;
    {
        uint32_t top = 0;                                         /* the largest key this thread read */
        int at = -1;
        const int here = min(span, V - base);                   /* ids of this CTA; negative: none */
        const auto take = [&](uint32_t bits, int i) {
            const uint32_t key = key_fast(bits);
            live += key != 0;
            if (key > top) { top = key; at = i; }
            return key;
        };
        const auto take_one = [&](int i) {
            const uint32_t bits = i < here ? (uint32_t)x[i] << (sizeof(K) == 2 ? 16 : 0) : 0xff800000u;
            keys[i] = (K)(take(bits, i) >> (sizeof(K) == 2 ? 16 : 0));
        };
        if (e * kPer < 16) {                                      /* few: every thread reads some, for the groups below */
#pragma unroll 4
            for (int i = tid; i < span; i += kT) take_one(i);
        } else {
            constexpr int kFlight = 4;                            /* loads of 16 bytes on their way at a time */
#pragma unroll 1
            for (int i0 = tid * kEach - lead; i0 < span; i0 += kFlight * kT * kEach) {
                uint4 w[kFlight];
#pragma unroll
                for (int j = 0; j < kFlight; ++j) {
                    const int i = i0 + j * kT * kEach;
                    if (i >= 0 && i + kEach <= here) w[j] = *(const uint4*)(x + i);
                }
#pragma unroll
                for (int j = 0; j < kFlight; ++j) {
                    const int i = i0 + j * kT * kEach;
                    if (i >= 0 && i + kEach <= here) {
                        uint32_t* const u = (uint32_t*)&w[j];
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            if (sizeof(K) == 2) {
                                const uint32_t a = take(u[c] << 16, i + 2 * c), b = take(u[c] & 0xffff0000u, i + 2 * c + 1);
                                u[c] = __byte_perm(a, b, 0x7632);
                            } else u[c] = take(u[c], i + c);
                        }
                        *(uint4*)(keys + i) = w[j];
                    } else if (i >= 0 && i >= here && i + kEach <= span) {
                        *(uint4*)(keys + i) = make_uint4(0u, 0u, 0u, 0u);
                    } else {
#pragma unroll 1
                        for (int c = 0; c < kEach; ++c) if (i + c >= 0 && i + c < span) take_one(i + c);
                    }
                }
            }
        }
        if (top) best_id = (u64)top << 32 | (0xffffffffu - (uint32_t)(base + at));
#pragma unroll 1
        for (int o = 1; o < kT / mine_groups; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (tid % (kT / mine_groups) == 0) s->my_tops[tid / (kT / mine_groups)] = top;
    }
    if (tid < lead) keys[tid - lead] = 0;
    if (tid < kEach - lead) keys[span + tid] = 0;
    if (tid < 128) s->powers.of[tid] = kPowers.of[tid];
    live = __reduce_add_sync(0xffffffffu, live);
#pragma unroll 1
    for (int o = 16; o; o >>= 1) best_id = max(best_id, (u64)__shfl_xor_sync(0xffffffffu, best_id, o));
    if ((tid & 31) == 0) { s->warp_w[tid >> 5] = best_id; s->warp_n[tid >> 5] = live; }
    __syncthreads();
    if (tid < 32) {
        best_id = tid < kWarps ? s->warp_w[tid] : 0;
        live = __reduce_add_sync(0xffffffffu, tid < kWarps ? s->warp_n[tid] : 0);
#pragma unroll 1
        for (int o = 16; o; o >>= 1) best_id = max(best_id, (u64)__shfl_xor_sync(0xffffffffu, best_id, o));
        if (tid == 0) { s->mine.key = best_id; s->mine.w[0] = (u64)live; s->gathered = 0; }
    } else if (tid < 64) {                                        /* one warp: a quotient and a logarithm in 64 bits */
        const double c = t > 0.0f ? 1.4426950408889634 / (double)t : 0.0, y = floor_of(low);
        if (tid == 32) { s->c = c; s->floor_y = y; s->drop = y / c; }
    }
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
#pragma unroll 1
    for (int i = tid; i < mine_groups * cl.size; i += kT)
        peer_put(peer_addr(&s->tops[cl.rank * mine_groups + i % mine_groups], i / mine_groups), s->my_tops[i % mine_groups]);
    {
        const Part* parts = cl.exchange();
        best_id = 0; live = 0;
#pragma unroll 1
        for (int r = 0; r < cl.size; ++r) { best_id = max(best_id, parts[r].key); live += (int)parts[r].w[0]; }
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
    Row R;
    R.c = s->c; R.mx = (double)val_of(best); R.inf = isinf(val_of(best)); R.S = P.shift;
    const bool by_k = k < live, by_p = p < 1.0f;
    if (tid == 0) s->weigh = Weigh{R.mx, R.c * 128.0, val_of(best), R.S, R.inf};
    __syncthreads();
    const auto weight = [&](uint32_t key) { return s->weigh.of(s->powers.of, val_of(key)); };
    const auto word = [&](int i, auto f) { word_of<K>(words, lead, i, f); };
    const auto each = [&](auto f) { each_of<K>(words, lead, e, f); };     /* of all, in any order */
    /* the least kept form that is `key` or more: (a bf16 key stands for one of 2^16) */
    const auto least_form = [&](uint32_t key) -> uint32_t {
        if (sizeof(K) == 4) return key;
        const uint32_t h = key >> 16;
        return wide((K)h) >= key ? h : h + 1;
    };
    /* the least key that min-p keeps: among the 32 next to where the bound falls, if it lies between two of them. Next to 0,
     * where f32 numbers lie closer together than x - mx is known, they may all be on one side of it (and T without end
     * keeps all keys): then it is searched, a warp looking at 32 keys a step. The largest logit is always kept. */
    uint32_t least_key = 1;
    if (low > 0.0f) {
        const double floor_y = s->floor_y;
        const uint32_t guess = R.inf || !(R.c > 0.0) ? best : key_of((float)fmax(R.mx + s->drop, -3.4e38));
        const uint32_t mine = max(min(guess, best), 32u) - 16 + (tid & 31);
        const uint32_t yes = __ballot_sync(0xffffffffu, mine >= best || exponent_of(R, mine) >= floor_y);
        least_key = min(best, mine - (tid & 31) + __ffs(yes) - 1);
        if (!yes || (yes & 1u)) least_key = R.inf ? best : least_kept(R, best, floor_y);
    }
    /* the tokens whose keys are `from` or more and below `to`, to the lists of the first `copies` CTAs, in any order */
    const auto gather = [&](int copies, uint32_t from, uint32_t to) {
        const uint32_t low_form = max(least_form(from), 1u), range = max(least_form(to), low_form) - low_form;
        int n = 0, n_cta;
        each([&](K key, float, int) { n += key - low_form < range; });
        int at = scan(n, &n_cta);
        if (tid == 0) {
            uint32_t first;
            asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(first) : "r"(peer_addr(&s->gathered, 0)), "r"(n_cta) : "memory");
            s->from = (int)first;
        }
        __syncthreads();
        at += s->from;
        if (n)
            each([&](K key, float, int i) {
                if (key - low_form >= range) return;
                if (at < kCap)
                    for (int r = 0; r < copies; ++r) peer_put(peer_addr(&s->list[at], r), (u64)wide(key) << 32 | (0xffffffffu - (uint32_t)(base + i)));
                ++at;
            });
    };

    /* what the first CTA has gathered if that is all that can be kept, at most a thread each: how many tokens, how many of
     * them top-k lets through, and the weight that top-p wants (0: of those) */
    int few = -1, most = 0;
    u64 want_few = 0;
    /* ---- top-k of a few */
    int sel = 128;                                                /* groups: at least twice k, which lets through 1.4 k tokens */
    while (sel < 2 * k && sel <= kT) sel *= 2;
    static_assert(2 * kSmallK == kT, "what `sel` lets through");
    if (by_k && sel <= kT) {
        /* a bound that k groups reach, and at most an eighth more: neighbours are taken together down to `sel` groups, one a
         * thread, and every step of the search is one barrier that counts */
        const int of = mine_groups * cl.size / sel;
        uint32_t g = 0;
        if (tid < sel)
#pragma unroll 1
            for (int j = 0; j < of; ++j) g = max(g, s->tops[tid * of + j]);
        uint32_t bound = __reduce_min_sync(0xffffffffu, tid < sel ? g : best);      /* the least group: all reach it */
        if ((tid & 31) == 0) s->warp_n[tid >> 5] = (int)bound;
        __syncthreads();
        bound = __reduce_min_sync(0xffffffffu, (tid & 31) < kWarps ? (uint32_t)s->warp_n[tid & 31] : best);
        uint32_t past = best + 1;
        for (int have = sel; have > k + k / 8 && past - bound > 1;) {
            const uint32_t mid = bound + (past - bound) / 2;
            const int n = __syncthreads_count(g >= mid);
            if (n >= k) { bound = mid; have = n; } else past = mid;
        }
        gather(1, bound, best + 1);
        meet();
        const int n = (int)peer_get(peer_addr(&s->gathered, 0));
        meet();                                                   /* all have read it */
        if (bound && n <= kT) {
            few = n;
            most = k;
        }
    }

    uint32_t cut = 1;                                             /* kept: keys above cut, and the first `ties` equal to it */
    int ties = V;
    if (few < 0 && (by_k || by_p)) {
        /* ---- histogram of the distance to the largest logit (key order and step order agree) */
        const float mx = val_of(best), inv = (float)((kBins - 1) / kRange * 1.4426950408889634) / t;
        const auto bin_of = [&](float x) {
            if (R.inf) return x == mx ? 0 : kBins - 1;
            const float d = __fsub_rn(mx, x) * inv;
            return d < (float)(kBins - 1) ? (int)d : d >= (float)(kBins - 1) ? kBins - 1 : 0;     /* not a number: 0 * inf, every weight is 1 */
        };
        __syncthreads();
        for (int i = tid; i < kBins; i += kT) s->hist[i] = 0;
        __syncthreads();
        each([&](K key, float x, int) { if (key) atomicAdd(&s->hist[bin_of(x)], 1u); });
        meet();
        /* each CTA sums its share of the steps, `size` threads a step, and tells all */
        const int seg = kBins / cl.size;
#pragma unroll
        for (int i = tid; i < kBins; i += kT) {
            const int b = cl.rank * seg + i / cl.size, r = i % cl.size;
            uint32_t n = peer_get(peer_addr(&s->hist[b], r));
#pragma unroll 1
            for (int o = 1; o < cl.size; o <<= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
            peer_put(peer_addr(&s->upto[b], r), n);
        }
        meet();
        uint32_t cnt[kBinsEach], n_own = 0;
        float est[kBinsEach], est_own = 0.0f;
        const float per_bin = (float)(kRange / (kBins - 1));       /* halvings a step */
#pragma unroll
        for (int j = 0; j < kBinsEach; ++j) {
            cnt[j] = s->upto[kBinsEach * tid + j];
            est[j] = (float)cnt[j] * exp2f(-per_bin * ((float)(kBinsEach * tid + j) + 0.5f));
            n_own += cnt[j]; est_own += est[j];
        }
        int dummy;
        int upto = scan((int)n_own, &dummy);
#pragma unroll
        for (int j = 0; j < kBinsEach; ++j) {
            const int before = upto;
            upto += (int)cnt[j];
            if (by_k && before < k && upto >= k) s->pick = kBinsEach * tid + j;       /* the step of the k-th token */
            s->upto[kBinsEach * tid + j] = (uint32_t)upto;
        }
        __syncthreads();
        const int k_step = s->pick;
        const auto count_to = [&](int b) { return b > 0 ? (int)s->upto[b - 1] : 0; };      /* tokens in steps below b */

        /* the least key in a step below b, by the warps' first and second, for two steps at once: a warp looks at 32 keys */
        const auto edges = [&](int b0, int b1) {
            __syncthreads();
            if (tid < 64) {
                const int b = tid < 32 ? b0 : b1;
                uint32_t lo = 0x00800000u, hi = best + 1;         /* from the least number on; the largest logit is in step 0 */
                if (b <= 0) lo = hi;
                else if (b >= kBins) { lo = 1; hi = 1; }
#pragma unroll 1
                while (lo < hi) {
                    const uint32_t step = (hi - lo + 31) / 32, at = lo + (tid & 31) * step;
                    const uint32_t yes = __ballot_sync(0xffffffffu, at >= hi || bin_of(val_of(at)) < b);
                    if (!yes) { lo += 31 * step + 1; continue; }
                    const int first = __ffs(yes) - 1;             /* the lane before says no, this one yes */
                    hi = min(hi, lo + first * step);
                    if (first) lo += (first - 1) * step + 1;
                }
                if ((tid & 31) == 0) s->edge[tid >> 5] = lo;
            }
            __syncthreads();
        };
        /* the largest key c of the keys [low_key, high_key) such that above + the value of those >= c reaches `need`;
         * *above moves on to what lies over c. The `many` tokens are gathered and ranked, or the key is searched */
        const auto key_at = [&](uint32_t low_key, uint32_t high_key, int many, u64 need, u64* above, bool ones) {
            const auto value = [&](float x) { return ones ? 1ull : s->weigh.of(s->powers.of, x); };
            /* ranking takes as many steps as the square of their number over the CTAs: a thousand on 4, 512 on one */
            if (many <= kCap && many * many <= cl.size << 18) {
                if (first_cta && tid == 0) s->gathered = 0;
                meet();
                gather(cl.size, low_key, high_key);
                if (tid == 0) s->mine.key = 0;
                meet();
                /* each CTA ranks its share of them */
                const int n = (int)peer_get(peer_addr(&s->gathered, 0));
                for (int i = tid; i < n; i += kT) s->weight[i] = value(val_of((uint32_t)(s->list[i] >> 32)));
                __syncthreads();
                const int here = (n + cl.size - 1) / cl.size, sh = share_of(here);
#pragma unroll 1
                for (int j = tid / sh; j - tid / sh < here; j += kT / sh) {
                    const int i = j < here ? cl.rank * here + j : n;
                    const u64 run = *above + sum_before(n, i, sh);
                    if (i < n && tid % sh == 0 && run < need && run + s->weight[i] >= need) s->mine.key = s->list[i] >> 32;
                }
                const Part* parts = cl.exchange();
                uint32_t found = 0;
#pragma unroll 1
                for (int r = 0; r < cl.size; ++r) found = max(found, (uint32_t)parts[r].key);
                u64 larger = 0, all;
                for (int i = tid; i < n; i += kT) larger += (uint32_t)(s->list[i] >> 32) > found ? s->weight[i] : 0;
                scan(larger, &all);
                *above += all;
                return found;
            }
            uint32_t lo = max(least_form(low_key), 1u), hi = least_form(high_key);
            u64 over = 0;                                         /* of the keys from hi on */
#pragma unroll 1
            while (hi - lo > 1) {
                const uint32_t d = max(1u, (hi - lo) / 4);
                const uint32_t c0 = min(lo + d, hi), c1 = min(lo + 2 * d, hi), c2 = min(lo + 3 * d, hi);
                Sum3 v{};
                each([&](K key, float x, int) {
                    if (key < c0 || key >= hi) return;
                    const u64 w = value(x);
                    v.w[0] += w;
                    if (key >= c1) v.w[1] += w;
                    if (key >= c2) v.w[2] += w;
                });
                v = cl.sum(v);
                const u64 have = *above + over;
                if (c2 < hi && have + v.w[2] >= need) lo = c2;
                else if (c1 < hi && have + v.w[1] >= need) { lo = c1; if (c2 < hi) { over += v.w[2]; hi = c2; } }
                else if (have + v.w[0] >= need) { lo = c0; if (c1 < hi) { over += v.w[1]; hi = c1; } }
                else { over += v.w[0]; hi = c0; }
            }
            *above += over;
            return wide((K)lo);
        };
        u64 above;
        if (by_k) {
            above = (u64)count_to(k_step);
            edges(k_step + 1, k_step);
            cut = key_at(s->edge[0], s->edge[1], count_to(k_step + 1) - count_to(k_step), (u64)k, &above, true);
            ties = (int)((u64)k - above);
        }
        if (by_p) {
            /* the window: where p of the middle weights ends, and up to two steps to either side if they hold few */
            float all;
            float run = scan(est_own, &all);
            if (by_k) {                                           /* of the first k tokens */
                float part = 0.0f;
#pragma unroll
                for (int j = 0; j < kBinsEach; ++j) if (kBinsEach * tid + j <= k_step) part += est[j];
                scan(part, &all);
            }
            if (tid == 0) s->pick = by_k ? k_step : kBins - 1;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < kBinsEach; ++j) {
                if (run < p * all && run + est[j] >= p * all) atomicMin(&s->pick, kBinsEach * tid + j);
                run += est[j];
            }
            __syncthreads();
            const int mid = min(s->pick, kBins - 1);
            int from = mid, to = mid + 1, width = 1;
            for (int d = 1; d <= 2; ++d)
                if (mid >= d && mid + d < kBins && count_to(mid + d + 1) - count_to(mid - d) <= 256) { from = mid - d; to = mid + d + 1; width = to - from; }
            const u64 tied = by_k ? (u64)ties * weight(cut) : 0;
#pragma unroll 1
            for (;;) {
                edges(to, from);
                const uint32_t low_key = s->edge[0], high_key = s->edge[1];
                /* over the cut; of those, in steps below from, below to */
                Sum3 v = weigh_all<K>(e, by_k ? least_form(cut) + 1 : 0u, least_form(high_key), least_form(low_key));
                v = cl.sum(v);
                const u64 want = want_of(p, v.w[0] + tied);
                above = v.w[0];
                if (by_k && want > v.w[0]) {                      /* it ends among the cut's ties */
                    const u64 one = weight(cut);
                    if (one) ties = (int)min((u64)ties, (want - above + one - 1) / one);
                    break;
                }
                if (!by_k && want <= v.w[2] && count_to(to) <= kT) {          /* it ends among a few */
                    gather(1, low_key, best + 1);
                    meet();
                    few = most = count_to(to);
                    want_few = want;
                    break;
                }
                if (want > v.w[1] && want <= v.w[2]) {
                    above = v.w[1];
                    cut = key_at(by_k ? max(cut + 1, low_key) : low_key, high_key, count_to(to) - count_to(from), want, &above, false);
                    const u64 one = weight(cut);
                    ties = one ? (int)min((u64)V, (want - above + one - 1) / one) : V;
                    break;
                }
                width *= 8;
                if (want <= v.w[1]) { to = from; from = max(from - width, 0); }
                else { from = to; to = min(to + width, kBins); }
            }
        }
    }

    if (few >= 0) {
        if (!first_cta) return;
        /* ---- in order, a thread each; what is kept is a first part */
        const int n = few;
        int sh = share_of(n), i = tid / sh;
        const int place = count_before(n, i, sh);
        if (i < n && tid % sh == 0) s->list[kT + place] = s->list[i];
        __syncthreads();
        const u64 me = s->list[kT + tid];
        uint32_t key = (uint32_t)(me >> 32);
        const bool in = tid < min(n, most);
        u64 w = in ? weight(key) : 0, sum;
        const u64 before = scan(w, &sum), want = want_few ? want_few : by_p ? want_of(p, sum) : ~0ull;
        const bool keep = in && (tid == 0 || (before < want && key >= least_key));
        /* by id, ascending: the low words are 0xffffffff - id */
        s->list[tid] = me << 32 | key;
        s->weight[tid] = w;
        const int n_kept = __syncthreads_count(keep);
        scan(keep ? w : 0ull, &sum);
        sh = share_of(n_kept); i = tid / sh;
        const u64 run = sum_before(n_kept, i, sh), point = point_of(u, sum);
        if (i < n_kept && tid % sh == 0 && run <= point && point < run + s->weight[i]) {
            key = (uint32_t)s->list[i];
            answer(P, m, (int)(0xffffffffu - (uint32_t)(s->list[i] >> 32)), n_kept, logprob_of(R, key, sum));
        }
        return;
    }

    /* ---- the kept ones by id */
    int tie_rank = 0;
    if (ties < V) {
        int n = 0, n_cta;
        own_of<K>(words, lead, e, [&](K key, float, int) { n += key == (K)(sizeof(K) == 2 ? cut >> 16 : cut); });
        tie_rank = scan(n, &n_cta);
        if (tid == 0) s->mine.w[0] = (u64)n_cta;
        const Part* parts = cl.exchange();
#pragma unroll 1
        for (int r = 0; r < cl.rank; ++r) tie_rank += (int)parts[r].w[0];
    }
    /* the least kept, and what is more than the cut, in the form of the keys */
    const uint32_t least = max(max(least_form(cut), least_form(least_key)), 1u), over = least_form(cut) + 1;
    const Sum mine = weigh_kept<K>(e, least, over, tie_rank, ties);
    const u64 w = mine.w;
    u64 w_cta;
    int n = mine.n;
    n = __reduce_add_sync(0xffffffffu, n);
    if ((tid & 31) == 0) s->warp_n[tid >> 5] = n;
    u64 before = scan(w, &w_cta);                      /* its barriers order the counts, too */
    if (tid < 32) {
        n = __reduce_add_sync(0xffffffffu, tid < kWarps ? s->warp_n[tid] : 0);
        if (tid == 0) { s->mine.w[0] = w_cta; s->mine.w[1] = (u64)n; }
    }
    const Part* parts = cl.exchange();
    u64 sum = 0;
    int n_kept = 0;
#pragma unroll 1
    for (int r = 0; r < cl.size; ++r) {
        if (r < cl.rank) before += parts[r].w[0];
        sum += parts[r].w[0]; n_kept += (int)parts[r].w[1];
    }
    const u64 point = point_of(u, sum);
    if (before <= point && point < before + w) {
        int rank = tie_rank;
        bool found = false;
#pragma unroll 1
        for (int i = tid * e; i < tid * e + e && !found; ++i)
            word(i, [&](K key, float x, int id) {
                if (found || key < least || (key < over && rank++ >= ties)) return;
                before += s->weigh.of(s->powers.of, x);
                if (before <= point) return;
                answer(P, m, base + id, n_kept, logprob_of(R, wide(key), sum));
                found = true;
            });
    }
}

constexpr size_t kRowSmem = 220 * 1024;
/* words of keys a thread: an odd number, and 16 bytes for the shift to the logits' grid */
int words_of(int vocab, int size, int ksz) {
    const int bytes = (vocab + size - 1) / size * ksz + 16;
    return (bytes + kT * 4 - 1) / (kT * 4) | 1;
}
size_t row_smem(int vocab, int size, int ksz) { return sizeof(Shared) + (size_t)kT * 4 * words_of(vocab, size, ksz); }

template <typename K>
int launch_row(const R3dNucleus& P, int size, cudaStream_t st) {
    const auto kernel = k_nucleus_row<K>;
    static std::atomic<bool> set[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return RAD_E_DEVICE;
    if (!set[dev].load(std::memory_order_relaxed)) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kRowSmem) != cudaSuccess ||
            cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return RAD_E_DEVICE;
        set[dev].store(true, std::memory_order_relaxed);
    }
    const int e = words_of(P.n_vocab, size, (int)sizeof(K));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)P.rows * (unsigned)size); cfg.blockDim = dim3(kT); cfg.stream = st;
    cfg.dynamicSmemBytes = row_smem(P.n_vocab, size, (int)sizeof(K));
    cudaLaunchAttribute at[2] = {};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)size; at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at; cfg.numAttrs = tc_pdl_on() ? 2 : 1;
    const int early = (long long)P.rows * size <= 2 * tc_sm_count(), reorder = !early && P.top_p && P.rows <= kT;
    return cudaLaunchKernelEx(&cfg, kernel, P, e, early, reorder) == cudaSuccess && cudaGetLastError() == cudaSuccess ? RAD_OK : RAD_E_DEVICE;
}

} /* namespace */

int launch_nucleus(const R3dNucleus& p, cudaStream_t st) {
    R3dNucleus P = p;
    int bits = 0;
    while ((1ll << bits) < (long long)p.n_vocab) ++bits;
    P.shift = 62 - bits < 50 ? 62 - bits : 50;
    count_launch();
    const int ksz = p.x_dtype == RAD_F32 ? 4 : 2;
    /* CTAs a row: what lets two be on an SM, and more where they are all resident still (a few over the SM count share one),
     * down to ten tokens a thread; rows of more than 70 tokens a thread may take a second wave. Measured, us, on 1 / 2 / 4 /
     * 8 / 16 CTAs a row, the rule's in brackets. Settings of their own: 1 x 151936 f32 - / - / 49 / 35 / [28], 30 x 65000
     * bf16 86 / 58 / 46 / [40] / 52, 64 x 32000 56 / 42 / [37] / 42 / 74, 64 x 151936 - / 132 / 93 / [63] / 90, 150 x 32000
     * 67 / [53] / 58 / 86 / 168, 256 x 32000 [73] / 68 / 85 / 142 / 283, 256 x 151936 - / 141 / [130] / 180 / 318. Top-k 50 and
     * top-p for all: 1 x 151936 f32 - / - / 19 / 15 / [13], 256 x 32000 [25] / 40 / 60 / 116 / 226. Which rows need every
     * token's weight is known on the device alone: a batch of 64 x 151936 without such rows would be faster on fewer CTAs
     * (- / 28 / 29 / [42] / 72). */
    const int sms = tc_sm_count();
    int size = 1;
    const auto each = [&]() { return words_of(p.n_vocab, size, ksz) * (4 / ksz); };
    const auto all = [&]() { return (long long)p.rows * size; };
    while (size < kMaxCluster && (row_smem(p.n_vocab, size, ksz) > 112 * 1024 || (64 * all() <= 65 * sms && each() > 10) ||
                                  (4 * all() <= 7 * sms && each() > 70))) size *= 2;
    if (row_smem(p.n_vocab, size, ksz) > kRowSmem) {
        k_nucleus_long<<<(unsigned)p.rows, 1024, 0, st>>>(P);
        return cudaGetLastError() == cudaSuccess ? RAD_OK : RAD_E_DEVICE;
    }
    return ksz == 4 ? launch_row<uint32_t>(P, size, st) : launch_row<uint16_t>(P, size, st);
}

} /* namespace r3d */

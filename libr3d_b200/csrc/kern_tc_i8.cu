/* kern_tc_i8.cu -- gemm_nt_q @ i8a8 on the tensor core (tcgen05 kind::i8, 32-bit integer accumulators in tensor
 * memory): y[m, n] = (sum_k a[m, k] b[n, k] * sa[m]) * sb[n]. The sum over the whole of K is one exact
 * accumulation, so the result does not depend on tiles, splits or order. An f32 result carries the first product's rounding
 * error on (scaled_once: 2 more operations a value, 8192 x 5120 x 5120 178 -> 179 us, 8192 x 8192 x 512 63 -> 65; with the
 * low bits of sums beyond 2^24, too, 184 and 69). A bf16 result is two f32 products, then narrowed: one in 195 thousand is
 * not the bf16 number next to the exact value.
 *
 * Tokens lie on the MMA's M axis (tensor-memory lanes), channels on its N axis (columns): a thread of the epilogue
 * owns a token, whose channels lie next to each other in registers as they do in y, and the channel tile can be any
 * multiple of 16, which is what balances a wave over 148 SMs.
 *
 * k_i8_stream (M <= 128, and more tokens on few channels): bound by the weights' bytes. One CTA a channel tile (and 128
 *   tokens), the channel tile chosen so that the tiles fill the device's slots (27648 channels: 288 tiles of 96 on 296
 *   slots), a deep TMA ring; rows of the token tile past M are whatever shared memory holds, their lanes are never read.
 *   Where the tiles do not fill the device, the CTAs of a cluster split K and add their 32-bit sums through distributed
 *   shared memory.
 *
 * k_i8_pair (M > 128): bound by the tensor pipe and by the operands' way from L2 into shared memory. CTA pairs
 *   (cta_group::2), 256 tokens x 512 channels a pair: 96 KiB of operands for 2 x 256 x 512 x 128 operations, two
 *   thirds of what 256 x 256 tiles fetch. The 512 accumulator columns fill tensor memory, so its two halves run
 *   `kLag` K steps apart: while one half is drained, the other half's MMAs still run. Persistent, 74 pairs.
 *
 * Every wait is bounded; on expiry a status word is set, the copies on their way are waited for (again with a bound), and
 * the CTA leaves without storing its tile, which no other share of it stores either.
 */
#include <atomic>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#define R3D_TC_STATUS_WORD ::r3d::g_tci8_status
namespace r3d { __device__ int g_tci8_status = 0; }
#include "tc_common.cuh"

namespace r3d {

namespace {
using namespace tcdev;

constexpr int kStageK = 128;                       /* K bytes of a stage: one 128-byte swizzle row */

struct I8Params {
    const float* as; int64_t as_pitch;
    const void* ws; int64_t ws_pitch; int ws_dtype;
    void* y; int64_t y_pitch; int y_f32;
    int m, n, nk;                                  /* nk: K stages */
    int nt;                                        /* channels of a tile */
    int tok_tiles, ch_tiles, workers, group;
    int whole, split, jobs;                        /* pair: jobs below `whole` are tiles, those above halves of one if `split` */
    int mb, stages, shares;                        /* stream: token rows of a box, ring, K shares */
    int tma_store, y_quads;                        /* pair: y's rows on the 16-byte grid (2: not their ends); stream: on that of four elements */
};

/* kind::i8: s32 accumulators (2 at bit 4), a and b signed (1 at bits 7 and 10), N >> 3 at bit 17, M >> 4 at bit 24 */
__device__ __forceinline__ uint32_t i8_idesc(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
template <int CG>
__device__ __forceinline__ void umma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if (CG == 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ uint32_t mapa_u32(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
                 "[%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void umma2_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld16u(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
}
/* pins uses of the loaded registers behind tcgen05.wait::ld */
template <int N>
__device__ __forceinline__ void pin_u32(uint32_t* r) {
#pragma unroll
    for (int i = 0; i < N; i += 8)
        asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}
__device__ __forceinline__ float scaled(uint32_t sum, float sa, float sb) { return __fmul_rn(__fmul_rn((float)(int)sum, sa), sb); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float channel_scale(const I8Params& P, int n) {
    return n < P.n ? ld_scale((const uint8_t*)P.ws, (int64_t)n * P.ws_pitch, P.ws_dtype) : 0.0f;
}

/* barrier `id` of 128 threads; true where all of them came with true */
__device__ __forceinline__ bool group_and(int id, bool v) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\t"
                 "barrier.cta.red.and.pred q, %1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"(id), "r"((uint32_t)v) : "memory");
    return r != 0;
}

/* a place in a ring of N slots, and its phase */
template <int N> struct Ring {
    int s = 0; uint32_t ph = 0;
    __device__ __forceinline__ void next() { if (++s == N) { s = 0; ph ^= 1u; } }
};

/* ------------------------------------------------------------------ M > 128: CTA pairs */
constexpr int kTokC = 128;                         /* tokens of a CTA; a pair has 256 */
constexpr int kHalf = 256;                         /* accumulator columns of a half */
constexpr int kLag = 2;                            /* K stages between the halves of a 512-channel tile */
constexpr int kOpBytes = 128 * kStageK;            /* one operand tile of a stage: 128 rows, 16 KiB */
constexpr int kPairThreads = 32 * 10;
constexpr int kStoreBytes = 32 * 128;              /* a warp's staging tile: 32 tokens x 128 bytes */

/* slots of the token ring and of the channel ring: a token tile is held until both halves have read it, a channel tile
 * for one half only */
constexpr int kSA = 6, kSB = 6;
constexpr size_t kPairSmem = (kSA + kSB) * (size_t)kOpBytes + 8 * kStoreBytes + 2 * kHalf * sizeof(float) + 256;
static_assert(kPairSmem <= 232448, "shared memory of a CTA");

/* job -> tile: blocks of `group` token tiles walk the channels, so that the tiles in flight
 * share both operands in L2 */
struct Job { int t0, n0, halves; };                /* first token and channel; how many halves of nt channels */
template <int NH>
__device__ __forceinline__ Job place(const I8Params& P, int job) {
    const bool half = P.split && job >= P.whole;
    const int tile = half ? P.whole + (job - P.whole) / 2 : job;
    const int block = P.group * P.ch_tiles, b = tile / block, r = tile - b * block;
    const int here = min(P.group, P.tok_tiles - b * P.group);
    const int first = half ? (job - P.whole) & 1 : 0;
    return Job{(b * P.group + r % here) * 2 * kTokC, (r / here * NH + first) * P.nt, half ? 1 : NH};
}

/* stores under a predicate, without a branch around them */
__device__ __forceinline__ void store_if(bool yes, char* at, uint32_t v) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p st.global.u32 [%0], %1;\n\t}" ::"l"(at), "r"(v), "r"((uint32_t)yes) : "memory");
}
__device__ __forceinline__ void store_half_if(bool yes, char* at, uint32_t v) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p st.global.u16 [%0], %1;\n\t}" ::"l"(at), "h"((uint16_t)v), "r"((uint32_t)yes) : "memory");
}
/* A warp's staging tile to rows of y off the 16-byte grid, a row at a time and a word a lane: 32 f32 channels, or 64 of bf16
 * as pairs, which in rows that begin at an odd pair are the lanes' second ones with the next lane's first; the channels at
 * either end go by themselves. Bound by the warp's own instructions: eight rows are read before they are written, and nothing
 * branches (2000 x 29118 x 896 f32 took 178 us with a row and a test at a time). */
__device__ __forceinline__ void store_rows(const I8Params& P, const uint8_t* out, int t0, int n0, int have, int lane) {
    const int rows = min(32, P.m - t0), esz = P.y_f32 ? 4 : 2;
    const int64_t step = P.y_pitch * esz;
    char* y = (char*)P.y + t0 * step + (int64_t)n0 * esz + 4 * lane;
#pragma unroll 1
    for (int r0 = 0; r0 < rows; r0 += 8) {
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = *(const uint32_t*)(out + (r0 + j) * 128 + ((((lane >> 2) ^ j) << 4) | (lane & 3) << 2));
        if (P.y_f32) {
#pragma unroll
            for (int j = 0; j < 8; ++j, y += step) store_if(r0 + j < rows && lane < have, y, w[j]);
            continue;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j, y += step) {
            const int odd = (int)((uintptr_t)y >> 1) & 1, c = 2 * lane + odd;      /* the channel this lane's word begins with */
            const uint32_t next = __shfl_down_sync(0xffffffffu, w[j], 1), v = __byte_perm(w[j], next, odd ? 0x5432 : 0x3210);
            const bool row = r0 + j < rows, two = c + 1 < have && c < 63;
            store_if(row && two, y + 2 * odd, v);
            store_half_if(row && !two && c < have, y + 2 * odd, v);
            store_half_if(row && odd && lane == 0 && have > 0, y, w[j]);
        }
    }
}

template <int NH>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
k_i8_pair(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
          const __grid_constant__ CUtensorMap tmY, const I8Params P) {
    extern __shared__ __align__(1024) uint8_t smem[];             /* kSA token tiles, kSB channel tiles */
    uint8_t* staging = smem + (kSA + kSB) * kOpBytes;
    float* sb_s = (float*)(staging + 8 * kStoreBytes);            /* [2][kHalf] channel scales of the half in each buffer */
    uint64_t* full_a = (uint64_t*)(sb_s + 2 * kHalf);
    uint64_t* empty_a = full_a + kSA;
    uint64_t* full_b = empty_a + kSA;
    uint64_t* empty_b = full_b + kSB;
    uint64_t* acc_full = empty_b + kSB;
    uint64_t* acc_empty = acc_full + 2;
    uint32_t* tmem_slot = (uint32_t*)(acc_empty + 2);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t crank = cluster_rank();
    const bool leader = crank == 0;
    const int pair = blockIdx.x >> 1;
    const int nk = P.nk, bc = P.nt / 2;                           /* bc: channels of a half that this CTA loads */
    bool alive = (smem_u32(smem) & 1023u) == 0;                   /* the operand tiles' swizzle needs it */

    if (threadIdx.x == 0) {
        for (int s = 0; s < 2 * (kSA + kSB); ++s) mbar_init(&full_a[s], 1);
        for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (!alive) atomicExch(&R3D_TC_STATUS_WORD, 90);
    }
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    dep_launch();
    dep_wait();

    if (warp == 0) {
        /* ---------------- TMA producer: this CTA's half of both operands ---------------- */
        if (elect_one()) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&tmA) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&tmB) : "memory");
            Ring<kSA> ra; Ring<kSB> rb;
            int na = 0, nb = 0;                                   /* loads issued */
            const auto load = [&](uint64_t* full, uint64_t* empty, int s, uint32_t ph, int slot, const CUtensorMap* map, int rows, int x, int y, int& n) {
                if (!mbar_wait(&empty[s], ph ^ 1u, 91)) return false;
                ++n;
                if (leader) mbar_expect_tx(&full[s], 2u * (uint32_t)rows * kStageK);
                tma_load_2d_pair(smem_u32(smem + slot * kOpBytes), map, x, y, mapa_u32(smem_u32(&full[s]), 0u));
                return true;
            };
            for (int job = pair; job < P.jobs && alive; job += P.workers) {
                const Job J = place<NH>(P, job);
                const int t0 = J.t0 + (int)crank * kTokC, n0 = J.n0 + (int)crank * bc;
                for (int it = 0; it < nk + (J.halves - 1) * kLag && alive; ++it) {     /* the order in which the MMAs read */
                    if (it < nk) {
                        alive = load(full_a, empty_a, ra.s, ra.ph, ra.s, &tmA, kTokC, it * kStageK, t0, na); ra.next();
                        alive = alive && load(full_b, empty_b, rb.s, rb.ph, kSA + rb.s, &tmB, bc, it * kStageK, n0, nb); rb.next();
                    }
                    if (NH == 2 && J.halves == 2 && it >= kLag && alive) {
                        alive = load(full_b, empty_b, rb.s, rb.ph, kSA + rb.s, &tmB, bc, (it - kLag) * kStageK, n0 + P.nt, nb); rb.next();
                    }
                }
            }
            /* where a wait ran out, the last loads into each slot are still to land (both CTAs' count on the leader's barriers);
             * else they have */
            bool landed = leader;
            for (int i = na > kSA ? na - kSA : 0; i < na && landed; ++i) landed = mbar_wait(&full_a[i % kSA], (i / kSA) & 1, 98);
            for (int i = nb > kSB ? nb - kSB : 0; i < nb && landed; ++i) landed = mbar_wait(&full_b[i % kSB], (i / kSB) & 1, 99);
        }
    } else if (warp == 1) {
        /* ---------------- MMA issuer (the pair's leader only) ---------------- */
        if (leader && elect_one()) {
            const uint32_t idesc = i8_idesc(2 * kTokC, P.nt);
            const uint64_t desc0 = smem_desc_sw128(smem_u32(smem));
            const auto mma = [&](int a, int b, int buf, bool first) {
                const uint64_t a0 = desc0 + a * (kOpBytes >> 4), b0 = desc0 + (kSA + b) * (kOpBytes >> 4);
#pragma unroll
                for (int k = 0; k < 4; ++k)                       /* 32 bytes of K on: two units of the descriptor's address */
                    umma_i8<2>(tmem_base + buf * kHalf, a0 + 2 * k, b0 + 2 * k, idesc, first && !k ? 0u : 1u);
            };
            const auto release = [&](uint64_t* bar) {
                umma2_commit(smem_u32(bar));
                umma2_commit(mapa_u32(smem_u32(bar), 1u));
            };
            Ring<kSA> ra, ra1; Ring<kSB> rb;                        /* ra1: the token tile half 1 reads next */
            int buf = 0; uint32_t aph = 0;
            for (int job = pair; job < P.jobs && alive; job += P.workers) {
                const int halves = place<NH>(P, job).halves;
                for (int it = 0; it < nk + (halves - 1) * kLag; ++it) {
                    if (it < nk) {
                        if (it == 0 && !mbar_wait(&acc_empty[buf], aph ^ 1u, 92)) { alive = false; break; }
                        if (!mbar_wait(&full_a[ra.s], ra.ph, 93) || !mbar_wait(&full_b[rb.s], rb.ph, 94)) { alive = false; break; }
                        tc_fence_after();
                        mma(ra.s, rb.s, buf, it == 0);
                        release(&empty_b[rb.s]);
                        if (halves == 1) release(&empty_a[ra.s]);
                        if (it == nk - 1) release(&acc_full[buf]);
                        ra.next(); rb.next();
                    }
                    if (NH == 2 && halves == 2 && it >= kLag) {
                        if (it == kLag && !mbar_wait(&acc_empty[1], aph ^ 1u, 95)) { alive = false; break; }
                        if (!mbar_wait(&full_b[rb.s], rb.ph, 96)) { alive = false; break; }
                        tc_fence_after();
                        mma(ra1.s, rb.s, 1, it == kLag);
                        release(&empty_b[rb.s]);
                        release(&empty_a[ra1.s]);
                        if (it == nk + kLag - 1) release(&acc_full[1]);
                        ra1.next(); rb.next();
                    }
                }
                if (NH == 2 || buf) aph ^= 1u;
                if (NH == 1) buf ^= 1;
            }
        }
    } else {
        /* ---------------- epilogue: thread = token; warps 2-5 drain buffer 0, warps 6-9 buffer 1 ---------------- */
        const int q = warp & 3, g = (warp - 2) >> 2, et = threadIdx.x - 64 - 128 * g;
        const uint32_t ta = tmem_base + ((uint32_t)(q * 32) << 16) + g * kHalf;
        const uint32_t acc_empty_leader = mapa_u32(smem_u32(&acc_empty[g]), 0u);
        uint8_t* const out = staging + (warp - 2) * kStoreBytes;
        float* const sb = sb_s + g * kHalf;
        const int esz = P.y_f32 ? 4 : 2, cols = 128 / esz;        /* channels of a 128-byte staging row */
        uint32_t aph = 0;
        int count = 0;
        for (int job = pair; job < P.jobs && alive; job += P.workers, ++count) {
            const Job J = place<NH>(P, job);
            if (NH == 1 ? (count & 1) != g : g >= J.halves) continue;
            const int tw = J.t0 + (int)crank * kTokC + q * 32, t = tw + lane;
            const int n0 = J.n0 + (NH == 2 ? g * P.nt : 0);
            for (int i = et; i < P.nt; i += 128) sb[i] = channel_scale(P, n0 + i);
            const float sa = t < P.m ? __ldg(P.as + (int64_t)t * P.as_pitch) : 0.0f;
            /* one answer for the four warps: they meet at a barrier again below */
            alive = group_and(1 + g, mbar_wait(&acc_full[g], aph, 97));
            if (!alive) break;
            tc_fence_after();
            aph ^= 1u;
            const bool live = tw < P.m;                           /* the warp has tokens at all */
            const bool tma = P.tma_store == 1 || (P.tma_store == 2 && n0 + P.nt <= P.n);
            uint32_t bufs[2][32];
            if (live) tmem_ld32(ta, bufs[0]);
#pragma unroll 1
            for (int c2 = 0; c2 < P.nt && live; c2 += 64)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int c = c2 + 32 * h;
                uint32_t* const r = bufs[h];
                tmem_ld_wait();
                pin_u32<32>(r);
                if (c + 32 < P.nt) tmem_ld32(ta + c + 32, bufs[h ^ 1]);
                else {                                            /* the last columns are in registers: the MMAs may go on */
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(acc_empty_leader);
                }
                if (c % cols == 0) {                              /* the staging tile's last store has read it */
                    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                    __syncwarp();
                }
                uint4* row = (uint4*)(out + lane * 128);
                if (P.y_f32) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float4 w = *(const float4*)(sb + c + 4 * j);
                        row[j ^ (lane & 7)] = make_uint4(__float_as_uint(scaled_once((int)r[4 * j], sa, w.x)), __float_as_uint(scaled_once((int)r[4 * j + 1], sa, w.y)),
                                                         __float_as_uint(scaled_once((int)r[4 * j + 2], sa, w.z)), __float_as_uint(scaled_once((int)r[4 * j + 3], sa, w.w)));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float4 w = *(const float4*)(sb + c + 8 * j), v = *(const float4*)(sb + c + 8 * j + 4);
                        row[(((c >> 5) & 1) * 4 + j) ^ (lane & 7)] = make_uint4(
                            pack_bf16(scaled(r[8 * j], sa, w.x), scaled(r[8 * j + 1], sa, w.y)), pack_bf16(scaled(r[8 * j + 2], sa, w.z), scaled(r[8 * j + 3], sa, w.w)),
                            pack_bf16(scaled(r[8 * j + 4], sa, v.x), scaled(r[8 * j + 5], sa, v.y)), pack_bf16(scaled(r[8 * j + 6], sa, v.z), scaled(r[8 * j + 7], sa, v.w)));
                    }
                }
                if ((c + 32) % cols && c + 32 < P.nt) continue;
                const int cb = c / cols * cols, have = min(c + 32 - cb, P.n - n0 - cb);   /* channels staged and inside y */
                if (tma) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0 && have > 0) {
                        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
                                     ::"l"(&tmY), "r"(smem_u32(out)), "r"(n0 + cb), "r"(tw) : "memory");
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                } else {
                    __syncwarp();
                    store_rows(P, out, tw, n0 + cb, have, lane);
                    __syncwarp();
                }
            }
            if (!live && lane == 0) mbar_arrive_cluster(acc_empty_leader);
            asm volatile("bar.sync %0, 128;" ::"r"(1 + g) : "memory");   /* sb is read before the next tile's scales */
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    tc_fence_before();
    __syncwarp();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
    }
}

/* ------------------------------------------------------------------ few tokens or few channels: the weights' stream */
constexpr int kStreamThreads = 32 * 6;
constexpr int kMaxShares = 8;                      /* a portable cluster */
constexpr size_t kStreamSmem = 220 * 1024;
constexpr int kMaxStages = 16;                     /* 88 KiB of 7 KiB or 190 KiB of 15 KiB: 12 */

/* a warp's wait ran out: the last copies into each stage land before the ring is given up, and all CTAs of the cluster are
 * told (they began together, a second ago) */
__device__ __forceinline__ void give_up(uint64_t* full, int issued, int stages, int* failed, int shares) {
    const int lane = threadIdx.x & 31;
    if (lane == 0)
        for (int i = issued > stages ? issued - stages : 0; i < issued && mbar_wait(&full[i % stages], (i / stages) & 1, 84); ++i) { }
    if (shares == 1) *(volatile int*)failed = 1;
    else if (lane < shares)
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapa_u32(smem_u32(failed), (uint32_t)lane)), "r"(1) : "memory");
}

__global__ void __launch_bounds__(kStreamThreads, 2)
k_i8_stream(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const I8Params P) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ uint64_t full[kMaxStages], empty[kMaxStages], done;
    __shared__ uint32_t tmem_slot;
    __shared__ int issued, failed;                                /* K blocks asked for; a wait of this CTA or of a peer ran out */
    __shared__ float sa_s[128];
    __shared__ __align__(16) float sb_s[256];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int shares = P.shares, crank = shares > 1 ? (int)cluster_rank() : 0;
    /* neighbours share a channel tile's weights in L2 */
    const int job = (int)(blockIdx.x / shares), n0 = job / P.tok_tiles * P.nt, t0 = job % P.tok_tiles * 128, m = min(128, P.m - t0);
    const int it0 = (int)((int64_t)P.nk * crank / shares), nk = (int)((int64_t)P.nk * (crank + 1) / shares) - it0;
    const int ablock = P.mb * kStageK, stage = ablock + P.nt * kStageK;
    const uint32_t cols = P.nt <= 32 ? 32u : P.nt <= 64 ? 64u : P.nt <= 128 ? 128u : 256u;
    uint8_t* const ring = (uint8_t*)(((uintptr_t)smem + 1023) & ~(uintptr_t)1023);

    if (threadIdx.x == 0) {
        for (int s = 0; s < P.stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        mbar_init(&done, 1);
        failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tmem_slot;
    dep_launch();
    dep_wait();

    if (warp == 0) {
        if (elect_one()) {
            int s = 0, it = 0; uint32_t ph = 0;
            for (; it < nk; ++it) {
                if (!mbar_wait(&empty[s], ph ^ 1u, 81)) break;
                uint8_t* const st = ring + s * stage;
                const int at = it0 + it;
                mbar_expect_tx(&full[s], (uint32_t)stage);
                tma_load_2d(st + ablock, &tmB, at * kStageK, n0, &full[s]);
                tma_load_2d(st, &tmA, at * kStageK, t0, &full[s]);
                if (++s == P.stages) { s = 0; ph ^= 1u; }
            }
            issued = it;
        }
        __syncwarp();
    } else if (warp == 1) {
        if (elect_one()) {
            const uint32_t idesc = i8_idesc(128, P.nt);
            const uint64_t desc0 = smem_desc_sw128(smem_u32(ring));
            int s = 0, it = 0; uint32_t ph = 0;
            for (; it < nk; ++it) {
                if (!mbar_wait(&full[s], ph, 82)) break;
                tc_fence_after();
                const uint64_t a = desc0 + s * (stage >> 4), b = a + (ablock >> 4);
#pragma unroll
                for (int k = 0; k < 4; ++k) umma_i8<1>(tmem_base, a + 2 * k, b + 2 * k, idesc, (it | k) ? 1u : 0u);
                umma_commit(&empty[s]);
                if (++s == P.stages) { s = 0; ph ^= 1u; }
            }
            if (it == nk) umma_commit(&done);                     /* else the wait for it runs out, too */
        }
        __syncwarp();
    } else {
        for (int i = threadIdx.x - 64; i < m; i += 128) sa_s[i] = __ldg(P.as + (int64_t)(t0 + i) * P.as_pitch);
        for (int i = threadIdx.x - 64; i < P.nt; i += 128) sb_s[i] = channel_scale(P, n0 + i);
    }
    /* the sums of the CTA's K share as [token][channel] words over the ring, whose stages are all consumed */
    const bool ok = __all_sync(0xffffffffu, mbar_wait(&done, 0, 83));
    __syncthreads();
    if (!ok) give_up(full, issued, P.stages, &failed, shares);
    const int pitch = P.nt + 4;                                   /* 16 bytes on: the lanes' rows fall into different banks */
    int* const sums = (int*)ring;
    if (warp >= 2 && ok) {
        const int q = warp & 3, t = q * 32 + lane;
        tc_fence_after();
        if (q * 32 < m)
            for (int c = 0; c < P.nt; c += 16) {
                uint32_t v[16];
                tmem_ld16u(tmem_base + ((uint32_t)(q * 32) << 16) + c, v);
                tmem_ld_wait();
                pin_u32<16>(v);
                if (t < m)
#pragma unroll
                    for (int j = 0; j < 4; ++j) *(uint4*)(sums + t * pitch + c + 4 * j) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            }
        tc_fence_before();
    }
    if (shares > 1) cluster_sync_all(); else __syncthreads();
    if (*(volatile int*)&failed == 0) {
        /* four channels of a token a thread, all of them spread over the threads of the cluster; the peers' words of two
         * such items are requested together (one at a time: 1.5 us more at 128 tokens and five shares) */
        const int quads = P.nt / 4, items = m * quads, step = kStreamThreads * shares;
        const auto finish = [&](int item, int4 v) {
            const int t = item / quads, c = 4 * (item - t * quads), live = P.n - n0 - c;
            const float sa = sa_s[t];
            const float4 sb = *(const float4*)(sb_s + c);
            const int64_t at = (int64_t)(t0 + t) * P.y_pitch + n0 + c;
            if (P.y_f32) {
                const float y[4] = {scaled_once(v.x, sa, sb.x), scaled_once(v.y, sa, sb.y), scaled_once(v.z, sa, sb.z), scaled_once(v.w, sa, sb.w)};
                float* const o = (float*)P.y + at;
                if (P.y_quads && live >= 4) *(float4*)o = make_float4(y[0], y[1], y[2], y[3]);
                else
#pragma unroll
                    for (int j = 0; j < 4; ++j) if (j < live) o[j] = y[j];
            } else {
                const float y[4] = {scaled((uint32_t)v.x, sa, sb.x), scaled((uint32_t)v.y, sa, sb.y), scaled((uint32_t)v.z, sa, sb.z), scaled((uint32_t)v.w, sa, sb.w)};
                uint16_t* const o = (uint16_t*)P.y + at;
                if (P.y_quads && live >= 4) *(uint2*)o = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
                else
#pragma unroll
                    for (int j = 0; j < 4; ++j) if (j < live) o[j] = f32_to_bf16(y[j]);
            }
        };
        const auto word_of = [&](int item) { const int t = item / quads; return sums + t * pitch + 4 * (item - t * quads); };
        if (shares == 1) {
            for (int i = threadIdx.x; i < items; i += step) finish(i, *(const int4*)word_of(i));
        } else {
            for (int i = crank * kStreamThreads + (int)threadIdx.x; i < items; i += 2 * step) {
                int4 w[2][kMaxShares];
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (i + h * step < items) {
                        const uint32_t mine = smem_u32(word_of(i + h * step));
#pragma unroll
                        for (int r = 0; r < kMaxShares; ++r)
                            if (r < shares)
                                asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                                             : "=r"(w[h][r].x), "=r"(w[h][r].y), "=r"(w[h][r].z), "=r"(w[h][r].w) : "r"(mapa_u32(mine, (uint32_t)r)));
                    }
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (i + h * step < items) {
                        int4 v = w[h][0];
#pragma unroll
                        for (int r = 1; r < kMaxShares; ++r)
                            if (r < shares) { v.x += w[h][r].x; v.y += w[h][r].y; v.z += w[h][r].z; v.w += w[h][r].w; }
                        finish(i + h * step, v);
                    }
            }
        }
    }
    if (shares > 1) cluster_sync_all(); else __syncthreads();    /* peers have read this CTA's sums */
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(cols) : "memory");
    }
}

/* ------------------------------------------------------------------ host */
bool grid16(const void* p, int64_t pitch_bytes) { return (((uintptr_t)p | (uintptr_t)pitch_bytes) & 15) == 0; }

/* maps are made for the call: encoding takes less than a microsecond and nothing outlives the launch */
bool rows_map(CUtensorMap* m, const void* p, int d0, int d1, int64_t pitch_bytes, CUtensorMapDataType dt, int box0, int box1) {
    const cuuint64_t dims[2] = {(cuuint64_t)d0, (cuuint64_t)d1}, strides[1] = {(cuuint64_t)pitch_bytes};
    const cuuint32_t box[2] = {(cuuint32_t)box0, (cuuint32_t)box1};
    return tc_encode_map(m, p, dt, 2, dims, strides, box);
}
bool codes_map(CUtensorMap* m, const void* p, int k, int rows, int64_t pitch, int box) {
    return rows_map(m, p, k, rows, pitch, CU_TENSOR_MAP_DATA_TYPE_UINT8, kStageK, box);
}

template <typename K, typename... A>
int launch(K kernel, int grid, int threads, size_t smem, int cluster, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid); cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute at[2];
    int n = 0;
    if (tc_pdl_on()) { at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization; at[n++].val.programmaticStreamSerializationAllowed = 1; }
    if (cluster > 1) { at[n].id = cudaLaunchAttributeClusterDimension; at[n].val.clusterDim.x = (unsigned)cluster; at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1; ++n; }
    cfg.attrs = at; cfg.numAttrs = (unsigned)n;
    count_launch();
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? RAD_OK : RAD_E_DEVICE;
}

/* host threads may come here at once */
template <typename K>
bool allow_smem(K kernel, size_t smem, std::atomic<bool> (&set)[kTcMaxDevices]) {
    const int dev = tc_device();
    if (dev < 0) return false;
    if (!set[dev].load(std::memory_order_acquire)) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return false;
        set[dev].store(true, std::memory_order_release);
    }
    return true;
}

I8Params params_of(const R3dGemmI8& p) {
    I8Params P{};
    P.as = p.a_scale; P.as_pitch = p.as_pitch;
    P.ws = p.b_scale; P.ws_pitch = p.bs_pitch; P.ws_dtype = p.bs_dtype;
    P.y = p.y; P.y_pitch = p.y_pitch; P.y_f32 = p.y_dtype == RAD_F32;
    P.m = p.m; P.n = p.n; P.nk = (p.k + kStageK - 1) / kStageK;
    return P;
}

template <int NH>
int run_pair(const I8Params& P, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& ty, cudaStream_t st) {
    static std::atomic<bool> set[kTcMaxDevices];
    if (!allow_smem(k_i8_pair<NH>, kPairSmem, set)) return RAD_E_DEVICE;
    return launch(k_i8_pair<NH>, 2 * P.workers, kPairThreads, kPairSmem, 1, st, ta, tb, ty, P);
}

/* a test's: operand boxes of fewer rows than are waited for */
int missing_rows() {
    static const int rows = getenv("R3D_TEST_I8_MISSING") ? 16 : 0;
    return rows;
}

int tc_i8_pair(const R3dGemmI8& p, cudaStream_t st) {
    I8Params P = params_of(p);
    const int pairs = tc_sm_count() / 2;
    P.tok_tiles = (p.m + 255) / 256;
    /* 512 channels a tile, or one half of 256 down to 64 (a staging row of bf16 is 64 channels): what ends first when
     * every pair works through its tiles. Where the last wave of 512-channel tiles fills no more than half the pairs, its
     * halves go to pairs of their own. */
    long best = -1; int nh = 1, nt = 256;
    for (int c = 512; c >= 64; c -= c > 256 ? 256 : 64) {
        const long tiles = (long)P.tok_tiles * ((p.n + c - 1) / c), rest = tiles % pairs;
        const long cost = c == 512 ? tiles / pairs * 512 + (rest == 0 ? 0 : 2 * rest <= pairs ? 300 : 512)
                                   : (tiles + pairs - 1) / pairs * (24 + (c * 9) / 8);
        if (best < 0 || cost < best) { best = cost; nh = c == 512 ? 2 : 1; nt = c == 512 ? 256 : c; }
    }
    P.nt = nt;
    P.ch_tiles = (p.n + nh * nt - 1) / (nh * nt);
    const int tiles = P.tok_tiles * P.ch_tiles;
    P.whole = tiles / pairs * pairs;
    P.split = nh == 2 && 2 * (tiles - P.whole) <= pairs;
    P.jobs = P.whole + (tiles - P.whole) * (P.split ? 2 : 1);
    P.workers = P.jobs < pairs ? P.jobs : pairs;
    P.group = 16;
    const int esz = P.y_f32 ? 4 : 2;
    /* a box is clipped to whole 16 bytes: where y's rows end inside one, the tiles at their end are stored by words */
    P.tma_store = !grid16(p.y, p.y_pitch * esz) ? 0 : (int64_t)p.n * esz % 16 == 0 ? 1 : 2;
    CUtensorMap ta, tb, ty;
    memset(&ty, 0, sizeof ty);
    if (!codes_map(&ta, p.a, p.k, p.m, p.a_pitch, kTokC) || !codes_map(&tb, p.b, p.k, p.n, p.b_pitch, P.nt / 2 - missing_rows()) ||
        (P.tma_store && !rows_map(&ty, p.y, p.n, p.m, p.y_pitch * esz,
                                  P.y_f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 128 / esz, 32)))
        return RAD_E_UNSUPPORTED;
    return nh == 2 ? run_pair<2>(P, ta, tb, ty, st) : run_pair<1>(P, ta, tb, ty, st);
}

/* clusters of `shares` CTAs that the device holds at once at one CTA an SM. Each lies in one GPC, so 27 clusters of five
 * do not fit 148 SMs (26 do; measured: a second wave, 28 instead of 17 us). Two CTAs an SM hold at least twice as
 * many; the query itself counts one for kernels that allocate tensor memory. */
int resident_clusters(int dev, int shares) {
    static std::atomic<int> known[kTcMaxDevices][kMaxShares + 1];
    int n = known[dev][shares].load(std::memory_order_relaxed);
    if (n) return n;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)shares); cfg.blockDim = dim3(kStreamThreads); cfg.dynamicSmemBytes = kStreamSmem;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)shares; at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at; cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, k_i8_stream, &cfg) != cudaSuccess || n < 1) { (void)cudaGetLastError(); n = 1; }
    known[dev][shares].store(n, std::memory_order_relaxed);
    return n;
}

int tc_i8_stream(const R3dGemmI8& p, cudaStream_t st) {
    static std::atomic<bool> set[kTcMaxDevices];
    if (!allow_smem(k_i8_stream, kStreamSmem, set)) return RAD_E_DEVICE;
    I8Params P = params_of(p);
    P.mb = p.m > 128 ? 128 : (p.m + 7) / 8 * 8;
    P.tok_tiles = (p.m + 127) / 128;
    const int sms = tc_sm_count();
    const int per_sm = P.mb <= 64 || (p.m <= 128 && p.n >= 160 * sms) ? 2 : 1, slots = sms * per_sm;
    P.shares = 1;
    if (per_sm == 1) {
        /* 65 tokens and more (fewer than 160 channels an SM up to 128): a CTA has an SM, and the channels of a tile and the K shares are
         * those with the lowest cost of a K block (its two operands' way into shared memory), of a tile's results, and of
         * adding the shares' sums. A ranking, not a time: launch, ring fill and drain, some 6 us, are the same for all
         * forms and left out (12288 channels, K = 4096, 128 tokens: cost 8.9, measured 14.6 us). Fitted to 540 forms of
         * thirteen sizes; against all forms of six sizes measured since, the choice is within 4 % of the best for five
         * (77 x 5119 x 13808 18.8 and 18.3 us, 128 x 5120 x 13824 18.7 and 18.7, 191 x 576 x 13568 8.9 and 8.6) and 11 % off
         * for one (457 x 2304 x 6272 14.5 us, 64 channels in one share 13.1). Beyond 160 channels an SM two CTAs, one's results under the other's loads
         * (27648, 5120, 128 tokens: 29.2 us, one CTA of 192 channels 31.4; 20480, 4096: 20.0 us and, with one, 19.7). */
        long best = -1;
        for (int nt = 48; nt <= 256; nt += 16)
            for (int sh = 1; sh <= kMaxShares && (sh == 1 || 5 * sh <= P.nk); ++sh) {
                const long tiles = (p.n + nt - 1) / nt * P.tok_tiles;
                if (sh > 1 && (tiles * sh > slots || tiles > resident_clusters(tc_device(), sh))) break;
                const long cost = (tiles * sh + slots - 1) / slots * ((P.nk + sh - 1) / sh * (61 + 5L * (P.mb + nt) / 8) + (long)P.mb * nt / 5) +
                                  (sh > 1 ? (long)P.mb * nt / 20 : 0);
                if (best < 0 || cost < best) { best = cost; P.nt = nt; P.shares = sh; }
            }
    } else {
        /* Two CTAs an SM with 96 channels each. A K block costs a CTA about 145 ns however few channels it has (measured
         * from 16 to 64), so where those tiles leave slots idle, the CTAs of a cluster share K instead of taking fewer
         * channels each: 5120 channels, K = 13824, 16 tokens take 15.0 us with 54 tiles x 4 shares, 22.4 us with 160 tiles
         * of 32 (other forms of 64 to 128 channels and 3 to 6 shares: 14.8 to 15.3). A share is at least eight K blocks
         * (4096 x 4096: 4 shares 6.6 us, 8 shares 6.9 us). Where they do not, the tile is the multiple of 16 with which the
         * last wave is fullest. */
        const int tiles0 = (p.n + 95) / 96;
        P.nt = 96;
        P.shares = slots / tiles0;
        if (P.shares > kMaxShares) P.shares = kMaxShares;
        if (P.shares > P.nk / 8) P.shares = P.nk / 8;
        while (P.shares > 1 && per_sm * resident_clusters(tc_device(), P.shares) < tiles0) --P.shares;
        if (P.shares < 2) {
            P.shares = 1;
            long best = -1;
            for (int nt = 48; nt <= 128; nt += 16) {
                const long tiles = (p.n + nt - 1) / nt, cost = (tiles + slots - 1) / slots * (nt + 16 + P.mb / 4);
                if (best < 0 || cost <= best) { best = cost; P.nt = nt; }
            }
        }
    }
    const int tiles = (p.n + P.nt - 1) / P.nt, stage = (P.mb + P.nt) * kStageK;
    P.stages = (per_sm == 2 ? 88 * 1024 : 190 * 1024) / stage;
    if (P.stages > kMaxStages) P.stages = kMaxStages;
    const int esz = P.y_f32 ? 4 : 2;
    P.y_quads = (((uintptr_t)p.y | (uintptr_t)(p.y_pitch * esz)) & (uintptr_t)(4 * esz - 1)) == 0;
    /* the MMA reads 128 token rows from wherever the token tile starts: the last stage's reach 16 KiB on */
    const size_t ring = (size_t)P.stages * stage + 128 * kStageK;
    const size_t sums = (size_t)(p.m < 128 ? p.m : 128) * (P.nt + 4) * 4;
    const size_t smem = 1024 + (ring > sums ? ring : sums);
    if (smem > kStreamSmem) return RAD_E_UNSUPPORTED;
    CUtensorMap ta, tb;
    if (!codes_map(&ta, p.a, p.k, p.m, p.a_pitch, P.mb) || !codes_map(&tb, p.b, p.k, p.n, p.b_pitch, P.nt - missing_rows())) return RAD_E_UNSUPPORTED;
    return launch(k_i8_stream, P.tok_tiles * tiles * P.shares, kStreamThreads, smem, P.shares, st, ta, tb, P);
}

} /* namespace */

bool tc_i8_ok(const R3dGemmI8& p) {
    return grid16(p.a, p.a_pitch) && grid16(p.b, p.b_pitch) && p.a_pitch >= p.k && p.b_pitch >= p.k && tc_have_encoder();
}
/* Above 128 tokens the streams, 128 tokens a CTA, where tiles of 256 tokens x 64 channels would not be enough for one and a half waves of pairs:
 * they split K instead (191 x 576, K = 13568: 9.0 us instead of 26.3; 687 x 900, 10112: 14.5 and 22.2; 457 x 2304, 6272, 72
 * tiles: 14.8 and 15.6; but 734 x 728, 1568: 7.8 and 6.7). With more tiles the pairs are faster (472 x 4800, 4096: 14.6 us,
 * 16.1; 764 x 12464, 2016: 18.5, 38.3). */
bool tc_i8_streams(const R3dGemmI8& p) { return p.m <= 128 || (long)((p.m + 255) / 256) * ((p.n + 63) / 64) * 2 <= tc_sm_count() / 2 * 3; }
int tc_i8(const R3dGemmI8& p, cudaStream_t st) { return tc_i8_streams(p) ? tc_i8_stream(p, st) : tc_i8_pair(p, st); }

int tc_i8_status() {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_tci8_status, sizeof(int)) != cudaSuccess) return -1;
    return v;
}

} /* namespace r3d */

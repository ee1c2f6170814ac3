/* entries_i8.cpp -- rows of the ops the reference does not have: gemm_nt_q @ i8a8, the int8 activation producers
 * (one scale a token) and sample_nucleus.
 *
 * Host C++ only. Operands by schema position. Unlike the reference's rows, an operand must have exactly the extents
 * the call names, its leading dimensions must fold into one row stride, and an output's rows must not overlap: what
 * cannot be walked that way is refused (RAD_E_SHAPE, RAD_E_STRIDE) instead of read flat.
 */
#include <cuda_runtime.h>
#include "entry_util.h"
#include "r3d_kernels.h"

using namespace r3d;

namespace {

bool act_type(uint32_t dt) { return dt == RAD_F32 || dt == RAD_BF16; }

/* the dimensions [0, rank) of t as one strided axis: *len elements, *pitch apart. RAD_E_STRIDE when they do not fold. */
int fold(const RadTensor* t, int rank, int64_t* len, int64_t* pitch) {
    *len = 1; *pitch = 0;
    for (int i = rank - 1; i >= 0; --i) {
        if (t->shape[i] <= 0) return RAD_E_SHAPE;
        if (t->shape[i] == 1) continue;
        if (t->stride[i] < 0) return RAD_E_STRIDE;
        if (*len == 1) *pitch = t->stride[i];
        else if (t->stride[i] != *pitch * *len) return RAD_E_STRIDE;
        if (t->shape[i] > INT64_MAX / *len) return RAD_E_SHAPE;
        *len *= t->shape[i];
    }
    return RAD_OK;
}

bool on_grid(const RadTensor* t) {
    return ((uintptr_t)t->data % (uintptr_t)rad_dtype_bytes(t->dtype, 1)) == 0;
}

enum Use { kIn, kOut };

/* a [rows, cols] operand with contiguous rows; rows < 0: take what is there */
int matrix(const RadTensor* t, int64_t* rows, int64_t cols, int64_t* pitch, Use use) {
    if (t->rank < 1 || t->rank > RAD_MAX_RANK) return RAD_E_SHAPE;
    const int last = (int)t->rank - 1;
    if (t->shape[last] != cols) return RAD_E_SHAPE;
    int64_t len;
    const int rc = fold(t, last, &len, pitch);
    if (rc != RAD_OK) return rc;
    if (*rows >= 0 && len != *rows) return RAD_E_SHAPE;
    *rows = len;
    if (cols > 1 && t->stride[last] != 1) return RAD_E_STRIDE;
    if (len == 1) *pitch = cols;
    if (use == kOut && *pitch < cols) return RAD_E_STRIDE;
    return on_grid(t) ? RAD_OK : RAD_E_STRIDE;
}

/* one value a row */
int column(const RadTensor* t, int64_t rows, int64_t* pitch, Use use) {
    if (t->rank > RAD_MAX_RANK) return RAD_E_SHAPE;
    int64_t len;
    const int rc = fold(t, (int)t->rank, &len, pitch);
    if (rc != RAD_OK) return rc;
    if (len != rows) return RAD_E_SHAPE;
    if (len == 1) *pitch = 1;
    if (use == kOut && *pitch < 1) return RAD_E_STRIDE;
    return on_grid(t) ? RAD_OK : RAD_E_STRIDE;
}

bool int_is(const RadArgs* a, const char* key, int64_t want) {
    long long v;
    return !rad_args_geti(a, key, &v) || v <= 0 || v == want;
}

#define CHECK(call) do { const int rc_ = (call); if (rc_ != RAD_OK) return rc_; } while (0)

} /* namespace */

extern "C" int r3d_rad_gemm_nt_q_i8(const RadArgs* a, RadStream s) {
    static const bool off = env_present("R3D_NO_I8A8");
    if (off) return RAD_E_UNSUPPORTED;                              /* backstop of the gate */
    const RadTensor* A = rad_arg_in(a, 0);
    const RadTensor* AS = rad_arg_in(a, 1);
    const RadTensor* B = rad_arg_in(a, 2);
    const RadTensor* BS = rad_arg_in(a, 3);
    const RadTensor* Y = rad_arg_in(a, 4);
    if (!A || !AS || !B || !BS || !Y) return RAD_E_UNSUPPORTED;
    if (rad_arg_in(a, 5) || rad_arg_in(a, 6)) return RAD_E_UNSUPPORTED;      /* a_sum, b_ref */
    const char* enc = rad_args_gets(a, "dtype");
    if (!enc || strcmp(enc, "i8a8") != 0) return RAD_E_UNSUPPORTED;
    long long part = 0;
    if (rad_args_geti(a, "pb1", &part) && part > 0) return RAD_E_UNSUPPORTED;
    if (rad_args_geti(a, "pb2", &part) && part > 0) return RAD_E_UNSUPPORTED;
    if (A->dtype != RAD_I8 || B->dtype != RAD_I8 || AS->dtype != RAD_F32 || !act_type(BS->dtype) || !act_type(Y->dtype))
        return RAD_E_UNSUPPORTED;
    long long N = 0, K = 0;
    if (!rad_args_geti(a, "N", &N) || !rad_args_geti(a, "K", &K)) return RAD_E_SHAPE;
    if (N <= 0 || K <= 0 || K > 131071 || N > kMaxExtent) return RAD_E_SHAPE;
    if (!int_is(a, "group", K)) return RAD_E_SHAPE;                 /* one scale over the whole of K */
    R3dGemmI8 q{};
    int64_t M = -1, n = N;
    CHECK(matrix(Y, &M, N, &q.y_pitch, kOut));
    if (M > kMaxExtent) return RAD_E_SHAPE;
    CHECK(matrix(A, &M, K, &q.a_pitch, kIn));
    CHECK(matrix(B, &n, K, &q.b_pitch, kIn));
    CHECK(column(AS, M, &q.as_pitch, kIn));
    CHECK(column(BS, N, &q.bs_pitch, kIn));
    q.a = A->data; q.a_scale = (const float*)AS->data; q.b = B->data; q.b_scale = BS->data; q.y = Y->data;
    q.m = (int32_t)M; q.n = (int32_t)N; q.k = (int32_t)K;
    q.bs_dtype = (int32_t)BS->dtype; q.y_dtype = (int32_t)Y->dtype;
    q.arm = R3D_ARM_AUTO;
    return r3d_b200_gemm_i8a8(&q, (void*)s);
}

/* the three producers: x at `xi`, residual and w (norm only), q, scale, out? */
static int token_i8(const RadArgs* a, RadStream s, int kind, int xi, int ri, int wi, int qi, int si, int oi) {
    static const bool off = env_present("R3D_NO_I8A8");
    if (off) return RAD_E_UNSUPPORTED;
    const RadTensor* X = rad_arg_in(a, xi);
    const RadTensor* R = ri >= 0 ? rad_arg_in(a, ri) : nullptr;
    const RadTensor* W = wi >= 0 ? rad_arg_in(a, wi) : nullptr;
    const RadTensor* Q = rad_arg_in(a, qi);
    const RadTensor* S = rad_arg_in(a, si);
    const RadTensor* O = oi >= 0 ? rad_arg_in(a, oi) : nullptr;
    if (!X || !Q || !S || (wi >= 0 && !W)) return RAD_E_INVAL;
    if (!act_type(X->dtype) || (W && !act_type(W->dtype)) || (R && R->dtype != X->dtype)) return RAD_E_DTYPE;
    if (Q->dtype != RAD_I8 || S->dtype != RAD_F32 || (O && !act_type(O->dtype))) return RAD_E_DTYPE;
    const bool gated = kind == R3D_TOKEN_SILU || kind == R3D_TOKEN_SIGMOID;
    if (Q->rank < 1) return RAD_E_SHAPE;
    const int64_t n = Q->shape[Q->rank - 1];
    if (n <= 0 || n > kMaxExtent / 2 || !int_is(a, "n", n)) return RAD_E_SHAPE;
    R3dTokenI8 p{};
    int64_t rows = -1, one = -1, w_pitch;
    CHECK(matrix(X, &rows, gated ? 2 * n : n, &p.x_pitch, kIn));
    if (rows > kMaxExtent) return RAD_E_SHAPE;
    CHECK(matrix(Q, &rows, n, &p.q_pitch, kOut));
    CHECK(column(S, rows, &p.s_pitch, kOut));
    if (W) {
        CHECK(matrix(W, &one, n, &w_pitch, kIn));
        if (one != 1) return RAD_E_SHAPE;
    }
    if (R) CHECK(matrix(R, &rows, n, &p.r_pitch, kOut));
    if (O) CHECK(matrix(O, &rows, n, &p.out_pitch, kOut));
    p.x = X->data; p.x_dtype = (int32_t)X->dtype;
    if (R) p.residual = R->data;
    if (W) { p.w = W->data; p.w_dtype = (int32_t)W->dtype; }
    p.q = Q->data; p.scale = (float*)S->data;
    if (O) { p.out = O->data; p.out_dtype = (int32_t)O->dtype; }
    p.kind = kind; p.rows = (int32_t)rows; p.n = (int32_t)n;
    p.eps = (float)rad_args_getf_or(a, "eps", 1e-6);
    p.wadd = (float)rad_args_getf_or(a, "wadd", 0.0);
    return r3d_b200_token_i8(&p, (void*)s);
}

extern "C" int r3d_rad_quant_token_i8(const RadArgs* a, RadStream s) {
    return token_i8(a, s, R3D_TOKEN_QUANT, 0, -1, -1, 1, 2, -1);
}

extern "C" int r3d_rad_gated_quant_token_i8(const RadArgs* a, RadStream s) {
    const char* act = rad_args_gets(a, "act");
    if (act && strcmp(act, "silu") != 0 && strcmp(act, "sigmoid") != 0) return RAD_E_UNSUPPORTED;
    return token_i8(a, s, act && !strcmp(act, "sigmoid") ? R3D_TOKEN_SIGMOID : R3D_TOKEN_SILU, 0, -1, -1, 1, 2, 3);
}

extern "C" int r3d_rad_rmsnorm_quant_token_i8(const RadArgs* a, RadStream s) {
    return token_i8(a, s, R3D_TOKEN_RMSNORM, 0, 1, 2, 3, 4, 5);
}

extern "C" int r3d_rad_sample_nucleus(const RadArgs* a, RadStream s) {
    static const bool off = env_present("R3D_NO_NUCLEUS");
    if (off) return RAD_E_UNSUPPORTED;
    const RadTensor* X = rad_arg_in(a, 0);
    const RadTensor* U = rad_arg_in(a, 1);
    const RadTensor* T = rad_arg_in(a, 2);
    const RadTensor* Kt = rad_arg_in(a, 3);
    const RadTensor* Pt = rad_arg_in(a, 4);
    const RadTensor* Mt = rad_arg_in(a, 5);
    const RadTensor* O = rad_arg_in(a, 6);
    const RadTensor* L = rad_arg_in(a, 7);
    const RadTensor* C = rad_arg_in(a, 8);
    if (!X || !U || !O) return RAD_E_INVAL;
    if (!act_type(X->dtype) || U->dtype != RAD_F32 || O->dtype != RAD_I32) return RAD_E_DTYPE;
    if ((T && T->dtype != RAD_F32) || (Kt && Kt->dtype != RAD_I32) || (Pt && Pt->dtype != RAD_F32) ||
        (Mt && Mt->dtype != RAD_F32) || (L && L->dtype != RAD_F32) || (C && C->dtype != RAD_I32))
        return RAD_E_DTYPE;
    if (X->rank < 1) return RAD_E_SHAPE;
    const int64_t V = X->shape[X->rank - 1];
    if (V <= 0 || V > kMaxExtent || !int_is(a, "n_vocab", V)) return RAD_E_SHAPE;
    R3dNucleus p{};
    int64_t M = -1;
    CHECK(matrix(X, &M, V, &p.x_pitch, kIn));
    if (M > kMaxExtent) return RAD_E_SHAPE;
    CHECK(column(U, M, &p.u_pitch, kIn));
    if (T) CHECK(column(T, M, &p.t_pitch, kIn));
    if (Kt) CHECK(column(Kt, M, &p.k_pitch, kIn));
    if (Pt) CHECK(column(Pt, M, &p.p_pitch, kIn));
    if (Mt) CHECK(column(Mt, M, &p.mp_pitch, kIn));
    CHECK(column(O, M, &p.token_pitch, kOut));
    if (L) CHECK(column(L, M, &p.lp_pitch, kOut));
    if (C) CHECK(column(C, M, &p.kept_pitch, kOut));
    p.logits = X->data; p.x_dtype = (int32_t)X->dtype;
    p.u = (const float*)U->data;
    p.temperature = T ? (const float*)T->data : nullptr;
    p.top_k = Kt ? (const int32_t*)Kt->data : nullptr;
    p.top_p = Pt ? (const float*)Pt->data : nullptr;
    p.min_p = Mt ? (const float*)Mt->data : nullptr;
    p.token = (int32_t*)O->data;
    p.logprob = L ? (float*)L->data : nullptr;
    p.kept = C ? (int32_t*)C->data : nullptr;
    p.rows = (int32_t)M; p.n_vocab = (int32_t)V;
    return r3d_b200_sample_nucleus(&p, (void*)s);
}

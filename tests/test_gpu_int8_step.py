"""The int8 band and its sampler on the GPU: gemm_i8a8, the three per-token producers and sample_nucleus against
plain implementations in 64 bits.

Tolerances. A product's sum is a whole number held exactly, so with f32 output the only roundings are the sum's
conversion and two multiplications (3 * 2^-24 relative), with bf16 output one more of 2^-8. Codes: h carries at most
`rounds` f32 roundings, so |h * step| moves by at most 127 * (rounds + 3) * 2^-24 and a code differs by one only where
the 64-bit quotient lies that near a half. Tokens and counts are whole numbers and have to be equal: the rows' running
sums lie further from every border than the fixed point's error."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from libr3d_b200 import abi, ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def no_wait_expired():
    yield
    torch.cuda.synchronize()
    assert ops.plugin().lib.r3d_b200_stream_status() == 0


def _rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i8(g, *shape):
    return torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int32).to(torch.int8)


# ---------------------------------------------------------------------- product
def _check_gemm(a, sa, b, sb, y):
    want = (a.double() @ b.double().t()) * sa.double().reshape(-1, 1) * sb.double().reshape(1, -1)
    eps = 3 * 2.0 ** -24 + (2.0 ** -8 if y.dtype == BF16 else 0)
    err = (y.double() - want).abs()
    assert bool((err <= eps * want.abs() + 1e-30).all()), float((err / want.abs().clamp_min(1e-30)).max())


GEMM = [(1, 1, 1), (1, 4096, 4096), (1, 130, 256), (2, 257, 5120), (3, 64, 16), (5, 100, 17), (8, 1000, 1040), (16, 333, 512),
        (17, 128, 384), (31, 4100, 130), (33, 640, 13824), (64, 5119, 208), (65, 1024, 1024), (77, 300, 5008), (100, 5120, 640),
        (128, 256, 100), (200, 96, 2048), (255, 513, 768), (256, 256, 128), (257, 512, 256), (300, 1024, 1040), (520, 768, 384),
        (777, 2049, 1280), (1024, 31, 512), (2000, 4608, 144)]


@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("M,N,K", GEMM)
def test_gemm_against_whole_numbers(M, N, K, out):
    g = _rng(M * 7 + N + K)
    a, b = _i8(g, M, K), _i8(g, N, K)
    sa = torch.rand(M, 1, generator=g, device="cuda") + 0.5
    sb = (torch.rand(N, generator=g, device="cuda") + 0.5).to(F32 if N % 2 else BF16)
    _check_gemm(a, sa, b, sb, ops.gemm_i8a8(a, sa, b, sb, out_dtype=out))


@pytest.mark.parametrize("M,N,K", [(65, 700, 5120), (72, 24001, 400), (96, 5119, 4112), (100, 2560, 8192), (113, 30000, 256), (127, 9000, 1296), (128, 96, 20000)])
def test_gemm_tiles_and_shares_up_to_128_tokens(M, N, K):
    test_gemm_against_whole_numbers(M, N, K, BF16)
    test_gemm_against_whole_numbers(M, N, K, F32)


@pytest.mark.parametrize("M,N,K", [(129, 700, 4112), (191, 576, 13568), (257, 64, 13824), (300, 513, 8192), (687, 900, 1040), (1000, 1000, 400), (2000, 128, 528),
                                   (300, 2304, 1024), (300, 2369, 1024), (5000, 64, 256), (640, 1001, 272)])
def test_gemm_many_tokens_on_few_channels(M, N, K):
    test_gemm_against_whole_numbers(M, N, K, BF16)
    test_gemm_against_whole_numbers(M, N, K, F32)


def test_gemm_extremes_stay_inside_32_bits():
    K = 131071
    a = torch.full((3, K), -128, dtype=torch.int8, device="cuda")
    b = torch.full((5, K), -128, dtype=torch.int8, device="cuda")
    b[1] = 127
    one = torch.ones(5, device="cuda")
    y = ops.gemm_i8a8(a, one[:3], b, one, out_dtype=F32)
    assert y[0, 0].item() == float(np.float32(K * 16384)) and y[2, 1].item() == float(np.float32(-K * 128 * 127))


@pytest.mark.parametrize("M,N,K,pa,pb,py,off", [(5, 200, 256, 272, 320, 208, 0), (70, 130, 512, 512, 528, 131, 16), (9, 64, 130, 133, 131, 65, 1),
                                                (300, 600, 384, 400, 384, 608, 32), (600, 515, 256, 256, 272, 515, 3)])
def test_gemm_views(M, N, K, pa, pb, py, off):
    """row pitches and starts of their own; what lies between the rows of y stays as it was"""
    g = _rng(M + pa)
    a = _i8(g, M * pa + off)[off:].view(M, pa)[:, :K]
    b = _i8(g, N * pb + off)[off:].view(N, pb)[:, :K]
    sa = (torch.rand(M, 3, generator=g, device="cuda") + 0.5)[:, 1]
    sb = (torch.rand(N, 2, generator=g, device="cuda") + 0.5)[:, :1]
    whole = torch.full((M, py), 7.0, dtype=BF16, device="cuda")
    ops.gemm_i8a8(a, sa, b, sb, whole[:, :N])
    _check_gemm(a, sa, b, sb, whole[:, :N])
    assert bool((whole[:, N:] == 7.0).all())


@pytest.mark.parametrize("M,N,K", [(1, 100, 128), (40, 5120, 1024), (100, 640, 5008), (300, 1000, 272), (600, 4700, 512)])
def test_gemm_arms_give_the_same_bits(M, N, K):
    g = _rng(M + N)
    a, b = _i8(g, M, K), _i8(g, N, K)
    sa, sb = torch.rand(M, generator=g, device="cuda"), torch.rand(N, generator=g, device="cuda")
    got = []
    for arm in (abi.R3D_ARM_EXACT, abi.R3D_ARM_TILE):
        y = torch.empty(M, N, dtype=BF16, device="cuda")
        q = abi.R3dGemmI8()
        q.a, q.a_scale, q.b, q.b_scale, q.y = (t.data_ptr() for t in (a, sa, b, sb, y))
        q.m, q.n, q.k, q.bs_dtype, q.y_dtype, q.arm = M, N, K, abi.RAD_F32, abi.RAD_BF16, arm
        q.a_pitch, q.b_pitch, q.y_pitch, q.as_pitch, q.bs_pitch = K, K, N, 1, 1
        assert ops.plugin().lib.r3d_b200_gemm_i8a8(C.byref(q), torch.cuda.current_stream().cuda_stream) == abi.RAD_OK
        got.append(y)
    assert torch.equal(*got)


def test_gemm_by_the_ops_general_entry_and_declared_once():
    g = _rng(6)
    M, N, K = 9, 200, 384
    a, b = _i8(g, M, K), _i8(g, N, K)
    sa, sb = torch.rand(M, 1, generator=g, device="cuda"), torch.rand(N, 1, generator=g, device="cuda")
    for out in (BF16, F32):
        want = ops.gemm_i8a8(a, sa, b, sb, out_dtype=out)
        y = torch.empty_like(want)
        assert ops.gemm_nt_q(a, sa, b, sb, y, dtype="i8a8", N=N, K=K).name == "gemm_nt_q_i8a8"
        assert torch.equal(y, want)
        y.zero_()
        ops.BoundGemm(a, sa, b, sb, y, dtype="i8a8", N=N, K=K).issue()
        assert torch.equal(y, want)
        y.zero_()
        ops.gemm_nt_q(a, sa, b, sb, y, dtype="i8a8", N=N, K=K, row="gemm_nt_q_i8a8")
        assert torch.equal(y, want)


def test_gemm_arms_give_the_same_bits_and_batches_fold():
    g = _rng(3)
    a, b = _i8(g, 2, 21, 640), _i8(g, 384, 640)
    sa, sb = torch.rand(2, 21, 1, generator=g, device="cuda"), torch.rand(384, generator=g, device="cuda")
    y = ops.gemm_i8a8(a, sa, b, sb)
    assert y.shape == (2, 21, 384) and torch.equal(y.view(42, 384), ops.gemm_i8a8(a.view(42, 640), sa.view(42), b, sb))
    for m in (0, 17):
        assert torch.equal(y[1, m], ops.gemm_i8a8(a[1, m:m + 1], sa[1, m:m + 1], b, sb)[0])
    assert ops.gemm_i8a8(a[:0].view(0, 640), sa[:0].view(0, 1), b, sb).shape == (0, 384)


def test_a_token_with_a_nan_scale_is_nan_and_alone():
    g = _rng(4)
    x = torch.randn(20, 256, generator=g, device="cuda")
    x[3, 7] = math.nan
    x[5, 9] = math.inf
    q, s = ops.quant_token_i8(x)
    y = ops.gemm_i8a8(q, s, _i8(g, 96, 256), torch.ones(96, device="cuda"))
    bad = ~torch.isfinite(y.float()).all(-1)
    assert torch.isnan(y[3]).all() and bad.nonzero().flatten().tolist() == [3, 5]


# ---------------------------------------------------------------------- producers
def _check_codes(h, q, scale, rounds):
    """h: the values in 64 bits"""
    amax = h.abs().amax(-1, keepdim=True)
    zero = amax < 2.0 ** -100
    want = torch.where(zero, 1.0, amax / 127)
    assert bool(((scale.double().reshape(want.shape) - want).abs() <= (rounds + 1) * 2.0 ** -24 * want).all())
    ratio = torch.where(zero, 0.0, h / want)
    slack = 127 * (rounds + 3) * 2.0 ** -24
    assert bool(((q.double() - ratio).abs() <= 0.5 + slack).all()), float((q.double() - ratio).abs().max())


WIDTHS = [1, 2, 7, 8, 31, 100, 128, 255, 256, 1000, 2048, 4100, 5120, 6144, 8191, 8192, 13824, 16384, 20000, 32768, 40000]


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("n", WIDTHS)
def test_quant_token(n, dt):
    g = _rng(n)
    x = (torch.randn(5, n, generator=g, device="cuda") * torch.tensor([[1.0], [1e-4], [3e4], [0.0], [1e-35]], device="cuda")).to(dt)
    q, s = ops.quant_token_i8(x)
    _check_codes(x.double(), q, s, 0)
    assert s[3].item() == 1.0 and not q[3].any() and s[4].item() == 1.0 and not q[4].any()


@pytest.mark.parametrize("act", ["silu", "sigmoid"])
@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("n", WIDTHS)
def test_gated_quant_token(n, dt, act):
    g = _rng(n + 1)
    gu = (torch.randn(3, 2 * n, generator=g, device="cuda") * 3).to(dt)
    if n > 4:
        gu[0, :4] = torch.tensor([-200.0, 200.0, -88.0, -30.0]).to(dt)
    out = torch.empty(3, n, dtype=F32 if n % 2 else BF16, device="cuda")
    q, s = ops.gated_quant_token_i8(gu, out=out, act=act)
    gate, up = gu.double().chunk(2, -1)
    h = (gate if act == "silu" else 1) * torch.sigmoid(gate) * up
    # the exponential is off by at most 2 + 1.173 |gate| ulp, the quotient by 2, the sum and two products by a half
    # each; an ulp is up to 2 * 2^-24. A sigmoid below 2^-126 may become 0
    rounds = 12 + 2.4 * gate.abs()
    err = rounds * 2.0 ** -24 * h.abs() + (gate * up).abs() * 2.0 ** -126 + up.abs() * 2.0 ** -126
    _check_codes(h, q, s, float(rounds.max()))
    assert bool(((out.double() - h).abs() <= err + h.abs() * (2.0 ** -8 if out.dtype == BF16 else 0)).all())


@pytest.mark.parametrize("res", [False, True])
@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("n", WIDTHS)
def test_rmsnorm_quant_token(n, dt, res):
    g = _rng(n + 2)
    M = 4
    x = torch.randn(M, n, generator=g, device="cuda").to(dt)
    r = (torch.randn(M, n, generator=g, device="cuda") * 2).to(dt) if res else None
    x[1] = 0
    if res:
        r[1] = 0
    w = (1 + 0.2 * torch.randn(n, generator=g, device="cuda")).to(BF16 if n % 3 else F32)
    out = torch.empty(M, n, dtype=F32, device="cuda")
    summed = (x.float() + r.float()).to(dt) if res else x
    before = x.clone()
    q, s = ops.rmsnorm_quant_token_i8(x, w, eps=1e-6, residual=r, out=out, wadd=0.5)
    if res:
        assert torch.equal(r, summed)
    assert torch.equal(x, before)
    v = summed.double()
    h = v / torch.sqrt(v.square().mean(-1, keepdim=True) + np.float32(1e-6)) * (w.double() + 0.5)
    # the mean of squares: runs of at most n / 64 values a thread, a tree of 5 steps and up to 32 warps' sums, their
    # rounding halved by the root; eight more for the rest
    rounds = 8 + (n / 64 + 37) / 2
    _check_codes(h, q, s, rounds)
    assert bool(((out.double() - h).abs() <= (rounds + 2) * 2.0 ** -24 * h.abs() + 1e-37).all())
    assert s[1].item() == 1.0 and not q[1].any()


@pytest.mark.parametrize("n", [512, 2056, 5120])
def test_many_rows_of_scales_far_apart(n):
    """a block walks many rows, one behind the other: each keeps its own largest value"""
    g = _rng(n + 3)
    M = 30000
    amp = 2.0 ** torch.randint(-40, 40, (M, 1), generator=g, device="cuda")
    x = (torch.randn(M, n, generator=g, device="cuda") * amp).to(BF16)
    q, s = ops.quant_token_i8(x)
    want = x.double().abs().amax(-1, keepdim=True) / 127           # one rounding to f32: half a step, 2^-24
    assert bool(((s.double() - want).abs() <= 2.0 ** -24 * want).all())
    assert bool((q.abs().amax(-1) == 127).all())
    q, s = ops.gated_quant_token_i8(x)
    assert bool((q.abs().amax(-1) == 127).all())
    for i in range(0, M, 5000):
        one_q, one_s = ops.gated_quant_token_i8(x[i:i + 3])
        assert torch.equal(one_q, q[i:i + 3]) and torch.equal(one_s, s[i:i + 3])


@pytest.mark.parametrize("n", [24000, 25613, 27641, 27648, 27649, 28000, 32753, 32760, 32761])
def test_wide_rows_of_two_f32_streams(n):
    """next to what the shared memory of a block holds"""
    test_gated_quant_token(n, F32, "silu")
    test_rmsnorm_quant_token(n, F32, True)
    test_gated_quant_token(n, BF16, "silu")


def test_producers_on_views_leave_the_rest():
    g = _rng(11)
    x = torch.randn(6, 3 * 200 + 5, generator=g, device="cuda").to(BF16)
    for start in (0, 1, 8):
        view = x[:, start:start + 400]
        q = torch.full((6, 220), 99, dtype=torch.int8, device="cuda")
        s = torch.full((6, 2), -1.0, device="cuda")
        ops.gated_quant_token_i8(view, q[:, 3:203], s[:, 1])
        want = ops.gated_quant_token_i8(view.contiguous())
        assert torch.equal(q[:, 3:203], want[0]) and torch.equal(s[:, 1:], want[1])
        assert bool((q[:, :3] == 99).all()) and bool((q[:, 203:] == 99).all()) and bool((s[:, 0] == -1).all())
    assert ops.quant_token_i8(x[:0])[0].shape == (0, 605)


# ---------------------------------------------------------------------- sampler
def _sample(x, u, t, k, p, low):
    """One row in 64 bits -> (token, logprob, kept)."""
    x = x.astype(np.float64).copy()
    x[np.isnan(x)] = -np.inf
    if not (x > -np.inf).any():
        return -1, -math.inf, 0
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if not t > 0:
        return int(order[0]), 0.0, 1
    if k > 0:
        order = order[:k]
    mx = x[order[0]]
    with np.errstate(invalid="ignore"):
        y = np.where(x[order] == mx, 0.0, (x[order] - mx) / t)
    w = np.exp(y)
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        n = max(1, int((before < p * w.sum()).sum()))
        order, w = order[:n], w[:n]
    n = max(1, int((w >= low).sum()))
    order, w = order[:n], w[:n]
    by_id = np.argsort(order)
    ids, wi = order[by_id], w[by_id]
    cum = np.cumsum(wi)
    at = min(int((cum <= u * cum[-1]).sum()), n - 1)
    return int(ids[at]), math.log(wi[at] / cum[-1]), n


def _check_sample(x, u, t=None, k=None, p=None, low=None):
    M = x.shape[0]
    lp, kept = torch.empty(M, device="cuda"), torch.empty(M, dtype=torch.int32, device="cuda")
    token = ops.sample_nucleus(x, u, temperature=t, top_k=k, top_p=p, min_p=low, logprob=lp, kept=kept)
    at = lambda v, m, d: d if v is None else v.cpu().numpy()[m].item()    # noqa: E731
    want = [_sample(x[m].float().cpu().numpy(), u[m].item(), at(t, m, 1.0), at(k, m, 0), at(p, m, 1.0), at(low, m, 0.0)) for m in range(M)]
    assert kept.tolist() == [w[2] for w in want]
    assert token.tolist() == [w[0] for w in want]
    # 64-bit arithmetic, narrowed once, and the fixed point's sum (within V * 2^-44 of a kept weight of at least 1)
    for a, (_, b, _) in zip(lp.tolist(), want):
        assert a == b or abs(a - b) <= 2.0 ** -23 * abs(b) + 2e-8


def _planes(g, M):
    i = torch.arange(M, device="cuda")
    t = torch.where(i % 7 == 6, 0.0, 0.4 + torch.rand(M, generator=g, device="cuda"))
    k = torch.where(i % 3 == 0, 0, torch.randint(1, 300, (M,), generator=g, device="cuda")).to(torch.int32)
    p = torch.where(i % 4 == 3, 1.0, 0.3 + 0.69 * torch.rand(M, generator=g, device="cuda"))
    low = torch.where(i % 2 == 0, 0.0, 0.2 * torch.rand(M, generator=g, device="cuda"))
    return t, k, p, low


VOCABS = [1, 2, 31, 100, 1000, 1025, 4096, 9999, 32000, 32001, 65537, 151936, 262144]


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("V", VOCABS)
def test_sample_rows_with_settings_of_their_own(V, dt):
    g = _rng(V)
    M = 22
    x = torch.randn(M, V, generator=g, device="cuda") * torch.linspace(0.5, 4, M, device="cuda")[:, None]
    x[1::3, : V // 2] -= 6
    x = x.to(dt)
    _check_sample(x, torch.rand(M, generator=g, device="cuda"), *_planes(g, M))


@pytest.mark.parametrize("only", ["none", "k", "p", "low", "t"])
@pytest.mark.parametrize("V,dt", [(1537, BF16), (32000, F32), (151936, BF16)])
def test_sample_one_filter(V, dt, only):
    g = _rng(V + 5)
    M = 6
    x = (torch.randn(M, V, generator=g, device="cuda") * 2.5).to(dt)
    t, k, p, low = _planes(g, M)
    t, k = t + 0.1, k.clamp_min(1)
    u = torch.rand(M, generator=g, device="cuda")
    _check_sample(x, u, t if only == "t" else None, k if only == "k" else None, p if only == "p" else None, low if only == "low" else None)


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("V,ks", [(3000, (257, 300, 1000, 2000, 2999)), (70000, (257, 999, 4000, 30000, 69000))])
def test_sample_large_k_alone_and_with_top_p(V, ks, dt):
    g = _rng(V + 1)
    M = len(ks)
    x = (torch.randn(M, V, generator=g, device="cuda") * 1.5).to(dt)
    u, k = torch.rand(M, generator=g, device="cuda"), torch.tensor(ks, dtype=torch.int32, device="cuda")
    for t in (0.05, 1.0, 20.0):
        t = torch.full((M,), t, device="cuda")
        _check_sample(x, u, t, k)
        _check_sample(x, u, t, k, torch.tensor([0.3, 0.99, 0.9, 0.5, 0.999], device="cuda"))


@pytest.mark.parametrize("V", [1200, 60000])
def test_sample_rows_whose_logits_lie_next_to_each_other(V):
    """more tokens in a step of the histogram than are gathered: the key is searched"""
    g = _rng(V)
    x = torch.stack([torch.rand(V, generator=g, device="cuda") * s + o for s, o in ((1e-3, 0.0), (1e-3, 5.0), (0.01, -3.0), (1e-30, 0.0))])
    x[3, 7] = -1e-3
    u = torch.rand(4, generator=g, device="cuda")
    p = torch.tensor([0.5, 0.9, 0.25, 0.7], device="cuda")
    k = torch.tensor([V // 2, V - 1, V // 3, V // 2], dtype=torch.int32, device="cuda")
    _check_sample(x, u, None, None, p)
    _check_sample(x, u, None, k, None)
    _check_sample(x, u, None, k, p)
    two = torch.where(torch.rand(4, V, generator=g, device="cuda") < 0.4, 2.0, 2.015625).to(BF16)
    _check_sample(two, u, None, None, p)
    _check_sample(two, u, None, k, p)


@pytest.mark.parametrize("M,V,dt", [(64, 151936, BF16), (300, 20001, F32), (512, 5003, BF16), (513, 5003, BF16), (700, 3001, F32)])
def test_sample_rows_of_long_batches_keep_their_places(M, V, dt):
    """batches of more than a wave: every row's answer is that of a call of its own rows"""
    g = _rng(M + V)
    x = (torch.randn(M, V, generator=g, device="cuda") * 3).to(dt)
    x[5::7, 1:] = -math.inf
    x[6::50] = math.nan
    u, (t, k, p, low) = torch.rand(M, generator=g, device="cuda"), _planes(g, M)
    kept, lp = torch.empty(M, dtype=torch.int32, device="cuda"), torch.empty(M, device="cuda")
    token = ops.sample_nucleus(x, u, temperature=t, top_k=k, top_p=p, min_p=low, kept=kept, logprob=lp)
    for at in range(0, M, 20):
        few = slice(at, at + 20)
        n, l = torch.empty_like(kept[few]), torch.empty_like(lp[few])
        one = ops.sample_nucleus(x[few], u[few], temperature=t[few], top_k=k[few], top_p=p[few], min_p=low[few], kept=n, logprob=l)
        assert torch.equal(one, token[few]) and torch.equal(n, kept[few]) and torch.equal(l, lp[few])
    assert bool((token[6::50] == -1).all()) and bool((token[5::7][token[5::7] >= 0] == 0).all())


def test_sample_temperatures_far_apart():
    g = _rng(77)
    M, V = 8, 20000
    x = torch.randn(M, V, generator=g, device="cuda") * 3
    t = torch.tensor([1e-4, 1e-2, 0.1, 0.3, 3.0, 30.0, 1e4, math.inf], device="cuda")
    u, p = torch.rand(M, generator=g, device="cuda"), torch.full((M,), 0.97, device="cuda")
    k = torch.full((M,), 60, dtype=torch.int32, device="cuda")
    _check_sample(x, u, t)
    _check_sample(x, u, t, None, p)
    _check_sample(x, u, t, k, p, torch.full((M,), 0.02, device="cuda"))


@pytest.mark.parametrize("V,dt", [(500001, F32), (700001, F32), (900001, F32), (1300001, BF16)])
def test_sample_long_vocabularies(V, dt):
    """from what sixteen CTAs keep to what they cannot"""
    g = _rng(V)
    x = (torch.randn(3, V, generator=g, device="cuda") * 2).to(dt)
    u = torch.rand(3, generator=g, device="cuda")
    k = torch.tensor([0, 50, 7000], dtype=torch.int32, device="cuda")
    _check_sample(x, u, None, k, torch.tensor([0.8, 0.9, 1.0], device="cuda"))


def test_sample_flat_and_tied_rows():
    """equal logits: the filters cut between ties, lower ids first; every sum is a whole number of equal weights"""
    V = 4096
    x = torch.zeros(8, V, device="cuda")
    x[1] = 3.0
    x[2, ::2] = 1.0
    x[3, 1::2] = 200.0
    x[4] = -0.0
    x[4, ::4] = 0.0
    x[5] = 88.0
    k = torch.tensor([0, 100, 50, 1000, 7, 0, 4096, 4095], dtype=torch.int32, device="cuda")
    p = torch.tensor([0.5, 1.0, 0.25, 0.5, 1.0, 0.125, 1.0, 0.5], device="cuda")
    for u in (0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24):
        _check_sample(x, torch.full((8,), u, device="cuda"), None, k, p, None)
        _check_sample(x.to(BF16), torch.full((8,), u, device="cuda"), None, k, p, None)


def test_sample_masks_infinities_and_settings_off_the_range():
    V = 5000
    g = _rng(9)
    x = torch.randn(14, V, generator=g, device="cuda")
    x[0] = -math.inf                                  # nothing left
    x[1] = -math.inf
    x[1, 4321] = -5.0                                 # one left
    x[2] = math.nan
    x[3, ::2] = math.nan
    x[4, 10] = x[4, 4000] = math.inf                  # infinities share the weight
    x[5] = torch.finfo(torch.float32).min             # a mask of the type's lowest value
    x[5, 17] = 0.0
    x[6] = torch.finfo(torch.float32).min             # ... in every place: all equal
    x[7] *= 1e30
    x[13] = -math.inf
    x[13, V - 3:] = torch.finfo(torch.float32).max
    u = torch.rand(14, generator=g, device="cuda")
    _check_sample(x, u)
    t = torch.full((14,), 0.7, device="cuda")
    _check_sample(x, u, t, torch.full((14,), 40, dtype=torch.int32, device="cuda"), torch.full((14,), 0.9, device="cuda"), torch.full((14,), 0.05, device="cuda"))
    _check_sample(x, u, torch.zeros(14, device="cuda"))
    t[8], t[9], t[10] = -1.0, 1e-30, 1e30
    k = torch.full((14,), 10 ** 9, dtype=torch.int32, device="cuda")
    k[11] = -3
    p = torch.full((14,), 0.0, device="cuda")
    p[9:12] = torch.tensor([7.0, 1.0, 1e-30], device="cuda")
    _check_sample(x, u, t, k, p, torch.full((14,), 2.0, device="cuda"))
    _check_sample(x, u, t, k, None, torch.full((14,), 1.0, device="cuda"))


def test_sample_strides_and_shared_settings():
    g = _rng(10)
    whole = torch.randn(5, 3, 2000, generator=g, device="cuda")
    x = whole[:, 1, 3:1990]
    u = torch.rand(5, 2, generator=g, device="cuda")[:, 1]
    t = torch.tensor(0.8, device="cuda").expand(5)
    k = torch.tensor([[30]], dtype=torch.int32, device="cuda").expand(5, 1)
    token = torch.full((5, 2), -7, dtype=torch.int32, device="cuda")
    ops.sample_nucleus(x, u, temperature=t, top_k=k, token=token[:, 0])
    want = ops.sample_nucleus(x.contiguous(), u.contiguous(), temperature=t.contiguous(), top_k=k[:, 0].contiguous())
    assert torch.equal(token[:, 0], want) and bool((token[:, 1] == -7).all())
    _check_sample(x, u, t, k[:, 0])


def test_sample_follows_the_distribution():
    """a million evenly spaced numbers give each token its share to within one of them a token"""
    x = torch.tensor([[0.3, -1.0, 2.0, 0.0, 1.1, -math.inf, 0.5]], device="cuda").expand(4096, 7)
    u = (torch.arange(4096, device="cuda") + 0.5) / 4096
    got = torch.bincount(ops.sample_nucleus(x, u).long(), minlength=7).double().cpu()
    want = torch.softmax(x[0].double().cpu(), 0) * 4096
    assert bool(((got - want).abs() <= 1).all())


# ---------------------------------------------------------------------- together
def test_a_step_of_them_captured_and_replayed():
    """norm -> gate_up -> gated -> down -> norm -> head -> sampler: eager, on another stream, and replayed from a graph"""
    g = _rng(20)
    M, H, I, V = 5, 512, 704, 4001
    x, res = torch.randn(M, H, generator=g, device="cuda").to(BF16), torch.randn(M, H, generator=g, device="cuda").to(BF16)
    w1, w2 = torch.ones(H, device="cuda", dtype=BF16), torch.ones(H, device="cuda", dtype=BF16)
    weights = [ops.quant_token_i8(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5) for n, k in ((2 * I, H), (H, I), (V, H))]
    u = torch.rand(M, generator=g, device="cuda")
    t = torch.full((M,), 0.9, device="cuda")
    k = torch.full((M,), 40, dtype=torch.int32, device="cuda")

    def step(x, res):
        q, s = ops.rmsnorm_quant_token_i8(x, w1, eps=1e-6, residual=res)
        q, s = ops.gated_quant_token_i8(ops.gemm_i8a8(q, s, *weights[0]))
        q, s = ops.rmsnorm_quant_token_i8(ops.gemm_i8a8(q, s, *weights[1]), w2, eps=1e-6, residual=res)
        logits = ops.gemm_i8a8(q, s, *weights[2], out_dtype=F32)
        return logits, ops.sample_nucleus(logits, u, temperature=t, top_k=k)

    want = step(x, res.clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(x, res.clone())
    side.synchronize()
    assert torch.equal(want[0], other[0]) and torch.equal(want[1], other[1])
    # against the same step in 64 bits
    def codes(h):
        s = h.abs().amax(-1, keepdim=True) / 127
        return torch.round(h / s) * s
    deq = [q.double() * s.double() for q, s in weights]
    norm = lambda r: r / torch.sqrt(r.square().mean(-1, keepdim=True) + 1e-6)      # noqa: E731
    r = x.double() + res.double()
    gu = codes(norm(r)) @ deq[0].t()
    r = r + codes(gu[:, :I] * torch.sigmoid(gu[:, :I]) * gu[:, I:]) @ deq[1].t()
    plain = codes(norm(r)) @ deq[2].t()
    # six bf16 roundings on the way and the codes that flip with them: a few steps of 2^-8 of the logits' size
    assert float((want[0].double() - plain).norm() / plain.norm()) < 6 * 2.0 ** -8
    xs, rs = x.clone(), res.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(xs, rs)
    for seed in (0, 1):
        xs.copy_(x * (1 + seed))
        rs.copy_(res)
        graph.replay()
        again = step(x * (1 + seed), res.clone())
        assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("M", [3, 90, 300])
def test_two_streams_at_once_and_again(M):
    """the same calls on two streams at a time, many times over: every answer is the first one's"""
    g = _rng(21 + M)
    H, N = 1280, 1536
    x = torch.randn(M, H, generator=g, device="cuda").to(BF16)
    w = torch.ones(H, device="cuda")
    b, sb = ops.quant_token_i8(torch.randn(N, H, generator=g, device="cuda"))
    c, sc = ops.quant_token_i8(torch.randn(6000, N // 2, generator=g, device="cuda"))
    u = torch.rand(M, generator=g, device="cuda")
    p = torch.full((M,), 0.8, device="cuda")

    def step():
        q, s = ops.rmsnorm_quant_token_i8(x, w, eps=1e-6)
        q, s = ops.gated_quant_token_i8(ops.gemm_i8a8(q, s, b, sb))
        logits = ops.gemm_i8a8(q, s, c, sc)
        return q, s, logits, ops.sample_nucleus(logits, u, top_p=p)

    want = step()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            got.append(step())
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(a, b) for a, b in zip(want, one))


def test_norm_written_over_its_input():
    g = _rng(30)
    x = torch.randn(700, 1000, generator=g, device="cuda").to(BF16)
    w = torch.rand(1000, generator=g, device="cuda")
    out = torch.empty_like(x)
    q, s = ops.rmsnorm_quant_token_i8(x, w, eps=1e-5, out=out)
    again = ops.rmsnorm_quant_token_i8(x, w, eps=1e-5, out=x)
    assert torch.equal(x, out) and torch.equal(q, again[0]) and torch.equal(s, again[1])


def test_rows_and_tokens_beyond_32_bit_offsets():
    """logits, codes and results of more than 2^31 elements: the last rows are those of a call of their own"""
    M, V = 70000, 32001
    x = torch.empty(M, V, dtype=BF16, device="cuda")
    g = _rng(31)
    x[-3:] = (torch.randn(3, V, generator=g, device="cuda") * 4).to(BF16)
    x[:-3] = x[-1:]
    u = torch.rand(M, generator=g, device="cuda")
    token = ops.sample_nucleus(x, u, top_k=torch.full((1,), 30, dtype=torch.int32, device="cuda").expand(M))
    assert torch.equal(token[-3:], ops.sample_nucleus(x[-3:].clone(), u[-3:], top_k=torch.full((3,), 30, dtype=torch.int32, device="cuda")))
    q, s = ops.quant_token_i8(x)
    one_q, one_s = ops.quant_token_i8(x[-3:].clone())
    assert torch.equal(q[-3:], one_q) and torch.equal(s[-3:], one_s)
    del x
    b, sb = _i8(g, 24, V), torch.rand(24, generator=g, device="cuda")
    assert torch.equal(ops.gemm_i8a8(q, s, b, sb)[-3:], ops.gemm_i8a8(one_q, one_s, b, sb))
    b, sb = _i8(_rng(32), 32768, 32), torch.rand(32768, generator=_rng(33), device="cuda")
    y = ops.gemm_i8a8(q[:, :32].contiguous(), s, b, sb)
    assert y.numel() > 2 ** 31
    assert torch.equal(y[-3:], ops.gemm_i8a8(one_q[:, :32].contiguous(), one_s, b, sb))

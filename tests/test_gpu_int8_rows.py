"""The int8 producers where a block walks several rows, the next one on its way while one is reduced: every kind, type and
alignment against 64 bits, the residual that is stored in place, and rows with a NaN or an infinity among others.

Roundings of a norm's factor: a thread adds up to 16 pairs of squares and the pair's halves, then five steps of a warp and
five of the block, halved by the root: 14; the mean, the epsilon, the quotient and the root 2; two products and w's sum 3."""
import math

import pytest
import torch

from libr3d_b200 import ops
from test_gpu_int8_step import _check_codes, _rng

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
ROUNDS = 19

# rows enough that each block has several: at most 32 blocks on each of 148 SMs
SHAPES = [(12000, 264), (12000, 251), (9000, 1001), (3000, 5120), (3000, 5121), (1200, 8195), (700, 16381), (600, 27641)]


def _view(x, off, pitch):
    """x's values in rows `pitch` apart that begin `off` elements into their memory"""
    M, n = x.shape
    room = torch.empty(off + M * pitch, dtype=x.dtype, device="cuda")
    v = room[off:].view(M, pitch)[:, :n]
    v.copy_(x)
    return v


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("res", [False, True])
@pytest.mark.parametrize("M,n", SHAPES)
def test_norm_of_many_rows(M, n, res, dt):
    g = _rng(n)
    size = 2.0 ** torch.randint(-20, 20, (M, 1), generator=g, device="cuda")
    x = (torch.randn(M, n, generator=g, device="cuda") * size).to(dt)
    r = (torch.randn(M, n, generator=g, device="cuda") * size).to(dt) if res else None
    w = (1 + 0.2 * torch.randn(n, generator=g, device="cuda")).to(BF16 if n % 3 else F32)
    summed = (x.float() + r.float()).to(dt) if res else x
    for off, pitch in ((0, n), (1, n + 3)):
        xs, rs = _view(x, off, pitch), _view(r, off, pitch + 2) if res else None
        q, s = ops.rmsnorm_quant_token_i8(xs, w, eps=1e-6, residual=rs)
        assert torch.equal(xs, x)
        if res:
            assert torch.equal(rs, summed)
        v = summed.double()
        v = v / torch.sqrt(v.square().mean(-1, keepdim=True) + torch.tensor(1e-6).double().item()) * w.double()
        _check_codes(v, q, s, ROUNDS)
        del v


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("M,n", SHAPES)
def test_codes_and_gated_product_of_many_rows(M, n, dt):
    g = _rng(n + 1)
    size = 2.0 ** torch.randint(-40, 40, (M, 1), generator=g, device="cuda")
    gate = (torch.randn(M, n, generator=g, device="cuda") * 3).to(dt)
    up = (torch.randn(M, n, generator=g, device="cuda") * size).to(dt)
    for off, pitch in ((0, n), (3, n + 5)):
        q, s = ops.quant_token_i8(_view(up, off, pitch))
        _check_codes(up.double(), q, s, 0)
        q, s = ops.gated_quant_token_i8(_view(torch.cat([gate, up], 1), off, n + pitch))
        _check_codes(gate.double() * torch.sigmoid(gate.double()) * up.double(), q, s, 12)


@pytest.mark.parametrize("kind", ["quant", "silu", "sigmoid", "norm", "residual"])
@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("M,n", [(9, 16), (9, 264), (9, 1201), (9, 33001), (6000, 264), (6000, 1201), (3000, 5120)])
def test_rows_with_nan_or_infinity_are_marked_and_alone(M, n, dt, kind):
    g = _rng(n + 2)
    x = torch.randn(M, n, generator=g, device="cuda").to(dt)
    other = torch.randn(M, n, generator=g, device="cuda").to(dt)      # the gate, or the residual
    w = torch.ones(n, device="cuda")

    def call(x):
        if kind == "quant":
            return ops.quant_token_i8(x)
        if kind in ("silu", "sigmoid"):
            return ops.gated_quant_token_i8(torch.cat([other, x], 1), act=kind)
        return ops.rmsnorm_quant_token_i8(x, w, eps=1e-6, residual=other.clone() if kind == "residual" else None)

    want_q, want_s = call(x)
    at = {1: (0, math.nan), 3: (n - 1, math.inf), 4: (n // 2, -math.inf), M - 1: (n // 3, math.nan), M - 3: (7, math.inf)}
    bad = x.clone()
    for m, (i, v) in at.items():
        bad[m, i] = v
    bad[M - 3, n - 2] = math.nan
    q, s = call(bad)
    marked = torch.zeros(M, dtype=torch.bool, device="cuda")
    marked[list(at)] = True
    assert not torch.isfinite(s[marked]).any() and not q[marked].any()
    assert torch.equal(q[~marked], want_q[~marked]) and torch.equal(s[~marked], want_s[~marked])

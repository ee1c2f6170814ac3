"""The gated producer's product in f32, all over the gate's range. Its roundings, in units of 2^-24 of the value: the
exponential 4 (2^-22) and two of its correction, the sum with 1 one, the quotient 2 (2^-23), two products one each: 11,
whatever the gate's size; 12 with what they add up to in second order. A sigmoid below 2^-126 may be 0."""
import math

import pytest
import torch

from libr3d_b200 import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("act", ["silu", "sigmoid"])
@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("n", [4096, 4097, 40000])
def test_product_of_gates_of_every_size(n, dt, act):
    g = torch.Generator(device="cuda").manual_seed(n)
    M = 40
    size = torch.logspace(-3, 1.95, M, device="cuda")[:, None]
    gate = (torch.rand(M, n, generator=g, device="cuda") * 2 - 1) * size
    up = torch.randn(M, n, generator=g, device="cuda")
    gate, up = gate.to(dt), up.to(dt)
    out = torch.empty(M, n, device="cuda")
    ops.gated_quant_token_i8(torch.cat([gate, up], 1), out=out, act=act)
    G, U = gate.double(), up.double()
    s = torch.sigmoid(G)
    want = (G if act == "silu" else 1) * s * U
    err = (out.double() - want).abs()
    tiny = (G * U).abs().clamp_min(U.abs()) * 2.0 ** -126 + 2.0 ** -126
    assert bool((err <= 12 * 2.0 ** -24 * want.abs() + tiny).all()), float((err / want.abs().clamp_min(1e-30)).max() * 2 ** 24)


@pytest.mark.parametrize("n", [16, 17])
def test_gates_at_the_ends_of_f32(n):
    big = torch.finfo(F32).max
    gate = torch.zeros(1, n, device="cuda")
    gate[0, :12] = torch.tensor([big, -big, 3e38, -3e38, 1e30, -1e30, 104.0, -104.0, 89.0, -200.0, 200.0, 1e-40])
    up = torch.full((1, n), 0.5, device="cuda")
    out = torch.empty(1, n, device="cuda")
    q, s = ops.gated_quant_token_i8(torch.cat([gate, up], 1), out=out)
    want = torch.nn.functional.silu(gate.double()) * 0.5
    assert bool(((out.double() - want).abs() <= 12 * 2.0 ** -24 * want.abs() + 2.0 ** -119).all())
    assert bool(torch.isfinite(s).all()) and q[0, 0].item() == 127


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("n", [16, 17, 40000])
def test_infinite_gates(n, dt):
    """sigmoid is 1 or 0 there, silu infinite or not a number; the row's other values are as without them"""
    g = torch.Generator(device="cuda").manual_seed(n)
    gate, up = ((torch.randn(2, n, generator=g, device="cuda") * 3).to(dt) for _ in range(2))
    out, plain = torch.empty(2, n, device="cuda"), torch.empty(2, n, device="cuda")
    for act in ("sigmoid", "silu"):
        ops.gated_quant_token_i8(torch.cat([gate, up], 1), out=plain, act=act)
        ends = gate.clone()
        ends[0, 3], ends[0, n - 2], ends[1, 5] = math.inf, math.inf, -math.inf
        q, s = ops.gated_quant_token_i8(torch.cat([ends, up], 1), out=out, act=act)
        same = ~torch.isinf(ends)
        assert torch.equal(out[same], plain[same])
        if act == "sigmoid":
            assert torch.equal(out[0, [3, n - 2]], up[0, [3, n - 2]].float()) and out[1, 5].item() == 0.0
            assert bool(torch.isfinite(s).all()) and bool((q.abs().amax(-1) == 127).all())
        else:
            assert torch.equal(out[0, [3, n - 2]], math.inf * up[0, [3, n - 2]].float().sign()) and math.isnan(out[1, 5].item())
            assert s[0].item() == math.inf and math.isnan(s[1].item()) and not q.any()

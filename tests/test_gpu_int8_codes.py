"""The int8 producers' codes where the quotient lies half way between two whole numbers: h * 127 / amax is a ratio of two
numbers of eight bits in bf16 rows, so a code is either decided by far more than the arithmetic's error or exactly at a
half, and a half goes to the even code. H * 127 / A = k + 1/2 asks for 127 to divide A (2 k + 1): it is 63.5, or A is 254."""
import pytest
import torch

from libr3d_b200 import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _rows(n, dt, size=60):
    """One row for each significand amax can have in eight bits, at sizes far apart; the row holds plus or minus amax,
    its half and numbers of eight bits below it."""
    g = torch.Generator().manual_seed(n)
    sig = torch.arange(128, 256, dtype=torch.int64)
    h = torch.randint(128, 256, (128, n), generator=g) << 8 >> torch.randint(0, 9, (128, n), generator=g)
    h = torch.where(h >= sig[:, None] << 8, h >> 1, h)
    h[:, 0::3] = sig[:, None] << 7
    h[:, n // 2] = sig << 8
    h *= torch.randint(0, 2, (128, n), generator=g) * 2 - 1
    x = h.double() * 2.0 ** torch.randint(-size, size, (128, 1), generator=g)
    assert torch.equal(x.to(dt).double(), x)
    num, den = 254 * h.abs(), sig[:, None] << 9                   # |h| * 127 / amax = num / den
    code = (num + (den >> 1)) // den
    code -= (((num + (den >> 1)) % den == 0) & (code % 2 == 1)).long()
    return x.to(dt).cuda(), (code * h.sign()).to(torch.int8).cuda()


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("n", [16, 264, 1201, 5120, 33001])
def test_codes_are_the_nearest_whole_numbers_and_halves_go_to_even(n, dt):
    x, code = _rows(n, dt)
    q, _ = ops.quant_token_i8(x)
    assert torch.equal(q, code)
    many = x.repeat(40, 1)                                        # blocks that walk several rows
    assert torch.equal(ops.quant_token_i8(many)[0], code.repeat(40, 1))


@pytest.mark.parametrize("n", [264, 1201, 33001])
def test_halves_of_the_norm_and_of_the_gated_form(n):
    x, code = _rows(n, BF16, 20)                                  # their squares stay inside f32
    half = code.abs() == 64
    x = torch.where(half | (code.abs() == 127), x, 0)
    w = torch.ones(n, device="cuda")
    # one factor for the row: amax / 2 stays that, but where A is 254 other halves lie on either side after the factor's rounding
    sure = (x.abs() == x.abs().amax(1, keepdim=True)) | (2 * x.abs() == x.abs().amax(1, keepdim=True)) | (torch.arange(128, 256, device="cuda") != 254)[:, None]
    q, _ = ops.rmsnorm_quant_token_i8(x, w, eps=0.0)
    assert torch.equal(q[sure], torch.where(x != 0, code, 0)[sure]) and int((~sure).sum()) <= n
    gate = torch.linspace(-3, 3, 128, device="cuda")[:, None].expand(128, n).to(BF16)
    q, _ = ops.gated_quant_token_i8(torch.cat([gate, x], 1), act="sigmoid")
    assert torch.equal(q[sure], torch.where(x != 0, code, 0)[sure])


@pytest.mark.parametrize("n", [5120, 1201, 40000])
def test_codes_of_f32_rows_lie_within_one_rounding_of_the_quotient(n):
    """quotients of f32 numbers lie anywhere: what decides between two codes is the quotient rounded to f32, off by at most
    half a step of the numbers below 128, 2^-18, and its factor's two parts, off by 2^-40 of it"""
    g = torch.Generator(device="cuda").manual_seed(n)
    for M in (20_000_000 // n, 40):
        x = torch.randn(M, n, generator=g, device="cuda") * 2.0 ** torch.randint(-40, 40, (M, 1), generator=g, device="cuda")
        q, _ = ops.quant_token_i8(x)
        ratio = x.double() * 127 / x.double().abs().amax(-1, keepdim=True)
        assert bool(((q.double() - ratio).abs() <= 0.5 + 2.0 ** -18 + 127 * 2.0 ** -40).all())

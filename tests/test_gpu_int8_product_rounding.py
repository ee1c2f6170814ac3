"""gemm_i8a8's f32 results are the exact value's rounded once: 2^-24 of it, and 2^-40 for what the correction itself
rounds. Sums of 2^24 and more are rounded to 24 bits before: twice that."""
import ctypes as C

import pytest
import torch

from libr3d_b200 import abi, ops

pytestmark = pytest.mark.gpu
F32 = torch.float32


def _product(a, sa, b, sb, arm):
    M, K = a.shape
    N = b.shape[0]
    y = torch.empty(M, N, device="cuda")
    q = abi.R3dGemmI8()
    q.a, q.a_scale, q.b, q.b_scale, q.y = (t.data_ptr() for t in (a, sa, b, sb, y))
    q.m, q.n, q.k, q.bs_dtype, q.y_dtype, q.arm = M, N, K, abi.RAD_F32, abi.RAD_F32, arm
    q.a_pitch, q.b_pitch, q.y_pitch, q.as_pitch, q.bs_pitch = K, K, N, 1, 1
    assert ops.plugin().lib.r3d_b200_gemm_i8a8(C.byref(q), torch.cuda.current_stream().cuda_stream) == abi.RAD_OK
    return y


@pytest.mark.parametrize("low,high", [(-128, 128), (-3, 4), (90, 128)])
@pytest.mark.parametrize("M,N,K", [(1, 4096, 16), (3, 4096, 4096), (100, 2000, 1040), (128, 30000, 256), (300, 4096, 1008), (1500, 5120, 2048), (40, 500, 80000)])
def test_f32_results_are_rounded_once(M, N, K, low, high):
    g = torch.Generator(device="cuda").manual_seed(M + N + K + low)
    a, b = (torch.randint(low, high, (r, K), generator=g, device="cuda", dtype=torch.int32).to(torch.int8) for r in (M, N))
    sa, sb = (torch.rand(r, generator=g, device="cuda") * 10.0 ** torch.randint(-9, 9, (r,), generator=g, device="cuda") for r in (M, N))
    total = a.double() @ b.double().t()
    want = total * sa.double()[:, None] * sb.double()
    eps = torch.where(total.abs() < 2 ** 24, 2.0 ** -24, 2.0 ** -23) + 2.0 ** -40
    y = _product(a, sa, b, sb, abi.R3D_ARM_TILE)
    assert bool(((y.double() - want).abs() <= eps * want.abs()).all()), float(((y.double() - want) / want).abs().nan_to_num().max() * 2 ** 24)
    assert torch.equal(y, _product(a, sa, b, sb, abi.R3D_ARM_EXACT))

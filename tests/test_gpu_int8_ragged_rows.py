"""gemm_i8a8 above 128 tokens into rows of y that begin on the 16-byte grid and end off it (the first columns of a wider
buffer): what lies behind them stays as it was, to the last element of the buffer."""
import pytest
import torch

from libr3d_b200 import ops
from test_gpu_int8_step import _check_gemm, _i8, _rng

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("off", [0, 8])
@pytest.mark.parametrize("ragged", range(1, 9))
@pytest.mark.parametrize("M,N,K", [(300, 8000, 256), (2000, 1200, 144), (257, 3264, 1024), (4096, 8192, 64)])
def test_columns_behind_y_stay(M, N, K, ragged, off, dt):
    g = _rng(N + ragged)
    N += ragged
    pitch = (N + 7) // 8 * 8
    a, b = _i8(g, M, K), _i8(g, N, K)
    sa, sb = torch.rand(M, generator=g, device="cuda") + 0.5, torch.rand(N, generator=g, device="cuda") + 0.5
    whole = torch.full((off + M * pitch + 64,), 7.0, dtype=dt, device="cuda")
    rows = whole[off:off + M * pitch].view(M, pitch)
    ops.gemm_i8a8(a, sa, b, sb, rows[:, :N])
    _check_gemm(a, sa, b, sb, rows[:, :N])
    assert bool((rows[:, N:] == 7.0).all()) and bool((whole[:off] == 7.0).all()) and bool((whole[off + M * pitch:] == 7.0).all())

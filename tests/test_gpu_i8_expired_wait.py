"""gemm_i8a8's tensor-core kernels when a wait runs out: its copies bring 16 rows fewer than are waited for. The call ends by
itself, reports through the status word and stores nothing. In a process of its own: the status word stays."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

CODE = """
import torch
from libr3d_b200 import ops
for M, N, K in ((3, 20000, 2048), (16, 512, 4096), (100, 640, 5008),          # streams: one share, and several
                (300, 4096, 1024), (4096, 8192, 512)):                            # CTA pairs: tiles of one half, and of two
    a = torch.ones(M, K, dtype=torch.int8, device="cuda")
    b = torch.ones(N, K, dtype=torch.int8, device="cuda")
    y = torch.full((M, N), 7.0, device="cuda")
    ops.gemm_i8a8(a, torch.ones(M, device="cuda"), b, torch.ones(N, device="cuda"), y)
    torch.cuda.synchronize()
    print(ops.plugin().lib.r3d_b200_stream_status() in (81, 82, 83, 84) + tuple(range(91, 100)), bool((y == 7.0).all()))
# other kernels are not touched: rows off the 16-byte grid
y = ops.gemm_i8a8(a[:, :17].contiguous(), torch.ones(M, device="cuda"), b[:, :17].contiguous(), torch.ones(N, device="cuda"))
print(bool((y == 17.0).all()))
"""


def test_tiles_whose_wait_ran_out_are_not_stored():
    env = os.environ | {"R3D_TEST_I8_MISSING": "1", "PYTHONPATH": str(ROOT)}
    r = subprocess.run([sys.executable, "-c", CODE], env=env, cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.split() == ["True"] * 11, r.stdout

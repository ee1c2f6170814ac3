"""The int8 step's first calls of a process, from several host threads at once: the binding gives up Python's lock around
the launch, so what the library finds out about a device on its first call is found out by all of them."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

CODE = """
import threading
import torch
from libr3d_b200 import ops
ops._load_bind()
g = torch.Generator(device="cuda").manual_seed(1)
x = torch.randn(300, 1024, generator=g, device="cuda")
w = torch.randn(4096, 1024, generator=g, device="cuda")
u = torch.rand(300, generator=g, device="cuda")
torch.cuda.synchronize()
start, got = threading.Barrier(8), [None] * 8

def step(i):
    start.wait()
    with torch.cuda.stream(torch.cuda.Stream()):
        q, s = ops.quant_token_i8(x)
        b, sb = ops.quant_token_i8(w)
        few = ops.gemm_i8a8(q[:9], s[:9], b, sb)
        many = ops.gemm_i8a8(q, s, b, sb)
        got[i] = (q, s, b, sb, few, many, ops.sample_nucleus(many, u))
        torch.cuda.current_stream().synchronize()

threads = [threading.Thread(target=step, args=(i,)) for i in range(8)]
for t in threads: t.start()
for t in threads: t.join()
q, s, b, sb, few, many, token = got[0]
want = (q.double() @ b.double().t()) * s.double() * sb.double().t()
print(bool(((many.double() - want).abs() <= (3 * 2.0 ** -24 + 2.0 ** -8) * want.abs()).all()), torch.equal(few, many[:9]))
print(all(torch.equal(a, c) for one in got for a, c in zip(one, got[0])))
"""


def test_first_calls_from_threads_at_once():
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.split() == ["True"] * 3, r.stdout

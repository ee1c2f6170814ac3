"""The general entries of gemm_nt_q with the i8a8 band, no GPU needed: operands that would be read as what they are not are
refused before any of them is described to the library."""
import pytest
import torch

from libr3d_b200 import ops

I8, F32, BF16 = torch.int8, torch.float32, torch.bfloat16


def _operands(**over):
    t = dict(a=torch.zeros(3, 64, dtype=I8), a_scale=torch.ones(3), b=torch.zeros(8, 64, dtype=I8), b_scale=torch.ones(8), y=torch.zeros(3, 8, dtype=BF16))
    return [(t[k].to(over[k]) if k in over else t[k]) for k in t]


def _bound(*operands, **kw):
    ops.BoundGemm(*operands, **kw).issue()


@pytest.mark.parametrize("call", [ops.gemm_nt_q, _bound])
@pytest.mark.parametrize("over", [dict(a=torch.uint8), dict(a=BF16), dict(a_scale=BF16), dict(a_scale=torch.float64), dict(a_scale=torch.float16), dict(b=torch.uint8),
                                  dict(b_scale=torch.float16), dict(b_scale=torch.float64), dict(y=torch.float16), dict(y=torch.float64), dict(y=I8)])
def test_operands_of_other_types_are_refused(plug, call, over):
    with pytest.raises(TypeError, match=f"{next(iter(over))} is"):
        call(*_operands(**over), dtype="i8a8", N=8, K=64)


@pytest.mark.parametrize("call", [ops.gemm_nt_q, _bound])
def test_operands_in_host_memory_are_refused(plug, call):
    with pytest.raises(ValueError, match="one CUDA device"):
        call(*_operands(), dtype="i8a8", N=8, K=64)


def test_a_launch_goes_to_its_operands_device(monkeypatch):
    entered = []

    class Device:
        def __init__(self, d):
            self.d = d

        def __enter__(self):
            entered.append(self.d.index)

        def __exit__(self, *a):
            entered.append("left")

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    assert ops._on_device(torch.device("cuda", 1), lambda: entered.append("launched") or 7) == 7
    assert entered == [1, "launched", "left"]
    assert ops._on_device(torch.device("cuda", 0), lambda: 5) == 5 and ops._on_device(None, lambda: 6) == 6 and len(entered) == 3


def test_resolution_reads_the_extension_rows_once(plug, monkeypatch):
    """they stand behind the loader's for every op: read for every call, they took 34 us of an old op's call on the host"""
    query = dict(M=4, N=4096, K=4096, group=128, dtype="fp8a8")
    row = plug.resolve("gemm_nt_q", query)
    read = []
    real = plug._rows
    monkeypatch.setattr(plug, "_rows", lambda count, at: read.append(count) or real(count, at))
    assert plug.resolve("gemm_nt_q", query).name == row.name and len(read) == 1
    rows = plug.ext_rows()
    assert len(rows) == 5 and rows is not plug.ext_rows()             # a list of the caller's own

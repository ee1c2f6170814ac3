"""Host side of the int8 band and the sampler, no GPU needed: their rows, levers and refusals (every call here is
refused before any device work)."""
import ctypes as C
import os
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from libr3d_b200 import abi, ops
from libr3d_b200.plugin import ArgPack, tensor_desc

ROOT = Path(__file__).resolve().parent.parent
NEW = {"gemm_nt_q_i8a8", "quant_token_i8_act", "gated_quant_token_i8_act", "rmsnorm_quant_token_i8", "sample_nucleus_row"}


def test_rows_stand_beside_the_loaders_table(plug):
    assert {r.name for r in plug.ext_rows()} == NEW
    assert not NEW & {r.name for r in plug.rows()}
    assert plug.resolve("gemm_nt_q", dict(M=3, N=7, K=131071, group=131071, dtype="i8a8")).name == "gemm_nt_q_i8a8"
    assert plug.resolve("gemm_nt_q", dict(M=3, N=7, K=131072, group=131072, dtype="i8a8")) is None
    assert plug.resolve("sample_nucleus", dict(M=3, n_vocab=7, dtype="bf16")).name == "sample_nucleus_row"
    assert plug.resolve("sample_nucleus", dict(M=3, n_vocab=7, dtype="f16")) is None
    for op in ("quant_token_i8", "gated_quant_token_i8", "rmsnorm_quant_token_i8", "sample_nucleus"):
        assert op in plug.schemas()


@pytest.mark.parametrize("env,table,ext", [({"R3D_EXT_ROWS": "1"}, NEW, NEW), ({"R3D_NO_I8A8": "1"}, set(), {"sample_nucleus_row"}),
                                           ({"R3D_NO_NUCLEUS": "", "R3D_EXT_ROWS": ""}, NEW - {"sample_nucleus_row"}, NEW - {"sample_nucleus_row"})])
def test_levers(env, table, ext):
    code = ("import sys; sys.path.insert(0, %r)\nfrom libr3d_b200.plugin import Plugin\np = Plugin()\n"
            "print(','.join(r.name for r in p.rows())); print(','.join(r.name for r in p.ext_rows()))" % str(ROOT))
    e = {k: v for k, v in os.environ.items() if not k.startswith("R3D_")} | env
    got = subprocess.run([sys.executable, "-c", code], env=e, capture_output=True, text=True, check=True).stdout.split("\n")
    assert set(got[0].split(",")) & NEW == table and set(got[1].split(",")) == ext


Z = np.zeros(64, np.uint8).ctypes.data                # a live host pointer: refusals precede any use
T = tensor_desc
F, B, I8, I32 = abi.RAD_F32, abi.RAD_BF16, abi.RAD_I8, abi.RAD_I32
INVAL, UNSUP, SHAPE, STRIDE, DTYPE = abi.RAD_E_INVAL, abi.RAD_E_UNSUPPORTED, abi.RAD_E_SHAPE, abi.RAD_E_STRIDE, abi.RAD_E_DTYPE


def _call(plug, entry, operands, params, over):
    t = {**operands, **{k: v for k, v in over.items() if k in operands}}
    p = {**params, **{k: v for k, v in over.items() if k not in operands}}
    return plug.entry(entry)(ArgPack(list(t.values()), {k: v for k, v in p.items() if v is not None}).args, None)


ABSENT = T(None, F, [])
GEMM = dict(a=T(Z, I8, [3, 64]), a_scale=T(Z, F, [3, 1]), b=T(Z, I8, [8, 64]), b_scale=T(Z, F, [8]), y=T(Z, B, [3, 8]), a_sum=ABSENT, b_ref=ABSENT)


@pytest.mark.parametrize("over,rc", [
    (dict(a=ABSENT), UNSUP), (dict(y=ABSENT), UNSUP), (dict(a_sum=T(Z, F, [3])), UNSUP), (dict(dtype="fp8a8"), UNSUP), (dict(pb1=1), UNSUP),
    (dict(a=T(Z, abi.RAD_U8, [3, 64])), UNSUP), (dict(a_scale=T(Z, B, [3])), UNSUP), (dict(y=T(Z, abi.RAD_F16, [3, 8])), UNSUP),
    (dict(N=None), SHAPE), (dict(K=63), SHAPE), (dict(N=9), SHAPE), (dict(K=131072), SHAPE), (dict(group=32), SHAPE), (dict(N=-8), SHAPE),
    (dict(a=T(Z, I8, [4, 64])), SHAPE), (dict(b=T(Z, I8, [7, 64])), SHAPE), (dict(a_scale=T(Z, F, [1])), SHAPE), (dict(b_scale=T(Z, F, [8, 2])), SHAPE),
    (dict(a=T(Z, I8, [3, 64], [64, 2])), STRIDE), (dict(y=T(Z, B, [3, 8], [7, 1])), STRIDE), (dict(y=T(Z, B, [3, 8], [0, 1])), STRIDE),
    (dict(y=T(Z, B, [3, 8], [1, 3])), STRIDE), (dict(a=T(Z, I8, [3, 64], [-64, 1])), STRIDE), (dict(y=T(Z + 1, B, [3, 8])), STRIDE),
    (dict(a_scale=T(Z + 2, F, [3])), STRIDE), (dict(a=T(Z, I8, [0, 64]), y=T(Z, B, [0, 8])), SHAPE),
])
def test_gemm_refusals(plug, over, rc):
    assert _call(plug, "r3d_rad_gemm_nt_q_i8", GEMM, dict(M=3, N=8, K=64, group=64, dtype="i8a8"), over) == rc


def test_leading_dimensions_have_to_fold(plug):
    ok = dict(a=T(Z, I8, [2, 3, 64], [384, 128, 1]), a_scale=T(Z, F, [2, 3]), y=T(Z, B, [2, 3, 8]))
    p = dict(M=6, N=8, K=64, group=64, dtype="i8a8")
    want = UNSUP if not torch.cuda.is_available() else None     # past every check: refused for want of a device
    if want is not None:
        assert _call(plug, "r3d_rad_gemm_nt_q_i8", GEMM, p, ok) == want
    assert _call(plug, "r3d_rad_gemm_nt_q_i8", GEMM, p, ok | dict(a=T(Z, I8, [2, 3, 64], [500, 128, 1]))) == STRIDE


NORM = dict(x=T(Z, B, [2, 8]), residual=ABSENT, w=T(Z, F, [8]), q=T(Z, I8, [2, 8]), scale=T(Z, F, [2, 1]), out=ABSENT)


@pytest.mark.parametrize("over,rc", [
    (dict(w=ABSENT), INVAL), (dict(q=ABSENT), INVAL), (dict(x=T(Z, abi.RAD_F16, [2, 8])), DTYPE), (dict(residual=T(Z, F, [2, 8])), DTYPE),
    (dict(q=T(Z, abi.RAD_U8, [2, 8])), DTYPE), (dict(scale=T(Z, B, [2])), DTYPE), (dict(out=T(Z, I8, [2, 8])), DTYPE), (dict(n=7), SHAPE),
    (dict(x=T(Z, B, [2, 9])), SHAPE), (dict(w=T(Z, F, [2, 8])), SHAPE), (dict(scale=T(Z, F, [2, 8])), SHAPE), (dict(residual=T(Z, B, [1, 8])), SHAPE),
    (dict(out=T(Z, B, [3, 8])), SHAPE), (dict(q=T(Z, I8, [2, 8], [4, 1])), STRIDE), (dict(residual=T(Z, B, [2, 8], [0, 1])), STRIDE),
    (dict(scale=T(Z, F, [2], [0])), STRIDE), (dict(x=T(Z, B, [2, 8], [16, 2])), STRIDE),
])
def test_norm_refusals(plug, over, rc):
    assert _call(plug, "r3d_rad_rmsnorm_quant_token_i8", NORM, dict(M=2, n=8, eps=1e-6, dtype="bf16"), over) == rc


def test_gated_refusals(plug):
    gated = dict(gate_up=T(Z, B, [2, 16]), q=T(Z, I8, [2, 8]), scale=T(Z, F, [2]), out=ABSENT)
    p = dict(M=2, n=8, dtype="bf16")
    assert _call(plug, "r3d_rad_gated_quant_token_i8", gated, p, dict(act="gelu")) == UNSUP
    assert _call(plug, "r3d_rad_gated_quant_token_i8", gated, p, dict(gate_up=T(Z, B, [2, 15]))) == SHAPE
    assert _call(plug, "r3d_rad_quant_token_i8", dict(list(gated.items())[:3]), p, {}) == SHAPE


SAMPLE = dict(logits=T(Z, F, [3, 9]), u=T(Z, F, [3]), temperature=ABSENT, top_k=ABSENT, top_p=ABSENT, min_p=ABSENT, token=T(Z, I32, [3]),
              logprob=ABSENT, kept=ABSENT)


@pytest.mark.parametrize("over,rc", [
    (dict(u=ABSENT), INVAL), (dict(token=ABSENT), INVAL), (dict(logits=T(Z, abi.RAD_F16, [3, 9])), DTYPE), (dict(token=T(Z, abi.RAD_I64, [3])), DTYPE),
    (dict(top_k=T(Z, F, [3])), DTYPE), (dict(top_p=T(Z, abi.RAD_F64, [3])), DTYPE), (dict(kept=T(Z, F, [3])), DTYPE), (dict(n_vocab=10), SHAPE),
    (dict(u=T(Z, F, [1])), SHAPE), (dict(temperature=T(Z, F, [3, 2])), SHAPE), (dict(token=T(Z, I32, [4])), SHAPE), (dict(logits=T(Z, F, [3, 0])), SHAPE),
    (dict(token=T(Z, I32, [3], [0])), STRIDE), (dict(logits=T(Z, F, [3, 9], [1, 3])), STRIDE), (dict(u=T(Z + 1, F, [3])), STRIDE),
])
def test_sample_refusals(plug, over, rc):
    assert _call(plug, "r3d_rad_sample_nucleus", SAMPLE, dict(M=3, n_vocab=9, dtype="f32"), over) == rc


def _struct(which, **over):
    fields = {
        "gemm": dict(a=Z, a_scale=Z, b=Z, b_scale=Z, y=Z, m=2, n=8, k=16, bs_dtype=F, y_dtype=B, arm=abi.R3D_ARM_AUTO, a_pitch=16, b_pitch=16, y_pitch=8,
                     as_pitch=1, bs_pitch=1),
        "norm": dict(x=Z, residual=None, w=Z, q=Z, scale=Z, out=None, kind=abi.R3D_TOKEN_RMSNORM, x_dtype=B, w_dtype=F, out_dtype=B, rows=2, n=8, eps=1e-6,
                     x_pitch=8, r_pitch=8, q_pitch=8, s_pitch=1, out_pitch=8),
        "sample": dict(logits=Z, u=Z, token=Z, logprob=None, kept=None, rows=2, n_vocab=8, x_dtype=F, x_pitch=8, u_pitch=1, token_pitch=1, lp_pitch=1, kept_pitch=1),
    }[which] | over
    s = {"gemm": abi.R3dGemmI8, "norm": abi.R3dTokenI8, "sample": abi.R3dNucleus}[which]()
    for k, v in fields.items():
        setattr(s, k, v)
    return s


@pytest.mark.parametrize("kind,over,rc", [
    ("gemm", dict(b=None), INVAL), ("gemm", dict(a_scale=None), INVAL), ("gemm", dict(m=0), SHAPE), ("gemm", dict(k=131072), SHAPE), ("gemm", dict(n=1 << 28), SHAPE),
    ("gemm", dict(a_pitch=-16), STRIDE), ("gemm", dict(y_pitch=7), STRIDE), ("gemm", dict(bs_dtype=abi.RAD_F16), DTYPE), ("gemm", dict(y_dtype=I8), DTYPE),
    ("norm", dict(w=None), INVAL), ("norm", dict(kind=4), INVAL), ("norm", dict(kind=-1), INVAL), ("norm", dict(kind=abi.R3D_TOKEN_QUANT), INVAL),
    ("norm", dict(x_dtype=abi.RAD_F16), DTYPE), ("norm", dict(w_dtype=I8), DTYPE), ("norm", dict(out=Z, out_dtype=I8), DTYPE), ("norm", dict(rows=0), SHAPE),
    ("norm", dict(q_pitch=7), STRIDE), ("norm", dict(residual=Z, r_pitch=0), STRIDE), ("norm", dict(s_pitch=0), STRIDE), ("norm", dict(x_pitch=-8), STRIDE),
    ("sample", dict(token=None), INVAL), ("sample", dict(x_dtype=abi.RAD_F16), DTYPE), ("sample", dict(n_vocab=0), SHAPE), ("sample", dict(rows=-1), SHAPE),
    ("gemm", dict(y=Z + 1), STRIDE), ("gemm", dict(a_scale=Z + 2), STRIDE), ("norm", dict(x=Z + 1), STRIDE), ("norm", dict(w=Z + 2), STRIDE),
    ("norm", dict(scale=Z + 1), STRIDE), ("sample", dict(logits=Z + 2), STRIDE), ("sample", dict(top_k=Z + 2), STRIDE), ("sample", dict(u=Z + 1), STRIDE),
    ("sample", dict(token_pitch=0), STRIDE), ("sample", dict(u_pitch=-1), STRIDE), ("sample", dict(kept=Z, kept_pitch=0), STRIDE),
])
def test_launch_layer_refusals(plug, kind, over, rc):
    call = {"gemm": plug.lib.r3d_b200_gemm_i8a8, "norm": plug.lib.r3d_b200_token_i8, "sample": plug.lib.r3d_b200_sample_nucleus}[kind]
    assert call(C.byref(_struct(kind, **over)), None) == rc


def test_ops_refuse_what_they_cannot_take():
    a, s = torch.zeros(2, 16, dtype=torch.int8), torch.ones(2)
    with pytest.raises(ValueError, match="one CUDA device"):
        ops.gemm_i8a8(a, s, a, s)
    with pytest.raises(TypeError):
        ops.quant_token_i8(torch.zeros(2, 16, dtype=torch.float16))
    with pytest.raises(TypeError):
        ops.sample_nucleus(torch.zeros(2, 16), torch.zeros(2, dtype=torch.float64))

"""The ops of the quantised-matmul path as a caller issues them: `gemm_nt_q` and
`logits_gemm`, the int8 step around `gemm_i8a8`, and the sampler behind the logits, with device tensors (torch is used
for device memory and streams only).

Each call does what the radiance engine does for the op: resolve the band to a row by the
rows' constraints and priorities, then call that row's `launch` with a RadArgs on the
current CUDA stream. Nothing is computed here.
"""
from __future__ import annotations

from pathlib import Path
from typing import Any

import torch

from . import abi
from .plugin import ArgPack, Plugin, Row, tensor_desc

_plugin: Plugin | None = None


def plugin() -> Plugin:
    global _plugin
    if _plugin is None:
        _plugin = Plugin()
    return _plugin


class RowRefused(RuntimeError):
    def __init__(self, row: str, rc: int):
        super().__init__(f"row {row} returned {abi.STATUS_NAMES[rc] if 0 <= rc < 7 else rc}")
        self.rc = rc


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _on_device(device: torch.device | None, launch) -> int:
    """launch() with `device` as the current one (None: the current one as it is)."""
    if device is None or device.index == torch.cuda.current_device():
        return launch()
    with torch.cuda.device(device):
        return launch()


def _desc(t: torch.Tensor | None, dtype: int, shape=None, stride=None) -> abi.RadTensor:
    if t is None:
        return tensor_desc(None, dtype, [])
    return tensor_desc(t.data_ptr(), dtype, shape if shape is not None else t.shape,
                       stride if stride is not None else t.stride())


def _group_of(dtype: str, K: int) -> int:
    return {"fp8a8": 128, "i8a8": K}.get(dtype, 32)


def _check_i8(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor, y: torch.Tensor) -> torch.device:
    """The i8a8 band's operands are what they will be read as, on one device (which is returned)."""
    wide = (torch.float32, torch.bfloat16)
    for name, t, types in (("a", a, (torch.int8,)), ("a_scale", a_scale, (torch.float32,)), ("b", b, (torch.int8,)),
                           ("b_scale", b_scale, wide), ("y", y, wide + (torch.uint16,))):
        if t.dtype not in types:
            raise TypeError(f"gemm_nt_q i8a8: {name} is {' or '.join(str(x) for x in types)}, got {t.dtype}")
    if not a.is_cuda or any(t.device != a.device for t in (a_scale, b, b_scale, y)):
        raise ValueError("gemm_nt_q i8a8: operands on one CUDA device are needed")
    return a.device


def _gemm_descs(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor, y: torch.Tensor,
                dtype: str, K: int) -> list[abi.RadTensor]:
    """gemm_nt_q's operands by schema position, a_sum and b_ref absent."""
    adt, ydt = abi.RAD_F8E4M3, abi.RAD_BF16
    sdt = abi.RAD_F32 if b_scale.dtype == torch.float32 else abi.RAD_BF16
    if dtype == "fp8a8":
        bdesc = _desc(b, abi.RAD_F8E4M3)
    elif dtype == "i8a8":
        adt, bdesc = abi.RAD_I8, _desc(b, abi.RAD_I8)
        ydt = abi.RAD_F32 if y.dtype == torch.float32 else abi.RAD_BF16
    else:
        bdesc = _desc(b, abi.RAD_FP4E2M1, shape=[b.shape[0], K], stride=[K, 1])
        sdt = abi.RAD_E8M0
    return [_desc(a, adt), _desc(a_scale, abi.RAD_F32), bdesc, _desc(b_scale, sdt), _desc(y, ydt),
            _desc(None, abi.RAD_F32), _desc(None, abi.RAD_BF16)]


def gemm_nt_q(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
              y: torch.Tensor, *, dtype: str, N: int, K: int, group: int | None = None,
              M_param: int | None = None, row: str | None = None) -> Row:
    """y[M,N] (bf16, given as a uint16/bfloat16 tensor) = a[M,K] @ dequant(b)[N,K]^T.

    a: uint8 e4m3 codes [M,K]; a_scale: float32 [M, K/128]
    dtype "fp8a8":   b uint8 e4m3 codes [N,K]; b_scale bf16 (or f32) [N/128 | N, K/128]
    dtype "mxfp4a8": b uint8 packed e2m1 [N,K/2] (low nibble = even k); b_scale uint8 E8M0 [N,K/32]
    dtype "i8a8":    a int8 codes, a_scale float32 [M] or [M,1]; b int8 codes [N,K]; b_scale f32 or bf16 [N] or [N,1];
                     y bf16 or f32 (gemm_i8a8 is the same with y made for the caller)
    `row` forces a row by name; otherwise the band is resolved like the engine would.
    Returns the row that served the call; raises RowRefused on a nonzero status.
    """
    device = _check_i8(a, a_scale, b, b_scale, y) if dtype == "i8a8" else None
    P = plugin()
    M = y.numel() // N
    if group is None:
        group = _group_of(dtype, K)
    query: dict[str, Any] = dict(M=M_param if M_param is not None else M, N=N, K=K,
                                 group=group, dtype=dtype)
    if row is None:
        r = P.resolve("gemm_nt_q", query)
        if r is None:
            raise RuntimeError(f"no row serves gemm_nt_q {query}")
    else:
        r = next(x for x in P.rows() + P.ext_rows() if x.name == row)
    pack = ArgPack(_gemm_descs(a, a_scale, b, b_scale, y, dtype, K), query)
    rc = _on_device(device, lambda: P.launch_row(r, pack, _stream()))
    if rc != abi.RAD_OK:
        raise RowRefused(r.name, rc)
    return r


def gemm_nt_q_gated(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
                    q: torch.Tensor, scale: torch.Tensor, *, N: int, K: int, act: str = "silu",
                    group: int = 128, out: torch.Tensor | None = None,
                    scratch: torch.Tensor | None = None) -> Row:
    """q[M, N/2] (e4m3 codes), scale[M, N/2/group] (f32) = gated_quant_fp8(a @ dequant(b)^T) for a
    [N = 2n, K] fp8a8 gate_up weight, gate half first; `out` optionally receives the gated product
    (bf16 or f32). `scratch` is the launch arena (default: what the row's scratch hook asks for)."""
    P = plugin()
    n = N // 2
    M = q.numel() // n
    query: dict[str, Any] = dict(M=M, N=N, K=K, group=group, dtype="fp8a8", act=act)
    r = P.resolve("gemm_nt_q_gated", query)
    if r is None:
        raise RuntimeError(f"no row serves gemm_nt_q_gated {query}")
    sdt = abi.RAD_F32 if b_scale.dtype == torch.float32 else abi.RAD_BF16
    odt = abi.RAD_F32 if (out is not None and out.dtype == torch.float32) else abi.RAD_BF16
    tensors = [_desc(a, abi.RAD_F8E4M3), _desc(a_scale, abi.RAD_F32), _desc(b, abi.RAD_F8E4M3),
               _desc(b_scale, sdt), _desc(q, abi.RAD_F8E4M3), _desc(scale, abi.RAD_F32),
               _desc(out, odt), _desc(None, abi.RAD_F32)]
    if scratch is None:
        probe = ArgPack(tensors, query)
        need = int(P.lib.r3d_rad_gemm_nt_q_gated_fp8_scratch(probe.args))
        scratch = torch.empty(need, dtype=torch.uint8, device=a.device)
    pack = ArgPack(tensors, query, scratch=scratch.data_ptr(), scratch_bytes=scratch.numel() * scratch.element_size())
    rc = P.launch_row(r, pack, _stream())
    if rc != abi.RAD_OK:
        raise RowRefused(r.name, rc)
    return r


def logits_gemm(x: torch.Tensor, head_blob: torch.Tensor, logits: torch.Tensor, *, n_vocab: int,
                n_embd: int) -> Row:
    """logits[M, n_vocab] f32 = x[M, n_embd] bf16 @ head^T, head a joined rad.planes blob
    (uint8 device tensor) of e4m3 codes + block scales."""
    P = plugin()
    M = logits.numel() // n_vocab
    query = dict(M=M, n_vocab=n_vocab, n_embd=n_embd, dtype="bf16")
    r = P.resolve("logits_gemm", query)
    if r is None:
        raise RuntimeError(f"no row serves logits_gemm {query}")
    tensors = [_desc(x, abi.RAD_BF16), _desc(head_blob, abi.RAD_U8), _desc(logits, abi.RAD_F32)]
    rc = P.launch_row(r, ArgPack(tensors, query), _stream())
    if rc != abi.RAD_OK:
        raise RowRefused(r.name, rc)
    return r


def gemm_w2a8(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, bs_blob: torch.Tensor, y: torch.Tensor,
              a_sum: torch.Tensor, *, N: int, K: int, M_param: int | None = None) -> Row:
    """y[M,N] bf16 = a[M,K] (int8, quant_act_i8's step order, f32 scale a row) @ dequant(b)[N,K]^T for the
    draft head's 2-bit weight: b uint8 [N, K/4] (four codes a byte), bs_blob the joined rad.planes blob of
    its f16 scale and u8/u4 zero per (row, 128 of K), a_sum f32 [K/128, mpad] the activation's group sums."""
    P = plugin()
    M = y.numel() // N
    query: dict[str, Any] = dict(M=M_param if M_param is not None else M, N=N, K=K, group=128, dtype="w2a8")
    r = P.resolve("gemm_nt_q", query)
    if r is None:
        raise RuntimeError(f"no row serves gemm_nt_q {query}")
    tensors = [_desc(a, abi.RAD_I8), _desc(a_scale, abi.RAD_F32), _desc(b, abi.RAD_U2, shape=[N, K], stride=[K, 1]),
               _desc(bs_blob, abi.RAD_U8), _desc(y, abi.RAD_BF16), _desc(a_sum, abi.RAD_F32), _desc(None, abi.RAD_BF16)]
    rc = P.launch_row(r, ArgPack(tensors, query), _stream())
    if rc != abi.RAD_OK:
        raise RowRefused(r.name, rc)
    return r


def logit_rerank(x: torch.Tensor, head_blob: torch.Tensor, idx_in: torch.Tensor, idx: torch.Tensor,
                 val: torch.Tensor, pairs: torch.Tensor | None = None, *, n_vocab: int, n_embd: int,
                 vocab_off: int = 0) -> Row:
    """R candidate ids a row (idx_in int32 [M, R], global ids) rescored exactly against the joined e4m3
    head and re-sorted: idx int32 [M, R], val f32 [M, R], optional pairs f32 [M, R, 2] (id bits, value).
    x is bf16 or f32 [M, n_embd]."""
    P = plugin()
    M, R = idx_in.shape
    query = dict(M=M, R=R, n_vocab=n_vocab, n_embd=n_embd, vocab_off=vocab_off, dtype="bf16")
    r = P.resolve("logit_rerank", query)
    if r is None:
        raise RuntimeError(f"no row serves logit_rerank {query}")
    xdt = abi.RAD_F32 if x.dtype == torch.float32 else abi.RAD_BF16
    tensors = [_desc(x, xdt), _desc(head_blob, abi.RAD_U8), _desc(idx_in, abi.RAD_I32), _desc(idx, abi.RAD_I32),
               _desc(val, abi.RAD_F32), _desc(pairs, abi.RAD_F32)]
    rc = P.launch_row(r, ArgPack(tensors, query), _stream())
    if rc != abi.RAD_OK:
        raise RowRefused(r.name, rc)
    return r


def quant_act_fp8(x: torch.Tensor, group: int = 128) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16/f32 activations [rows, n] -> (e4m3 codes uint8 [rows, n], f32 scale [rows, n/group])."""
    P = plugin()
    rows, n = x.shape
    ngrp = (n + group - 1) // group
    q = torch.empty((rows, n), dtype=torch.uint8, device=x.device)
    s = torch.empty((rows, ngrp), dtype=torch.float32, device=x.device)
    xdt = abi.RAD_F32 if x.dtype == torch.float32 else abi.RAD_BF16
    rc = P.lib.r3d_b200_quant_act_fp8(x.data_ptr(), xdt, x.stride(0), q.data_ptr(), q.stride(0),
                                      s.data_ptr(), s.stride(0), rows, n, group, _stream())
    if rc != abi.RAD_OK:
        raise RowRefused("quant_act_fp8", rc)
    return q, s


def _act_dt(t: torch.Tensor) -> tuple[int, str]:
    return (abi.RAD_F32, "f32") if t.dtype == torch.float32 else (abi.RAD_BF16, "bf16")


_ARENA: dict[tuple[int, int], torch.Tensor] = {}


def _arena(nbytes: int, device: torch.device) -> torch.Tensor:
    """the launch arena an engine hands a row whose scratch hook asks for one: kept per device, grown only"""
    key = (device.index or 0, 0)
    t = _ARENA.get(key)
    if t is None or t.numel() < nbytes:
        t = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _ARENA[key] = t
    return t


def _issue(op: str, query: dict, tensors: list, scratch_hook=None, device: torch.device | None = None) -> Row:
    P = plugin()
    r = P.resolve(op, query)
    if r is None:
        raise RuntimeError(f"no row serves {op} {query}")
    pack = ArgPack(tensors, query)
    if scratch_hook is not None and device is not None:
        need = int(scratch_hook(pack.args))
        if need > 0:
            arena = _arena(need, device)
            pack = ArgPack(tensors, query, scratch=arena.data_ptr(), scratch_bytes=arena.numel())
    rc = P.launch_row(r, pack, _stream())
    if rc != abi.RAD_OK:
        raise RowRefused(r.name, rc)
    return r


def quant_act_fp8_row(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor, *, group: int = 128) -> Row:
    """The quant_act_fp8 op through its row: x [M, n] bf16/f32 -> q e4m3 (uint8) [M, n], scale f32."""
    dt, name = _act_dt(x)
    query = dict(M=x.shape[0], n=x.shape[-1], group=group, dtype=name)
    return _issue("quant_act_fp8", query, [_desc(x, dt), _desc(q, abi.RAD_F8E4M3), _desc(scale, abi.RAD_F32)])


def gated_quant_fp8_row(gate_up: torch.Tensor, q: torch.Tensor, scale: torch.Tensor,
                        out: torch.Tensor | None = None, *, group: int = 128, act: str | None = None) -> Row:
    """The gated_quant_fp8 op through its row: gate_up [M, 2n] (gate half first) -> q [M, n], scale and,
    when `out` is given, the bf16/f32 gated product."""
    dt, name = _act_dt(gate_up)
    query = dict(M=gate_up.shape[0], n=gate_up.shape[-1] // 2, group=group, dtype=name)
    if act is not None:
        query["act"] = act
    odt = _act_dt(out)[0] if out is not None else abi.RAD_BF16
    return _issue("gated_quant_fp8", query, [_desc(gate_up, dt), _desc(q, abi.RAD_F8E4M3),
                                             _desc(scale, abi.RAD_F32), _desc(out, odt)])


def rmsnorm_quant_fp8(x: torch.Tensor, w: torch.Tensor, q: torch.Tensor, scale: torch.Tensor, *, eps: float,
                      residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
                      group: int = 128, wadd: float | None = None) -> Row:
    """The rmsnorm_quant_fp8 op through its row: x [M, n] bf16, w [n]; `residual` (bf16, updated in place
    with the narrowed sum) selects the fused-add form; `out` receives the bf16/f32 norm output."""
    query = dict(M=x.shape[0], n=x.shape[-1], eps=float(eps), group=group, dtype="bf16")
    if wadd is not None:
        query["wadd"] = float(wadd)
    odt = _act_dt(out)[0] if out is not None else abi.RAD_BF16
    return _issue("rmsnorm_quant_fp8", query, [_desc(x, abi.RAD_BF16), _desc(residual, abi.RAD_BF16),
                                               _desc(w, _act_dt(w)[0]), _desc(q, abi.RAD_F8E4M3),
                                               _desc(scale, abi.RAD_F32), _desc(out, odt)])


def row_topk(x: torch.Tensor, idx: torch.Tensor, val: torch.Tensor, pairs: torch.Tensor | None = None, *,
             R: int, vocab_off: int | None = None, arena: bool = True) -> Row:
    """The row_topk op through its row: x [M, N] bf16 -> idx i32 [M, R], val f32 [M, R] and, when given,
    pairs f32 [M, R, 2] holding (bits of the int32 id, value). `arena`: hand the row the launch arena its
    scratch hook asks for (as an engine does); without it the row uses planes of its own."""
    query = dict(M=x.shape[0], N=x.shape[-1], R=R, dtype="bf16")
    if vocab_off is not None:
        query["vocab_off"] = int(vocab_off)
    return _issue("row_topk", query, [_desc(x, abi.RAD_BF16), _desc(idx, abi.RAD_I32), _desc(val, abi.RAD_F32),
                                      _desc(pairs, abi.RAD_F32)],
                  plugin().lib.r3d_rad_row_topk_scratch if arena else None, x.device)


def sample_argmax(logits: torch.Tensor, token: torch.Tensor, params: torch.Tensor | None = None) -> Row:
    """The sample_argmax op through its row: logits f32 [M, n_vocab] -> token i32 [M] (greedy, ties to the
    lower id). `params` is the engine's per-row parameter blob; the row does not read it."""
    query = dict(M=logits.shape[0], n_vocab=logits.shape[1])
    return _issue("sample_argmax", query, [_desc(logits, abi.RAD_F32), _desc(params, abi.RAD_U8),
                                           _desc(token, abi.RAD_I32)],
                  plugin().lib.r3d_rad_sample_argmax_scratch, logits.device)


# ---------------------------------------------------------------------- the int8 band and its sampler
_NAME_OF = {torch.float32: "f32", torch.bfloat16: "bf16"}
_KIND_OF = {torch.float32: 0, torch.bfloat16: 1}
_I8, _F32, _I32 = 2, 0, 3
_bind = None


def _load_bind():
    """_bind.so stands beside the plugin and uses the same loaded library."""
    global _bind
    plugin()
    try:
        from . import _bind as loaded
    except ImportError as e:
        built = Path(__file__).with_name("_bind.so").exists()
        why = f"does not load with this torch ({e})" if built else "is not built"
        raise ImportError(f"libr3d_b200/_bind.so {why}: run `python -m libr3d_b200.build`") from e
    _bind = loaded
    return loaded


def _run(op: str, params: tuple, *tensors) -> None:
    """One call of `op` on the operands' device, on that device's current stream. `params`: (key, value) pairs;
    `tensors`: by schema position, None where an optional one is absent."""
    not_taken = (_bind or _load_bind()).issue(op, params, *tensors)
    if not_taken is not None:
        row, rc = not_taken
        if row is None:
            raise RuntimeError(f"no row serves {op} {dict(params)}")
        raise RowRefused(row, rc)


def gemm_i8a8(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
              y: torch.Tensor | None = None, *, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """y[..., N] = (sum_k a[..., k] * b[n, k]) * a_scale[...] * b_scale[n]: int8 codes [..., K] and [N, K], one f32
    scale a token ([...] or [..., 1]) and one f32 or bf16 scale a channel ([N] or [N, 1]). The sum is exact (K at
    most 131071). The result is of `out_dtype` (bf16 or f32), or of y's type where y is given: f32 rounds once (twice
    where the sum is 2^24 or more), bf16 narrows the two products in f32. Rows off the 16-byte grid (K not a multiple of
    16) are served by a kernel some 10 to 50 times slower."""
    N, K = b.shape
    if y is None:
        if out_dtype not in _KIND_OF:
            raise TypeError(f"gemm_i8a8: bf16 or f32 results, got {out_dtype}")
        y = (_bind or _load_bind()).rows(a, N, _KIND_OF[out_dtype])
    M = a.numel() // K if K else 0
    if M or not K:                                  # no tokens: nothing to do
        _run("gemm_nt_q", (("M", M), ("N", N), ("K", K), ("group", K), ("dtype", "i8a8")), a, a_scale, b, b_scale, y)
    return y


def _codes_for(x: torch.Tensor, n: int, q: torch.Tensor | None, scale: torch.Tensor | None):
    bind = _bind or _load_bind()
    if q is None and scale is None:
        return bind.codes(x, n)
    return bind.rows(x, n, _I8) if q is None else q, bind.rows(x, 1, _F32) if scale is None else scale


def _act_name(op: str, x: torch.Tensor) -> str:
    if x.dtype not in _NAME_OF:
        raise TypeError(f"{op}: bf16 or f32 activations, got {x.dtype}")
    return _NAME_OF[x.dtype]


def quant_token_i8(x: torch.Tensor, q: torch.Tensor | None = None,
                   scale: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16/f32 activations [..., n] -> int8 codes [..., n] and one f32 scale a token [..., 1]:
    scale = max|x| / 127, q = x * 127 / max|x| to the nearest whole number, halves to even; a row whose values all lie
    below 2^-100 has scale 1 and codes 0."""
    n, size = x.shape[-1], x.numel()
    q, scale = _codes_for(x, n, q, scale)
    if size or not n:
        _run("quant_token_i8", (("M", size // max(n, 1)), ("n", n), ("dtype", _NAME_OF.get(x.dtype) or _act_name("quant_token_i8", x))), x, q, scale)
    return q, scale


def gated_quant_token_i8(gate_up: torch.Tensor, q: torch.Tensor | None = None, scale: torch.Tensor | None = None,
                         out: torch.Tensor | None = None, *, act: str = "silu") -> tuple[torch.Tensor, torch.Tensor]:
    """silu(gate) * up (act "sigmoid": sigmoid(gate) * up) of gate_up [..., 2n], gate half first, quantised per token
    as by quant_token_i8 from its f32 values; `out` (bf16 or f32 [..., n]) receives the product itself."""
    n = gate_up.shape[-1] // 2
    q, scale = _codes_for(gate_up, n, q, scale)
    if gate_up.numel() or not n:
        _run("gated_quant_token_i8", (("M", gate_up.numel() // max(2 * n, 1)), ("n", n),
                                      ("dtype", _act_name("gated_quant_token_i8", gate_up)), ("act", act)), gate_up, q, scale, out)
    return q, scale


def rmsnorm_quant_token_i8(x: torch.Tensor, w: torch.Tensor, q: torch.Tensor | None = None,
                           scale: torch.Tensor | None = None, *, eps: float, residual: torch.Tensor | None = None,
                           out: torch.Tensor | None = None, wadd: float = 0.0) -> tuple[torch.Tensor, torch.Tensor]:
    """x / sqrt(mean(x^2) + eps) * (w + wadd) over [..., n], quantised per token as by quant_token_i8 from its f32
    values. `residual` (x's type, updated in place with x + residual) selects the fused-add form, whose norm reads
    the stored sum; `out` (bf16 or f32) receives the norm itself."""
    n = x.shape[-1]
    q, scale = _codes_for(x, n, q, scale)
    if x.numel() or not n:
        _run("rmsnorm_quant_token_i8",
             (("M", x.numel() // max(n, 1)), ("n", n), ("eps", float(eps)), ("wadd", float(wadd)),
              ("dtype", _act_name("rmsnorm_quant_token_i8", x))), x, residual, w, q, scale, out)
    return q, scale


def sample_nucleus(logits: torch.Tensor, u: torch.Tensor, *, temperature: torch.Tensor | None = None,
                   top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None,
                   min_p: torch.Tensor | None = None, token: torch.Tensor | None = None,
                   logprob: torch.Tensor | None = None, kept: torch.Tensor | None = None) -> torch.Tensor:
    """One token a row of logits (f32 or bf16 [..., n_vocab]) from the row's number u in [0, 1) -> int32 [...].

    Tokens are ordered by logit, ties to the lower id. top_k (int32) keeps the first k (k <= 0: all), top_p the
    shortest first part that holds p of what top_k left (p >= 1: all), min_p those at least min_p times as likely as
    the first; the first always stays. The answer is the first kept id, ascending, at which the running share of the
    kept probability exceeds u. temperature <= 0 is greedy. Every parameter is a plane with one value a row (f32
    but for top_k), or None. -inf and NaN logits are masked; a row with nothing left reports -1. A token
    less than some 2^-45 times as likely as the first has no share.
    `logprob` (f32) receives the log of the token's share of what was kept, `kept` (int32) how many tokens were."""
    V = logits.shape[-1]
    if token is None:
        token = (_bind or _load_bind()).rows(logits, -1, _I32)
    if logits.numel() or not V:
        _run("sample_nucleus", (("M", logits.numel() // max(V, 1)), ("n_vocab", V), ("dtype", _act_name("sample_nucleus", logits))),
             logits, u, temperature, top_k, top_p, min_p, token, logprob, kept)
    return token


class BoundGemm:
    """A gemm_nt_q band declared once and issued many times, the way the engine uses a row:
    the row is resolved and the RadArgs built at declare time over fixed device buffers; each
    `issue()` is one call of the row's launch pointer on the current stream. Buffers must
    outlive the object."""

    def __init__(self, a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor,
                 b_scale: torch.Tensor, y: torch.Tensor, *, dtype: str, N: int, K: int,
                 row: str | None = None):
        self._device = _check_i8(a, a_scale, b, b_scale, y) if dtype == "i8a8" else None
        P = plugin()
        M = y.numel() // N
        group = _group_of(dtype, K)
        query: dict[str, Any] = dict(M=M, N=N, K=K, group=group, dtype=dtype)
        self.row = (P.resolve("gemm_nt_q", query) if row is None
                    else next(x for x in P.rows() + P.ext_rows() if x.name == row))
        if self.row is None:
            raise RuntimeError(f"no row serves gemm_nt_q {query}")
        self._keep = (a, a_scale, b, b_scale, y)
        self.pack = ArgPack(_gemm_descs(a, a_scale, b, b_scale, y, dtype, K), query)
        self._fn = P._launch_t(self.row.launch)
        import ctypes as _C
        self._argp = _C.byref(self.pack.args)
        self._C = _C

    def issue(self) -> None:
        rc = _on_device(self._device, lambda: self._fn(self._argp, self._C.c_void_p(_stream())))
        if rc != abi.RAD_OK:
            raise RowRefused(self.row.name, rc)

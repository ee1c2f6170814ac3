"""The operators of the int8 step and its sampler: what is measured, and their plain forms.

  gemm         ops.gemm_i8a8               y[M, N] = (sum_k a[m, k] * b[n, k]) * a_scale[m] * b_scale[n], int8 codes, one scale a token and a channel
  rmsnorm      ops.rmsnorm_quant_token_i8  residual += x; h = residual * rsqrt(mean(residual^2) + eps) * w; int8 codes of h, one scale a token
  gated        ops.gated_quant_token_i8    h = silu(gate) * up; int8 codes of h, one scale a token
  quant        ops.quant_token_i8          int8 codes of x, one scale a token
  sample       ops.sample_nucleus          a token a row: temperature, top-k, top-p, min-p and the given random number

Each function below is the operator in elementary torch operations; where `own` is set the framework's call takes its
place. Codes are returned as the values they stand for.
"""
import math

import torch

own = False

_LARGEST = 8192 * 27648 * 5120


# ------------------------------------------------------------------ cases
def listed():
    return [
        # a single sequence's step through a square projection: latency
        dict(name="gemm 1x4096x4096", op="gemm", M=1, N=4096, K=4096, out="bf16"),
        # sixteen tokens (four sequences with three drafted tokens each) through gate and up
        dict(name="gemm 16x27648x5120", op="gemm", M=16, N=27648, K=5120, out="bf16"),
        # a ragged batch through an odd vocabulary-like width, f32 out, K not a multiple of 128
        dict(name="gemm 77x5119x13808 f32", op="gemm", M=77, N=5119, K=13808, out="f32"),
        # a prompt through gate and up
        dict(name="gemm 8192x27648x5120", op="gemm", M=8192, N=27648, K=5120, out="bf16"),
        # the norm in front of a projection, decode and prompt
        dict(name="rmsnorm 4x5120", op="rmsnorm", M=4, n=5120, x="bf16", residual=True),
        dict(name="rmsnorm 8192x5120", op="rmsnorm", M=8192, n=5120, x="bf16", residual=True),
        # the activation between gate_up and down, decode and prompt
        dict(name="gated 16x13824", op="gated", M=16, n=13824, x="bf16"),
        dict(name="gated 8192x13824", op="gated", M=8192, n=13824, x="bf16"),
        # the attention's output in front of its projection: a few tokens, and a ragged prompt
        dict(name="quant 3x6144", op="quant", M=3, n=6144, x="bf16"),
        dict(name="quant 4099x5120", op="quant", M=4099, n=5120, x="bf16"),
        # one sequence with one setting; a batch whose rows have settings of their own, some of them masked
        dict(name="sample 1x151936", op="sample", M=1, V=151936, x="f32", rows="one"),
        dict(name="sample 64x151936 mixed", op="sample", M=64, V=151936, x="bf16", rows="mixed"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gemm", "gemm", "gemm", "rmsnorm", "gated", "quant", "sample", "sample"])
    if op == "gemm":
        while True:
            M, N = _log(rng, 1, 8192), _log(rng, 512, 32000)
            K = 16 * _log(rng, 32, 1024)
            if rng.random() < 0.5:
                K = -(-K // 128) * 128
            if rng.random() < 0.5:
                N = -(-N // 64) * 64
            if M * N * K <= _LARGEST:
                return dict(op=op, M=M, N=N, K=K, out=rng.choice(["bf16", "bf16", "f32"]))
    if op == "sample":
        return dict(op=op, M=_log(rng, 1, 256), V=_log(rng, 1000, 262144), x=rng.choice(["f32", "bf16"]),
                    rows=rng.choice(["one", "mixed", "plain"]))
    n = _log(rng, 256, 16384)
    if rng.random() < 0.7:
        n = -(-n // 64) * 64
    case = dict(op=op, M=min(_log(rng, 1, 16384), 8192 * 13824 // n), n=n, x=rng.choice(["bf16", "bf16", "f32"]))
    if op == "rmsnorm":
        case["residual"] = rng.random() < 0.7
    return case


_TYPE = {"bf16": torch.bfloat16, "f32": torch.float32}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda", dtype=torch.float32)

    op = case["op"]
    s = dict(case)
    if op == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        s["a"] = (randn(M, K) * 30).round_().clamp_(-127, 127).to(torch.int8)
        s["b"] = (randn(N, K) * 32).round_().clamp_(-127, 127).to(torch.int8)
        s["a_scale"] = rand(M, 1) * 0.03 + 0.02
        s["b_scale"] = rand(N, 1) * 3e-4 + 4e-4
    elif op == "sample":
        M, V, t = case["M"], case["V"], _TYPE[case["x"]]
        x = randn(M, V) * 2
        # a head of likely tokens over the bulk of the vocabulary
        at = torch.randint(0, V, (M, 96), generator=g, device="cuda")
        x.scatter_add_(1, at, rand(M, 96) * 12)
        if case["rows"] == "mixed":
            # every fifth row follows a grammar that leaves a few tokens
            masked = (torch.arange(M, device="cuda") % 5 == 4)[:, None] & (rand(M, V) > 0.002)
            masked[:, 0] = False
            x.masked_fill_(masked, -math.inf)
        s["logits"] = x.to(t)
        s["u"] = rand(M)
        if case["rows"] == "one":
            s["temperature"] = torch.full((M,), 0.8, device="cuda")
            s["top_k"] = torch.full((M,), 50, device="cuda", dtype=torch.int32)
            s["top_p"] = torch.full((M,), 0.95, device="cuda")
            s["min_p"] = None
        elif case["rows"] == "plain":
            s["temperature"] = torch.full((M,), 1.0, device="cuda")
            s["top_k"] = s["top_p"] = s["min_p"] = None
        else:
            i = torch.arange(M, device="cuda")
            s["temperature"] = torch.where(i % 7 == 6, 0.0, 0.5 + rand(M))
            s["top_k"] = torch.where(i % 3 == 0, 0, torch.randint(1, 200, (M,), generator=g, device="cuda")).to(torch.int32)
            s["top_p"] = torch.where(i % 4 == 3, 1.0, 0.5 + 0.49 * rand(M))
            s["min_p"] = torch.where(i % 2 == 0, 0.0, 0.1 * rand(M))
    else:
        M, n, t = case["M"], case["n"], _TYPE[case["x"]]
        # token-dependent sizes and a few large channels, as hidden states have them
        size = 0.5 + rand(M, 1)
        if op == "gated":
            s["gate_up"] = (randn(M, 2 * n) * size).to(t)
        else:
            wide = 1 + 15 * (rand(n) > 0.995)
            s["x"] = (randn(M, n) * size * wide).to(t)
        if op == "rmsnorm":
            s["w"] = (1 + 0.1 * randn(n)).to(t)
            s["residual"] = (randn(M, n) * 2).to(t) if case["residual"] else None
            s["eps"] = 1e-6
    return s


# ------------------------------------------------------------------ plain forms
def _codes(h):
    """The int8 codes of the rows of h (f32) and their scale: amax / 127, or 1 where the row is all zeros."""
    amax = h.abs().amax(-1, keepdim=True)
    zero = amax == 0
    scale = torch.where(zero, 1.0, amax / 127)
    step = torch.where(zero, 0.0, 127 / amax)
    return torch.round(h * step).clamp(-127, 127).to(torch.int8), scale


def _values(q, scale):
    return torch.mul(q, scale, out=torch.empty(q.shape, dtype=torch.bfloat16, device=q.device))


def _gemm(s):
    # sums of products of codes pass 2^24: 64 bits
    y = s["a"].double() @ s["b"].double().t()
    return (y * s["a_scale"].double() * s["b_scale"].double().t()).to(_TYPE[s["out"]])


def _rmsnorm(s):
    h = s["x"]
    if s["residual"] is not None:
        h = s["residual"].copy_(h.float() + s["residual"].float())
    h = h.float()
    h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + s["eps"]) * s["w"].float()
    return _codes(h)


def _gated(s):
    gate, up = s["gate_up"].float().chunk(2, dim=-1)
    return _codes(gate / (1 + torch.exp(-gate)) * up)


def _sample(s):
    x, V = s["logits"].double(), s["V"]
    off = torch.zeros(s["M"], 1, device=x.device, dtype=torch.float64)
    t = s["temperature"][:, None].double()
    k = s["top_k"][:, None] if s["top_k"] is not None else off
    p = s["top_p"][:, None].double() if s["top_p"] is not None else off + 1
    low = s["min_p"][:, None].double() if s["min_p"] is not None else off
    k = torch.where(t > 0, torch.where(k > 0, k, V), 1)
    best = x.amax(-1, keepdim=True)
    w = torch.exp((x - best) / torch.where(t > 0, t, 1.0))
    order = x.argsort(dim=-1, descending=True, stable=True)
    ws, rank = w.gather(1, order), torch.arange(V, device=x.device)
    keep = (rank < k) & (x.gather(1, order) > -math.inf)
    part = ws * keep
    before = part.cumsum(-1) - part
    keep &= (p >= 1) | (rank == 0) | (before < p * part.sum(-1, keepdim=True))
    keep &= (rank == 0) | (ws >= low)
    w = w * torch.zeros_like(keep).scatter_(1, order, keep)
    cum = w.cumsum(-1)
    total = w.sum(-1, keepdim=True)
    token = ((cum > s["u"][:, None].double() * total) & (w > 0)).int().argmax(-1)
    logprob = torch.log(w.gather(1, token[:, None]) / total)[:, 0]
    return token.int(), logprob.float(), keep.sum(-1).int()


def run(s):
    op = s["op"]
    if own:
        from libr3d_b200 import ops
    if op == "gemm":
        if own:
            return ops.gemm_i8a8(s["a"], s["a_scale"], s["b"], s["b_scale"], out_dtype=_TYPE[s["out"]])
        return _gemm(s)
    if op == "sample":
        if own:
            x = s["logits"]
            logprob = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
            kept = torch.empty(x.shape[0], dtype=torch.int32, device=x.device)
            token = ops.sample_nucleus(x, s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                       min_p=s["min_p"], logprob=logprob, kept=kept)
            return dict(token=token, logprob=logprob, kept=kept)
        token, logprob, kept = _sample(s)
        return dict(token=token, logprob=logprob, kept=kept)
    if op == "rmsnorm":
        if own:
            q, scale = ops.rmsnorm_quant_token_i8(s["x"], s["w"], eps=s["eps"], residual=s["residual"])
        else:
            q, scale = _rmsnorm(s)
    elif op == "gated":
        q, scale = ops.gated_quant_token_i8(s["gate_up"]) if own else _gated(s)
    else:
        q, scale = ops.quant_token_i8(s["x"]) if own else _codes(s["x"].float())
    out = dict(values=_values(q, scale), scale=scale)
    if op == "rmsnorm" and s["residual"] is not None:
        out["residual"] = s["residual"]
    return out


# ------------------------------------------------------------------ the work of a pass
def work(case):
    op = case["op"]
    if op == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        return dict(bytes=M * K + N * K + 4 * (M + N) + M * N * (2 if case["out"] == "bf16" else 4), flops=2 * M * N * K)
    size = 2 if case["x"] == "bf16" else 4
    if op == "sample":
        M, V = case["M"], case["V"]
        return dict(bytes=M * V * size + M * 32, flops=4 * M * V)
    M, n = case["M"], case["n"]
    if op == "rmsnorm":
        return dict(bytes=M * n * (size + 1 + (2 * size if case["residual"] else 0)) + n * size + 4 * M, flops=8 * M * n)
    if op == "gated":
        return dict(bytes=M * n * (2 * size + 1) + 4 * M, flops=10 * M * n)
    return dict(bytes=M * n * (size + 1) + 4 * M, flops=4 * M * n)


# ------------------------------------------------------------------ 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "gemm":
        # whole numbers below 2^53, a part of K at a time: every sum is exact in 64 bits
        total = torch.zeros(case["M"], case["N"], dtype=torch.float64, device="cuda")
        for at in range(0, case["K"], 2048):
            total += torch.matmul(s["a"][:, at:at + 2048].to(torch.float64), s["b"][:, at:at + 2048].to(torch.float64).T)
        total *= s["a_scale"].to(torch.float64)
        total *= s["b_scale"].to(torch.float64).reshape(1, -1)
        return total
    if op == "sample":
        got = []
        # row by row on sorted values: the kept ones are the first of the sorted row
        for m in range(case["M"]):
            value, ids = torch.sort(s["logits"][m].to(torch.float64), descending=True, stable=True)
            t = float(s["temperature"][m])
            if t <= 0:
                got.append(0.0)
                continue
            weight = torch.exp(value / t - value[0] / t)
            n = int((value > -math.inf).sum())
            if s["top_k"] is not None and int(s["top_k"][m]) > 0:
                n = min(n, int(s["top_k"][m]))
            mass = torch.cumsum(weight[:n], 0)
            if s["top_p"] is not None and float(s["top_p"][m]) < 1:
                n = min(n, int((mass < float(s["top_p"][m]) * mass[-1]).sum()) + 1)
            if s["min_p"] is not None:
                n = min(n, max(1, int((weight >= float(s["min_p"][m])).sum())))
            weight = weight[torch.sort(ids[:n]).indices]
            mass = torch.cumsum(weight, 0)
            at = min(int((mass <= float(s["u"][m]) * mass[-1]).sum()), n - 1)
            got.append(float(torch.log(weight[at] / mass[-1])))
        return dict(token=None, logprob=torch.tensor(got, dtype=torch.float64), kept=None)
    if op == "gated":
        v = s["gate_up"].to(torch.float64)
        v = v[:, :case["n"]] * torch.sigmoid(v[:, :case["n"]]) * v[:, case["n"]:]
    elif op == "rmsnorm":
        v = s["x"].to(torch.float64)
        if case["residual"]:
            v = (v + s["residual"].to(torch.float64)).to(s["x"].dtype).to(torch.float64)
        stored = v
        v = v / torch.sqrt((v * v).sum(1, keepdim=True) / case["n"] + s["eps"]) * s["w"].to(torch.float64)
    else:
        v = s["x"].to(torch.float64)
    largest = torch.max(v.max(1, keepdim=True).values, -v.min(1, keepdim=True).values)
    scale = torch.where(largest > 0, largest / 127, torch.ones_like(largest))
    out = dict(values=torch.round(v / scale) * scale, scale=scale)
    if op == "rmsnorm" and case["residual"]:
        out["residual"] = stored
    return out

"""sample_nucleus where min-p's bound falls next to a logit of 0: f32 numbers lie closer together there than the bound
itself is known, which has to leave every other token on its side of it."""
import pytest
import torch

from test_gpu_int8_step import _check_sample, _rng

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32

# largest logit, min-p, temperature: mx + T log(min-p) lies within 1e-9 of 0
BOUNDS = [(2.416025161743164, 0.0892757698893547, 1.0), (2.361177682876587, 0.09430909156799316, 1.0),
          (0.6148342490196228, 0.6637235879898071, 1.5), (0.9523961544036865, 0.38581544160842896, 1.0),
          (0.6007784008979797, 0.5483846068382263, 1.0), (0.9649723768234253, 0.38099372386932373, 1.0),
          (0.3650858402252197, 0.6335874199867249, 0.8), (0.7425498962402344, 0.34618374705314636, 0.7),
          (1.0696794986724854, 0.26260629296302795, 0.8), (0.9692445993423462, 0.5240526795387268, 1.5),
          (0.9324755668640137, 0.2639203369617462, 0.7), (0.3788808584213257, 0.6846271753311157, 1.0),
          (0.6007820963859558, 0.548382580280304, 1.0), (0.5372607111930847, 0.5109028220176697, 0.8),
          (0.18495401740074158, 0.7935866713523865, 0.8), (1.9893803596496582, 0.05831056460738182, 0.7)]


@pytest.mark.parametrize("others", ["none", "top-p", "few", "many", "few and top-p", "many and top-p"])
@pytest.mark.parametrize("V", [50, 3000, 70000, 900001])
def test_min_p_bound_next_to_zero(V, others):
    g = _rng(V)
    M = len(BOUNDS)
    mx, low, t = (torch.tensor(c, dtype=F32, device="cuda") for c in zip(*BOUNDS))
    # tokens on both sides of the bound, all of them further from it than 1e-3
    x = torch.rand(M, V, generator=g, device="cuda") * 2 - 1
    x = torch.where(x > 0, 1e-3 + x * (mx[:, None] - 2e-3), -1e-3 + 3 * x)
    x.scatter_(1, torch.randint(0, V, (M, 1), generator=g, device="cuda"), mx[:, None])
    k = torch.full((M,), 40 if "few" in others else V - V // 4, dtype=torch.int32, device="cuda") if "few" in others or "many" in others else None
    p = torch.full((M,), 0.9, device="cuda") if "top-p" in others else None
    for _ in range(3 if V < 100000 else 1):
        _check_sample(x, torch.rand(M, generator=g, device="cuda"), t, k, p, low)

"""8-bit optimizer states on the GPU where a step's arithmetic leaves the ordinary
range, and where calls are mixed. Oracle: oracle/state8_ref.py."""
import math

import pytest
import torch

from oracle import state8_ref as ref
from sol_b200 import AdamW, EmaWeights, _lib, state8

pytestmark = pytest.mark.gpu

KEYS = ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _optimizer(ps, **kw):
    return AdamW(ps, **{"lr": 1.2e-2, "betas": (0.9, 0.95), "eps": 1e-8, "weight_decay": 0.0, "state_dtype": torch.int8,
                        "min_8bit_numel": 0, **kw})


FORMS = [(torch.float32, "none"), (torch.bfloat16, "none"), (torch.bfloat16, "bf16_mt")]


# ------------------------------------------- second moments that overflow --
@pytest.mark.parametrize("dtype,master", FORMS)
@pytest.mark.parametrize("wd,cautious", [(0.0, False), (0.1, False), (0.1, True)])
@pytest.mark.parametrize("n", [1000, 16384])
def test_an_overflowed_second_moment_leaves_the_weight(cuda, dtype, master, wd, cautious, n):
    """g = 1e30: g^2 is infinite, m is not, and m / inf is 0. Only decay moves that weight in this step; its neighbours'
    steps are those without it. (n: the tail path, and whole chunks with vector accesses.) The pass with wide moments
    gives NaN here: it makes v as torch's fused pass does, fma(-beta2, g^2, g^2), inf - inf."""
    hot = torch.tensor([0, 300, n - 1])
    w0 = (torch.randn(n, generator=_gen(0)) * 0.02).to(dtype)
    g = (torch.randn(n, generator=_gen(1)) * 1e-3).to(dtype)
    got = []
    for size, eps in ((1e30, 1e-8), (-1e30, 1e-8), (1e30, 0.0), (1.0, 1e-8)):
        p = torch.nn.Parameter(w0.cuda())
        opt = _optimizer([p], master=master, weight_decay=wd, cautious_wd=cautious, eps=eps)
        p.grad = g.clone().index_fill_(0, hot, size).cuda()
        avg = EmaWeights(torch.nn.ParameterList([p]), 0.999)
        avg.update()
        opt.step()
        avg.update()
        w = p.detach().double().cpu()
        if master == "bf16_mt":
            w += opt.state[p]["mant_rem"].double().cpu()
        assert w.isfinite().all() and avg.shadow[0].isfinite().all(), (size, eps)
        got.append((size, eps, w))
    _, _, calm = got.pop()
    rest = torch.ones(n, dtype=torch.bool)
    rest[hot] = False
    for size, eps, w in got:
        m = math.copysign(1.0, size)
        down = wd != 0 and (not cautious)
        keep = w0.double()[hot]
        factor = torch.full_like(keep, 1 - 1.2e-2 * wd) if down else torch.where(keep * m > 0, 1 - 1.2e-2 * wd, 1.0)
        want = keep * factor
        # lr wd, its product and the sum: three halves of an fp32 step; then the stored type (2^-16 with a remainder)
        half = 2.0 ** -16 if master == "bf16_mt" else torch.finfo(dtype).eps / 2
        assert ((w[hot] - want).abs() <= (4 * 2.0 ** -24 + half * (1 + 2.0 ** -8)) * keep.abs()).all(), (size, eps)
        if not wd:
            assert torch.equal(w[hot], keep)
        if eps:
            assert torch.equal(w[rest], calm[rest]), (size, eps)


@pytest.mark.parametrize("dtype,master", FORMS)
def test_a_gradient_that_is_not_finite_makes_its_weight_nan(cuda, dtype, master):
    """m itself is infinite or NaN: inf / inf is NaN; no other weight takes part in this step."""
    for bad in (math.inf, -math.inf, math.nan):
        p = torch.nn.Parameter(torch.zeros(1000, dtype=dtype, device=cuda))
        opt = _optimizer([p], master=master)
        p.grad = torch.full((1000,), 1e-3, dtype=dtype, device=cuda)
        p.grad[300] = bad
        opt.step()
        assert torch.equal(p.detach().isnan().nonzero().flatten().cpu(), torch.tensor([300]))

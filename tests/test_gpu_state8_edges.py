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


# ----------------------------- an eps that does not cover the smallest roots --
def _state(n):
    return {"exp_avg": torch.zeros(n, dtype=torch.int8), "exp_avg_sq": torch.zeros(n, dtype=torch.uint8),
            "exp_avg_scale": torch.zeros(state8.blocks(n)), "exp_avg_sq_scale": torch.zeros(state8.blocks(n))}


@pytest.mark.parametrize("dtype,master", FORMS)
@pytest.mark.parametrize("wd,cautious,ema,clip", [(0.0, False, False, None), (0.1, False, True, None), (0.1, True, False, 0.37),
                                                  (0.0, False, True, 0.37)])
@pytest.mark.parametrize("eps", [0.0, 1e-13])
def test_a_tiny_eps_matches_the_restatement(cuda, dtype, master, wd, cautious, ema, clip, eps):
    """Tolerance: codes and scales equal. The update: m and v each carry at most four roundings of 2^-24 of the sum of
    their positive parts, root, quotient, products and coefficients fewer than 24 more, doubled: 64 x 2^-24 of the
    update with nothing cancelled; decay and the sum 4 x 2^-24 of the weight; then the stored type: half a step, or
    2^-16 with a remainder."""
    n = 8192 + 999
    cpu = (torch.randn(n, generator=_gen(2)) * 0.02).to(dtype)
    p = torch.nn.Parameter(cpu.cuda())
    opt = _optimizer([p], master=master, eps=eps, weight_decay=wd, cautious_wd=cautious)
    avg = None
    if ema:
        avg = EmaWeights(torch.nn.ParameterList([p]), 0.999)
        avg.update()
    st = _state(n)
    coef = None if clip is None else torch.tensor(clip, device=cuda)
    for step in range(1, 4):
        x = torch.randn(n, generator=_gen(100 + step)) * torch.exp(2 * torch.randn(n, generator=_gen(200 + step))) * 1e-3
        x[::7] = torch.where(x[::7] < 0, -1e-18, 1e-18)  # squares below every eps here
        x = x.to(dtype)
        p0, rem = p.detach().cpu(), opt.state[p]["mant_rem"].cpu() if "mant_rem" in opt.state[p] else None
        shadow = avg.shadow[0].cpu() if ema else None
        if rem is None and master == "bf16_mt":
            rem = torch.zeros_like(p0)
        p.grad = x.cuda()
        opt._grad_scale = coef
        opt.step()
        if ema:
            avg.update()
        if clip is not None:
            x = (x.float() * torch.tensor(clip)).to(dtype)
        m0 = ref.decode(st["exp_avg"], st["exp_avg_scale"], False).double().abs()
        v0 = ref.decode(st["exp_avg_sq"], st["exp_avg_sq_scale"], True).double()
        w = ref.adamw_step(p0, rem, x, st, lr=1.2e-2, betas=(0.9, 0.95), eps=eps, wd=wd, cautious=cautious, step=step)
        for k in KEYS:
            assert torch.equal(opt.state[p][k].cpu(), st[k]), (k, step)
        a, v = 0.9 * m0 + 0.1 * x.double().abs(), 0.95 * v0 + 0.05 * x.double() ** 2
        up = 1.2e-2 / (1 - 0.9 ** step) * a / (v.sqrt() / math.sqrt(1 - 0.95 ** step) + eps)
        tol = 64 * 2.0 ** -24 * up + 4 * 2.0 ** -24 * (p0.double().abs() + w.abs()) + 1e-42
        got = p.detach().cpu()
        whole = got.double() + opt.state[p]["mant_rem"].cpu().double() if master == "bf16_mt" else got.double()
        half = 2.0 ** -16 if master == "bf16_mt" else torch.finfo(dtype).eps / 2
        # a second moment that is subnormal in fp32 (below 1e-38) keeps fewer bits than the tolerance counts
        held = v > 1e-36
        assert held.float().mean() > 0.8 and ((whole - w).abs() <= tol + half * (w.abs() + tol))[held].all(), step
        if ema:
            want = shadow.double() + (1.0 - 0.999) * (got.double() - shadow.double())
            assert ((avg.shadow[0].cpu().double() - want).abs() <= 4 * 2.0 ** -24 * (shadow.abs() + got.float().abs())).all()


@pytest.mark.parametrize("dtype,master", FORMS)
def test_a_tensors_step_does_not_depend_on_what_shares_its_call(cuda, dtype, master):
    """Groups with eps 1e-8 give the same bits alone and beside groups whose eps is 0 or tiny, decayed or not."""
    n = 3 * 8192 + 77
    def params(k):
        # weights of 0: the update's last places stand in the stored bits
        return [torch.nn.Parameter(torch.zeros(n, dtype=dtype, device=cuda)) for _ in range(k)]
    mixed, alone = params(4), params(4)
    groups = [dict(eps=1e-8), dict(eps=0.0), dict(eps=1e-8, weight_decay=0.1), dict(eps=1e-14, weight_decay=0.1)]
    opts = [_optimizer([{"params": [p], **g} for p, g in zip(mixed, groups)], master=master)]
    opts += [_optimizer([{"params": [p], **g}], master=master) for p, g in zip(alone, groups)]
    for step in range(1, 6):
        for k, (p, q) in enumerate(zip(mixed, alone)):
            p.grad = ((torch.randn(n, generator=_gen(10 * step + k)) + 0.01) * 1e-3).to(dtype).cuda()
            q.grad = p.grad.clone()
        for o in opts:
            o.step()
    for k, (p, q, o) in enumerate(zip(mixed, alone, opts[1:])):
        assert torch.equal(p, q), k
        assert all(torch.equal(opts[0].state[p][x], o.state[q][x]) for x in o.state[q]), k


@pytest.mark.parametrize("dtype,master", FORMS)
@pytest.mark.parametrize("eps", [1e-8, 0.0])
@pytest.mark.parametrize("size", [1e-22, 1e-20, 1e-19, 3e-19, 1e-18, 1e-15])
def test_codes_of_second_moments_near_the_smallest_numbers(cuda, dtype, master, eps, size):
    """Squares that are subnormal, 0 or just normal, in blocks of their own and beside each other: codes and scales are
    the restatement's in every form (bf16 keeps such gradients, and a remainder changes how the roots are taken)."""
    n = 8192 + 1000
    p = torch.nn.Parameter(torch.zeros(n, dtype=dtype, device=cuda))
    opt = _optimizer([p], master=master, eps=eps)
    st = _state(n)
    for step in range(1, 4):
        g = _gen(int(-math.log10(size)) * 10 + step)
        x = torch.randn(n, generator=g) * size * torch.where(torch.rand(n, generator=g) < 0.1, 30.0, 1.0)
        x = x.to(dtype)
        p.grad = x.cuda()
        opt.step()
        ref.adamw_step(torch.zeros(n, dtype=dtype), None, x, st, lr=0.0, betas=(0.9, 0.95), eps=1.0, wd=0.0, cautious=False, step=step)
        for k in KEYS:
            assert torch.equal(opt.state[p][k].cpu(), st[k]), (k, step)

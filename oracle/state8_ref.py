"""8-bit optimizer states restated: the format's definition, one AdamW step and
one momentum pass on it, with torch on the CPU.

What is stored is a function of fp32 states (each product and sum of the
moments rounded by itself), so those run in fp32 and the codes, decided in
float64, have to be equal; the update that follows runs in float64.
"""
import math

import torch

BLOCK = 128


def offset(n, step, root, first=0):
    """u of elements first .. first + n in a step (None: a conversion, 1/2)."""
    if step is None:
        return torch.full((n,), 0.5, dtype=torch.float64)
    h = (torch.arange(first, first + n) * 0x9E3779B9 + step * 0x6A09E667 + (0 if root else 1 << 31)) & 0xFFFFFFFF
    return (h >> 9).double() / (1 << 23)


def encode(x, root, step=None, first=0):
    """(codes in the shape of x, scales) of an fp32 or bf16 tensor."""
    flat = x.detach().float().reshape(-1)
    n = flat.numel()
    nb = -(-n // BLOCK)
    pad = torch.zeros(nb * BLOCK)
    pad[:n] = flat
    rows = pad.view(nb, BLOCK)
    bad = ~rows.isfinite().all(1)
    if root:
        bad |= (rows < 0).any(1)
    size = rows.clamp(min=0).double().sqrt().float() if root else rows.abs()  # the fp32 root, correctly rounded
    s = size.nan_to_num(0.0, 0.0, 0.0).amax(1) if nb else torch.zeros(0)
    if not root:
        s = torch.where(s < 2.0 ** -126, torch.zeros(()), s)
    s = torch.where(bad, torch.full((), math.nan), s)
    levels = 255 if root else 127
    u = torch.zeros(nb * BLOCK, dtype=torch.float64)
    u[:n] = offset(n, step, root, first)
    live = (s > 0)[:, None]
    y = levels * (size.double() / torch.where(s > 0, s, torch.ones(())).double()[:, None]).sqrt()
    q = torch.where(live, (y + u.view(nb, BLOCK)).floor().clamp(max=levels), torch.zeros((), dtype=torch.float64))
    if root:
        q = torch.where(live & (rows > 0), q.clamp(min=1), q)
        codes = q.to(torch.uint8)
    else:
        codes = torch.where(rows < 0, -q, q).to(torch.int8)
    return codes.view(-1)[:n].view(x.shape), s


def decode(codes, scales, root):
    """fp32 values, each product rounded by itself."""
    n = codes.numel()
    s = scales.repeat_interleave(BLOCK)[:n].view(codes.shape)
    q = codes.float()
    if root:
        r = q * q * torch.tensor(1 / 65025) * s
        return r * r
    return q * q.abs() * torch.tensor(1 / 16129) * s


def f32(x):
    return torch.tensor(x, dtype=torch.float64).float()


def adamw_step(p, rem, g, state, *, lr, betas, eps, wd, cautious, step, first=0):
    """One step. state: dict of exp_avg, exp_avg_scale, exp_avg_sq,
    exp_avg_sq_scale, replaced. Returns the updated weight in float64."""
    b1, b2 = betas
    gf = g.float()
    m = f32(b1) * decode(state["exp_avg"], state["exp_avg_scale"], False) + f32(1 - b1) * gf
    v = f32(b2) * decode(state["exp_avg_sq"], state["exp_avg_sq_scale"], True) + f32(1 - b2) * (gf * gf)
    w = p.double() if rem is None else p.double() + rem.double()
    md, vd = m.double(), v.double()
    if wd:
        keep = (md * w > 0) if cautious else torch.ones_like(w, dtype=torch.bool)
        w = torch.where(keep, w - lr * wd * w, w)
    w = w - lr / (1 - b1 ** step) * md / (vd.sqrt() / math.sqrt(1 - b2 ** step) + eps)
    state["exp_avg"], state["exp_avg_scale"] = encode(m, False, step, first)
    state["exp_avg_sq"], state["exp_avg_sq_scale"] = encode(v, True, step, first)
    return w


def momentum_step(g, codes, scales, *, beta, nesterov, step):
    """(u in bf16, codes, scales) of one matrix."""
    gf = g.float()
    m = f32(beta) * decode(codes, scales, False) + f32(1 - beta) * gf
    codes, scales = encode(m, False, step)
    val = decode(codes, scales, False)
    u = f32(beta) * val + f32(1 - beta) * gf if nesterov else val
    return u.to(torch.bfloat16), codes, scales

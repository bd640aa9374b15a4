"""How far training with 8-bit states is from 64-bit ones, on the restatement in
state8_ref.py: updates, the drift of elements that get no gradient any more, the
value bias of second moments, and the orthogonalised update of a matrix.

``python -m oracle.state8_accuracy`` prints the tables (under a minute).
Gradients are normal; an element's standard deviation is 1e-3 times a lognormal
factor of the given spread (sigma), so a block of 128 holds elements of such
different sizes."""
import math

import torch

from . import state8_ref as ref


def gradients(n, spread, seed=0):
    """(standard deviations of n elements, a function that draws the next gradient)."""
    g = torch.Generator().manual_seed(seed)
    std = 1e-3 * torch.exp(spread * torch.randn(n, generator=g))
    return std, lambda: torch.randn(n, generator=g) * std


class Wide:
    """Moments in 64 bits."""

    def __init__(self, n, betas):
        self.m, self.v, self.betas = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64), betas

    def step(self, g, t):
        b1, b2 = self.betas
        self.m, self.v = b1 * self.m + (1 - b1) * g.double(), b2 * self.v + (1 - b2) * g.double() ** 2
        return self.m, self.v


class Eight:
    """Moments in 8 bits. offset: the codes' running offset; else they are rounded to nearest."""

    def __init__(self, n, betas, offset=True):
        nb = -(-n // ref.BLOCK)
        self.m = torch.zeros(n, dtype=torch.int8), torch.zeros(nb)
        self.v = torch.zeros(n, dtype=torch.uint8), torch.zeros(nb)
        self.betas, self.offset = betas, offset

    def step(self, g, t):
        """The moments before they are rounded, which the update uses."""
        b1, b2 = self.betas
        m = ref.f32(b1) * ref.decode(*self.m, False) + ref.f32(1 - b1) * g
        v = ref.f32(b2) * ref.decode(*self.v, True) + ref.f32(1 - b2) * (g * g)
        u = t if self.offset else None
        self.m, self.v = ref.encode(m, False, u), ref.encode(v, True, u)
        return m.double(), v.double()


def update(m, v, betas, t, eps=1e-8):
    """The step in units of lr."""
    return m / (1 - betas[0] ** t) / ((v / (1 - betas[1] ** t)).sqrt() + eps)


def update_error(betas, spread, offset, n=64 * 128, steps=600, seed=0):
    """rms of the update's error over rms of the update, over every 25th of the last 200 steps."""
    _, draw = gradients(n, spread, seed)
    wide, eight = Wide(n, betas), Eight(n, betas, offset)
    num = den = 0.0
    for t in range(1, steps + 1):
        g = draw()
        a, b = update(*wide.step(g, t), betas, t), update(*eight.step(g, t), betas, t)
        if t > steps - 200 and t % 25 == 0:
            num, den = num + float((a - b).square().sum()), den + float(a.square().sum())
    return math.sqrt(num / den)


def drift(betas, spread, offset, n=64 * 128, live=100, steps=600, seed=0):
    """Elements (a tenth) whose gradient is zero after ``live`` steps: mean distance that they move in the ``steps``
    that follow, in units of lr. offset None: 64-bit moments."""
    std, draw = gradients(n, spread, seed)
    dead = torch.rand(n, generator=torch.Generator().manual_seed(seed + 1)) < 0.1
    state = Wide(n, betas) if offset is None else Eight(n, betas, offset)
    moved = torch.zeros(n, dtype=torch.float64)
    for t in range(1, live + steps + 1):
        g = draw()
        if t > live:
            g[dead] = 0
        x = update(*state.step(g, t), betas, t)
        if t > live:
            moved += x
    return float(moved[dead].abs().mean())


def value_bias(beta2, spread, n=256 * 128, steps=400, average=100, seed=0):
    """[(band of an element's root against its block's largest, stored second moment over the 64-bit one)], averages
    over elements and the last steps."""
    betas = (0.9, beta2)
    _, draw = gradients(n, spread, seed)
    wide, eight = Wide(n, betas), Eight(n, betas)
    got, want = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
    for t in range(1, steps + 1):
        g = draw()
        wide.step(g, t)
        eight.step(g, t)
        if t > steps - average:
            got += ref.decode(*eight.v, True).double()
            want += wide.v
    root = want.sqrt().view(-1, ref.BLOCK)
    part = (root / root.amax(1, keepdim=True)).view(-1)
    out = []
    for lo, hi in ((0.3, 1.0), (0.03, 0.3), (0.003, 0.03), (0.0, 0.003)):
        at = (part > lo) & (part <= hi)
        if at.sum() >= 100:
            out.append(((lo, hi), float((got[at] / want[at]).mean())))
    return out


def polar(x):
    u, _, vh = torch.linalg.svd(x.double(), full_matrices=False)
    return u @ vh


def orthogonalised_error(r=128, c=512, steps=40, beta=0.95, seed=0):
    """Relative Frobenius error of the orthogonal factor of NorMuon's u: (8-bit momentum, 64-bit momentum with u rounded to bf16)."""
    g = torch.Generator().manual_seed(seed)
    codes, scales = torch.zeros(r, c, dtype=torch.int8), torch.zeros(r * c // ref.BLOCK)
    m = torch.zeros(r, c, dtype=torch.float64)
    for t in range(1, steps + 1):
        grad = torch.randn(r, c, generator=g) * 1e-3
        u8, codes, scales = ref.momentum_step(grad, codes, scales, beta=beta, nesterov=True, step=t)
        m = beta * m + (1 - beta) * grad.double()
    u = beta * m + (1 - beta) * grad.double()
    want = polar(u)
    return tuple(float((polar(x) - want).norm() / want.norm()) for x in (u8, u.to(torch.bfloat16)))


def main():
    torch.set_num_threads(4)
    print("update error (rms, %): offset / nearest")
    for b2 in (0.95, 0.99, 0.999):
        row = [f"{100 * update_error((0.9, b2), s, True):5.1f} /{100 * update_error((0.9, b2), s, False):5.1f}" for s in (0.3, 1.0, 1.5)]
        print(f"  beta2 {b2:<6}", "   ".join(row), "  (spread 0.3, 1.0, 1.5)", flush=True)
    print("drift without gradient (lr, 600 steps): offset / nearest / 64 bits")
    for b2 in (0.95, 0.99, 0.999):
        row = ["/".join(f"{drift((0.9, b2), s, o):6.1f}" for o in (True, False, None)) for s in (0.3, 1.0, 1.5)]
        print(f"  beta2 {b2:<6}", "   ".join(row), flush=True)
    print("stored second moment / 64-bit one, by the root's part of the block's largest")
    for b2 in (0.95, 0.999):
        for s in (1.0, 1.5):
            print(f"  beta2 {b2} spread {s}:", ", ".join(f"{lo}-{hi}: {x:.3f}" for (lo, hi), x in value_bias(b2, s)), flush=True)
    print("orthogonalised update (relative): 8-bit momentum %.4f, u in bf16 %.4f" % orthogonalised_error())


if __name__ == "__main__":
    main()

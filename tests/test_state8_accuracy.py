"""8-bit moments against 64-bit ones over many steps, on the restatement
(the kernels are held to that one bit for bit)."""
import math

import pytest
import torch

from oracle import state8_accuracy as acc
from oracle import state8_ref as ref

E = 2.0 ** -24


@pytest.mark.parametrize("spread", [0.3, 1.0, 1.5])
@pytest.mark.parametrize("betas", [(0.9, 0.95), (0.9, 0.999), (0.0, 0.0)])
@pytest.mark.parametrize("offset", [True, False])
def test_moments_stay_within_their_codes_errors(spread, betas, offset):
    """A stored moment differs from what was stored by at most one code step, and a step multiplies that by beta.

    First moment, Y = 127 sqrt(|m| / s): the code q is less than 1 from Y, so the value s q^2 / 127^2 is at most
    s (2 Y + 1) / 127^2 off. Second moment, root r, Y = 255 sqrt(r / s): its root's value is at most
    d = s (2 Y + 1) / 255^2 off (a code raised to 1 too), and its value d (2 r + d). Roundings to fp32: three of the
    decoded value (five for a second moment, whose root's count twice, and one of the root that is coded), one of each
    coefficient, product and sum, and one of g^2: at most 8 (16) x 2^-24 of the positive parts."""
    n = 16 * 128 + 77
    _, draw = acc.gradients(n, spread)
    wide, eight = acc.Wide(n, betas), acc.Eight(n, betas, offset)
    err_m = err_v = code_m = code_v = torch.zeros(n, dtype=torch.float64)
    b1, b2 = betas
    block = torch.arange(n) // ref.BLOCK
    for t in range(1, 151):
        g = draw()
        if t > 60:
            g[::9] = 0  # elements whose gradient stops
        m_was, v_was = wide.m.abs() + err_m + code_m, wide.v + err_v + code_v
        a, v = wide.step(g, t)
        m8, v8 = eight.step(g, t)
        err_m = b1 * (err_m + code_m) + 8 * E * (b1 * m_was + (1 - b1) * g.double().abs())
        err_v = b2 * (err_v + code_v) + 16 * E * (b2 * v_was + (1 - b2) * g.double() ** 2)
        assert ((m8 - a).abs() <= err_m).all() and ((v8 - v).abs() <= err_v).all(), t
        s = eight.m[1].double()[block]
        code_m = s * (2 * 127 * (m8.abs() / s.clamp(min=1e-300)).sqrt() + 1) / 127 ** 2
        s, r = eight.v[1].double()[block], v8.sqrt()
        d = s * (2 * 255 * (r / s.clamp(min=1e-300)).sqrt() + 1) / 255 ** 2
        code_v = d * (2 * r + d)


def test_the_tables_come_out():
    b = (0.9, 0.95)
    assert all(math.isfinite(acc.update_error(b, 1.0, o, n=256, steps=250)) for o in (True, False))
    assert all(math.isfinite(acc.drift(b, 1.0, o, n=256, live=10, steps=20)) for o in (True, False, None))
    assert acc.value_bias(0.95, 1.0, n=1024, steps=20, average=5)
    assert all(math.isfinite(x) for x in acc.orthogonalised_error(16, 64, 3))

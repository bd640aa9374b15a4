"""8-bit optimizer states on the GPU against the restatement in
oracle/state8_ref.py.

Tolerances. Codes and scales: equal (both sides decide them exactly from the
same fp32 states). Updated weights against float64: m and v each carry at most
four roundings of half an fp32 step (2^-24) relative to the sum of their two
positive parts, the root, the quotient (two steps of 2^-23 by its
documentation) and the products a few more: 32 x 2^-24 of the update, doubled
for the parts of m that cancel being bounded by |b1 m| + |w1 g| in the test
itself; then the roundings of the stored weight: half a step of its type, and
2^-16 of it for a bf16 weight with a remainder: bf16 keeps 8 bits, so half a
step of w in [2^e, 2^(e+1)) is 2^(e-8) <= 2^-8 |w|; the remainder is at most
that, and its own rounding at most 2^-8 of the remainder."""
import ctypes
import math

import pytest
import torch

from oracle import state8_ref as ref
from sol_b200 import AdamW, EmaWeights, NorMuonGNS, _lib, build_optimizers, clip_grad_norm_, state8, synth
from sol_b200.checkpoint import load_checkpoint, save_checkpoint

pytestmark = pytest.mark.gpu

SIZES = [1, 2, 7, 8, 9, 127, 128, 129, 255, 256, 257, 1000, 8191, 8192, 8193, 20011]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _values(n, root, what, seed=0):
    g = _gen(seed)
    x = torch.randn(n, generator=g) * torch.exp(2 * torch.randn(n, generator=g))
    if what == "zeros":
        x.zero_()
    elif what == "spike":
        x *= 1e-12
        x[n // 2] = 3.0
    elif what == "subnormal":
        x *= 1e-42
    elif what == "tiny":
        x *= 1e-34
    elif what == "huge":
        x = (x / x.abs().max()) * 3.4e38
    elif what == "quarters":  # the middle between two codes, exactly
        x = torch.where(torch.rand(n, generator=g) < 0.5, 0.25, -0.25)
        x[::97] = 1.0
    elif what == "least":  # ties and scales where a quarter is no longer exact
        x = torch.where(torch.rand(n, generator=g) < 0.5, 2.0 ** -128, 2.0 ** -126 * (1 + 2.0 ** -23)) * (1 + (x > 0))
    elif what == "same":
        x.fill_(-0.37)
    elif what == "sparse":
        x *= torch.rand(n, generator=g) < 0.1
    return x.abs() * (x.abs() if what == "quarters" else 1) if root else x


def _same(a, b):
    """Equal, a NaN to a NaN."""
    return a.dtype == b.dtype and a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


# ------------------------------------------------------------ encode/decode --
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("root", [False, True])
@pytest.mark.parametrize("what", ["normal", "zeros", "spike", "subnormal", "tiny", "huge", "quarters", "least", "same", "sparse"])
def test_encode_and_decode_match_the_definition(cuda, what, root, dtype):
    kind = "root" if root else "signed"
    xs = [_values(n, root, what, seed=n).to(dtype) for n in SIZES]
    got = state8.encode([(x.cuda(), kind) for x in xs])
    vals = state8.decode([(q, s, kind) for q, s in got])
    half = state8.decode([(q, s, kind) for q, s in got], dtype=torch.bfloat16)
    for x, (q, s), v, h in zip(xs, got, vals, half):
        rq, rs = ref.encode(x, root)
        assert _same(s.cpu(), rs), (x.numel(), "scale")
        assert torch.equal(q.cpu(), rq), (x.numel(), "codes")
        rv = ref.decode(rq, rs, root)
        assert _same(v.cpu(), rv)
        assert _same(h.cpu(), rv.to(torch.bfloat16))
        # no value is off by more than half a code step and its fp32 roundings
        ok = x.float().abs() > 0
        top = rs.repeat_interleave(128)[:x.numel()].double()
        y = (255 if root else 127) * ((x.double().sqrt() if root else x.double().abs()) / top.clamp(min=1e-300)).sqrt()
        yv = (255 if root else 127) * ((rv.double().sqrt() if root else rv.double().abs()) / top.clamp(min=1e-300)).sqrt()
        live = ok & (top > 0) & (rv != 0)
        assert ((y - yv).abs()[live] <= torch.where(y < 0.5, 1.0, 0.5001)[live]).all() or what in ("subnormal", "tiny", "least")


@pytest.mark.parametrize("root", [False, True])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_block_with_a_value_that_is_not_finite_reads_as_nan(cuda, bad, root):
    x = _values(1000, root, "normal")
    x[300] = bad
    kind = "root" if root else "signed"
    (q, s), = state8.encode([(x.cuda(), kind)])
    v, = state8.decode([(q, s, kind)])
    hit = torch.zeros(1000, dtype=torch.bool)
    hit[256:384] = True
    assert torch.equal(v.cpu().isnan(), hit)
    rq, rs = ref.encode(x, root)
    assert torch.equal(q.cpu(), rq) and torch.equal(s.cpu().isnan(), rs.isnan())


def test_a_negative_second_moment_reads_as_nan(cuda):
    x = _values(300, True, "normal")
    x[5] = -1e-30
    x[200] = -0.0  # is zero
    (q, s), = state8.encode([(x.cuda(), "root")])
    v, = state8.decode([(q, s, "root")])
    assert v[:128].isnan().all() and not v[128:].isnan().any() and v[200] == 0


@pytest.mark.parametrize("root", [False, True])
def test_decoded_values_encode_to_their_codes(cuda, root):
    codes = torch.arange(256).to(torch.uint8) if root else torch.arange(-127, 128).to(torch.int8)
    codes = torch.cat([codes, codes, codes])[: 3 * 253].clone()
    codes[::128] = 255 if root else 127
    kind = "root" if root else "signed"
    scales = torch.tensor([1.0, 1e-5, 3.3e6, 2.0 ** -60, 17.0, 5e-20])
    v, = state8.decode([(codes.cuda(), scales.cuda(), kind)])
    (q, s), = state8.encode([(v, kind)])
    assert torch.equal(q.cpu(), codes)


def test_pairs_split_and_join(cuda):
    ws = [_values(n, False, "normal", seed=n) for n in SIZES]
    got = state8.encode([(w.cuda(), "pair") for w in ws])
    back = state8.decode([(p, r, "pair") for p, r in got])
    for w, (p, r), b in zip(ws, got, back):
        pe = w.to(torch.bfloat16)
        re = (w - pe.float()).to(torch.bfloat16)
        assert torch.equal(p.cpu(), pe) and torch.equal(r.cpu(), re) and torch.equal(b.cpu(), pe.float() + re.float())


@pytest.mark.parametrize("off", [1, 3, 8])
def test_unaligned_views_and_their_surroundings(cuda, off):
    """Views that start inside an allocation: same codes, and nothing written around them."""
    n = 1003
    for kind, cdt, sdt, sn in (("signed", torch.int8, torch.float32, 8), ("root", torch.uint8, torch.float32, 8),
                               ("pair", torch.bfloat16, torch.bfloat16, n)):
        for dt in (torch.float32, torch.bfloat16):
            x = _values(n, kind == "root", "normal", seed=off).to(dt)
            big = torch.full((n + 64,), 7.0, dtype=dt, device=cuda)
            big[off:off + n] = x.cuda()
            whole, = state8.encode([(x.cuda(), kind)])
            q, s = torch.full((n + 64,), 3, dtype=cdt, device=cuda), torch.full((sn + 8,), 5.0, dtype=sdt, device=cuda)
            arr = (_lib.StateTensor * 1)(_lib.StateTensor(
                big[off:].data_ptr(), q[off:].data_ptr(), s[1:].data_ptr(), n, state8._KINDS[kind], _lib.dtype_code(dt)))
            _lib.check(_lib.load().b2o_state_encode(arr, 1, _lib.stream_ptr()), "encode")
            assert torch.equal(q[off:off + n], whole[0]) and torch.equal(s[1:1 + sn], whole[1])
            assert (q[:off] == 3).all() and (q[off + n:] == 3).all() and s[0] == 5 and (s[1 + sn:] == 5).all()
            out = torch.full((n + 64,), 9.0, dtype=dt, device=cuda)
            ref_v, = state8.decode([(whole[0], whole[1], kind)], dtype=dt)
            state8.decode([(q[off:off + n], s[1:1 + sn], kind)], out=[out[off:off + n]])
            assert torch.equal(out[off:off + n], ref_v) and (out[:off] == 9).all() and (out[off + n:] == 9).all()


def test_more_tensors_than_one_launch_takes(cuda):
    xs = [_values(1 + 37 * i, i % 2 == 1, "normal", seed=i) for i in range(205)]
    kinds = ["root" if i % 2 else "signed" for i in range(205)]
    got = state8.encode([(x.cuda(), k) for x, k in zip(xs, kinds)])
    for x, k, (q, s) in zip(xs, kinds, got):
        rq, rs = ref.encode(x, k == "root")
        assert torch.equal(q.cpu(), rq) and torch.equal(s.cpu(), rs)
    # empty tensors take no part
    (q, s), (e, es) = state8.encode([(xs[3].cuda(), kinds[3]), (torch.zeros(0, 4, device=cuda), "signed")])
    assert torch.equal(q, got[3][0]) and e.shape == (0, 4) and es.numel() == 0
    assert state8.decode([(e, es, "signed")])[0].shape == (0, 4)


def test_conversions_refuse_what_does_not_fit(cuda):
    x = torch.randn(300, device=cuda)
    (q, s), = state8.encode([(x, "signed")])
    with pytest.raises(ValueError, match="scales"):
        state8.decode([(q, s[:2], "signed")])
    with pytest.raises(ValueError, match="codes"):
        state8.decode([(q, s, "root")])
    with pytest.raises(ValueError, match="contiguous"):
        state8.decode([(q[::2], s, "signed")])
    with pytest.raises(ValueError, match="contiguous"):
        state8.encode([(torch.randn(8, 8, device=cuda).t(), "signed")])
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        state8.encode([(x.half(), "signed")])
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        state8.decode([(q, s, "signed")], dtype=torch.float64)
    with pytest.raises(ValueError, match="size"):
        state8.decode([(q, s, "signed")], out=[x[:299]])
    with pytest.raises(ValueError, match="twice"):
        state8.decode([(q, s, "signed"), (q, s, "signed")], out=[x, x])


# -------------------------------------------------------------------- AdamW --
SHAPES = [(1,), (8,), (77,), (128,), (3, 43), (33, 77), (4099,), (5, 64, 33)]


def _tensors(dtype, seed, shapes=SHAPES):
    g = _gen(seed)
    return [(torch.randn(s, generator=g) * 0.02).to(dtype) for s in shapes]


def _grads(ps, seed):
    g = _gen(1000 + seed)
    out = []
    for p in ps:
        x = torch.randn(p.shape, generator=g) * 1e-3
        flat = x.view(-1)
        flat[::50] *= 30
        flat[torch.rand(flat.shape, generator=g) < 0.05] = 0
        out.append(x.to(p.dtype))
    return out


def _optimizer(ps, **kw):
    kw = {"lr": 1.2e-2, "betas": (0.9, 0.95), "eps": 1e-8, "weight_decay": 0.0, "state_dtype": torch.int8,
          "min_8bit_numel": 0, **kw}
    return AdamW(ps, **kw)


KEYS = ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale")


@pytest.mark.parametrize("dtype,master", [(torch.float32, "none"), (torch.bfloat16, "none"), (torch.bfloat16, "bf16_mt")])
@pytest.mark.parametrize("wd,cautious,betas,ema", [(0.0, False, (0.9, 0.95), True), (0.1, False, (0.9, 0.999), False),
                                                   (0.1, True, (0.75, 0.95), True), (0.0, False, (0.0, 0.0), False)])
def test_adamw_step_matches_the_restatement(cuda, dtype, master, wd, cautious, betas, ema):
    cpu = _tensors(dtype, 0)
    ps = [torch.nn.Parameter(x.cuda()) for x in cpu]
    opt = _optimizer(ps, betas=betas, weight_decay=wd, cautious_wd=cautious, master=master)
    avg = None
    if ema:
        avg = EmaWeights(torch.nn.ParameterList(ps), 0.999)
        avg.update()
    states = [{"exp_avg": torch.zeros(x.shape, dtype=torch.int8), "exp_avg_sq": torch.zeros(x.shape, dtype=torch.uint8),
               "exp_avg_scale": torch.zeros(state8.blocks(x.numel())),
               "exp_avg_sq_scale": torch.zeros(state8.blocks(x.numel()))} for x in cpu]
    for step in range(1, 7):
        grads = _grads(cpu, step)
        before = [(p.detach().cpu(), opt.state[p]["mant_rem"].cpu() if "mant_rem" in opt.state[p] else None,
                   avg.shadow[i].cpu() if ema else None) for i, p in enumerate(ps)]
        for p, x in zip(ps, grads):
            p.grad = x.cuda()
        opt.step()
        if ema:
            avg.update()
        torch.cuda.synchronize()
        for i, (p, x, st) in enumerate(zip(ps, grads, states)):
            p0, rem, shadow = before[i]
            if rem is None and master == "bf16_mt":
                rem = torch.zeros_like(p0)
            m0 = ref.decode(st["exp_avg"], st["exp_avg_scale"], False).double().abs()
            v0 = ref.decode(st["exp_avg_sq"], st["exp_avg_sq_scale"], True).double()
            w = ref.adamw_step(p0, rem, x, st, lr=1.2e-2, betas=betas, eps=1e-8, wd=wd, cautious=cautious, step=step)
            for k in KEYS:
                assert torch.equal(opt.state[p][k].cpu(), st[k]), (k, tuple(p.shape), step)
            assert float(opt.state[p]["step"]) == step
            # size of the update with nothing cancelled
            a = betas[0] * m0 + (1 - betas[0]) * x.double().abs()
            v = betas[1] * v0 + (1 - betas[1]) * x.double() ** 2
            up = 1.2e-2 / (1 - betas[0] ** step) * a / (v.sqrt() / math.sqrt(1 - betas[1] ** step) + 1e-8)
            tol = 64 * 2.0 ** -24 * up + 4 * 2.0 ** -24 * (p0.double().abs() + w.abs()) + 1e-42
            got = p.detach().cpu()
            if master == "bf16_mt":
                r = opt.state[p]["mant_rem"].cpu()
                assert ((got.double() + r.double() - w).abs() <= tol + 2.0 ** -16 * (w.abs() + tol)).all()
                assert torch.equal(got, (got.float() + r.float()).to(torch.bfloat16)) or \
                    ((got.double() - w).abs() <= tol + 2.0 ** -8 * (w.abs() + tol)).all()
            else:
                half = torch.finfo(dtype).eps / 2
                assert ((got.double() - w).abs() <= tol + half * (w.abs() + tol)).all()
            if ema:
                want = shadow.double() + (1.0 - 0.999) * (got.double() - shadow.double())
                # the weight 1 - decay, the difference, the product and the sum: four halves of a step
                assert ((avg.shadow[i].cpu().double() - want).abs() <= 4 * 2.0 ** -24 * (shadow.abs() + got.float().abs())).all()


def test_the_step_uses_moments_before_their_rounding(cuda):
    """One step from zero state: the first update is lr g / (|g| + eps) whatever the codes lose."""
    g = _gen(0)
    x = torch.randn(1000, generator=g) * torch.exp(3 * torch.randn(1000, generator=g)) * 1e-3
    p = torch.nn.Parameter(torch.zeros(1000, device=cuda))
    opt = _optimizer([p], lr=0.5)
    p.grad = x.cuda()
    opt.step()
    want = -0.5 * x.double() / (x.double().abs() + 1e-8)
    assert ((p.detach().cpu().double() - want).abs() <= 32 * 2.0 ** -24 * want.abs()).all()


def test_clip_coefficient_is_applied_as_the_eager_clip_does(cuda):
    for dtype, master in ((torch.float32, "none"), (torch.bfloat16, "bf16_mt")):
        res = []
        for defer in (False, True):
            ps = [torch.nn.Parameter(x.cuda()) for x in _tensors(dtype, 1)]
            opt = _optimizer(ps, master=master)
            for step in range(3):
                for p, x in zip(ps, _grads(ps, step)):
                    p.grad = x.cuda()
                clip_grad_norm_(ps, 0.01, defer_to=(opt,) if defer else None)
                opt.step()
            res.append([t for p in ps for t in (p.detach(), *(opt.state[p][k] for k in KEYS))])
        assert all(torch.equal(a, b) for a, b in zip(*res))


def test_slices_give_what_the_whole_tensor_gives(cuda):
    n = 5 * 1024 + 77
    res = []
    for cuts in ([0, n], [0, 128, 1024, 4096, n]):
        p = torch.nn.Parameter((torch.randn(n, generator=_gen(2)) * 0.02).to(torch.bfloat16).cuda())
        opt = _optimizer([p], master="bf16_mt")
        for step in range(3):
            p.grad = (torch.randn(n, generator=_gen(50 + step)) * 1e-3).to(torch.bfloat16).cuda()
            for a, b in zip(cuts, cuts[1:]):
                opt._owned_slices = {id(p): (a, b - a)}
                if a:
                    opt._steps[id(p)] -= 1
                opt.step()
        res.append([p.detach(), *(opt.state[p][k] for k in KEYS), opt.state[p]["mant_rem"]])
    assert all(torch.equal(a, b) for a, b in zip(*res))
    for bad in ((64, 128), (0, 100), (128, 200)):
        opt._owned_slices = {id(p): bad}
        with pytest.raises(ValueError, match="multiples of 128"):
            opt.step()


def test_unaligned_gradients_and_parameters(cuda):
    """A gradient view that starts inside an allocation gives the same step."""
    n = 3001
    res = []
    for off in (0, 1, 5):
        buf = torch.zeros(2, n + 16, dtype=torch.bfloat16, device=cuda)
        p = torch.nn.Parameter(buf[0, off:off + n])
        p.data.copy_(torch.randn(n, generator=_gen(3)) * 0.02)
        opt = _optimizer([p], master="bf16_mt")
        for step in range(3):
            p.grad = buf[1, off:off + n]
            p.grad.copy_(torch.randn(n, generator=_gen(60 + step)) * 1e-3)
            opt.step()
        assert (buf[0, :off] == 0).all() and (buf[0, off + n:] == 0).all()
        res.append([p.detach().clone(), *(opt.state[p][k] for k in KEYS), opt.state[p]["mant_rem"]])
    for other in res[1:]:
        assert all(torch.equal(a, b) for a, b in zip(res[0], other))


def test_a_gradient_that_is_not_finite_stays_in_its_block(cuda):
    for bad in (math.inf, math.nan, 1e30):  # 1e30 squared overflows
        p = torch.nn.Parameter(torch.zeros(1000, device=cuda))
        opt = _optimizer([p])
        g = torch.full((1000,), 1e-3, device=cuda)
        p.grad = g.clone()
        p.grad[300] = bad
        opt.step()
        ok = torch.ones(1000, dtype=torch.bool, device=cuda)
        ok[300] = False
        assert p.detach()[ok].isfinite().all()  # this step's update does not read the codes it writes
        p.grad = g.clone()
        opt.step()
        ok[256:384] = False
        assert p.detach()[ok].isfinite().all()
        m, = [x["exp_avg_sq"] for x in opt.expanded_state()]
        assert m[256:384].isnan().all() and m[ok].isfinite().all()


@pytest.mark.parametrize("size", [1e-20, 3e-19, 1e-12, 1e10])
def test_moments_at_the_ends_of_the_range(cuda, size):
    """Gradients whose squares are subnormal, and an eps of 0 that does not cover them; and large ones."""
    g = _gen(6)
    x = torch.randn(2000, generator=g) * size
    x[torch.rand(2000, generator=g) < 0.1] *= 1e-3
    p = torch.nn.Parameter(torch.zeros(2000, device=cuda))
    opt = _optimizer([p], eps=0.0, lr=0.25)
    st = {"exp_avg": torch.zeros(2000, dtype=torch.int8), "exp_avg_sq": torch.zeros(2000, dtype=torch.uint8),
          "exp_avg_scale": torch.zeros(16), "exp_avg_sq_scale": torch.zeros(16)}
    for step in range(1, 4):
        before = p.detach().cpu()
        p.grad = x.cuda()
        opt.step()
        w = ref.adamw_step(before, None, x, st, lr=0.25, betas=(0.9, 0.95), eps=0.0, wd=0.0, cautious=False, step=step)
        for k in KEYS:
            assert torch.equal(opt.state[p][k].cpu(), st[k]), (k, step)
        got, up = p.detach().cpu().double(), (w - before.double()).abs()
        ok = w.isfinite()  # a square that has become 0 leaves m / 0, as in 32 bits
        assert ((got - w).abs() <= 64 * 2.0 ** -24 * up + 4 * 2.0 ** -24 * (before.double().abs() + w.abs()))[ok].all()
        assert ok.any()
        if not ok.all():
            break


def test_the_update_is_the_rounded_quotient(cuda):
    """Second moments of 0 (denominator eps): w - fl(fl(c m) / eps), rounded as torch's operations round it. The
    quotient's residual step leaves a wrong last place in about one of 2^21 quotients."""
    n = 5000
    g = _gen(8)
    m = torch.randn(n, generator=g) * 1e-3
    p = torch.nn.Parameter((torch.randn(n, generator=g) * 0.02).cuda())
    w0 = p.detach().cpu()
    opt = _optimizer([p], lr=1.2e-2)
    opt._init_state(p)
    q, s = ref.encode(m, False)
    opt.state[p]["exp_avg"].copy_(q)
    opt.state[p]["exp_avg_scale"].copy_(s)
    p.grad = torch.zeros_like(p)
    opt.step()
    m1 = ref.f32(0.9) * ref.decode(q, s, False)
    want = w0 - ref.f32(1.2e-2 / (1 - 0.9)) * m1 / ref.f32(1e-8)
    differ = p.detach().cpu() != want
    assert differ.float().mean() < 1e-3
    assert ((p.detach().cpu() - want).abs() <= 2 * 2.0 ** -23 * want.abs()).all()


def test_a_master_weight_is_the_rounded_update(cuda):
    """With a remainder every operation of the update is rounded as torch's are, so weight and remainder are those of
    the fp32 formula (but for about one wrong last place in 2^20 of quotient or root)."""
    n = 20_000
    cpu = _tensors(torch.bfloat16, 21, [(n,)])[0]
    for wd, cautious in ((0.0, False), (0.1, False), (0.1, True)):
        p = torch.nn.Parameter(cpu.cuda())
        opt = _optimizer([p], master="bf16_mt", weight_decay=wd, cautious_wd=cautious)
        st = {"exp_avg": torch.zeros(n, dtype=torch.int8), "exp_avg_sq": torch.zeros(n, dtype=torch.uint8),
              "exp_avg_scale": torch.zeros(state8.blocks(n)), "exp_avg_sq_scale": torch.zeros(state8.blocks(n))}
        w, rem = cpu.clone(), torch.zeros_like(cpu)
        for step in range(1, 4):
            x = _grads([cpu], step)[0]
            p.grad = x.cuda()
            opt.step()
            m = ref.f32(0.9) * ref.decode(st["exp_avg"], st["exp_avg_scale"], False) + ref.f32(1 - 0.9) * x.float()
            v = ref.f32(0.95) * ref.decode(st["exp_avg_sq"], st["exp_avg_sq_scale"], True) + \
                ref.f32(1 - 0.95) * (x.float() * x.float())
            st["exp_avg"], st["exp_avg_scale"] = ref.encode(m, False, step)
            st["exp_avg_sq"], st["exp_avg_sq_scale"] = ref.encode(v, True, step)
            full = w.float() + rem.float()
            if wd and cautious:
                full = torch.where(m * full > 0, full * (1 - ref.f32(1.2e-2 * wd)), full)
            elif wd:
                full = full - ref.f32(1.2e-2 * wd) * full
            d = v.double().sqrt().float() * (1 / ref.f32(math.sqrt(1 - 0.95 ** step))) + ref.f32(1e-8)
            full = full - ref.f32(1.2e-2 / (1 - 0.9 ** step)) * m / d
            w = full.to(torch.bfloat16)
            rem = (full - w.float()).to(torch.bfloat16)
            assert (p.detach().cpu() != w).sum() <= 2 and (opt.state[p]["mant_rem"].cpu() != rem).sum() <= 2, (wd, step)


def test_a_state_of_another_size_is_refused(cuda):
    """Codes or scales that do not belong to the parameter (a damaged checkpoint) never reach a kernel."""
    p = torch.nn.Parameter(torch.zeros(64, 128, device=cuda))
    p.grad = torch.ones_like(p)
    opt, muon = _optimizer([p]), NorMuonGNS([p], momentum_dtype=torch.int8)
    opt.step()
    muon.step()
    for o, keys in ((opt, ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale")),
                    (muon, ("momentum_buffer", "momentum_scale"))):
        for k in keys:
            good = o.state[p][k]
            for bad in (good[:-1].clone(), good.to(torch.int16 if good.dtype != torch.float32 else torch.bfloat16)):
                o.state[p][k] = bad
                o.invalidate_plan()
                with pytest.raises((ValueError, TypeError)):
                    o.step()
            o.state[p][k] = good
        o.invalidate_plan()
        o.step()
    opt.state[p]["exp_avg"] = torch.zeros(64, 128, device=cuda)  # wide beside 8 bits
    opt.invalidate_plan()
    with pytest.raises(ValueError, match="one dtype"):
        opt.step()


def test_a_parameter_twice_is_refused(cuda):
    p = torch.nn.Parameter(torch.zeros(64, 128, device=cuda))
    p.grad = torch.ones_like(p)
    with pytest.warns(UserWarning, match="duplicate"):
        opt = _optimizer([p, p])
    with pytest.raises(ValueError, match="twice"):
        opt.step()
    with pytest.warns(UserWarning, match="duplicate"):
        muon = NorMuonGNS([p, p], momentum_dtype=torch.int8)
    with pytest.raises(ValueError, match="twice"):
        muon.step()


def test_two_optimizers_take_turns(cuda):
    """Steps of two optimizers in turn, with a conversion between them, equal each run alone."""
    def make(seed):
        ps = [torch.nn.Parameter(x.cuda()) for x in _tensors(torch.bfloat16, seed, [(64, 300), (4099,)])]
        return ps, _optimizer(ps, master="bf16_mt")
    alone = []
    for seed in (1, 2):
        ps, opt = make(seed)
        for step in range(3):
            for p, x in zip(ps, _grads(ps, 10 * seed + step)):
                p.grad = x.cuda()
            opt.step()
        alone.append([p.detach() for p in ps])
    pair = [make(1), make(2)]
    for step in range(3):
        for seed, (ps, opt) in zip((1, 2), pair):
            for p, x in zip(ps, _grads(ps, 10 * seed + step)):
                p.grad = x.cuda()
            opt.step()
            opt.expanded_state(dtype=torch.bfloat16)
    assert all(torch.equal(a, p) for ps, b in zip([x[0] for x in pair], alone) for a, p in zip(b, ps))


def test_small_tensors_keep_wide_moments(cuda):
    big, small = (torch.nn.Parameter(torch.zeros(s, dtype=torch.bfloat16, device=cuda)) for s in ((64, 64), (64,)))
    opt = AdamW([big, small], master="bf16_mt", state_dtype=torch.int8)
    wide = AdamW([torch.nn.Parameter(torch.zeros(64, dtype=torch.bfloat16, device=cuda))], master="bf16_mt")
    for step in range(3):
        for p in (big, small, wide.param_groups[0]["params"][0]):
            p.grad = (torch.randn(p.shape, generator=_gen(step)) * 1e-3).to(torch.bfloat16).cuda()
        opt.step()
        wide.step()
    w = wide.param_groups[0]["params"][0]
    assert opt.state[big]["exp_avg"].dtype == torch.int8
    for k in ("exp_avg", "exp_avg_sq", "mant_rem"):
        assert torch.equal(opt.state[small][k], wide.state[w][k])
    assert torch.equal(small, w)
    assert torch.equal(wide.expanded_state()[0]["exp_avg_sq"], wide.state[w]["exp_avg_sq"])  # nothing to expand
    x = opt.expanded_state()
    assert torch.equal(x[1]["exp_avg"], wide.state[w]["exp_avg"])
    assert torch.equal(x[0]["master"], big.detach().float() + opt.state[big]["mant_rem"].float())


def test_more_tensors_than_one_launch_takes_and_groups(cuda):
    def make():
        ps = [torch.nn.Parameter(x.cuda()) for x in _tensors(torch.float32, 5, [(1 + 13 * i,) for i in range(200)])]
        return ps
    ps, qs = make(), make()
    groups = lambda x: [{"params": x[:90], "lr": 1e-2}, {"params": x[90:150], "betas": (0.75, 0.95)},  # noqa: E731
                        {"params": x[150:], "weight_decay": 0.3}]
    opt = _optimizer(groups(ps))
    one = [_optimizer([{**g, "params": [p]}]) for g in groups(qs) for p in g["params"]]
    for step in range(2):
        for p, q, x in zip(ps, qs, _grads(ps, step)):
            p.grad, q.grad = x.cuda(), x.cuda()
        opt.step()
        for o in one:
            o.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    assert all(torch.equal(opt.state[p][k], o.state[q][k]) for p, q, o in zip(ps, qs, one) for k in KEYS)


def test_steps_follow_the_current_stream(cuda):
    """A plan built on one stream steps on another: everything runs in that stream's order."""
    res = []
    side = torch.cuda.Stream()
    for use in (False, True):
        p = torch.nn.Parameter((torch.randn(1 << 20, generator=_gen(7)) * 0.02).cuda())
        q = torch.nn.Parameter((torch.randn(256, 512, generator=_gen(8)) * 0.02).to(torch.bfloat16).cuda())
        opt = _optimizer([p])
        muon = NorMuonGNS([q], momentum_dtype=torch.int8, bf16_master=True)
        for step in range(4):
            torch.cuda.synchronize()
            with torch.cuda.stream(side if use and step >= 2 else torch.cuda.current_stream()):
                big = torch.randn(4096, 4096, device=cuda)
                for _ in range(20):
                    big = big @ big * 1e-2  # work ahead of the gradient on the same stream
                p.grad = (torch.randn(1 << 20, generator=_gen(70 + step)) * 1e-3).cuda() + 0 * big.view(-1)[:1 << 20].nan_to_num(0, 0, 0)
                q.grad = (torch.randn(256, 512, generator=_gen(80 + step)) * 1e-3).to(torch.bfloat16).cuda()
                opt.step()
                muon.step()
                out = [p.detach().clone(), q.detach().clone(), *(opt.state[p][k].clone() for k in KEYS)]
            torch.cuda.synchronize()
        res.append(out)
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_captured_step_and_expansion_replay(cuda):
    """The library call captured into a graph and replayed equals the call made as often (same step number)."""
    n = 10_007
    lib = _lib.load()

    def setup():
        p = (torch.randn(n, generator=_gen(1)) * 0.02).cuda()
        g = (torch.randn(n, generator=_gen(2)) * 1e-3).cuda()
        st = [torch.zeros(n, dtype=torch.int8, device=cuda), torch.zeros(n, dtype=torch.uint8, device=cuda),
              torch.zeros(state8.blocks(n), device=cuda), torch.zeros(state8.blocks(n), device=cuda)]
        out = torch.zeros(n, device=cuda)
        arr = (_lib.Adamw8Tensor * 1)(_lib.Adamw8Tensor(p.data_ptr(), None, g.data_ptr(), *[x.data_ptr() for x in st], None,
                                                        n, 0, 0, 0, None))
        grp = (_lib.Adamw8Group * 1)(_lib.Adamw8Group(1e-2, 0.9, 0.95, 1e-8, 0.0, 3.0, None, 0))

        def call():
            _lib.check(lib.b2o_adamw8_step(arr, 1, grp, 1, _lib.F32, 0.0, _lib.stream_ptr()), "adamw8")
            state8.decode([(st[0], st[2], "signed")], out=[out])
        return (p, *st, out), g, call
    a, ga, call_a = setup()
    b, gb, call_b = setup()
    for _ in range(4):
        call_a()
        ga.mul_(-0.7)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call_b()
    for _ in range(4):
        graph.replay()
        gb.mul_(-0.7)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_steps_repeat_bit_for_bit(cuda):
    res = []
    for _ in range(2):
        ps = [torch.nn.Parameter(x.cuda()) for x in _tensors(torch.bfloat16, 9, [(300, 1024), (77, 33)])]
        opt = _optimizer(ps, master="bf16_mt")
        for step in range(5):
            for p, x in zip(ps, _grads(ps, step)):
                p.grad = x.cuda()
            opt.step()
        res.append([t for p in ps for t in (p.detach(), *(opt.state[p][k] for k in KEYS))])
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_elements_behind_2_to_the_31(cuda):
    """The last elements of tensors whose offsets pass 32 bits: codes, values and the step."""
    n, tail = 2 ** 31 + 128 * 5 + 77, 1000
    lib = _lib.load()
    first = (n - tail) // 128 * 128
    cut = n - first
    x = torch.zeros(n, dtype=torch.bfloat16, device=cuda)
    t = (torch.randn(cut, generator=_gen(4)) * 1e-3).to(torch.bfloat16)
    x[first:] = t.cuda()
    (q, s), = state8.encode([(x, "signed")])
    (tq, ts), = state8.encode([(t.cuda(), "signed")])
    assert torch.equal(q[first:], tq) and torch.equal(s[first // 128:], ts) and not s[:first // 128].any()
    out = torch.ones(n, dtype=torch.bfloat16, device=cuda)
    state8.decode([(q, s, "signed")], out=[out])
    assert torch.equal(out[first:], state8.decode([(tq, ts, "signed")], dtype=torch.bfloat16)[0]) and out[first - 1] == 0
    del out
    # the step, as a whole and as a slice
    v, vs = torch.zeros(n, dtype=torch.uint8, device=cuda), torch.zeros_like(s)
    p = torch.zeros(n, dtype=torch.bfloat16, device=cuda)
    sl = [p[first:].clone(), x[first:].clone(), q[first:].clone(), v[first:].clone(), s[first // 128:].clone(),
          vs[first // 128:].clone()]
    grp = (_lib.Adamw8Group * 1)(_lib.Adamw8Group(1e-2, 0.9, 0.95, 1e-8, 0.0, 3.0, None, 0))
    for (a, b, c, d, e, f), m, o in (((p, x, q, v, s, vs), n, 0), (sl, cut, first)):
        arr = (_lib.Adamw8Tensor * 1)(_lib.Adamw8Tensor(a.data_ptr(), None, b.data_ptr(), c.data_ptr(), d.data_ptr(),
                                                        e.data_ptr(), f.data_ptr(), None, m, o, 0, 0, None))
        _lib.check(lib.b2o_adamw8_step(arr, 1, grp, 1, _lib.BF16, 0.0, _lib.stream_ptr()), "adamw8")
    torch.cuda.synchronize()
    whole = [p[first:], x[first:], q[first:], v[first:], s[first // 128:], vs[first // 128:]]
    assert all(torch.equal(a, b) for a, b in zip(whole, sl)) and sl[3].any()


# ------------------------------------------------- loading and checkpoints --
def test_wide_states_load_into_8_bits_and_back(cuda):
    shapes = [(64, 128), (33, 200), (100,)]
    ps = [torch.nn.Parameter(x.cuda()) for x in _tensors(torch.bfloat16, 11, shapes)]
    wide = AdamW(ps, master="bf16_mt", lr=1e-2)
    for step in range(3):
        for p, x in zip(ps, _grads(ps, step)):
            p.grad = x.cuda()
        wide.step()
    narrow = AdamW(ps, master="bf16_mt", lr=1e-2, state_dtype=torch.int8)
    narrow.load_state_dict(wide.state_dict())
    for p in ps[:2]:
        for k, root in (("exp_avg", False), ("exp_avg_sq", True)):
            rq, rs = ref.encode(wide.state[p][k].cpu(), root)
            assert torch.equal(narrow.state[p][k].cpu(), rq) and torch.equal(narrow.state[p][k + "_scale"].cpu(), rs)
        assert torch.equal(narrow.state[p]["mant_rem"], wide.state[p]["mant_rem"])
    assert narrow._steps[id(ps[0])] == 3 and narrow.state[ps[2]]["exp_avg"].dtype == torch.float32
    # back to wide, directly and through the expanded state dict
    again = AdamW(ps, master="bf16_mt", lr=1e-2)
    again.load_state_dict(narrow.state_dict())
    other = AdamW(ps, master="bf16_mt", lr=1e-2)
    other.load_state_dict(narrow.expanded_state_dict())
    torch_one = torch.optim.AdamW(ps, lr=1e-2, fused=True)
    sd = narrow.expanded_state_dict()
    torch_one.load_state_dict({"state": {k: {n: v for n, v in st.items() if n != "mant_rem"} for k, st in sd["state"].items()},
                               "param_groups": torch_one.state_dict()["param_groups"]})
    for p in ps[:2]:
        for k, root in (("exp_avg", False), ("exp_avg_sq", True)):
            want = ref.decode(narrow.state[p][k].cpu(), narrow.state[p][k + "_scale"].cpu(), root)
            for o in (again, other):
                assert set(o.state[p]) == {"step", "exp_avg", "exp_avg_sq", "mant_rem"}
                assert torch.equal(o.state[p][k].cpu(), want)
            assert torch.equal(torch_one.state[p][k].cpu(), want.to(torch.bfloat16))
    for p, x in zip(ps, _grads(ps, 9)):
        p.grad = x.cuda()
    narrow.step()
    again.step()


def _train(model, muon, adamw, ema, steps, seed=0):
    for step in steps:
        synth.set_grads(model, [g.cuda() for g in synth.make_grads(synth.SyntheticLM(synth.MICRO, seed=0), step, seed)])
        clip_grad_norm_(list(model.parameters()), 1.0, defer_to=(muon, adamw))
        muon.step()
        adamw.step()
        ema.update()
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


KW = dict(muon_lr=8e-3, adam_lr=1.2e-2, embed_lr=2.4e-2, weight_decay=0.1, cautious_wd=True, bf16_master=True,
          adam_master="bf16_mt", adam_state_dtype=torch.int8, momentum_dtype=torch.int8)


def _setup():
    model = synth.SyntheticLM(synth.MICRO, seed=0).cuda()
    return (model, *build_optimizers(model, **KW), EmaWeights(model, 0.999))


def test_training_resumes_bit_for_bit(cuda, tmp_path):
    """Clip, NorMuon, AdamW and EMA with every state in 8 bits: 5 steps are 3, a checkpoint, and 2."""
    a = _setup()
    _train(*a, range(3))
    save_checkpoint(a[0], a[1], 3, tmp_path / "c.pt", adamw=a[2])
    shadow = [s.clone() for s in a[3].shadow]
    _train(*a, range(3, 5))
    b = _setup()
    assert load_checkpoint(tmp_path / "c.pt", b[0], b[1], adamw=b[2]) == 3
    b[3].update()
    for s, t in zip(b[3].shadow, shadow):
        s.copy_(t)
    _train(*b, range(3, 5))
    assert all(torch.equal(p, q) for p, q in zip(a[0].parameters(), b[0].parameters()))
    assert all(torch.equal(s, t) for s, t in zip(a[3].shadow, b[3].shadow))
    for o, r in zip(a[1:3], b[1:3]):
        for p, q in zip([p for g in o.param_groups for p in g["params"]], [p for g in r.param_groups for p in g["params"]]):
            assert all(torch.equal(v, r.state[q][k]) if torch.is_tensor(v) else v == r.state[q][k] for k, v in o.state[p].items())


def test_expanded_checkpoint_has_the_reference_layout(cuda, tmp_path):
    model, muon, adamw, ema = _setup()
    _train(model, muon, adamw, ema, range(2))
    save_checkpoint(model, muon, 2, tmp_path / "c.pt", adamw=adamw, expand_state=True)
    obj = torch.load(tmp_path / "c.pt", weights_only=False)
    for st in obj["optimizer"]["state"].values():
        assert set(st) == {"momentum_buffer", "v_row", "mant_rem"} and st["momentum_buffer"].dtype == torch.bfloat16
    for st in obj["adamw"]["state"].values():
        assert not any(k.endswith("_scale") for k in st) and st["exp_avg"].dtype in (torch.float32, torch.bfloat16)
    plain = synth.SyntheticLM(synth.MICRO, seed=0).cuda()
    wide = build_optimizers(plain, **{**KW, "adam_state_dtype": None, "momentum_dtype": None})
    load_checkpoint(tmp_path / "c.pt", plain, wide[0], adamw=wide[1])
    narrow = _setup()
    load_checkpoint(tmp_path / "c.pt", narrow[0], narrow[1], adamw=narrow[2])
    for p, q in zip([p for g in muon.param_groups for p in g["params"]], [p for g in narrow[1].param_groups for p in g["params"]]):
        assert narrow[1].state[q]["momentum_buffer"].dtype == torch.int8 and narrow[1].state[q]["momentum_step"] == 0
    _train(narrow[0], narrow[1], narrow[2], narrow[3], range(1))


def test_the_ranks_of_a_sharded_step_give_the_whole_step(cuda):
    """Each of two ranks' own part of a step (run one after the other, without the exchange) is the part of the
    unsharded step, bit for bit: parameters, codes, scales, remainders, momenta."""
    from sol_b200.sharding import ShardedStep
    grads = [[g.cuda() for g in synth.make_grads(synth.SyntheticLM(synth.MICRO, seed=0), 0, 0)]]
    whole = _setup()
    ranks = []
    for rank in range(2):
        model, muon, adamw, ema = _setup()
        sh = ShardedStep(model, muon, adamw, ema, 2, rank, min_rows_shard=16, exchange="nccl")
        ranks.append((model, muon, adamw, sh))
    assert any(adamw.holds_8bit(p) for p in ranks[0][3].row_sharded)
    # one step: the next would need the weights and states that the ranks exchange
    for model, muon, adamw, _ in [(whole[0], whole[1], whole[2], None)] + ranks:
        synth.set_grads(model, [g.clone() for g in grads[0]])
        adamw.step()
        muon.step()
    torch.cuda.synchronize()
    for rank, (model, muon, adamw, sh) in enumerate(ranks):
        pairs = list(zip([p for g in adamw.param_groups for p in g["params"]],
                         [p for g in whole[2].param_groups for p in g["params"]]))
        for p, q in pairs:
            start, n = adamw._owned_slices[id(p)]
            for k, v in {**whole[2].state[q], "p": q.detach()}.items():
                w = adamw.state[p][k] if k != "p" else p.detach()
                lo, hi = (start // 128, -(-(start + n) // 128)) if k.endswith("_scale") else (start, start + n)
                if k == "step":
                    lo, hi = 0, 1
                assert torch.equal(w.reshape(-1)[lo:hi], v.reshape(-1)[lo:hi]), (rank, tuple(p.shape), k)
        for p, q in zip([p for g in muon.param_groups for p in g["params"]], [p for g in whole[1].param_groups for p in g["params"]]):
            if sh.owner[id(p)] == rank:
                assert torch.equal(p, q)
                for k, v in whole[1].state[q].items():
                    w = muon.state[p][k]
                    assert torch.equal(w, v) if torch.is_tensor(v) else w == v, (rank, k)


# ---------------------------------------------------------- NorMuon momentum --
def _front8(cuda, shapes, dtype, nesterov, steps, x0=False, coef=None, seed=0, beta=0.9, scale_of=lambda t: 1e-3):
    """Runs the front (and, with x0, the prescale) call over several steps and checks each against the restatement."""
    lib = _lib.load()
    items, keep = [], []
    arr = (_lib.NormuonBatch * len(shapes))()
    scs, sts = [], []
    for k, (S, r, c) in enumerate(shapes):
        d = dict(S=S, r=r, c=c, g=[torch.zeros(r, c, dtype=dtype, device=cuda) for _ in range(S)],
                 q=[torch.zeros(r, c, dtype=torch.int8, device=cuda) for _ in range(S)],
                 s=[torch.zeros(state8.blocks(r * c), device=cuda) for _ in range(S)],
                 u=torch.zeros(S, r, c, dtype=torch.float16 if x0 else torch.bfloat16, device=cuda),
                 part=torch.zeros(S, lib.b2o_normuon_front_parts(r * c), device=cuda),
                 pre=torch.zeros(S, device=cuda), xs=torch.zeros(2 * S, device=cuda),
                 fl=torch.zeros(S, dtype=torch.int32, device=cuda),
                 ref=[(torch.zeros(r, c, dtype=torch.int8), torch.zeros(state8.blocks(r * c))) for _ in range(S)])
        items.append(d)
        gp, qp, sp = (_lib.ptr_array([x.data_ptr() for x in d[n]]) for n in ("g", "q", "s"))
        st = (ctypes.c_uint32 * S)()
        keep += [gp, qp, sp]
        scs.append(_lib.addr(sp))
        sts.append(st)
        arr[k] = _lib.NormuonBatch(S=S, r=r, c=c, grads=_lib.addr(gp), bufs=_lib.addr(qp), u=d["u"].data_ptr(),
                                   partial=d["part"].data_ptr(), prescale=d["pre"].data_ptr(), xscale=d["xs"].data_ptr(),
                                   flags=d["fl"].data_ptr(), x0_half=int(x0))
    scp, stp = _lib.ptr_array(scs), _lib.ptr_array([_lib.addr(x) for x in sts])
    gsc = torch.tensor([coef], device=cuda) if coef is not None else None
    gptr = gsc.data_ptr() if gsc is not None else None
    g = _gen(seed)
    for t in range(1, steps + 1):
        for k, d in enumerate(items):
            for j in range(d["S"]):
                sts[k][j] = t + j  # matrices may have stepped a different number of times
                d["g"][j].copy_((torch.randn(d["r"], d["c"], generator=g) * scale_of(t)).to(dtype))
        _lib.check(lib.b2o_normuon_front8_multi(arr, scp, stp, len(shapes), _lib.dtype_code(dtype), beta, nesterov, gptr,
                                                _lib.stream_ptr()), "front8")
        if x0:
            _lib.check(lib.b2o_normuon_prescale8(arr, scp, len(shapes), _lib.dtype_code(dtype), beta, nesterov, gptr,
                                                 1e-7, 1.0, _lib.stream_ptr()), "prescale8")
        torch.cuda.synchronize()
        for d in items:
            for j in range(d["S"]):
                gr = d["g"][j].cpu()
                if coef is not None:
                    gr = (gr.float() * torch.tensor(coef)).to(dtype)
                u, q, s = ref.momentum_step(gr, *d["ref"][j], beta=beta, nesterov=nesterov, step=t + j)
                d["ref"][j] = (q, s)
                assert torch.equal(d["q"][j].cpu(), q) and torch.equal(d["s"][j].cpu(), s), (t, d["r"], d["c"])
                sq = u.double().square().view(-1)
                want = torch.nn.functional.pad(sq, (0, -sq.numel() % 16384)).view(-1, 16384).sum(1)
                # 8 x 8 sums a lane, then 5 + 8 more of half a step each
                assert ((d["part"][j].cpu().double() - want).abs() <= 80 * 2.0 ** -24 * want).all()
                if not x0:
                    assert torch.equal(d["u"][j].cpu(), u)
                elif u.any():
                    # X0 = u k, exact, with the k that leaves ||X0|| between 4 and 16384
                    f = d["xs"][j].cpu().double() * want.sum().sqrt()  # s_norm ||u|| / k = 1 / k
                    k2 = 2.0 ** round(math.log2(1.0 / f))
                    assert torch.equal(d["u"][j].cpu(), (u.float() * k2).to(torch.float16)), t
                    assert 4 <= float(want.sum().sqrt()) * k2 <= 16384
    assert _lib.device_error() == 0


SHAPES8 = [(3, 128, 128), (2, 33, 77), (1, 1, 1), (2, 1, 5), (1, 129, 257), (4, 8, 1024), (2, 64, 300)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nesterov", [0, 1])
def test_front8_matches_the_restatement(cuda, dtype, nesterov):
    _front8(cuda, SHAPES8, dtype, nesterov, 4)


def test_front8_with_clip_and_no_momentum(cuda):
    _front8(cuda, SHAPES8[:4], torch.bfloat16, 1, 3, coef=0.37)
    _front8(cuda, SHAPES8[:4], torch.float32, 1, 3, coef=0.37, beta=0.0)


def test_front8_half_input_and_its_repair(cuda):
    """X0 in binary16 with the power of two kept from the step before; gradients that grow and shrink by 10^4 force a rewrite."""
    _front8(cuda, [(2, 128, 128), (1, 33, 77), (2, 64, 300)], torch.bfloat16, 1, 6, x0=True,
            scale_of=lambda t: (1e-3, 1e-3, 10.0, 1e-6, 1e-6, 1e-3)[t - 1])
    _front8(cuda, [(2, 128, 128), (1, 33, 77)], torch.float32, 0, 3, x0=True)


def test_muon_step_runs_on_the_8_bit_momentum(cuda):
    """muon.step() takes u from the 8-bit momentum: a hook sees the restatement's u, and the update through the
    production path agrees with the one computed from that u by the engine's own orthogonaliser."""
    shapes = [(128, 384), (384, 128), (128, 128), (128, 384), (8, 128)]
    base = [(torch.randn(s, generator=_gen(20 + i)) * 0.02).to(torch.bfloat16) for i, s in enumerate(shapes)]
    mk = lambda: [torch.nn.Parameter(x.cuda()) for x in base]  # noqa: E731
    pa, pb = mk(), mk()
    kw = dict(lr=8e-3, weight_decay=0.1, cautious_wd=True, bf16_master=True, momentum_dtype=torch.int8)
    prod, hooked = NorMuonGNS(pa, **kw), NorMuonGNS(pb, **kw)
    seen = []
    inner = hooked._orthogonalize_batch
    hooked._orthogonalize_batch = lambda U, n: (seen.append(U.clone()), inner(U, n))[1]
    refs = [(torch.zeros(s, dtype=torch.int8), torch.zeros(state8.blocks(s[0] * s[1]))) for s in shapes]
    for step in range(1, 5):
        grads = [(torch.randn(s, generator=_gen(100 * step + i)) * (1e-3 if step != 3 else 5.0)).to(torch.bfloat16)
                 for i, s in enumerate(shapes)]
        for p, q, x in zip(pa, pb, grads):
            p.grad, q.grad = x.cuda(), x.cuda()
        seen.clear()
        prod.step()
        hooked.step()
        torch.cuda.synchronize()
        us = []
        for i, x in enumerate(grads):
            u, q, s = ref.momentum_step(x, *refs[i], beta=0.95, nesterov=True, step=step)
            refs[i] = (q, s)
            us.append(u)
            for o, p in ((prod, pa[i]), (hooked, pb[i])):
                assert torch.equal(o.state[p]["momentum_buffer"].cpu(), q) and o.state[p]["momentum_step"] == step
                assert torch.equal(o.state[p]["momentum_scale"].cpu(), s)
        order = [0, 3, 1, 2, 4]  # exact-shape batches in parameter order
        got = torch.cat([b.reshape(-1) for b in seen]).cpu()
        assert torch.equal(got, torch.cat([us[i].reshape(-1) for i in order]))
    assert _lib.device_error() == 0
    num = sum(((p.float() - q.float()) ** 2).sum() for p, q in zip(pa, pb))
    den = sum(((p.detach().cpu().float() - b.float()) ** 2).sum() for p, b in zip(pa, base))
    # both run the same binary16 iteration from the same u, one from u 2^k and one from u / ||u|| rounded
    # to binary16; the suite allows 1e-2 between either and exact arithmetic, so two of them may be
    # 1e-2 + 1e-2 apart
    assert float((num.cpu() / den).detach()) ** 0.5 <= 2e-2


def test_momentum_widens_when_loaded_elsewhere(cuda):
    p = torch.nn.Parameter((torch.randn(128, 256, generator=_gen(1)) * 0.02).to(torch.bfloat16).cuda())
    a = NorMuonGNS([p], momentum_dtype=torch.int8)
    p.grad = (torch.randn(128, 256, generator=_gen(2)) * 1e-3).to(torch.bfloat16).cuda()
    a.step()
    want = ref.decode(a.state[p]["momentum_buffer"].cpu(), a.state[p]["momentum_scale"].cpu(), False).to(torch.bfloat16)
    for sd in (a.state_dict(), a.expanded_state_dict()):
        b = NorMuonGNS([p])
        b.load_state_dict(sd)
        assert set(b.state[p]) == {"momentum_buffer", "v_row"} and torch.equal(b.state[p]["momentum_buffer"].cpu(), want)
    c = NorMuonGNS([p], momentum_dtype=torch.int8)
    c.load_state_dict(b.state_dict())
    rq, rs = ref.encode(want, False)
    assert torch.equal(c.state[p]["momentum_buffer"].cpu(), rq) and torch.equal(c.state[p]["momentum_scale"].cpu(), rs)

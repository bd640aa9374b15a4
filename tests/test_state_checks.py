"""States that do not fit their parameter are refused before a kernel gets their
pointers. Everything runs on the host: the launches are replaced, so that a state
that slips through is seen in the descriptors and touches no memory."""
import contextlib
import ctypes
import io

import pytest
import torch

from sol_b200 import AdamW, NorMuonGNS, _lib, build_optimizers, state8, synth
from sol_b200.checkpoint import save_checkpoint


class _Library:
    """Stands in for libb2o: launches are recorded by name and succeed (or fail, for ``fail``)."""

    def __init__(self, real):
        self.real, self.calls, self.fail = real, [], None

    def __getattr__(self, name):
        if any(x in name for x in ("_blocks", "_parts", "_bytes", "_floats")):
            return getattr(self.real, name)

        def call(*args):
            self.calls.append(name)
            return -1 if name == self.fail else 0
        return call


@pytest.fixture
def host(monkeypatch):
    lib = _Library(_lib.load())
    lib.rows = []
    monkeypatch.setattr(_lib, "load", lambda *a: lib)
    monkeypatch.setattr(_lib, "require_cuda", lambda *a: None)
    monkeypatch.setattr(_lib, "on_device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "stream_ptr", lambda dev=None: 0)
    monkeypatch.setattr(state8.Rows, "launch", lambda self, fn, what: lib.rows.extend(self.by.values()))
    return lib


def _adamw(shape=(64, 128), dtype=torch.bfloat16, **kw):
    p = torch.nn.Parameter(torch.zeros(shape, dtype=dtype))
    p.grad = torch.ones_like(p)
    kw = {"state_dtype": torch.int8, "master": "bf16_mt" if dtype == torch.bfloat16 else "none", **kw}
    return p, AdamW([p], **kw)


def _cut(t):
    return t.reshape(-1)[: t.numel() // 2].clone()


BAD_ADAMW = [("exp_avg", _cut), ("exp_avg_sq", _cut), ("exp_avg_scale", _cut), ("exp_avg_sq_scale", _cut),
             ("mant_rem", _cut), ("exp_avg_sq", lambda t: t.float()), ("exp_avg", lambda t: t.to(torch.uint8)),
             ("exp_avg_scale", lambda t: t.bfloat16()), ("exp_avg_scale", lambda t: None),
             ("exp_avg_sq_scale", lambda t: None), ("mant_rem", lambda t: t.to(torch.int8)),
             ("exp_avg", lambda t: t.t().contiguous().t()), ("mant_rem", lambda t: t.t().contiguous().t())]


# ------------------------------------------------------------- expanded_state --
def test_a_state_that_fits_is_expanded(host):
    p, opt = _adamw()
    x, = opt.expanded_state()
    assert set(x) == {"exp_avg", "exp_avg_sq", "master"} and all(t.shape == p.shape for t in x.values())
    assert [len(r) for r in host.rows] == [3 * state8._WORDS]
    assert [r[3::state8._WORDS].tolist() for r in host.rows] == [[8192] * 3]


@pytest.mark.parametrize("key,change", BAD_ADAMW)
@pytest.mark.parametrize("seen", [False, True])
def test_expanded_state_refuses_a_state_that_does_not_fit(host, key, change, seen):
    p, opt = _adamw()
    opt._init_state(p)
    if seen:  # a state of another size comes after one that fitted
        opt.expanded_state()
    host.rows.clear()
    bad = change(opt.state[p][key])
    if bad is None:
        del opt.state[p][key]
    else:
        opt.state[p][key] = bad
    for call in (opt.expanded_state, opt.expanded_state_dict, lambda: opt.expanded_state([p], torch.bfloat16)):
        with pytest.raises(ValueError, match=key.replace("_scale", "")):
            call()
    assert host.rows == []


def test_a_parameter_that_grew_is_refused(host):
    p, opt = _adamw()
    opt.expanded_state()
    host.rows.clear()
    p.grad = None
    p.data = torch.zeros(128, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="exp_avg"):
        opt.expanded_state()
    assert host.rows == []


def test_an_expanded_checkpoint_refuses_a_state_that_does_not_fit(host):
    model = synth.SyntheticLM(synth.MICRO, seed=0)
    muon, adamw = build_optimizers(model, muon_lr=8e-3, adam_lr=1.2e-2, embed_lr=2.4e-2, weight_decay=0.1,
                                   bf16_master=True, adam_master="bf16_mt", adam_state_dtype=torch.int8)
    p = next(p for g in adamw.param_groups for p in g["params"] if adamw.holds_8bit(p))
    adamw._init_state(p)["exp_avg_sq"] = torch.zeros(p.numel() // 2, dtype=torch.uint8)
    with pytest.raises(ValueError, match="exp_avg_sq"):
        save_checkpoint(model, muon, 1, io.BytesIO(), adamw=adamw, expand_state=True)
    assert host.rows == []


def test_a_remainder_beside_an_fp32_parameter_is_not_expanded(host):
    p, opt = _adamw(dtype=torch.float32)
    opt._init_state(p)["mant_rem"] = torch.zeros(64, 128, dtype=torch.bfloat16)
    assert set(opt.expanded_state()[0]) == {"exp_avg", "exp_avg_sq"}


# ----------------------------------------------------------------- AdamW.step --
def test_a_step_on_states_that_fit_is_launched(host):
    for dt in (torch.int8, torch.float32, torch.bfloat16):
        p, opt = _adamw(state_dtype=dt)
        opt.step()
        opt.step()
    assert host.calls == ["b2o_adamw8_step"] * 2 + ["b2o_adamw_step"] * 4


@pytest.mark.parametrize("key,change", BAD_ADAMW + [("step", lambda t: t.double()), ("step", lambda t: t.expand(2))])
def test_adamw_step_refuses_a_state_that_does_not_fit(host, key, change):
    p, opt = _adamw()
    opt._init_state(p)
    bad = change(opt.state[p][key])
    if bad is None:
        del opt.state[p][key]
    else:
        opt.state[p][key] = bad
    with pytest.raises(ValueError, match=key.replace("_scale", "")):
        opt.step()
    assert host.calls == []


def test_adamw_step_refuses_one_wide_moment_beside_8_bits(host):
    p, opt = _adamw()
    st = opt._init_state(p)
    st["exp_avg"] = st["exp_avg"].float()
    with pytest.raises(ValueError, match="one dtype"):
        opt.step()
    assert host.calls == []


@pytest.mark.parametrize("key,change", [("exp_avg", _cut), ("exp_avg_sq", _cut), ("mant_rem", _cut),
                                        ("exp_avg_sq", lambda t: t.bfloat16()), ("mant_rem", lambda t: t.float()),
                                        ("exp_avg", lambda t: t.t().contiguous().t()), ("step", lambda t: t.double())])
def test_adamw_step_refuses_a_wide_state_that_does_not_fit(host, key, change):
    p, opt = _adamw(state_dtype=torch.float32)
    opt._init_state(p)
    opt.state[p][key] = change(opt.state[p][key])
    with pytest.raises(ValueError, match=key):
        opt.step()
    assert host.calls == []


# ------------------------------------------------------------ NorMuonGNS.step --
def _muon(**kw):
    p = torch.nn.Parameter(torch.zeros(64, 128, dtype=torch.bfloat16))
    p.grad = torch.ones_like(p)
    return p, NorMuonGNS([p], bf16_master=True, **kw)


@pytest.mark.parametrize("kw", [{}, dict(momentum_dtype=torch.int8)])
@pytest.mark.parametrize("hooked", [False, True])
def test_a_muon_step_on_states_that_fit_is_launched(host, kw, hooked):
    p, opt = _muon(**kw)
    if hooked:
        opt._orthogonalize_batch = lambda U, n: torch.zeros_like(U)
    opt.step()
    opt.step()
    assert sum("front" in c for c in host.calls) == 2 and sum("apply" in c for c in host.calls) == 2


@pytest.mark.parametrize("kw,key,change", [
    ({}, "momentum_buffer", _cut), ({}, "momentum_buffer", lambda t: t.float()), ({}, "momentum_buffer", lambda t: t.to(torch.int8)),
    ({}, "v_row", _cut), ({}, "v_row", lambda t: t.bfloat16()), ({}, "mant_rem", _cut), ({}, "mant_rem", lambda t: t.float()),
    ({}, "mant_rem", lambda t: t.t().contiguous().t()),
    (dict(momentum_dtype=torch.int8), "momentum_buffer", _cut), (dict(momentum_dtype=torch.int8), "momentum_scale", _cut),
    (dict(momentum_dtype=torch.int8), "momentum_scale", lambda t: None),
    (dict(momentum_dtype=torch.int8), "momentum_buffer", lambda t: t.float()), (dict(momentum_dtype=torch.int8), "v_row", _cut)])
@pytest.mark.parametrize("hooked", [False, True])
def test_muon_step_refuses_a_state_that_does_not_fit(host, kw, key, change, hooked):
    p, opt = _muon(**kw)
    if hooked:
        opt._orthogonalize_batch = lambda U, n: torch.zeros_like(U)
    opt._init_state(p)
    bad = change(opt.state[p][key])
    if bad is None:
        del opt.state[p][key]
    else:
        opt.state[p][key] = bad
    with pytest.raises(ValueError, match=key.replace("scale", "buffer")):
        opt.step()
    assert host.calls == []


# -------------------------------------------------------------------- loading --
def _saved(opt, p, step=3.0):
    st = opt._init_state(p)
    if "step" in st:
        st["step"].fill_(step)
    return opt.state_dict()


def _snapshot(opt):
    return {k: {n: (t, t._version) if torch.is_tensor(t) else t for n, t in st.items()} for k, st in opt.state.items()}


def _same(a, b):
    """The same states, and each value the same tensor (and not written), or equal."""
    return set(map(id, a)) == set(map(id, b)) and all(
        set(a[p]) == set(b[p]) and all(x[0] is y[0] and x[1] == y[1] if isinstance(x, tuple) else x == y
                                       for x, y in ((a[p][n], b[p][n]) for n in a[p])) for p in a)


@pytest.mark.parametrize("make,kw", [(_adamw, {}), (_adamw, dict(state_dtype=torch.float32)), (_muon, {}),
                                     (_muon, dict(momentum_dtype=torch.int8))])
@pytest.mark.parametrize("shape", [(32, 128), (128, 128), (64, 130)])
def test_a_state_of_another_parameter_is_not_loaded(host, make, kw, shape):
    """Before, the state of a 32 x 128 tensor loaded into an optimizer over 64 x 128."""
    p, opt = make(**kw)
    opt._init_state(p)
    before, groups = _snapshot(opt), opt.state_dict()["param_groups"]
    q = torch.nn.Parameter(torch.zeros(shape, dtype=torch.bfloat16))
    other = AdamW([q], master="bf16_mt", lr=0.5, **{"state_dtype": torch.int8, **kw}) if make is _adamw else \
        NorMuonGNS([q], bf16_master=True, lr=0.5, **kw)
    with pytest.raises(ValueError, match="loaded"):
        opt.load_state_dict(_saved(other, q))
    assert _same(before, _snapshot(opt)) and opt.state_dict()["param_groups"] == groups


@pytest.mark.parametrize("make,kw,bad", [(_adamw, {}, BAD_ADAMW[:10] + [("step", lambda t: torch.zeros(2))]),
                                         (_adamw, dict(state_dtype=torch.float32),
                                          [(k, _cut) for k in ("exp_avg", "exp_avg_sq", "mant_rem")] +
                                          [("exp_avg", lambda t: t.to(torch.int16)), ("mant_rem", lambda t: t.to(torch.int8))]),
                                         (_muon, {}, [(k, _cut) for k in ("momentum_buffer", "v_row", "mant_rem")] +
                                          [("mant_rem", lambda t: t.float())]),
                                         (_muon, dict(momentum_dtype=torch.int8),
                                          [(k, _cut) for k in ("momentum_buffer", "momentum_scale", "v_row", "mant_rem")] +
                                          [("momentum_scale", lambda t: None), ("momentum_scale", lambda t: t.bfloat16())])])
def test_each_part_of_a_loaded_state_is_checked(host, make, kw, bad):
    for key, change in bad:
        p, opt = make(**kw)
        sd = _saved(opt, p)
        x = change(sd["state"][0][key])
        sd["state"][0] = {k: v for k, v in {**sd["state"][0], key: x}.items() if v is not None}
        before = _snapshot(opt)
        with pytest.raises(ValueError, match="|".join(("loaded", "without scales"))):
            opt.load_state_dict(sd)
        assert _same(before, _snapshot(opt)), key


@pytest.mark.parametrize("make,kw", [(_adamw, {}), (_adamw, dict(state_dtype=torch.float32)), (_muon, {}),
                                     (_muon, dict(momentum_dtype=torch.int8))])
def test_a_state_that_fits_is_loaded_and_steps(host, make, kw):
    p, opt = make(**kw)
    sd = _saved(opt, p)
    opt.load_state_dict(sd)
    opt.step()
    assert host.calls and (make is _muon or opt._steps[id(p)] == 4)
    with pytest.raises(ValueError, match="group"):  # torch's own refusal keeps its form
        opt.load_state_dict({"state": {5: sd["state"][0]}, "param_groups": sd["param_groups"] * 2})


def test_loaded_types_become_those_that_the_kernels_read(host):
    """torch's loader in the reference leaves v_row in bf16 when a run is resumed, and a state saved from a transposed
    parameter keeps its strides."""
    p, opt = _muon()
    st = opt._init_state(p)
    x = torch.arange(64 * 128).view(64, 128).float() / 64
    sd = {"state": {0: {"momentum_buffer": x.clone(), "v_row": torch.full((64, 1), 0.5, dtype=torch.bfloat16),
                        "mant_rem": x.bfloat16().t().contiguous().t()}}, "param_groups": opt.state_dict()["param_groups"]}
    opt.load_state_dict(sd)
    st = opt.state[p]
    assert st["v_row"].dtype == torch.float32 and st["momentum_buffer"].dtype == torch.bfloat16
    assert torch.equal(st["momentum_buffer"], x.bfloat16()) and torch.equal(st["mant_rem"], x.bfloat16())
    opt.step()
    q, adam = _adamw(state_dtype=torch.float32)
    sd = _saved(adam, q)
    sd["state"][0] = {**sd["state"][0], "step": torch.tensor(3.0, dtype=torch.float64), "exp_avg": x.t().contiguous().t()}
    adam.load_state_dict(sd)
    assert torch.equal(adam.state[q]["exp_avg"], x) and adam._steps[id(q)] == 3
    adam.step()


# -------------------------------------------------------------- refused calls --
@pytest.mark.parametrize("hooked", [False, True])
def test_a_refused_front_call_leaves_the_step_counts(host, hooked):
    """The count is the t of the codes: after a refusal a step has to be the one that it would have been."""
    p, opt = _muon(momentum_dtype=torch.int8)
    if hooked:
        opt._orthogonalize_batch = lambda U, n: torch.zeros_like(U)
    opt.step()
    host.fail = "b2o_normuon_front8_multi"
    for _ in range(3):
        with pytest.raises(RuntimeError, match="front8"):
            opt.step()
    assert opt.state[p]["momentum_step"] == 1
    host.fail = None
    opt.step()
    assert opt.state[p]["momentum_step"] == 2


def test_the_counts_that_the_front_call_gets(host):
    p, opt = _muon(momentum_dtype=torch.int8)
    q = torch.nn.Parameter(torch.zeros(64, 128, dtype=torch.bfloat16))
    q.grad = torch.ones_like(q)
    opt.add_param_group({"params": [q]})
    opt._init_state(q)["momentum_step"] = 2 ** 32 - 1
    seen = []
    real = host.__getattr__

    def look(name):
        call = real(name)
        if name != "b2o_normuon_front8_multi":
            return call
        return lambda arr, scales, steps, n, *a: seen.append(
            [ctypes.cast(steps[0], ctypes.POINTER(ctypes.c_uint32))[0]]) or call(arr, scales, steps, n, *a)
    type(host).__getattr__, keep = lambda self, name: look(name), type(host).__getattr__
    try:
        opt.step()
        opt.step()
    finally:
        type(host).__getattr__ = keep
    assert seen == [[1], [0], [2], [1]] and opt.state[q]["momentum_step"] == 2 ** 32 + 1


def test_momentum_out_of_range_is_refused_before_any_group_steps(host):
    p, opt = _muon(momentum_dtype=torch.int8)
    q = torch.nn.Parameter(torch.zeros(64, 128, dtype=torch.bfloat16))
    q.grad = torch.ones_like(q)
    opt.add_param_group({"params": [q]})
    for bad in (1.0, -0.1, float("nan")):
        opt.param_groups[1]["momentum"] = bad
        with pytest.raises(ValueError, match="momentum in"):
            opt.step()
    assert host.calls == []
    q.grad = None  # takes no part
    opt.step()
    wide = NorMuonGNS([torch.nn.Parameter(torch.zeros(4, 4))], momentum=1.0)
    assert wide.param_groups[0]["momentum"] == 1.0


@pytest.mark.parametrize("state_dtype,call", [(torch.int8, "b2o_adamw8_step"), (torch.float32, "b2o_adamw_step")])
def test_a_refused_adamw_call_leaves_the_step_counts(host, state_dtype, call):
    p, opt = _adamw(state_dtype=state_dtype)
    opt.step()
    host.fail = call
    for _ in range(3):
        with pytest.raises(RuntimeError, match="adamw"):
            opt.step()
    assert opt._steps[id(p)] == 1
    host.fail = None
    opt.step()
    assert opt._steps[id(p)] == 2


# ------------------------------------------------------------------ the device --
@pytest.mark.parametrize("kw", [{}, dict(momentum_dtype=torch.int8)])
@pytest.mark.parametrize("hooked", [False, True])
def test_every_launch_of_a_muon_step_runs_on_its_parameters_device(host, monkeypatch, kw, hooked):
    """With an overridden _orthogonalize_batch too, which calls the engine's own here."""
    current = []

    @contextlib.contextmanager
    def on_device(dev):
        current.append(dev)
        yield
        current.pop()
    monkeypatch.setattr(_lib, "on_device", on_device)
    p, opt = _muon(**kw)
    if hooked:
        inner = opt._orthogonalize_batch
        opt._orthogonalize_batch = lambda U, n: inner(U, n)
    real, where = host.__getattr__, []

    def look(name):
        call = real(name)
        return call if call.__name__ != "call" else lambda *a: where.append((name, list(current))) or call(*a)
    type(host).__getattr__, keep = lambda self, name: look(name), type(host).__getattr__
    try:
        opt.step()
    finally:
        type(host).__getattr__ = keep
    assert any("front" in n for n, _ in where) and any("orthogonalize" in n for n, _ in where)
    assert all(on == [p.device] for _, on in where), where


def test_expanded_state_refuses_a_parameter_of_another_optimizer(host):
    """It would get a state here, and state_dict() could no longer name its parameter."""
    p, opt = _adamw()
    q, _ = _adamw()
    with pytest.raises(ValueError, match="not this optimizer"):
        opt.expanded_state([p, q])
    assert q not in opt.state and host.rows == []
    assert set(opt.state_dict()["state"]) == {0}
    opt.expanded_state([p, p])

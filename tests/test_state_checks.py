"""States that do not fit their parameter are refused before a kernel gets their
pointers. Everything runs on the host: the launches are replaced, so that a state
that slips through is seen in the descriptors and touches no memory."""
import contextlib
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

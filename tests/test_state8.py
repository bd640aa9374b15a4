"""8-bit optimizer states on the host: the format's restatement, refusals of the
C entry points and of the Python layer, checkpoints and the sharded layout."""
import ctypes
import datetime
import io
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from oracle import state8_ref as ref
from sol_b200 import AdamW, EmaWeights, NorMuonGNS, _lib, build_optimizers, state8, synth
from sol_b200.checkpoint import load_checkpoint, save_checkpoint
from sol_b200.sharding import ShardedStep

KW = dict(muon_lr=8e-3, adam_lr=1.2e-2, embed_lr=2.4e-2, weight_decay=0.1, cautious_wd=True, bf16_master=True)


# ------------------------------------------------------------------- format --
@pytest.mark.parametrize("root", [False, True])
def test_every_code_stands_for_a_value_that_encodes_to_it(root):
    codes = torch.arange(256).to(torch.uint8) if root else torch.arange(-127, 128).to(torch.int8)
    codes = torch.cat([codes, codes[-1:].expand((-len(codes)) % 128)])
    for s in (1.0, 3.1e-5, 7e12):
        scales = torch.full((codes.numel() // 128,), s)
        # every block needs its largest code for its scale to be found again
        c = codes.clone().view(-1, 128)
        c[:, 0] = 255 if root else 127
        back, again = ref.encode(ref.decode(c.view(-1), scales, root), root)
        assert torch.equal(back, c.view(-1))
        # the largest value is s by two (root: and squared and rooted, two more) roundings of half a step
        assert torch.allclose(again, scales, rtol=4 * 2.0 ** -24, atol=0)


def test_a_steps_offset_is_even_over_steps():
    """Over 4096 steps the offsets of an element leave no gap wider than 4 / 4096
    (a rotation by an irrational-like turn), so a state's expected code is the state."""
    for i in (0, 1, 77, 10 ** 9):
        u = torch.stack([ref.offset(1, t, True, i)[0] for t in range(1, 4097)]).sort().values
        assert torch.diff(u).max() < 4 / 4096 and u[0] < 4 / 4096 and u[-1] > 1 - 4 / 4096


def test_a_first_moment_without_gradient_decays():
    """An element whose gradient stays zero inside a live block: to nearest its
    code would stay where 10 % of decay is below half a step; here it reaches 0."""
    g = torch.Generator().manual_seed(0)
    codes, scales = torch.zeros(128, dtype=torch.int8), torch.zeros(1)
    for t in range(1, 300):
        grad = torch.randn(128, generator=g)
        if t > 20:
            grad[5] = 0
        _, codes, scales = ref.momentum_step(grad, codes, scales, beta=0.9, nesterov=False, step=t)
    assert codes[5] == 0 and scales[0] > 0


# ----------------------------------------------------------------- refusals --
def test_ctypes_structs_match_header_layout():
    assert ctypes.sizeof(_lib.Adamw8Tensor) == 8 * 8 + 2 * 8 + 2 * 4 + 8
    assert ctypes.sizeof(_lib.Adamw8Group) == 6 * 8 + 8 + 2 * 4
    assert ctypes.sizeof(_lib.StateTensor) == 3 * 8 + 8 + 2 * 4


def test_state_blocks():
    lib = _lib.load()
    assert [lib.b2o_state_blocks(n) for n in (-1, 0, 1, 128, 129, 2 ** 33 + 1)] == [0, 0, 1, 1, 2, 2 ** 26 + 1]
    assert state8.BLOCK == 128 and state8.blocks(129) == 2


def _state(**kw):
    d = dict(value=16, codes=16, scales=16, numel=8, kind=0, value_dtype=_lib.F32)
    return _lib.StateTensor(**{**d, **kw})


@pytest.mark.parametrize("bad,msg", [(dict(value=None), "null pointer"), (dict(codes=None), "null pointer"),
                                     (dict(scales=None), "null pointer"), (dict(numel=-1), "null pointer"),
                                     (dict(kind=3), "unknown kind"), (dict(value_dtype=_lib.F16), "fp32 or bf16"),
                                     (dict(numel=2 ** 50), "too large")])
def test_conversions_refuse_on_the_host(bad, msg):
    lib = _lib.load()
    for fn in (lib.b2o_state_encode, lib.b2o_state_decode):
        arr = (_lib.StateTensor * 2)(_state(numel=0), _state(**bad))
        assert fn(arr, 2, None) < 0 and msg in _lib.last_error()
        assert fn(None, 1, None) < 0 and fn(arr, -1, None) < 0
        assert fn(None, 0, None) == 0


def _adam(**kw):
    d = dict(param=16, rem=None, grad=16, exp_avg=16, exp_avg_sq=16, exp_avg_scale=16, exp_avg_sq_scale=16, ema=None,
             numel=8, first=0, group=0, step_out=None)
    return _lib.Adamw8Tensor(**{**d, **kw})


def _group(**kw):
    d = dict(lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0, step=1.0, grad_scale=None, cautious=0)
    return _lib.Adamw8Group(**{**d, **kw})


@pytest.mark.parametrize("tensor,group,dtype,msg", [
    (dict(grad=None), {}, 1, "null pointer"), (dict(exp_avg_scale=None), {}, 1, "null pointer"),
    (dict(numel=-5), {}, 1, "negative size"), (dict(first=-128), {}, 1, "negative size"),
    (dict(first=64), {}, 1, "multiple of 128"), (dict(group=1), {}, 1, "group out of range"),
    (dict(rem=16), {}, 0, "remainder needs bf16"), ({}, {}, 2, "bad param dtype"),
    (dict(numel=2 ** 50), {}, 1, "too large"),
    ({}, dict(beta1=1.0), 1, "betas"), ({}, dict(beta2=-0.1), 1, "betas"), ({}, dict(beta2=float("nan")), 1, "betas"),
    ({}, dict(eps=-1.0), 1, "eps"), ({}, dict(step=0.0), 1, "step"), ({}, dict(step=1e16), 1, "step")])
def test_adamw8_refuses_on_the_host(tensor, group, dtype, msg):
    lib = _lib.load()
    rc = lib.b2o_adamw8_step((_lib.Adamw8Tensor * 1)(_adam(**tensor)), 1, (_lib.Adamw8Group * 1)(_group(**group)), 1,
                             dtype, 0.0, None)
    assert rc < 0 and msg in _lib.last_error()


def test_adamw8_refuses_bad_lists():
    lib = _lib.load()
    g = (_lib.Adamw8Group * 9)(*[_group() for _ in range(9)])
    assert lib.b2o_adamw8_step(None, 1, g, 1, 1, 0.0, None) < 0
    assert lib.b2o_adamw8_step(None, 0, g, 0, 1, 0.0, None) < 0
    assert lib.b2o_adamw8_step(None, 0, g, 9, 1, 0.0, None) < 0
    assert lib.b2o_adamw8_step(None, 0, g, 8, 1, 0.0, None) == 0


def test_front8_refuses_on_the_host():
    lib = _lib.load()
    ptr = _lib.ptr_array([16])
    steps = (ctypes.c_uint32 * 1)(1)
    good = dict(S=1, r=4, c=4, grads=_lib.addr(ptr), bufs=_lib.addr(ptr), u=16, partial=16)

    def call(batch=None, scales=True, step=True, dtype=1, beta=0.9):
        arr = (_lib.NormuonBatch * 1)(_lib.NormuonBatch(**{**good, **(batch or {})}))
        sc = _lib.ptr_array([_lib.addr(ptr) if scales is True else scales])
        return lib.b2o_normuon_front8_multi(arr, None if scales is None else sc,
                                            _lib.ptr_array([ctypes.addressof(steps) if step else None]), 1, dtype, beta, 1,
                                            None, None)
    null = _lib.ptr_array([None])
    for kw, msg in ((dict(batch=dict(S=0)), "1..64"), (dict(batch=dict(u=None)), "bad args"),
                    (dict(batch=dict(bufs=_lib.addr(null))), "null matrix"), (dict(scales=None), "no scales"),
                    (dict(scales=0), "null scale"), (dict(scales=_lib.addr(null)), "null scale"),
                    (dict(step=False), "null step"), (dict(dtype=2), "bad dtype"), (dict(beta=1.0), "momentum"),
                    (dict(beta=float("nan")), "momentum"), (dict(batch=dict(x0_half=1)), "x0_half")):
        assert call(**kw) < 0 and msg in _lib.last_error(), kw


def test_python_layer_refuses():
    p = torch.nn.Parameter(torch.randn(64, 128))
    p.grad = torch.randn(64, 128)
    with pytest.raises(ValueError, match="state_dtype"):
        AdamW([p], state_dtype=torch.float16)
    with pytest.raises(ValueError, match="betas"):
        AdamW([p], state_dtype=torch.int8, betas=(0.9, 1.0))
    with pytest.raises(ValueError, match="momentum_dtype"):
        NorMuonGNS([p], momentum_dtype=torch.uint8)
    with pytest.raises(ValueError, match="momentum in"):
        NorMuonGNS([p], momentum=1.0, momentum_dtype=torch.int8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        AdamW([p], state_dtype=torch.int8).step()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        NorMuonGNS([p], momentum_dtype=torch.int8).step()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        AdamW([p], state_dtype=torch.int8).expanded_state()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        state8.encode([(torch.zeros(4), "signed")])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        state8.decode([(torch.zeros(4, dtype=torch.int8), torch.zeros(1), "signed")])
    with pytest.raises(ValueError, match="kind"):
        state8.encode([(torch.zeros(4), "unsigned")])
    with pytest.raises(ValueError, match="outputs"):
        state8.decode([], out=[torch.zeros(1)])
    with pytest.raises(ValueError, match="dtypes"):
        state8.decode([], dtype=[torch.float32])
    assert state8.encode([]) == [] and state8.decode([]) == []


# ------------------------------------------------------- layout, checkpoints --
def test_which_parameters_hold_8_bits():
    model = synth.SyntheticLM(synth.MICRO, device="meta")
    muon, adamw = build_optimizers(model, adam_state_dtype=torch.int8, momentum_dtype=torch.int8, **KW)
    held = [p for g in adamw.param_groups for p in g["params"] if adamw.holds_8bit(p)]
    assert held and all(p.numel() >= 4096 for p in held)
    assert muon.momentum_dtype == torch.int8
    assert not any(AdamW([p]).holds_8bit(p) for p in held)


def _fill(muon, adamw):
    g = torch.Generator().manual_seed(3)
    for opt in (muon, adamw):
        for group in opt.param_groups:
            for p in group["params"]:
                st = opt._init_state(p)
                for k in sorted(st):
                    if not torch.is_tensor(st[k]):
                        st[k] = 7
                    elif st[k].dtype in (torch.int8, torch.uint8):
                        st[k].copy_(torch.randint(0, 127, st[k].shape, generator=g))
                    elif k != "step":
                        st[k].copy_(torch.rand(st[k].shape, generator=g))
                    else:
                        st[k].fill_(7.0)
                if opt is adamw:
                    adamw._steps[id(p)] = 7


def test_checkpoint_keeps_8_bit_states():
    opts = []
    for seed in (0, 1):
        model = synth.SyntheticLM(synth.MICRO, seed=seed)
        opts.append((model, *build_optimizers(model, adam_master="bf16_mt", adam_state_dtype=torch.int8,
                                              momentum_dtype=torch.int8, **KW)))
    _fill(*opts[0][1:])
    buf = io.BytesIO()
    save_checkpoint(opts[0][0], opts[0][1], 5, buf, adamw=opts[0][2])
    buf.seek(0)
    assert load_checkpoint(buf, opts[1][0], opts[1][1], adamw=opts[1][2]) == 5
    for a, b in zip(opts[0][1:], opts[1][1:]):
        for p, q in zip([p for g in a.param_groups for p in g["params"]], [p for g in b.param_groups for p in g["params"]]):
            assert set(a.state[p]) == set(b.state[q])
            for k, v in a.state[p].items():
                w = b.state[q][k]
                assert (w == v) if not torch.is_tensor(v) else (w.dtype == v.dtype and torch.equal(w, v)), k


def _port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _gather_worker(rank, world, port, q):
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    try:
        dist.init_process_group("gloo", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=60))
        model = synth.SyntheticLM(synth.MICRO, seed=0)
        muon, adamw = build_optimizers(model, adam_master="bf16_mt", adam_state_dtype=torch.int8,
                                       momentum_dtype=torch.int8, **KW)
        ema = EmaWeights(model, 0.999)
        whole = synth.SyntheticLM(synth.MICRO, seed=0)
        wm, wa = build_optimizers(whole, adam_master="bf16_mt", adam_state_dtype=torch.int8, momentum_dtype=torch.int8, **KW)
        _fill(wm, wa)
        sh = ShardedStep(model, muon, adamw, ema, world, rank, min_rows_shard=16)
        assert sh.row_sharded
        for a, b in ((muon, wm), (adamw, wa)):
            for p, r in zip([p for g in a.param_groups for p in g["params"]], [p for g in b.param_groups for p in g["params"]]):
                st = a._init_state(p)
                if a is muon:
                    if sh.owner[id(p)] == rank:
                        for k, v in b.state[r].items():
                            st[k] = v.clone() if torch.is_tensor(v) else v
                    continue
                start, n = adamw._owned_slices[id(p)]
                assert start % 128 == 0 and (n % 128 == 0 or start + n == p.numel()) or not adamw.holds_8bit(p)
                for k, v in b.state[r].items():
                    flat, src = st[k].view(-1), v.view(-1)
                    lo, hi = (start // 128, -(-(start + n) // 128)) if k.endswith("_scale") else (start, start + n)
                    if k == "step":
                        lo, hi = 0, 1
                    flat[lo:hi] = src[lo:hi]
        sh.gather_state()
        bad = []
        for a, b in ((muon, wm), (adamw, wa)):
            for p, r in zip([p for g in a.param_groups for p in g["params"]], [p for g in b.param_groups for p in g["params"]]):
                for k, v in b.state[r].items():
                    w = a.state[p][k]
                    if not (torch.equal(w, v) if torch.is_tensor(v) else w == v):
                        bad.append((tuple(p.shape), k))
        q.put((rank, bad))
    except Exception as e:  # the parent reports it
        q.put((rank, repr(e)))
    finally:
        if dist.is_initialized():
            dist.destroy_process_group()


def test_sharded_ranks_gather_8_bit_states():
    ctx = mp.get_context("spawn")
    q, port = ctx.Queue(), _port()
    ps = [ctx.Process(target=_gather_worker, args=(r, 2, port, q)) for r in range(2)]
    for p in ps:
        p.start()
    got = [q.get(timeout=180) for _ in ps]
    for p in ps:
        p.join(timeout=60)
    assert all(bad == [] for _, bad in got), got


def test_row_slices_hold_whole_blocks():
    """A table that divides by the world size but not into whole blocks stays whole on every rank."""
    class M(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.token_embeddings = torch.nn.Parameter(torch.zeros(66, 100, dtype=torch.bfloat16))
            self.w = torch.nn.Parameter(torch.zeros(64, 64, dtype=torch.bfloat16))
    for dt, want in ((torch.int8, (0, 6600)), (None, (3300, 3300))):
        model = M()
        muon, adamw = build_optimizers(model, adam_state_dtype=dt, **KW)
        ShardedStep(model, muon, adamw, None, 2, 1, min_rows_shard=16, exchange="nccl")
        assert adamw._owned_slices[id(model.token_embeddings)] == want

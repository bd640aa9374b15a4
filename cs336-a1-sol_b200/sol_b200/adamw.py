"""Fused AdamW (+ EMA) on the B200 engine.

Drop-in for the ``torch.optim.AdamW(groups, betas=..., eps=..., fused=True)``
built by ``build_optimizers`` (transformer_lm/sol_modules.py:468-476). Same
defaults, param-group keys (lr, betas, eps, weight_decay, amsgrad, maximize,
foreach, capturable, differentiable, fused) and per-parameter state
(``step`` fp32 0-d tensor, ``exp_avg``, ``exp_avg_sq``).

Storage modes:
  * reference (default): moments in the parameter dtype, exactly what torch's
    fused AdamW keeps for bf16 parameters; the arithmetic is torch's fused
    formula (ATen/native/cuda/fused_adam_utils.cuh, ADAMW mode) in fp32.
  * master="bf16_mt": bf16 parameter plus a bf16 low-mantissa remainder
    (``mant_rem``, the NorMuonGNS trick at sol_modules.py:406-424) and fp32
    moments (state_dtype=torch.float32); optional cautious weight decay.
  * state_dtype=torch.int8 (with either of the above): both moments in 8 bits
    with one fp32 scale per 128 elements (format in state8.py; state keys
    ``exp_avg`` int8, ``exp_avg_sq`` uint8, ``exp_avg_scale``,
    ``exp_avg_sq_scale``): 2.06 bytes per element instead of 4 or 8, and 22
    bytes moved per element of the recipe's tables instead of 34. Parameters
    with fewer than ``min_8bit_numel`` elements (gains, gates, scalars: nothing
    to save there) keep fp32 moments. The rounding is even over steps and a
    function of element and step alone, so results repeat and a sharded step
    gives what one GPU gives.
One streaming kernel pass updates parameter, remainder, moments and (when an
EmaWeights object has armed folding) the fp32 EMA shadow.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import _lib, state8
from .ema import register_optimizer

MAX_GROUPS = 8
# b2o_adamw_tensor as 64-bit words (the gradient pointer is refreshed in place each step)
_DESC_WORDS = C.sizeof(_lib.AdamwTensor) // 8
_GRAD_WORD = _lib.AdamwTensor.grad.offset // 8
assert C.sizeof(_lib.AdamwTensor) % 8 == 0 and _lib.AdamwTensor.grad.offset % 8 == 0
_DESC8_WORDS = C.sizeof(_lib.Adamw8Tensor) // 8
_GRAD8_WORD = _lib.Adamw8Tensor.grad.offset // 8


class AdamW(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, amsgrad=False, *,
                 maximize=False, foreach=None, capturable=False, differentiable=False, fused=None,
                 decoupled_weight_decay=True, master="none", state_dtype=None, cautious_wd=False,
                 min_8bit_numel=4096):
        if amsgrad or maximize or capturable or differentiable or not decoupled_weight_decay:
            raise ValueError("the B200 AdamW implements the recipe's configuration: no amsgrad/maximize/"
                             "capturable/differentiable")
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=amsgrad,
                        maximize=maximize, foreach=foreach, capturable=capturable, differentiable=differentiable,
                        fused=fused, decoupled_weight_decay=True)
        super().__init__(params, defaults)
        if master not in ("none", "bf16_mt"):
            raise ValueError("master must be 'none' or 'bf16_mt'")
        if state_dtype not in (None, torch.float32, torch.bfloat16, torch.int8):
            raise ValueError("state_dtype must be None, torch.float32, torch.bfloat16 or torch.int8")
        if state_dtype == torch.int8:
            for group in self.param_groups:
                self._check_8bit_group(group)
        self.master = master
        self.min_8bit_numel = int(min_8bit_numel)
        self.state_dtype = state_dtype
        self.cautious_wd = cautious_wd
        self._steps = {}           # id(param) -> int step count (mirrors state["step"])
        self._owned_slices = None  # id(param) -> (start_elem, numel) this rank updates
        self._ema = None           # EmaWeights folded into the pass (set when it arms)
        self._ema_weight = 0.0
        self._grad_scale = None    # device fp32 clip coefficient for the next step (clip_grad_norm_ defer_to)
        self._plan = None          # cached launch descriptors (see step)
        self._checked = {}         # id(param) -> what expanded_state last found to fit it
        register_optimizer(self)

    @staticmethod
    def _check_8bit_group(group):
        b1, b2 = group["betas"]
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and group["eps"] >= 0.0):
            raise ValueError("AdamW with 8-bit moments needs betas in [0, 1) and eps >= 0")

    def holds_8bit(self, p) -> bool:
        """Whether this optimizer keeps p's moments in 8 bits."""
        return self.state_dtype == torch.int8 and p.numel() >= max(1, self.min_8bit_numel)

    def _init_state(self, p):
        st = self.state[p]
        if "step" not in st and self.holds_8bit(p):
            st["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
            nb = state8.blocks(p.numel())
            st["exp_avg"] = torch.zeros_like(p, dtype=torch.int8, memory_format=torch.preserve_format)
            st["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.uint8, memory_format=torch.preserve_format)
            st["exp_avg_scale"] = torch.zeros(nb, dtype=torch.float32, device=p.device)
            st["exp_avg_sq_scale"] = torch.zeros(nb, dtype=torch.float32, device=p.device)
            if self.master == "bf16_mt" and p.dtype == torch.bfloat16:
                st["mant_rem"] = torch.zeros_like(p)
            self._steps[id(p)] = 0
        if "step" not in st:
            st["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
            sdt = torch.float32 if self.state_dtype == torch.int8 else self.state_dtype or p.dtype
            if self.master == "bf16_mt" and p.dtype == torch.bfloat16 and self.state_dtype is None:
                sdt = torch.float32
            st["exp_avg"] = torch.zeros_like(p, dtype=sdt, memory_format=torch.preserve_format)
            st["exp_avg_sq"] = torch.zeros_like(p, dtype=sdt, memory_format=torch.preserve_format)
            if self.master == "bf16_mt" and p.dtype == torch.bfloat16:
                st["mant_rem"] = torch.zeros_like(p)
            self._steps[id(p)] = int(st["step"].item()) if st["step"].device.type == "cpu" else 0
        return st


    def load_state_dict(self, state_dict):
        """Keeps each saved state tensor's dtype (fp32 moments of bf16 parameters
        in master mode; torch's loader would cast them to bf16), except between
        8-bit and wider moments: those are converted to what this optimizer
        holds (on the GPU; needs the parameters there). A state that does not
        fit its parameter is refused, and nothing is loaded."""
        from .normuon import _load_state_keep_dtypes
        _load_state_keep_dtypes(self, state_dict, self._check_loaded)
        self.invalidate_plan()
        self._convert_loaded()
        for group in self.param_groups:
            for p in group["params"]:
                st = self.state.get(p)
                if st and "step" in st:
                    st["step"] = st["step"].float()
                    self._steps[id(p)] = int(float(st["step"].item()))

    @staticmethod
    def _check_loaded(p, st):
        from .normuon import _check_loaded_size
        n, m, v = p.numel(), st.get("exp_avg"), st.get("exp_avg_sq")
        if m is not None and v is not None and (m.dtype == torch.int8 or v.dtype == torch.uint8):
            state8.check_sizes(n, m, st.get("exp_avg_scale"), "signed", "AdamW: the loaded exp_avg")
            state8.check_sizes(n, v, st.get("exp_avg_sq_scale"), "root", "AdamW: the loaded exp_avg_sq")
        else:
            _check_loaded_size(st, "exp_avg", n, None, "AdamW")
            _check_loaded_size(st, "exp_avg_sq", n, None, "AdamW")
        if p.dtype == torch.bfloat16:
            _check_loaded_size(st, "mant_rem", n, (torch.bfloat16,), "AdamW")
        if torch.is_tensor(st.get("step")):
            _check_loaded_size(st, "step", 1, None, "AdamW")

    def _convert_loaded(self):
        narrow, widen = [], []
        for group in self.param_groups:
            for p in group["params"]:
                st = self.state.get(p)
                if not st or "exp_avg" not in st:
                    continue
                if self.holds_8bit(p) and st["exp_avg"].dtype != torch.int8:
                    narrow.append(st)
                elif not self.holds_8bit(p) and st["exp_avg"].dtype == torch.int8:
                    widen.append((p, st))
        if narrow:
            kept = state8.encode([x for st in narrow for x in ((st["exp_avg"].contiguous(), "signed"),
                                                               (st["exp_avg_sq"].contiguous(), "root"))])
            for i, st in enumerate(narrow):
                st["exp_avg"], st["exp_avg_scale"] = kept[2 * i]
                st["exp_avg_sq"], st["exp_avg_sq_scale"] = kept[2 * i + 1]
        for p, st in widen:
            dt = self.state_dtype if self.state_dtype in (torch.float32, torch.bfloat16) else torch.float32
            if self.state_dtype is None and self.master == "none":
                dt = p.dtype
            st["exp_avg"], st["exp_avg_sq"] = state8.decode(
                [(st["exp_avg"], st.pop("exp_avg_scale"), "signed"),
                 (st["exp_avg_sq"], st.pop("exp_avg_sq_scale"), "root")], dtype=dt)

    @staticmethod
    def _check_narrow(p, st):
        """Refuses 8-bit moments and a remainder that are not those of parameter p."""
        m, v = st["exp_avg"], st["exp_avg_sq"]
        if m.dtype == torch.int8 or v.dtype == torch.uint8:
            state8.check_state(p, m, st.get("exp_avg_scale"), "signed", "AdamW: exp_avg")
            state8.check_state(p, v, st.get("exp_avg_sq_scale"), "root", "AdamW: exp_avg_sq")
        rem = st.get("mant_rem")
        if rem is not None and p.dtype == torch.bfloat16:
            _lib.require_match(rem, p, p.numel(), (torch.bfloat16,), "AdamW: mant_rem")

    @torch.no_grad()
    def expanded_state(self, params=None, dtype=torch.float32):
        """The moments as ``dtype`` (fp32 or bf16) tensors, and the fp32 master
        weight where a bf16 parameter has a remainder: one dict per parameter
        with "exp_avg", "exp_avg_sq" and, there, "master". A state that does not
        fit its parameter is refused. 8-bit moments and
        master weights of all parameters are expanded in one launch; moments
        that are wide already are cast by torch. (In a sharded step a rank's
        moments are those of its own rows until ``gather_state``.)"""
        if params is None:
            params = [p for g in self.param_groups for p in g["params"]]
        value_code = state8._VALUE_CODE.get(dtype)
        if value_code is None:
            raise TypeError(f"AdamW.expanded_state: float32 or bfloat16 (got {dtype})")
        signed, root = value_code << 32, 1 | value_code << 32
        pair = 2 | _lib.F32 << 32
        out, rows, last, extend = [], state8.Rows(), None, None
        empty, eight, f32, states = torch.empty_like, torch.int8, torch.float32, self.state
        checked, unseen, mine = self._checked, (None,) * 9, None
        for p in params:
            index = p.get_device()
            if index != last:
                _lib.require_cuda(p, "AdamW.expanded_state")
                last, extend = index, rows.extend(index)
            st = states.get(p)
            if not st or "exp_avg" not in st:
                if mine is None:
                    mine = {id(q) for g in self.param_groups for q in g["params"]}
                if id(p) not in mine:
                    raise ValueError("AdamW.expanded_state: a parameter that is not this optimizer's")
                st = self._init_state(p)
            m, v, n = st["exp_avg"], st["exp_avg_sq"], p.numel()
            get = st.get
            ms, vs, rem = get("exp_avg_scale"), get("exp_avg_sq_scale"), get("mant_rem")
            # The kernel takes n elements of each. The same tensors are looked over once.
            m0, v0, ms0, vs0, rem0, n0, index0, narrow, pair_of = checked.get(id(p), unseen)
            if not (m is m0 and v is v0 and ms is ms0 and vs is vs0 and rem is rem0 and n == n0 and index == index0):
                self._check_narrow(p, st)
                narrow, pair_of = m.dtype is eight, rem if p.dtype is torch.bfloat16 else None
                checked[id(p)] = (m, v, ms, vs, rem, n, index, narrow, pair_of)
            if narrow:
                a, b = empty(m, dtype=dtype), empty(v, dtype=dtype)
                if n:
                    extend((a.data_ptr(), m.data_ptr(), ms.data_ptr(), n, signed,
                            b.data_ptr(), v.data_ptr(), vs.data_ptr(), n, root))
            else:
                a, b = m.to(dtype, copy=True), v.to(dtype, copy=True)
            wide = {"exp_avg": a, "exp_avg_sq": b}
            if pair_of is not None:
                if not p.is_contiguous():
                    raise ValueError("AdamW.expanded_state: contiguous parameters only")
                wide["master"] = w = empty(rem, dtype=f32)
                if n:
                    extend((w.data_ptr(), p.data_ptr(), rem.data_ptr(), n, pair))
            out.append(wide)
        rows.launch(_lib.load().b2o_state_decode, "state_decode")
        return out

    def expanded_state_dict(self):
        """state_dict() with 8-bit moments expanded to fp32 (the layout of torch's AdamW)."""
        sd = self.state_dict()
        for p, key in self._state_keys(sd):
            st = sd["state"].get(key)
            if st and "exp_avg" in st and (st["exp_avg"].dtype == torch.int8 or st["exp_avg_sq"].dtype == torch.uint8):
                wide = self.expanded_state([p])[0]
                sd["state"][key] = {k: wide.get(k, v) for k, v in st.items()
                                    if k not in ("exp_avg_scale", "exp_avg_sq_scale")}
        return sd

    def _state_keys(self, sd):
        params = [p for g in self.param_groups for p in g["params"]]
        return list(zip(params, [k for g in sd["param_groups"] for k in g["params"]]))

    def invalidate_plan(self) -> None:
        """Drops the cached launch descriptors (rebuilt on the next step). Needed
        only after replacing a parameter's state dict or one of its state
        tensors by hand (load_state_dict does this itself); steps detect new
        parameters, moved parameter storage, gradients appearing or vanishing,
        EMA folding and shard changes themselves."""
        self._plan = None
        self._checked = {}

    def _build_plan(self, ps, gis, key):
        """Launch descriptors for the parameters (with gradients) of this step:
        one b2o_adamw_tensor array per (device, param dtype, state dtype)
        bucket, with every pointer except the gradient's filled in."""
        buckets = {}
        step_of = {}
        for gi, p in zip(gis, ps):
            _lib.require_cuda(p, "AdamW.step")
            if not p.is_contiguous():
                raise ValueError("AdamW needs contiguous params and grads of the param dtype")
            st = self._init_state(p)
            if step_of.setdefault(gi, self._steps.get(id(p), 0)) != self._steps.get(id(p), 0):
                raise RuntimeError("params of one group have different step counts")
            buckets.setdefault((p.device, p.dtype, st["exp_avg"].dtype), []).append((gi, p, st))
        for (_, _, sdt), members in buckets.items():
            if sdt == torch.int8 and len({id(p) for _, p, _ in members}) != len(members):
                raise ValueError("AdamW: a parameter with 8-bit moments appears twice")
        launches, ema_idx = [], set()
        pos = {id(p): i for i, p in enumerate(ps)}
        # (gradient words of a descriptor array, the items' positions in ps, byte offsets)
        refresh = []
        for (dev, pdt, sdt), members in buckets.items():
            descs, owners = [], []
            for gi, p, st in members:
                shadow = self._ema._lookup(p) if self._ema is not None else None
                rem = st.get("mant_rem")
                start, n = 0, p.numel()
                if self._owned_slices is not None:
                    sl = self._owned_slices.get(id(p))
                    if sl is None:
                        continue
                    start, n = sl
                if sdt != torch.int8 and st["exp_avg_sq"].dtype != sdt:
                    raise ValueError("AdamW: exp_avg and exp_avg_sq of one dtype (or both in 8 bits)")
                self._check_narrow(p, st)
                _lib.require_match(st["step"], p, 1, (torch.float32,), "AdamW: step")
                esz = p.element_size()
                ssz = st["exp_avg"].element_size()
                if sdt == torch.int8:
                    if start % state8.BLOCK or ((start + n) % state8.BLOCK and start + n != p.numel()):
                        raise ValueError("AdamW: a slice of 8-bit moments starts and ends at multiples of "
                                         f"{state8.BLOCK} elements (got {start}, {n} of {p.numel()})")
                    sc = 4 * (start // state8.BLOCK)
                    descs.append(_lib.Adamw8Tensor(
                        p.data_ptr() + start * esz,
                        (rem.data_ptr() + start * 2) if rem is not None else None,
                        None,
                        st["exp_avg"].data_ptr() + start,
                        st["exp_avg_sq"].data_ptr() + start,
                        st["exp_avg_scale"].data_ptr() + sc,
                        st["exp_avg_sq_scale"].data_ptr() + sc,
                        (shadow.data_ptr() + start * 4) if shadow is not None else None,
                        n, start, gi, 0, st["step"].data_ptr()))
                else:
                    for k in ("exp_avg", "exp_avg_sq"):
                        _lib.require_match(st[k], p, p.numel(), (sdt,), f"AdamW: {k}")
                    descs.append(_lib.AdamwTensor(
                        p.data_ptr() + start * esz,
                        (rem.data_ptr() + start * 2) if rem is not None else None,
                        None,
                        st["exp_avg"].data_ptr() + start * ssz,
                        st["exp_avg_sq"].data_ptr() + start * ssz,
                        (shadow.data_ptr() + start * 4) if shadow is not None else None,
                        n, gi, 0, st["step"].data_ptr()))
                owners.append((p, start * esz))
                if shadow is not None:
                    ema_idx.add(self._ema._index[id(p)])
            if not descs:
                continue
            eight = sdt == torch.int8
            arr = ((_lib.Adamw8Tensor if eight else _lib.AdamwTensor) * len(descs))(*descs)
            words = np.frombuffer(arr, dtype=np.uint64).reshape(len(descs), _DESC8_WORDS if eight else _DESC_WORDS)
            refresh.append((words[:, _GRAD8_WORD if eight else _GRAD_WORD], np.array([pos[id(p)] for p, _ in owners]),
                            np.array([off for _, off in owners], dtype=np.uint64)))
            launches.append((arr, len(descs), _lib.dtype_code(pdt), None if eight else _lib.dtype_code(sdt), dev))
        by_group = {}
        for gi, p in zip(gis, ps):
            by_group.setdefault(gi, []).append(id(p))
        return {"key": key, "ema": self._ema, "owned": self._owned_slices, "state": self.state,
                "keep": ps, "launches": launches, "refresh": refresh, "groups": by_group,
                "ema_idx": frozenset(ema_idx)}

    def _groups(self, steps_of, grad_scale):
        """Group table of the pass with wide moments; a group that does not step keeps a row of zeros."""
        tab = (_lib.AdamwGroup * max(1, len(self.param_groups)))()
        for gi, group in enumerate(self.param_groups):
            if gi not in steps_of:
                continue
            b1, b2 = group["betas"]
            lr, wd = float(group["lr"]), float(group["weight_decay"])
            # torch's fused kernel multiplies fp32(lr) * fp32(weight_decay)
            lr_wd = float(C.c_float(float(C.c_float(lr).value) * float(C.c_float(wd).value)).value)
            tab[gi] = _lib.AdamwGroup(lr, float(b1), float(b2), float(group["eps"]), wd, lr_wd, float(steps_of[gi]),
                                      int(bool(self.cautious_wd)), grad_scale)
        return tab

    def _groups8(self, steps_of, grad_scale):
        """Group table of the 8-bit pass; a group that does not step gets a neutral row."""
        tab = (_lib.Adamw8Group * max(1, len(self.param_groups)))()
        for gi, group in enumerate(self.param_groups):
            if gi not in steps_of:
                tab[gi].step = 1.0
                continue
            b1, b2 = group["betas"]
            tab[gi] = _lib.Adamw8Group(float(group["lr"]), float(b1), float(b2), float(group["eps"]),
                                       float(group["weight_decay"]), float(steps_of[gi]), grad_scale,
                                       int(bool(self.cautious_wd)))
        return tab

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        lib = _lib.load()
        ps, gs_, gis = [], [], []
        for gi, group in enumerate(self.param_groups):
            if gi >= MAX_GROUPS:
                raise ValueError("at most 8 param groups")
            for p in group["params"]:
                g = p.grad
                if g is not None:
                    if g.dtype != p.dtype or not g.is_contiguous():
                        raise ValueError("AdamW needs contiguous params and grads of the param dtype")
                    ps.append(p)
                    gs_.append(g)
                    gis.append(gi)
        if self.state_dtype == torch.int8:
            for gi in set(gis):
                self._check_8bit_group(self.param_groups[gi])
        # The launch descriptors depend only on which parameters step, where
        # their storage and state live, the EMA folding and the shard: cached
        # across steps; the gradient pointers are written into them each step.
        key = (tuple(gis), tuple(map(id, ps)), tuple([p.data_ptr() for p in ps]), len(self.state))
        plan = self._plan
        if (plan is None or plan["key"] != key or plan["ema"] is not self._ema or plan["owned"] is not
                self._owned_slices or plan["state"] is not self.state):
            plan = self._plan = self._build_plan(ps, gis, key)
        gptr = np.fromiter((g.data_ptr() for g in gs_), dtype=np.uint64, count=len(gs_))
        for words, where, offs in plan["refresh"]:
            words[:] = gptr[where] + offs
        steps_of = {gi: self._steps.get(ids[0], 0) + 1 for gi, ids in plan["groups"].items()}
        gsc = self._grad_scale.data_ptr() if self._grad_scale is not None else None
        groups = groups8 = None
        ngroups = len(self.param_groups)
        for arr, n, pdt, sdt, dev in plan["launches"]:
            with _lib.on_device(dev):
                if sdt is None:
                    if groups8 is None:
                        groups8 = self._groups8(steps_of, gsc)
                    rc = lib.b2o_adamw8_step(arr, n, groups8, ngroups, pdt, self._ema_weight, _lib.stream_ptr(dev))
                    _lib.check(rc, "adamw8_step")
                else:
                    if groups is None:
                        groups = self._groups(steps_of, gsc)
                    rc = lib.b2o_adamw_step(arr, n, groups, ngroups, pdt, sdt, self._ema_weight, _lib.stream_ptr(dev))
                    _lib.check(rc, "adamw_step")
        for gi, ids in plan["groups"].items():  # a refused call leaves them
            self._steps.update(dict.fromkeys(ids, steps_of[gi]))
        if self._ema is not None and plan["ema_idx"]:
            self._ema._folded |= plan["ema_idx"]
        self._grad_scale = None
        return loss

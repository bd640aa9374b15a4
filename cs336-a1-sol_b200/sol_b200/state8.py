"""Optimizer states in 8 bits: conversion to and from fp32 / bf16 tensors.

A state is cut into blocks of 128 consecutive elements of the flattened tensor
(the last may be shorter), each with one fp32 scale s. Kinds:

  "signed" (first moments, momentum): int8 codes, s = max |x|,
           q = sgn(x) floor(127 sqrt(|x| / s) + 1/2), value s q |q| / 127^2
  "root"   (second moments, x >= 0): uint8 codes, s = max sqrt(x),
           q = floor(255 sqrt(sqrt(x) / s) + 1/2), at least 1 where x > 0, value (s (q / 255)^2)^2
  "pair"   (bf16 master weights): bf16 weight and bf16 remainder, value their sum

In an optimizer's step the 1/2 is an offset that runs evenly over [0, 1) with
the element and the step (include/b2o.h), so that changes below a code step are
kept on average. A block with a value that is not finite ("root": or negative) reads back as
NaN. The reference keeps every state in the parameter dtype
(transformer_lm/sol_modules.py:384-398,468-476); this is the engine's own form,
used by ``AdamW(state_dtype=torch.int8)`` and ``NorMuonGNS(momentum_dtype=torch.int8)``.

Every call takes a list and converts all of it in one kernel launch per 96
tensors of a device, on that device's current stream.
"""
from __future__ import annotations

import torch

from . import _lib

BLOCK = 128
_KINDS = {"signed": 0, "root": 1, "pair": 2}
_CODE_DTYPE = {"signed": torch.int8, "root": torch.uint8, "pair": torch.bfloat16}


def blocks(numel: int) -> int:
    """Scales of a tensor of ``numel`` elements."""
    return -(-numel // BLOCK)


def _kind(kind) -> int:
    if kind not in _KINDS:
        raise ValueError(f"state kind must be 'signed', 'root' or 'pair' (got {kind!r})")
    return _KINDS[kind]


def _check_value(t, what):
    _lib.require_cuda(t, what)
    if t.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"{what}: values are float32 or bfloat16 (got {t.dtype})")
    if not t.is_contiguous():
        raise ValueError(f"{what}: contiguous tensors only")


def _check_codes(codes, scales, kind, what):
    for t in (codes, scales):
        _lib.require_cuda(t, what)
        if not t.is_contiguous() or t.device != codes.device:
            raise ValueError(f"{what}: contiguous codes and scales on one device")
    n = codes.numel()
    want = (torch.bfloat16, n) if kind == "pair" else (torch.float32, blocks(n))
    if codes.dtype != _CODE_DTYPE[kind] or (scales.dtype, scales.numel()) != want:
        raise ValueError(f"{what}: a {kind!r} state of {n} elements has {_CODE_DTYPE[kind]} codes and "
                         f"{want[1]} {want[0]} scales (got {codes.dtype}, {scales.numel()} {scales.dtype})")


def _launch(fn, what, rows):
    """rows: (device, value, codes, scales, kind code); one call per device."""
    by = {}
    for dev, value, codes, scales, kind in rows:
        by.setdefault(dev, []).append((value.data_ptr(), codes.data_ptr(), scales.data_ptr(), value.numel(), kind,
                                       _lib.dtype_code(value.dtype)))
    for dev, descs in by.items():
        arr = (_lib.StateTensor * len(descs))(*descs)
        with _lib.on_device(dev):
            _lib.check(fn(arr, len(descs), _lib.stream_ptr(dev)), what)


@torch.no_grad()
def encode(items):
    """[(tensor, kind), ...] -> [(codes, scales), ...] ("pair": (bf16 weight, bf16
    remainder)). ``tensor``: contiguous fp32 or bf16 CUDA tensor; codes keep its shape."""
    out, rows = [], []
    for value, kind in items:
        code = _kind(kind)
        _check_value(value, "state8.encode")
        codes = torch.empty_like(value, dtype=_CODE_DTYPE[kind])
        if kind == "pair":
            scales = torch.empty_like(codes)
        else:
            scales = torch.empty(blocks(value.numel()), dtype=torch.float32, device=value.device)
        out.append((codes, scales))
        if value.numel():
            rows.append((value.device, value, codes, scales, code))
    _launch(_lib.load().b2o_state_encode, "state_encode", rows)
    return out


@torch.no_grad()
def decode(items, dtype=torch.float32, out=None):
    """[(codes, scales, kind), ...] -> values, in the shape of the codes.

    ``dtype``: torch.float32 or torch.bfloat16 (nearest), one for all or a list.
    ``out``: contiguous tensors to write instead of new ones (their dtype counts)."""
    items = list(items)
    if out is not None and len(out) != len(items):
        raise ValueError(f"state8.decode: {len(items)} states and {len(out)} outputs")
    if isinstance(dtype, (list, tuple)) and len(dtype) != len(items):
        raise ValueError(f"state8.decode: {len(items)} states and {len(dtype)} dtypes")
    values, rows = [], []
    for i, (codes, scales, kind) in enumerate(items):
        code = _kind(kind)
        _check_codes(codes, scales, kind, "state8.decode")
        if out is not None:
            value = out[i]
        else:
            value = torch.empty_like(codes, dtype=dtype[i] if isinstance(dtype, (list, tuple)) else dtype)
        _check_value(value, "state8.decode")
        if value.numel() != codes.numel() or value.device != codes.device:
            raise ValueError("state8.decode: an output has its codes' size and device")
        values.append(value)
        if value.numel():
            rows.append((value.device, value, codes, scales, code))
    _launch(_lib.load().b2o_state_decode, "state_decode", rows)
    return values

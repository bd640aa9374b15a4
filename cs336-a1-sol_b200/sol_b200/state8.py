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

import ctypes as C
from array import array

import torch

from . import _lib

BLOCK = 128
_WORDS = C.sizeof(_lib.StateTensor) // 8
_VALUE_CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
_KINDS = {"signed": 0, "root": 1, "pair": 2}
_CODE_DTYPE = {"signed": torch.int8, "root": torch.uint8, "pair": torch.bfloat16}


def blocks(numel: int) -> int:
    """Scales of a tensor of ``numel`` elements."""
    return -(-numel // BLOCK)


def _kind(kind) -> int:
    try:
        return _KINDS[kind]
    except (KeyError, TypeError):
        raise ValueError(f"state kind must be 'signed', 'root' or 'pair' (got {kind!r})") from None


def _value_code(t, what) -> int:
    """Checks a tensor of values; its dtype code."""
    if not t.is_cuda:
        _lib.require_cuda(t, what)
    code = _VALUE_CODE.get(t.dtype)
    if code is None:
        raise TypeError(f"{what}: values are float32 or bfloat16 (got {t.dtype})")
    if not t.is_contiguous():
        raise ValueError(f"{what}: contiguous tensors only")
    return code


def check_sizes(n, codes, scales, kind, what):
    """Refuses codes and scales that are not those of a state of n elements: their
    types and numbers, on whatever device."""
    if scales is None:
        raise ValueError(f"{what}: a {kind!r} state without scales")
    want = (torch.bfloat16, n) if kind == "pair" else (torch.float32, blocks(n))
    if (codes.dtype, codes.numel(), scales.dtype, scales.numel()) != (_CODE_DTYPE[kind], n, *want):
        raise ValueError(f"{what}: a {kind!r} state of {n} elements has {n} {_CODE_DTYPE[kind]} codes and "
                         f"{want[1]} {want[0]} scales (got {codes.numel()} {codes.dtype}, {scales.numel()} {scales.dtype})")


def _check_codes(codes, scales, kind, n, what):
    pair = kind == "pair"
    if (codes.dtype is _CODE_DTYPE[kind] and scales.dtype is (torch.bfloat16 if pair else torch.float32) and
            scales.numel() == (n if pair else (n + BLOCK - 1) // BLOCK) and codes.is_cuda and
            codes.get_device() == scales.get_device() and codes.is_contiguous() and scales.is_contiguous()):
        return
    _lib.require_cuda(codes, what)
    _lib.require_cuda(scales, what)
    if not (codes.is_contiguous() and scales.is_contiguous() and codes.get_device() == scales.get_device()):
        raise ValueError(f"{what}: contiguous codes and scales on one device")
    check_sizes(n, codes, scales, kind, what)


def check_state(p, codes, scales, kind, what):
    """Refuses a state that does not belong to parameter p (a loaded one may not)."""
    if codes.numel() != p.numel() or codes.get_device() != p.get_device():
        raise ValueError(f"{what}: {codes.numel()} codes for a parameter of {p.numel()} elements, or on another device")
    if scales is None:
        raise ValueError(f"{what}: a {kind!r} state without scales")
    _check_codes(codes, scales, kind, p.numel(), what)


class Rows:
    """Descriptors of one call (b2o_state_tensor as 64-bit words), by device.
    ``extend(index)`` gives the function that appends value pointer, codes
    pointer, scales pointer, numel and kind | value code << 32."""
    __slots__ = ("by",)

    def __init__(self):
        self.by = {}

    def extend(self, index):
        words = self.by.get(index)
        if words is None:
            words = self.by[index] = array("Q")
        return words.extend

    def launch(self, fn, what):
        for index, words in self.by.items():
            n = len(words) // _WORDS
            if not n:
                continue
            dev = torch.device("cuda", index)
            with _lib.on_device(dev):
                _lib.check(fn((_lib.StateTensor * n).from_buffer(words), n, _lib.stream_ptr(dev)), what)


@torch.no_grad()
def encode(items):
    """[(tensor, kind), ...] -> [(codes, scales), ...] ("pair": (bf16 weight, bf16
    remainder)). ``tensor``: contiguous fp32 or bf16 CUDA tensor; codes keep its shape."""
    out, rows, last, extend = [], Rows(), None, None
    empty, empty_like, f32 = torch.empty, torch.empty_like, torch.float32
    for value, kind in items:
        code = _kind(kind)
        value_code = _value_code(value, "state8.encode")
        n, index = value.numel(), value.get_device()
        codes = empty_like(value, dtype=_CODE_DTYPE[kind])
        scales = empty_like(codes) if kind == "pair" else empty((n + BLOCK - 1) // BLOCK, dtype=f32, device=value.device)
        out.append((codes, scales))
        if n:
            if index != last:
                last, extend = index, rows.extend(index)
            extend((value.data_ptr(), codes.data_ptr(), scales.data_ptr(), n, code | value_code << 32))
    rows.launch(_lib.load().b2o_state_encode, "state_encode")
    return out


@torch.no_grad()
def decode(items, dtype=torch.float32, out=None):
    """[(codes, scales, kind), ...] -> values, in the shape of the codes.

    ``dtype``: torch.float32 or torch.bfloat16 (nearest), one for all or a list.
    ``out``: contiguous tensors to write instead of new ones (their dtype counts);
    they may not overlap."""
    items = list(items)
    if out is not None:
        if len(out) != len(items):
            raise ValueError(f"state8.decode: {len(items)} states and {len(out)} outputs")
        at = [t.data_ptr() for t in out if t.numel()]
        if len(set(at)) != len(at):
            raise ValueError("state8.decode: an output appears twice")
    many = isinstance(dtype, (list, tuple))
    if many and len(dtype) != len(items):
        raise ValueError(f"state8.decode: {len(items)} states and {len(dtype)} dtypes")
    values, rows, last, extend, empty_like = [], Rows(), None, None, torch.empty_like
    for i, (codes, scales, kind) in enumerate(items):
        code = _kind(kind)
        n, index = codes.numel(), codes.get_device()
        _check_codes(codes, scales, kind, n, "state8.decode")
        if out is not None:
            value = out[i]
            value_code = _value_code(value, "state8.decode")
            if value.numel() != n or value.get_device() != index:
                raise ValueError("state8.decode: an output has its codes' size and device")
        else:
            dt = dtype[i] if many else dtype
            value_code = _VALUE_CODE.get(dt)
            if value_code is None:
                raise TypeError(f"state8.decode: values are float32 or bfloat16 (got {dt})")
            value = empty_like(codes, dtype=dt)
        values.append(value)
        if n:
            if index != last:
                last, extend = index, rows.extend(index)
            extend((value.data_ptr(), codes.data_ptr(), scales.data_ptr(), n, code | value_code << 32))
    rows.launch(_lib.load().b2o_state_decode, "state_decode")
    return values

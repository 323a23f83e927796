"""Rotary positions and attention over an int8 paged key / value cache (acfun_rope, acfun_kv8_*).

Activations are torch tensors or numpy arrays [tokens, heads, dim] whose last dimension is
contiguous (fp32, fp16 or bf16; numpy has no bf16); the cache is a set of CUDA tensors.  Calls
on device tensors are stream-ordered on the library's stream, as everywhere in this package.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import AcfunError, check, lib

_TYPES = {"float32": 0, "float16": 1, "bfloat16": 2, "int32": 10, "int8": 11}
_F32, _I32, _I8 = 0, 10, 11
_codes = {}  # by dtype object: these calls cost a few microseconds, and naming a dtype is one of them


def _code(dt):
    code = _codes.get(dt)
    if code is None:
        code = _codes[dt] = _TYPES.get(str(dt).replace("torch.", ""), -1)
    return code


def _dtype_code(dt):
    code = _code(dt)
    if not 0 <= code <= 2:
        raise TypeError(f"dtype {dt} is not float32, float16 or bfloat16")
    return code


_calls = {}  # the library's functions by name, bound at their first use


def _fn(name):
    f = _calls.get(name)
    if f is None:
        f = _calls[name] = getattr(lib(), name)
    return f


class _Cache(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("pages", C.c_int), ("heads", C.c_int), ("page", C.c_int), ("dim", C.c_int)]


class _Batch(C.Structure):
    _fields_ = [("table", C.c_void_p), ("start", C.c_void_p), ("length", C.c_void_p), ("seqs", C.c_int),
                ("table_cols", C.c_int), ("tokens", C.c_int), ("max_new", C.c_int), ("max_len", C.c_int)]


class _Rope(C.Structure):
    _fields_ = [("freq", C.c_void_p), ("rot", C.c_int), ("interleaved", C.c_int), ("amplitude", C.c_float)]


def _address(x):
    return x.ctypes.data if isinstance(x, np.ndarray) else x.data_ptr()


def _flat(x, code, what):
    """The address of a contiguous array of the given element type."""
    if not (x.flags["C_CONTIGUOUS"] if isinstance(x, np.ndarray) else x.is_contiguous()) or _code(x.dtype) != code:
        raise ValueError(f"{what} must be contiguous {[k for k, v in _TYPES.items() if v == code][0]}")
    return _address(x)


_INT = 0x7fffffff


def _int(x, what):
    """x as a C int; ctypes would cut it to its low 32 bits."""
    x = int(x)
    if not -_INT <= x <= _INT:
        raise ValueError(f"{what} {x} does not fit 32 bits")
    return x


def _rows(x, what):
    """(address, dtype code, shape, token stride, head stride) of [tokens, heads, dim]; strides in
    elements."""
    shape = x.shape
    if len(shape) != 3:
        raise ValueError(f"{what} must be [tokens, heads, dim], got {tuple(shape)}")
    if shape[0] > _INT:
        raise ValueError(f"{what}: {shape[0]} tokens do not fit 32 bits")
    if isinstance(x, np.ndarray):
        if any(s % x.itemsize for s in x.strides):
            raise ValueError(f"{what}: strides {x.strides} are not whole elements of {x.itemsize} bytes")
        t, h, d = (s // x.itemsize for s in x.strides)
        at = x.ctypes.data
    else:
        t, h, d = x.stride()
        at = x.data_ptr()
    if d != 1 and shape[2] != 1:
        raise ValueError(f"{what}: the last dimension must be contiguous")
    return at, _dtype_code(x.dtype), shape, t, h


_empty_like = None  # torch's, once a torch tensor has come by


def _out(out, x, shape, code, what):
    """(out, address, token stride, head stride) of an output like x, made when it is None."""
    if out is None and not isinstance(x, np.ndarray):
        global _empty_like
        if _empty_like is None:
            from torch import empty_like as _empty_like
        out = _empty_like(x)
        t, h, d = out.stride()
        if d == 1 or shape[2] == 1:
            return out, out.data_ptr(), t, h
        out = out.contiguous()  # x's dimensions overlap or repeat
    elif out is None:
        out = np.empty(shape, x.dtype)
    at, out_code, out_shape, t, h = _rows(out, "out")
    if out_shape != shape or out_code != code:
        raise ValueError(f"out must have {what}'s shape and dtype")
    return out, at, t, h


def _done(code):
    if code:
        check()
        raise AcfunError(f"acfun error {code}")


class Rope:
    """Rotary positions: pair i of a head's first 2 * len(freq) elements turns by position *
    freq[i]; freq is fp32 and is kept by reference.  See rope_frequencies()."""

    def __init__(self, freq, interleaved=False, amplitude=1.0):
        if freq.ndim != 1:
            raise ValueError("freq must have one dimension")
        self.freq = freq
        self.c = _Rope(_flat(freq, _F32, "freq"), 2 * freq.shape[0], int(bool(interleaved)), float(amplitude))
        self.ref = C.byref(self.c)


def rope_frequencies(rot, base=10000.0, scaling=None, factor=1.0, trained=0, fast=32.0, slow=1.0):
    """(freq, amplitude): numpy fp32 [rot / 2] and a float.  scaling: None; "linear" (positions
    divided by factor); "base" (base enlarged so that the lowest frequency is divided by factor);
    "by_parts", "by_whole_parts" or "by_turns" (frequencies kept, divided or mixed by how often a pair
    turns within the `trained` length: above `fast` turns, below `slow`, between; mixed linearly in the
    pair's index, in it between ends rounded outward to whole pairs, as checkpoints of this scaling
    commonly have it, or in the turns)."""
    kinds = {None: 0, "linear": 1, "base": 2, "by_parts": 3, "by_turns": 4, "by_whole_parts": 5}
    if scaling not in kinds:
        raise ValueError(f"scaling {scaling!r} is not one of {sorted(k for k in kinds if k)}")
    if _int(rot, "rot") <= 0:
        raise ValueError("rot must be positive")
    freq = np.empty(rot // 2, np.float32)
    amp = C.c_float()
    _done(_fn("acfun_rope_frequencies")(rot, base, kinds[scaling], factor, trained, fast, slow, freq.ctypes.data,
                                       C.byref(amp)))
    return freq, amp.value


def rope(x, positions, spec: Rope, out=None):
    """x [tokens, heads, dim] at int32 positions [tokens]; out may be x."""
    at, code, shape, t, h = _rows(x, "x")
    tokens, heads, dim = shape
    if positions.shape != (tokens,):
        raise ValueError("positions must be [tokens]")
    out, out_at, ot, oh = _out(out, x, shape, code, "x")
    err = _fn("acfun_rope")(at, out_at, code, tokens, heads, dim, t, h, ot, oh, _flat(positions, _I32, "positions"), spec.ref)
    if err:
        _done(err)
    return out


class KvBatch:
    """Sequences of one step: table int32 [seqs, columns] of page numbers, start int32 [seqs + 1]
    (offsets of the sequences' new tokens in the packed activations), length int32 [seqs] (tokens
    in the cache, the new ones last), and on the host the number of packed tokens and bounds on
    any sequence's new tokens and length.  The arrays are kept by reference and read when a call's
    kernels run."""

    def __init__(self, table, start, length, tokens, max_new, max_len):
        if table.ndim != 2 or length.shape != (table.shape[0],) or start.shape != (table.shape[0] + 1,):
            raise ValueError("table must be [seqs, columns], start [seqs + 1] and length [seqs]")
        self.arrays = (table, start, length)
        self.likes = {}
        self.tokens = _int(tokens, "tokens")
        self.c = _Batch(_flat(table, _I32, "table"), _flat(start, _I32, "start"),
                        _flat(length, _I32, "length"), table.shape[0], table.shape[1], self.tokens,
                        _int(max_new, "max_new"), _int(max_len, "max_len"))
        self.ref = C.byref(self.c)


class KvCache8:
    """Keys and values as int8 codes [pages, heads, page, dim] with fp32 scales [pages, heads] (CUDA
    tensors, kept by reference)."""

    def __init__(self, k, v, k_scale, v_scale):
        if k.ndim != 4 or v.shape != k.shape or k_scale.shape != k.shape[:2] or v_scale.shape != k.shape[:2]:
            raise ValueError("codes must be [pages, heads, page, dim], scales [pages, heads]")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.heads, self.page, self.dim = k.shape
        self.c = _Cache(_flat(k, _I8, "k"), _flat(v, _I8, "v"), _flat(k_scale, _F32, "k_scale"),
                        _flat(v_scale, _F32, "v_scale"), *k.shape)
        self.ref = C.byref(self.c)

    @classmethod
    def empty(cls, pages, heads, dim, page=64, device="cuda"):
        """A cache of `pages` unwritten pages."""
        import torch
        codes = [torch.zeros((pages, heads, page, dim), dtype=torch.int8, device=device) for _ in range(2)]
        scales = [torch.zeros((pages, heads), dtype=torch.float32, device=device) for _ in range(2)]
        return cls(*codes, *scales)

    def _new(self, x, batch, what):
        rows = _rows(x, what)
        if rows[2] != (batch.tokens, self.heads, self.dim):
            raise ValueError(f"{what} must be [{batch.tokens}, {self.heads}, {self.dim}], got {tuple(rows[2])}")
        return rows

    def append(self, k, v, batch: KvBatch, rope: Rope | None = None):
        """Quantise the batch's new keys (rotated by their position in the sequence when rope is
        given) and values into their pages."""
        k_at, code, _, kt, kh = self._new(k, batch, "k")
        v_at, v_code, _, vt, vh = self._new(v, batch, "v")
        if code != v_code:
            raise ValueError("k and v must have one dtype")
        err = _fn("acfun_kv8_append")(self.ref, batch.ref, k_at, v_at, code, kt, kh, vt, vh,
                                      rope.ref if rope is not None else None)
        if err:
            _done(err)

    def read(self, batch: KvBatch, dtype):
        """(k, v) [tokens, heads, dim]: the last start[i + 1] - start[i] tokens of each sequence."""
        code = _dtype_code(dtype)
        key = dtype, self.heads, self.dim, self.k.device
        like = batch.likes.get(key)
        if like is None:  # one element that has the outputs' shape: making them like it is the shortest call
            like = batch.likes[key] = self.k.new_empty(1, dtype=dtype).expand(batch.tokens, self.heads, self.dim)
        global _empty_like
        if _empty_like is None:
            from torch import empty_like as _empty_like
        k, v = _empty_like(like), _empty_like(like)
        err = _fn("acfun_kv8_read")(self.ref, batch.ref, k.data_ptr(), v.data_ptr(), code)
        if err:
            _done(err)
        return k, v

    def attention(self, q, batch: KvBatch, scale=None, causal=True, window=0, out=None, lse=None):
        """softmax(scale * q k^T) v for q [tokens, q_heads, dim]; scale defaults to dim ** -0.5.  lse
        (fp32 [tokens, q_heads]) receives the logarithm of the softmax denominators."""
        at, code, shape, qt, qh = _rows(q, "q")
        if shape[0] != batch.tokens or shape[2] != self.dim:
            raise ValueError(f"q must be [{batch.tokens}, q_heads, {self.dim}], got {tuple(shape)}")
        if lse is not None and tuple(lse.shape) != tuple(shape[:2]):
            raise ValueError("lse must be [tokens, q_heads]")
        if window and not 0 < window <= _INT:  # beyond: no limit, as the longest
            window = _INT if window > 0 else -1
        out, out_at, ot, oh = _out(out, q, shape, code, "q")
        err = _fn("acfun_kv8_attention")(self.ref, batch.ref, at, out_at, code, shape[1], qt, qh, ot, oh,
                                         self.dim ** -0.5 if scale is None else scale, int(bool(causal)), window,
                                         _flat(lse, _F32, "lse") if lse is not None else None)
        if err:
            _done(err)
        return out

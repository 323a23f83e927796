"""CPU: refusals of the int8 cache's functions (argument checks come before any GPU work) and the
rotary frequencies."""
import ctypes as C
import math

import numpy as np
import pytest

import acfun_b200 as acf
from acfun_b200 import kv8


def freqs(rot, base=10000.0):
    return np.array([base ** (-2 * i / rot) for i in range(rot // 2)])


def test_frequencies():
    f, a = acf.rope_frequencies(64, 5e5)
    assert f.dtype == np.float32 and a == 1.0 and np.allclose(f, freqs(64, 5e5), rtol=1e-7)
    f, a = acf.rope_frequencies(64, scaling="linear", factor=4.0)
    assert a == 1.0 and np.allclose(f, freqs(64) / 4, rtol=1e-7)
    f, a = acf.rope_frequencies(64, scaling="base", factor=4.0)
    assert f[0] == 1.0 and np.isclose(f[-1], freqs(64)[-1] / 4, rtol=1e-6)
    for kind in ("by_parts", "by_turns"):
        f, a = acf.rope_frequencies(128, scaling=kind, factor=8.0, trained=8192, fast=32.0, slow=1.0)
        plain = freqs(128)
        turns = 8192 * plain / (2 * math.pi)
        assert np.allclose(f[turns >= 32], plain[turns >= 32], rtol=1e-7)
        assert np.allclose(f[turns <= 1], plain[turns <= 1] / 8, rtol=1e-7)
        between = (turns < 32) & (turns > 1)
        assert between.sum() > 4 and (f[between] < plain[between]).all() and (f[between] > plain[between] / 8).all()
        keep = (f / plain - 1 / 8) / (1 - 1 / 8)
        if kind == "by_turns":
            assert np.isclose(a, 1.0) and np.allclose(keep[between], (turns[between] - 1) / 31, atol=1e-5)
        else:
            assert np.isclose(a, 0.1 * math.log(8) + 1)
            assert np.allclose(np.diff(keep[between]), np.diff(keep[between])[0], atol=1e-5)


@pytest.mark.parametrize("args", [dict(rot=0), dict(rot=7), dict(rot=64, base=1.0), dict(rot=64, base=float("nan")),
                                  dict(rot=64, scaling="linear", factor=0.5), dict(rot=2, scaling="base", factor=2.0),
                                  dict(rot=64, scaling="by_parts", factor=2.0, trained=0),
                                  dict(rot=64, scaling="by_turns", factor=2.0, trained=100, fast=1.0, slow=1.0),
                                  dict(rot=64, scaling="other")])
def test_frequencies_refuse(args):
    with pytest.raises((acf.AcfunError, ValueError)):
        acf.rope_frequencies(**args)
    assert acf.lib().acfun_last_error_code() == 0


def refused(code, words):
    L = acf.lib()
    assert code == 1 and L.acfun_last_error_code() == 1
    msg = L.acfun_last_error().decode()
    L.acfun_clear_error()
    assert words in msg, msg


def rope_call(**kw):
    x, pos, f = np.zeros((2, 3, 64), np.float32), np.zeros(2, np.int32), np.ones(32, np.float32)
    a = dict(x=x.ctypes.data, y=x.ctypes.data, dtype=0, tokens=2, heads=3, dim=64, xt=192, xh=64, yt=192, yh=64,
             pos=pos.ctypes.data, spec=kv8._Rope(f.ctypes.data, 64, 0, 1.0))
    a.update(kw)
    spec = a.pop("spec")
    return acf.lib().acfun_rope(*a.values(), C.byref(spec) if spec is not None else None)


@pytest.mark.parametrize("kw,words", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(tokens=-1), "tokens"), (dict(heads=0), "heads"),
    (dict(dim=0), "dim"), (dict(x=None), "NULL"), (dict(pos=None), "NULL"), (dict(spec=None), "NULL"),
    (dict(spec=kv8._Rope(None, 64, 0, 1.0)), "freq"), (dict(spec=kv8._Rope(8, 66, 0, 1.0)), "rot"),
    (dict(spec=kv8._Rope(8, 31, 0, 1.0)), "rot"), (dict(xt=-1), "strides"), (dict(yt=100, xt=100), "overlap"),
    (dict(xt=200), "equal strides")])
def test_rope_refuses(kw, words):
    refused(rope_call(**kw), words)


def structs(**kw):
    """A cache and a batch whose addresses are never followed: every call here is refused first."""
    c = kv8._Cache(k=4096, v=4096, k_scale=4096, v_scale=4096, pages=4, heads=2, page=16, dim=64)
    b = kv8._Batch(table=4096, start=4096, length=4096, seqs=2, table_cols=4, tokens=3, max_new=2, max_len=60)
    for k, v in kw.items():
        setattr(c if hasattr(c, k) else b, k, v)
    return C.byref(c), C.byref(b)


def attention_call(cb=None, **kw):
    a = dict(q=4096, out=4096, dtype=1, q_heads=4, qt=256, qh=64, ot=256, oh=64, scale=0.125, causal=1, window=0, lse=None)
    a.update(kw)
    return acf.lib().acfun_kv8_attention(*(cb or structs()), *a.values())


CACHE = [(dict(k=None), "NULL"), (dict(v_scale=None), "NULL"), (dict(page=24), "page"), (dict(dim=96), "dim"),
         (dict(pages=0), "pages"), (dict(heads=0), "heads"), (dict(heads=5000), "heads"), (dict(k=4097), "aligned"),
         (dict(k_scale=4098), "aligned"), (dict(), "device memory")]


@pytest.mark.parametrize("kw,words", CACHE)
def test_cache_is_checked_by_every_call(kw, words):
    c, b = structs(**kw)
    L = acf.lib()
    refused(L.acfun_kv8_append(c, b, 4096, 4096, 1, 128, 64, 128, 64, None), words)
    refused(L.acfun_kv8_read(c, b, 4096, 4096, 1), words)
    refused(attention_call((c, b)), words)
    refused(L.acfun_kv8_read(None, b, 4096, 4096, 1), "NULL")


def test_dtypes_refused():
    c, b = structs()
    L = acf.lib()
    refused(L.acfun_kv8_append(c, b, 4096, 4096, 7, 128, 64, 128, 64, None), "dtype")
    refused(L.acfun_kv8_read(c, b, 4096, 4096, 3), "dtype")
    refused(attention_call(dtype=0), "dtype")

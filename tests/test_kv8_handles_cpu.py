"""CPU: what the Python handles of the int8 cache keep and pass on, with the library's calls replaced."""
import numpy as np
import pytest
import torch

import acfun_b200 as acf
from acfun_b200 import kv8


@pytest.fixture
def calls(monkeypatch):
    """Name -> arguments of the last call, which does nothing and succeeds."""
    seen = {}
    for name in ("acfun_rope", "acfun_kv8_append", "acfun_kv8_read", "acfun_kv8_attention"):
        monkeypatch.setitem(kv8._calls, name, lambda *a, name=name: seen.update({name: a}) and 0)
    return seen


def batch(tokens=3, max_new=3, max_len=9):
    return acf.KvBatch(np.zeros((1, 1), np.int32), np.array([0, tokens], np.int32), np.array([max_len], np.int32), tokens, max_new, max_len)


def test_one_batch_for_caches_on_two_devices(calls):
    """Index arrays may be host memory, so one batch can serve the layers of several devices: what is read
    is on the device of the cache it was read from."""
    b = batch()
    for _ in range(2):
        for device in ("cpu", "meta"):
            for heads, dim in ((2, 64), (2, 128)):
                cache = acf.KvCache8.empty(1, heads, dim, 16, device=device)
                for dtype in (torch.float16, torch.float32):
                    for x in cache.read(b, dtype):
                        assert x.device.type == device and x.dtype == dtype and x.shape == (3, heads, dim) and x.is_contiguous()


def test_byte_strides_that_are_not_whole_elements_are_refused(calls):
    """Rows of a record array whose records end in an odd byte: no stride in elements says where they are."""
    x = np.zeros(3, np.dtype([("x", np.float16, (2, 64)), ("flag", np.uint8)]))["x"]
    even = np.zeros(3, np.dtype([("x", np.float16, (2, 64)), ("flag", np.uint16)]))["x"]
    cache = acf.KvCache8.empty(1, 2, 64, 16, device="cpu")
    spec, pos, b = acf.Rope(np.ones(32, np.float32)), np.zeros(3, np.int32), batch()
    for call in (lambda v: acf.rope(v, pos, spec), lambda v: acf.rope(np.zeros((3, 2, 64), np.float16), pos, spec, out=v),
                 lambda v: cache.append(v, even, b), lambda v: cache.append(even, v, b), lambda v: cache.attention(v, b)):
        with pytest.raises(ValueError, match="stride"):
            call(x)
        call(even)
    assert calls["acfun_rope"][6] == 2 * 64 and calls["acfun_kv8_attention"][6] == 2 * 64 + 1


def test_sizes_past_32_bits_are_not_cut(calls):
    for sizes in (dict(tokens=2 ** 32 + 3), dict(max_new=2 ** 32 + 3), dict(max_len=2 ** 31), dict(max_len=-2 ** 32 + 9)):
        with pytest.raises(ValueError, match="32 bits"):
            acf.KvBatch(np.zeros((1, 1), np.int32), np.zeros(2, np.int32), np.zeros(1, np.int32), **dict(dict(tokens=3, max_new=3, max_len=9), **sizes))
    cache = acf.KvCache8.empty(1, 2, 64, 16, device="cpu")
    q = np.zeros((3, 2, 64), np.float16)
    for window, passed in ((0, 0), (5, 5), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 32 + 5, 2 ** 31 - 1), (2 ** 63, 2 ** 31 - 1), (-1, -1), (-2 ** 32 + 5, -1)):
        cache.attention(q, batch(), window=window)
        assert calls["acfun_kv8_attention"][12] == passed
    long = torch.zeros(1, dtype=torch.float16).expand(2 ** 32 + 1, 1, 8)
    with pytest.raises(ValueError, match="32 bits"):
        acf.rope(long, torch.zeros(1, dtype=torch.int32).expand(2 ** 32 + 1), acf.Rope(np.ones(4, np.float32)), out=long)
    with pytest.raises(ValueError, match="32 bits"):
        acf.rope_frequencies(2 ** 32 + 64)

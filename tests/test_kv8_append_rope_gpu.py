"""GPU: append with rotation where a page's cosines and sines fill much of the shared memory: wide
heads, long pages, and each such size as the first call of its kernel in a process."""
import os
import subprocess
import sys

import pytest
import torch

import kv8_plain as P

pytestmark = pytest.mark.gpu

# dtype, heads, dim, page, new, length, rot, interleaved, elements off a 16-byte boundary.  Cosines
# and sines take min(page, max_new) * rot * 4 bytes: some of these are just below 48 KiB, at it and above.
SIZES = [
    ("bf16", 2, 128, 128, [96], [96], 128, False, 0), ("f16", 1, 128, 128, [130, 7], [260, 9], 96, False, 0),
    ("f32", 1, 128, 128, [128], [200], 96, True, 0), ("bf16", 1, 256, 64, [48, 3], [50, 3], 256, True, 0),
    ("f16", 2, 256, 64, [64], [300], 192, False, 0), ("f32", 1, 256, 128, [48], [48], 256, False, 0),
    ("bf16", 1, 128, 128, [96], [97], 128, True, 1), ("f16", 3, 256, 128, [48], [48], 256, False, 1),
    ("f32", 1, 128, 128, [97], [97], 128, False, 1), ("bf16", 2, 256, 64, [70, 64], [71, 64], 192, False, 1)]
MORE = [
    ("bf16", 3, 128, 128, [95], [95], 128, False, 0), ("f16", 1, 128, 128, [97], [160], 128, True, 0),
    ("f32", 2, 128, 128, [300, 1], [300, 128], 128, False, 0), ("bf16", 1, 256, 128, [128, 47], [128, 200], 256, False, 0),
    ("f16", 1, 256, 128, [260], [261], 256, True, 0), ("f32", 1, 256, 16, [40], [70], 16, False, 0),
    ("f16", 9, 64, 128, [128], [128], 64, False, 0), ("bf16", 1, 128, 32, [33], [64], 112, False, 0)]


def check(acf, dtype, heads, dim, page, new, length, rot, inter, off):
    """An angle is computed once per run of a page's tokens and turned on by at most 127 products.  The
    start, the angle of one position and each complex product are within 3 units of 2^-23, so a
    rotated element is within 2 * 128 * 3 * 2^-23 of the pair's larger side and so of the page's largest;
    the scale is within that share of its value, and a code adds half a unit."""
    b = P.Batch(acf, new, length, page, seed=41)
    cache = P.random_cache(acf, b.pages, heads, dim, page, 42)
    cache.k_scale.fill_(1e-6)            # pages in use take the new tokens' scale
    g = torch.Generator(device="cuda").manual_seed(43)
    wide = torch.randn(b.tokens * 2 * heads * dim + 8, generator=g, device="cuda").to(P.DT[dtype])
    kv = wide[off:off + b.tokens * 2 * heads * dim].view(b.tokens, 2, heads, dim)
    freq = torch.from_numpy(acf.rope_frequencies(rot)[0]).cuda()
    cache.append(kv[:, 0], kv[:, 1], b.h, rope=acf.Rope(freq, inter, 1.1))
    acf.synchronize()
    share = 2 * 128 * 3 * 2.0 ** -23
    for i in range(len(new)):
        first = length[i] - new[i]
        rows = slice(b.start[i], b.start[i + 1])
        pos = torch.arange(first, length[i], device="cuda")
        want = P.rope64(kv[rows, 0].double(), pos, freq, 1.1, inter)
        got = b.whole(cache.k, cache.k_scale, i)[first:]
        for p in range(first // page, -(-length[i] // page)):
            t = slice(max(0, p * page - first), min(new[i], (p + 1) * page - first))
            top = want[t].abs().amax((0, 2))
            pid = int(b.table[i, p])
            assert ((cache.k_scale[pid].double() - top / 127).abs() <= top / 127 * (share + 2.0 ** -22)).all()
            assert ((got[t] - want[t]).abs().amax((0, 2)) <= top / 127 * 0.5 * (1 + 2 * share) + top * share).all()


@pytest.mark.parametrize("size", SIZES + MORE, ids=str)
def test_append_rotates_wide_heads(acf, size):
    check(acf, *size)


def test_each_size_as_the_first_call_of_its_kernel():
    """The sizes above are of ten different instances; a call of one must not need an earlier, larger one."""
    here = os.path.dirname(os.path.abspath(__file__))
    code = (f"import sys; sys.path[:0] = [{os.path.dirname(here)!r}, {here!r}]\n"
            "import acfun_b200 as acf, test_kv8_append_rope_gpu as t\n"
            "bad = []\n"
            "for s in t.SIZES:\n"
            "    try: t.check(acf, *s)\n"
            "    except acf.AcfunError as e: bad.append((s, str(e)))\n"
            "print(bad); sys.exit(bool(bad))\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout + r.stderr

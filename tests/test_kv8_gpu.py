"""GPU: rotary positions, the int8 paged cache and attention over it, against plain 64-bit
implementations (kv8_plain.py)."""
import numpy as np
import pytest
import torch

import kv8_plain as P

pytestmark = pytest.mark.gpu


def randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


# ------------------------------------------------------------------ rope
ROPE = [  # dtype, tokens, heads, dim, rot, interleaved, largest position
    ("bf16", 1, 1, 64, 64, False, 10), ("f16", 7, 5, 128, 32, True, 100000), ("f32", 33, 3, 80, 20, False, 4000),
    ("f32", 300, 9, 64, 64, True, 1 << 30), ("bf16", 2100, 2, 128, 128, False, 131072), ("f16", 5, 3, 6, 6, True, 50),
    ("f32", 4, 2, 7, 4, False, 9), ("bf16", 3, 70, 256, 0, False, 9), ("f16", 2500, 3, 96, 48, False, 70000),
    ("f32", 1300, 2, 72, 72, True, 70000), ("bf16", 9, 3, 192, 96, False, 5000), ("f16", 6, 2, 120, 104, True, 5000)]


def check_rope(got, x, pos, freq, amp, inter, dtype):
    want = P.rope64(x.double(), pos, freq, amp, inter)
    # cosine, sine and their product with amp within 4 units of 2^-23; then the sum and the rounding
    reach = P.rope64(x.double().abs(), torch.zeros_like(pos), freq, amp, inter).abs()
    r = 2 * len(freq)
    pair = reach.clone()
    i, j = (slice(0, r, 2), slice(1, r, 2)) if inter else (slice(0, r // 2), slice(r // 2, r))
    pair[..., i] = pair[..., j] = reach[..., i] + reach[..., j]
    tol = P.HALF_ULP[dtype] * want.abs() + P.SMALLEST[dtype] + 2.0 ** -20 * pair
    off = (got.double() - want).abs()
    assert (off <= tol).all(), float((off / tol).max())
    assert torch.equal(got[..., r:], x[..., r:])


@pytest.mark.parametrize("dtype,tokens,heads,dim,rot,inter,most", ROPE)
def test_rope(acf, dtype, tokens, heads, dim, rot, inter, most):
    x = randn(1, tokens, heads, dim).to(P.DT[dtype])
    pos = torch.randint(0, most, (tokens,), device="cuda", dtype=torch.int32)
    f, _ = acf.rope_frequencies(rot) if rot else (np.empty(0, np.float32), 1.0)
    freq = torch.from_numpy(f).cuda()
    got = acf.rope(x, pos, acf.Rope(freq, inter, 1.25))
    acf.synchronize()
    check_rope(got, x, pos, freq, 1.25, inter, dtype)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("shift", [0, 1])
def test_rope_strides_in_place_and_host(acf, inter, shift):
    freq = torch.from_numpy(acf.rope_frequencies(64)[0]).cuda()
    spec = acf.Rope(freq, inter)
    pos = torch.arange(11, device="cuda", dtype=torch.int32) * 1000
    wide = randn(2, 11 * 9 * 64 + 1).to(torch.bfloat16)[shift:shift + 11 * 8 * 64 + 0].view(11, 8, 64)
    part = wide[:, 2:5]                                  # a slice of a packed row, in place
    before = wide.clone()
    acf.rope(part, pos, spec, out=part)
    acf.synchronize()
    check_rope(part, before[:, 2:5], pos, freq, 1.0, inter, "bf16")
    assert torch.equal(wide[:, :2], before[:, :2]) and torch.equal(wide[:, 5:], before[:, 5:])
    by_head = before.permute(1, 0, 2)                    # heads outermost
    out = torch.empty((8, 11, 64), dtype=torch.bfloat16, device="cuda")
    acf.rope(before, pos, spec, out=out.permute(1, 0, 2))
    acf.synchronize()
    check_rope(out.permute(1, 0, 2), before, pos, freq, 1.0, inter, "bf16")
    assert by_head.shape == out.shape
    host = np.random.default_rng(0).standard_normal((11, 2, 64)).astype(np.float32)
    hspec = acf.Rope(freq.cpu().numpy(), inter)
    got = acf.rope(host, pos.cpu().numpy(), hspec)
    check_rope(torch.from_numpy(got), torch.from_numpy(host), pos.cpu(), freq.cpu(), 1.0, inter, "f32")


# ------------------------------------------------------------------ append and read
def codes32(x, scale):
    """The codes of x under one scale, in the documented 32-bit steps."""
    unit = np.float32(1) / np.float32(scale)
    return np.clip(np.rint((x.astype(np.float32) * unit).astype(np.float32)), -127, 127).astype(np.int8)


def append_plain(codes, scale, b, x):
    """Writes x (float32 [tokens, heads, dim] numpy) into numpy codes / scale as documented."""
    page = b.page
    tiny = np.float32(127.0 * 2.0 ** -60)
    for i in range(len(b.new)):
        first = b.length[i] - b.new[i]
        for g in range(first // page, -(-b.length[i] // page) if b.new[i] else 0):
            lo, hi = max(first - g * page, 0), min(b.length[i] - g * page, page)
            rows = x[b.start[i] + g * page + lo - first: b.start[i] + g * page + hi - first]
            pid = int(b.table[i, g])
            for h in range(x.shape[1]):
                v = rows[:, h].copy()
                v[np.isnan(v)] = 0
                fin = np.abs(v[np.isfinite(v)])
                s = np.float32(max(tiny, fin.max() if fin.size else tiny)) / np.float32(127)
                if lo > 0:
                    old = scale[pid, h]
                    if s > old:
                        f = np.float32(old) / np.float32(s)
                        codes[pid, h, :lo] = np.rint((codes[pid, h, :lo].astype(np.float32) * f).astype(np.float32))
                    else:
                        s = old
                with np.errstate(over="ignore", invalid="ignore"):
                    codes[pid, h, lo:hi] = codes32(v, s)
                scale[pid, h] = s


@pytest.mark.parametrize("dtype,heads,dim,page,new,length", [
    ("f32", 1, 64, 16, [1], [1]), ("bf16", 3, 128, 64, [1, 1, 1], [64, 65, 128]), ("f16", 2, 64, 32, [0, 5, 33], [7, 5, 90]),
    ("bf16", 5, 256, 128, [129, 0, 1], [129, 0, 128]), ("f32", 4, 128, 16, [50, 15, 17], [61, 31, 17]),
    ("f16", 2, 256, 16, [300], [301]), ("bf16", 7, 64, 128, [700, 3, 128], [700, 300, 256])])
def test_append_codes_and_scales_exactly(acf, dtype, heads, dim, page, new, length):
    b = P.Batch(acf, new, length, page, seed=3)
    cache = P.random_cache(acf, b.pages, heads, dim, page, 4)
    # packed as a projection leaves them; magnitudes over two decades so that page scales both grow and stay
    kv = randn(5, b.tokens, 2, heads, dim) * 10 ** (2 * torch.rand((b.tokens, 2, heads, 1), device="cuda") - 1)
    kv = kv.to(P.DT[dtype])
    want = [(cache.k.cpu().numpy(), cache.k_scale.cpu().numpy()), (cache.v.cpu().numpy(), cache.v_scale.cpu().numpy())]
    for w, (codes, scale) in enumerate(want):
        append_plain(codes, scale, b, kv[:, w].float().cpu().numpy())
    cache.append(kv[:, 0], kv[:, 1], b.h)
    acf.synchronize()
    for got, (codes, scale) in zip(((cache.k, cache.k_scale), (cache.v, cache.v_scale)), want):
        assert np.array_equal(got[1].cpu().numpy(), scale)
        assert np.array_equal(got[0].cpu().numpy(), codes)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_append_from_unaligned_rows(acf, dtype):
    """Keys and values one element off a 16-byte boundary, at odd strides; the cosines' path too."""
    b = P.Batch(acf, [20, 1, 7], [33, 1, 40], 16, seed=3)
    caches = [P.random_cache(acf, b.pages, 2, 64, 16, 4) for _ in range(2)]
    freq = torch.from_numpy(acf.rope_frequencies(32)[0]).cuda()
    for rope in (None, acf.Rope(freq), acf.Rope(freq, True)):
        wide = randn(5, b.tokens * 301 + 1).to(P.DT[dtype])
        kv = wide[1:].view(b.tokens, 301)[:, :256].unflatten(1, (2, 2, 64))
        caches[0].append(kv[:, 0], kv[:, 1], b.h, rope=rope)
        whole = kv.contiguous()
        caches[1].append(whole[:, 0], whole[:, 1], b.h, rope=rope)
        acf.synchronize()
        for x, y in zip(*((c.k, c.v, c.k_scale, c.v_scale) for c in caches)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("inter,rot", [(False, 64), (True, 64), (False, 16), (True, 32), (False, 0), (False, 48)])
def test_append_rotates_keys(acf, inter, rot):
    b = P.Batch(acf, [40, 1, 17], [100, 77, 17], 32, seed=6)
    cache = P.random_cache(acf, b.pages, 2, 64, 32, 7)
    cache.k_scale.fill_(1e-6)            # pages in use take the new tokens' scale
    k, v = randn(8, b.tokens, 2, 64).to(torch.bfloat16), randn(9, b.tokens, 2, 64).to(torch.bfloat16)
    freq = torch.from_numpy(acf.rope_frequencies(rot)[0] if rot else np.empty(0, np.float32)).cuda()
    cache.append(k, v, b.h, rope=acf.Rope(freq, inter, 1.1))
    acf.synchronize()
    for i in range(3):
        first = b.length[i] - b.new[i]
        rows = slice(b.start[i], b.start[i + 1])
        pos = torch.arange(first, b.length[i], device="cuda")
        want = P.rope64(k[rows].double(), pos, freq, 1.1, inter)
        got = b.whole(cache.k, cache.k_scale, i)[first:]
        for g in range(first // 32, -(-b.length[i] // 32)):
            t = slice(max(0, g * 32 - first), min(b.new[i], (g + 1) * 32 - first))
            top = want[t].abs().amax((0, 2))
            pid = int(b.table[i, g])
            assert (cache.k_scale[pid].double() - top / 127).abs().max() <= 1e-6 * top.max()
            # half a code, and the 32-bit rotation's own error
            assert ((got[t] - want[t]).abs().amax((0, 2)) <= top / 127 * (0.5 + 1e-3)).all()


def test_append_special_values(acf):
    b = P.Batch(acf, [20], [20], 16, seed=1)
    cache = P.random_cache(acf, b.pages, 2, 64, 16, 2)
    x = randn(3, 20, 2, 64)
    x[3, 0, 5], x[4, 0, 6], x[5, 0, 7] = float("inf"), float("-inf"), float("nan")
    x[16:, 1] = 0.0
    x[:16, 1] = 1e-30
    want = cache.k.cpu().numpy(), cache.k_scale.cpu().numpy()
    append_plain(*want, b, x.cpu().numpy())
    cache.append(x, x, b.h)
    acf.synchronize()
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        for pid, slots in zip(b.table[0, :2].tolist(), (16, 4)):   # the slots that were written
            assert np.array_equal(codes[pid, :, :slots].cpu().numpy(), want[0][pid, :, :slots])
            assert np.array_equal(scale[pid].cpu().numpy(), want[1][pid])
    k, v = cache.read(b.h, torch.float32)
    acf.synchronize()
    assert torch.isfinite(k).all() and (k[:, 1] == 0).all() and float(k[3, 0, 5]) == float(x[:16, 0][torch.isfinite(x[:16, 0])].abs().max())


def test_append_one_by_one_stays_within_the_last_scale(acf):
    """Codes moved to a growing scale again and again: each move rounds by at most half a code of the
    scale of its time, and all of those are at most the last scale."""
    page, n = 32, 50
    x = randn(11, n, 1, 64) * torch.linspace(0.1, 3, n, device="cuda")[:, None, None]
    cache = acf.KvCache8.empty(4, 1, 64, page)
    for t in range(n):
        b = P.Batch(acf, [1], [t + 1], page, spare_pages=0)
        b.table[0, : t // page + 1] = torch.arange(t // page + 1, dtype=torch.int32) + 1
        b.dev[0].copy_(b.table)
        cache.append(x[t:t + 1], x[t:t + 1], b.h)
    acf.synchronize()
    got = b.whole(cache.k, cache.k_scale, 0)
    moves = torch.tensor([page - t % page for t in range(n)], device="cuda").double()[:, None, None]
    last = cache.k_scale[1:3, 0].double().repeat_interleave(page)[:n, None, None]
    assert ((got - x.double()).abs() <= (moves + 1) * 0.5 * last * 1.001).all()
    assert torch.equal(cache.k, cache.v)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,dim,page", [(1, 64, 16), (5, 128, 64), (3, 256, 128)])
def test_read(acf, dtype, heads, dim, page):
    b = P.Batch(acf, [0, 1, 200, 37, 130], [300, 1, 200, 161, 258], page, seed=8)
    cache = P.random_cache(acf, b.pages, heads, dim, page, 9)
    k, v = cache.read(b.h, P.DT[dtype])
    acf.synchronize()
    for i in range(5):
        rows = slice(b.start[i], b.start[i + 1])
        for got, codes, scale in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
            want = b.whole(codes, scale, i)[b.length[i] - b.new[i]:].float().to(P.DT[dtype])  # one 32-bit rounding, then the type's
            assert torch.equal(got[rows], want)


def test_read_into_memory_that_is_only_16_byte_aligned_and_one_of_the_two(acf):
    b = P.Batch(acf, [37, 3], [100, 3], 32, seed=8)
    cache = P.random_cache(acf, b.pages, 2, 64, 32, 9)
    k, v = cache.read(b.h, torch.float16)
    out = torch.zeros(2 * k.numel() + 24, dtype=torch.float16, device="cuda")
    ko, vo = out[8:8 + k.numel()], out[16 + k.numel():16 + 2 * k.numel()]
    for kp, vp in ((ko.data_ptr(), vo.data_ptr()), (ko.data_ptr(), None), (None, vo.data_ptr())):
        out.zero_()
        assert acf.lib().acfun_kv8_read(cache.ref, b.h.ref, kp, vp, 1) == 0
        acf.synchronize()
        assert torch.equal(ko, k.flatten() if kp else torch.zeros_like(ko))
        assert torch.equal(vo, v.flatten() if vp else torch.zeros_like(vo))
        assert (out[:8] == 0).all() and (out[8 + k.numel():16 + k.numel()] == 0).all() and (out[16 + 2 * k.numel():] == 0).all()
    assert acf.lib().acfun_kv8_read(cache.ref, b.h.ref, ko.data_ptr() + 2, None, 1) == 1
    acf.lib().acfun_clear_error()


# ------------------------------------------------------------------ attention
ATTN = [  # dtype, q_heads, heads, dim, page, new, length, causal, window
    ("bf16", 1, 1, 64, 16, [1], [1], True, 0),
    ("f16", 8, 8, 64, 16, [1], [777], True, 0),
    ("bf16", 8, 2, 128, 64, [1, 1, 1, 1], [1, 64, 65, 3000], True, 0),
    ("f16", 3, 1, 128, 32, [1, 0, 2, 5], [31, 40, 2, 33], True, 0),
    ("bf16", 10, 2, 256, 128, [1, 4], [129, 700], True, 0),
    ("f16", 64, 4, 128, 16, [3, 1], [1000, 0], True, 0),
    ("bf16", 7, 7, 64, 32, [40, 7], [40, 400], False, 0),
    ("f16", 4, 2, 128, 64, [9, 100], [4, 120], True, 0),              # more new tokens than the cache holds: empty rows
    ("bf16", 4, 1, 64, 16, [1, 3, 50], [500, 260, 90], True, 1),
    ("f16", 6, 2, 128, 32, [1, 70], [2000, 300], True, 100),
    ("bf16", 8, 2, 128, 64, [300, 1, 129], [300, 513, 1000], True, 0),
    ("f16", 12, 4, 64, 128, [513], [513], True, 0),
    ("f16", 5, 1, 64, 32, [260, 77], [700, 77], True, 33),
    ("bf16", 16, 2, 128, 16, [150, 260], [1150, 261], False, 0),
    ("bf16", 2, 2, 256, 32, [200], [333], True, 0),
    ("f16", 2, 1, 128, 128, [1], [40001], True, 0),
    ("bf16", 48, 1, 64, 64, [30], [900], True, 500),
    ("f16", 130, 1, 128, 64, [3, 2], [200, 130], True, 0)]


@pytest.mark.parametrize("dtype,hq,heads,dim,page,new,length,causal,window", ATTN)
def test_attention(acf, dtype, hq, heads, dim, page, new, length, causal, window):
    b = P.Batch(acf, new, length, page, seed=10)
    cache = P.random_cache(acf, b.pages, heads, dim, page, 11)
    q = (randn(12, b.tokens, hq, dim) * 0.3).to(P.DT[dtype])
    lse = torch.full((b.tokens, hq), 7.0, device="cuda")
    got = cache.attention(q, b.h, causal=causal, window=window, lse=lse)
    acf.synchronize()
    P.check_attention(got, lse, P.attention64(cache, b, q, dim ** -0.5, causal, window), dtype)
    again = cache.attention(q, b.h, causal=causal, window=window)
    acf.synchronize()
    assert torch.equal(got, again)     # joined in a fixed order


# many rows per cache head: the key tiles are made before the kernel
MANY = [  # dtype, q_heads, heads, dim, page, new, length, causal, window, scale
    ("bf16", 48, 1, 128, 64, [130], [130], True, 0, None), ("f16", 48, 1, 64, 16, [131, 2], [700, 300], True, 0, None),
    ("bf16", 50, 1, 64, 32, [125], [1000], True, 77, -0.1), ("f16", 98, 2, 128, 128, [129, 0, 128], [129, 9, 500], False, 0, 0.2),
    ("f16", 48, 1, 128, 32, [140, 100], [100, 101], True, 0, -0.2), ("bf16", 16, 1, 128, 16, [400, 1], [1500, 3000], True, 0, None)]


@pytest.mark.parametrize("dtype,hq,heads,dim,page,new,length,causal,window,scale", MANY)
def test_attention_many_rows(acf, dtype, hq, heads, dim, page, new, length, causal, window, scale):
    b = P.Batch(acf, new, length, page, seed=20)
    cache = P.random_cache(acf, b.pages, heads, dim, page, 21)
    q = (randn(22, b.tokens, hq, dim) * 0.3).to(P.DT[dtype])
    lse = torch.full((b.tokens, hq), 7.0, device="cuda")
    got = cache.attention(q, b.h, scale=scale, causal=causal, window=window, lse=lse)
    acf.synchronize()
    P.check_attention(got, lse, P.attention64(cache, b, q, dim ** -0.5 if scale is None else scale, causal, window), dtype)


@pytest.mark.parametrize("new,length", [([1], [400]), ([5], [300]), ([300], [400])])
def test_attention_negative_scale(acf, new, length):
    b = P.Batch(acf, new, length, 32, seed=23)
    cache = P.random_cache(acf, b.pages, 2, 64, 32, 24)
    for dtype in ("f16", "bf16"):
        q = randn(25, b.tokens, 6, 64).to(P.DT[dtype])
        got = cache.attention(q, b.h, scale=-0.15)
        acf.synchronize()
        P.check_attention(got, None, P.attention64(cache, b, q, -0.15, True, 0), dtype)


@pytest.mark.parametrize("dtype,hq,heads,dim", [("bf16", 8, 2, 128), ("f16", 3, 3, 64), ("bf16", 40, 1, 64)])
def test_attention_decode_steps_beside_prompts(acf, dtype, hq, heads, dim):
    """One batch for both kernels: sequences with one new token, a few, none and many."""
    b = P.Batch(acf, [1, 200, 0, 8, 1, 9, 513, 33], [900, 200, 50, 77, 1, 2000, 600, 33], 64, seed=26)
    cache = P.random_cache(acf, b.pages, heads, dim, 64, 27)
    q = (randn(28, b.tokens, hq, dim) * 0.5).to(P.DT[dtype])
    lse = torch.full((b.tokens, hq), 7.0, device="cuda")
    got = cache.attention(q, b.h, lse=lse)
    acf.synchronize()
    P.check_attention(got, lse, P.attention64(cache, b, q, dim ** -0.5, True, 0), dtype)


@pytest.mark.parametrize("hq,heads,most", [(4, 1, 70), (3, 1, 300), (40, 1, 9)])
def test_attention_of_many_ragged_sequences(acf, hq, heads, most):
    """300 sequences, of which many have no new token and many few: row tiles are found by counting."""
    rng = np.random.default_rng(most)
    new = [int(x) for x in rng.integers(0, most + 1, 300) * (rng.random(300) < 0.6)]
    new[0], new[127], new[128], new[299] = 0, most, most, most
    b = P.Batch(acf, new, [n + int(x) for n, x in zip(new, rng.integers(0, 90, 300))], 16, seed=32)
    cache = P.random_cache(acf, b.pages, heads, 64, 16, 33)
    q = (randn(34, b.tokens, hq, 64) * 0.3).to(torch.float16)
    got = cache.attention(q, b.h)
    acf.synchronize()
    P.check_attention(got, None, P.attention64(cache, b, q, 64 ** -0.5, True, 0), "f16")


@pytest.mark.parametrize("dtype,dim,window,new,length", [
    ("f16", 64, 700, [260], [3000]), ("bf16", 128, 1023, [87, 1], [4096, 900]), ("f16", 128, 1 << 30, [60], [2000]),
    ("bf16", 64, 513, [333], [333]), ("f16", 64, 1, [100], [5000])])
def test_attention_windows_in_parts(acf, dtype, dim, window, new, length):
    """Few row tiles, whose windows are divided among blocks."""
    b = P.Batch(acf, new, length, 32, seed=35)
    cache = P.random_cache(acf, b.pages, 2, dim, 32, 36)
    q = (randn(37, b.tokens, 6, dim) * 0.3).to(P.DT[dtype])
    lse = torch.full((b.tokens, 6), 7.0, device="cuda")
    got = cache.attention(q, b.h, window=window, lse=lse)
    acf.synchronize()
    P.check_attention(got, lse, P.attention64(cache, b, q, dim ** -0.5, True, window), dtype)


def test_attention_of_very_many_sequences(acf):
    """More (sequence, head) pairs than the standing tickets, one of them split by the bound on a
    chunk's pages."""
    n = 2100
    b = P.Batch(acf, [1] * n, [1 + i % 3 for i in range(n - 1)] + [17000], 16, seed=29)
    cache = P.random_cache(acf, b.pages, 32, 64, 16, 30)
    q = (randn(31, n, 32, 64) * 0.3).to(torch.float16)
    got = cache.attention(q, b.h)
    acf.synchronize()
    pick = P.Batch.__new__(P.Batch)      # the reference for some of them
    some = [0, 1, 2, 1000, n - 1]
    pick.new, pick.length, pick.page, pick.start = [1] * 5, [b.length[i] for i in some], 16, list(range(6))
    pick.table = b.table[some]
    P.check_attention(got[some], None, P.attention64(cache, pick, q[some], 64 ** -0.5, True, 0), "f16")


@pytest.mark.parametrize("new,length", [([1, 1], [700, 90]), ([200], [260])])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_strides_and_alignment(acf, new, length, dim):
    b = P.Batch(acf, new, length, 32, seed=1)
    cache = P.random_cache(acf, b.pages, 2, dim, 32, 2)
    for shift in (0, 1):
        flat = (randn(3, b.tokens * 10 * dim + 8) * 0.5).to(torch.bfloat16)
        q = flat[shift:shift + b.tokens * 10 * dim].view(b.tokens, 10, dim)[:, 3:9]
        out = torch.zeros(b.tokens * 7 * dim + 8, dtype=torch.bfloat16, device="cuda")[shift:shift + b.tokens * 7 * dim].view(6 + 1, b.tokens, dim)[:6].permute(1, 0, 2)
        cache.attention(q, b.h, scale=0.2, out=out)
        acf.synchronize()
        P.check_attention(out, None, P.attention64(cache, b, q, 0.2, True, 0), "bf16")


@pytest.mark.parametrize("new,length", [([1], [333]), ([5, 250], [333, 600])])
def test_attention_never_reads_what_is_not_seen(acf, new, length):
    """Scales of pages outside the window are NaN, codes past the length are extreme, and the table
    has -1 for pages that no row sees."""
    page, window = 16, 64
    b = P.Batch(acf, new, length, page, seed=4)
    cache = P.random_cache(acf, b.pages, 2, 128, page, 5)
    q = randn(6, b.tokens, 6, 128).to(torch.float16)
    want = P.attention64(cache, b, q, 128 ** -0.5, True, window)
    for i in range(len(new)):
        first = max(0, length[i] - new[i] - window + 1) // page
        for g in range(first):
            pid = int(b.table[i, g])
            cache.k_scale[pid] = cache.v_scale[pid] = float("nan")
        if first > 1:
            b.dev[0][i, : first // 2] = -1
        tail = length[i] % page
        if tail:
            pid = int(b.table[i, length[i] // page])
            cache.k[pid, :, tail:] = cache.v[pid, :, tail:] = -128
    got = cache.attention(q, b.h, window=window)
    acf.synchronize()
    P.check_attention(got, None, want, "f16")


@pytest.mark.parametrize("new,length,hq", [([1, 2], [300, 5000], 4), ([300], [450], 4)])
def test_attention_extreme_scores_and_scales(acf, new, length, hq):
    """Scores in the hundreds, pages whose values differ by 10^3, queries near both ends of bf16."""
    b = P.Batch(acf, new, length, 32, seed=4)
    for factor, spread in ((30.0, 3.0), (1e30, 0.0), (1e-30, 3.0)):
        cache = P.random_cache(acf, b.pages, 2, 128, 32, 5, spread)
        q = (randn(6, b.tokens, hq, 128) * factor).to(torch.bfloat16)
        scale = (1.0 if factor == 30.0 else 1.0 / factor) * 128 ** -0.5
        got = cache.attention(q, b.h, scale=scale)
        acf.synchronize()
        P.check_attention(got, None, P.attention64(cache, b, q, scale, True, 0), "bf16")


@pytest.mark.parametrize("new,length", [([1], [300]), ([200], [300])])
def test_attention_nonfinite_queries_stay_in_their_rows(acf, new, length):
    b = P.Batch(acf, new, length, 64, seed=4)
    cache = P.random_cache(acf, b.pages, 2, 64, 64, 5)
    q = randn(6, b.tokens, 4, 64).to(torch.bfloat16)
    clean = cache.attention(q, b.h)
    q[0, 1, 3], q[0, 2, 5] = float("nan"), float("inf")
    got = cache.attention(q, b.h)
    acf.synchronize()
    assert torch.isnan(got[0, 1]).all() and torch.isnan(got[0, 2]).all()
    assert torch.equal(got[0, 0], clean[0, 0]) and torch.equal(got[0, 3], clean[0, 3]) and torch.equal(got[1:], clean[1:])


def test_append_then_attention_on_another_stream(acf):
    """A stream of the caller's own, ordered by it behind the tensors' stream."""
    s = torch.cuda.Stream()
    b = P.Batch(acf, [1, 70], [100, 70], 32, seed=2)
    cache = P.random_cache(acf, b.pages, 2, 64, 32, 3)
    k, v, q = (randn(i, b.tokens, h, 64).to(torch.bfloat16) for i, h in ((1, 2), (2, 2), (3, 6)))
    out = torch.empty_like(q)
    s.wait_stream(torch.cuda.current_stream())
    acf.lib().acfun_set_stream(s.cuda_stream)
    try:
        cache.append(k, v, b.h)
        cache.attention(q, b.h, out=out)
        acf.synchronize()
    finally:
        acf.lib().acfun_set_stream(None)
    P.check_attention(out, None, P.attention64(cache, b, q, 64 ** -0.5, True, 0), "bf16")


def test_host_activations(acf):
    b = P.Batch(acf, [3, 1], [40, 21], 16, seed=2)
    cache = P.random_cache(acf, b.pages, 1, 64, 16, 3)
    hb = acf.KvBatch(b.table.numpy(), np.array(b.start, np.int32), np.array(b.length, np.int32), b.tokens, 3, 40)
    q = np.random.default_rng(1).standard_normal((4, 2, 64)).astype(np.float16)
    got = cache.attention(q, hb)
    P.check_attention(torch.from_numpy(got), None, [t.cpu() for t in P.attention64(cache, b, torch.from_numpy(q).cuda(), 64 ** -0.5, True, 0)], "f16")


def test_offsets_past_32_bits(acf):
    """A cache of 2.3 GB of codes each for keys and values, whose last pages are the ones in use."""
    pages, heads, page, dim = 70000, 8, 64, 64
    assert pages * heads * page * dim > 2 ** 31
    codes = [torch.empty((pages, heads, page, dim), dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.full((pages, heads), 0.01, device="cuda") for _ in range(2)]
    cache = acf.KvCache8(*codes, *scales)
    for new, length in (([3, 1], [3, 700]), ([100, 1], [650, 40])):
        b = P.Batch(acf, new, length, page, seed=33, spare_pages=0)
        b.table = torch.where(b.table >= 0, pages - 1 - b.table, b.table)
        b.dev[0].copy_(b.table)
        for codes_of in (cache.k, cache.v):   # what is in the cache already
            used = b.table[b.table >= 0].long().cuda()
            codes_of[used] = torch.randint(-127, 128, (len(used), heads, page, dim), device="cuda").to(torch.int8)
        kv = randn(34, b.tokens, 2, heads, dim).to(torch.bfloat16)
        q = randn(35, b.tokens, 2 * heads, dim).to(torch.bfloat16)
        cache.append(kv[:, 0], kv[:, 1], b.h)
        k, _ = cache.read(b.h, torch.float32)
        got = cache.attention(q, b.h, scale=0.1)
        acf.synchronize()
        for i in range(2):
            rows = slice(b.start[i], b.start[i + 1])
            want = b.whole(cache.k, cache.k_scale, i)[b.length[i] - b.new[i]:]
            assert torch.equal(k[rows].double(), want.float().double())
            assert ((want - kv[rows, 0].double()).abs() <= cache.k_scale[b.table[i, 0].item()].max().double() * 4).all()
        P.check_attention(got, None, P.attention64(cache, b, q, 0.1, True, 0), "bf16")


# ------------------------------------------------------------------ bad device data is reported, not read
def test_bad_entries_are_reported(acf):
    b = P.Batch(acf, [2, 2, 40], [40, 50, 60], 16, seed=2)
    cache = P.random_cache(acf, b.pages, 1, 64, 16, 3)
    q = randn(4, b.tokens, 1, 64).to(torch.float16)
    want = cache.attention(q, b.h)
    kv = q.clone()
    acf.synchronize()
    for which, at, bad in ((0, (1, 3), b.pages), (0, (1, 3), -7), (2, 1, 10 ** 6), (2, 1, -1), (1, 1, 1), (1, 2, 10 ** 6)):
        kept = b.dev[which].clone()
        b.dev[which][at] = bad
        for call in (lambda: cache.attention(q, b.h), lambda: cache.read(b.h, torch.float16), lambda: cache.append(kv, kv, b.h)):
            if which == 1 and bad == 1:
                continue
            got = call()
            with pytest.raises(acf.AcfunError, match="argument check"):
                acf.synchronize()
            if got is not None and not isinstance(got, tuple) and which != 1:
                assert torch.equal(got[:2], want[:2]) and torch.equal(got[4:], want[4:])
                cache_before = cache.k.clone()
        b.dev[which].copy_(kept)
        cache.k.copy_(cache_before)
        want = cache.attention(q, b.h)
        acf.synchronize()


def test_bounds_that_are_too_small_are_reported(acf):
    b = P.Batch(acf, [5], [300], 16, seed=2)
    cache = P.random_cache(acf, b.pages, 1, 64, 16, 3)
    q = randn(4, 5, 1, 64).to(torch.float16)
    for max_new, max_len in ((3, 300), (5, 299)):
        h = acf.KvBatch(*b.dev, 5, max_new, max_len)
        for call in (lambda: cache.attention(q, h), lambda: cache.read(h, torch.float16), lambda: cache.append(q, q, h)):
            call()
            with pytest.raises(acf.AcfunError, match="argument check"):
                acf.synchronize()


# ------------------------------------------------------------------ refusals that need a device cache
def test_refusals(acf):
    b = P.Batch(acf, [2, 1], [40, 21], 16, seed=2)
    cache = P.random_cache(acf, b.pages, 2, 64, 16, 3)
    q, kv = randn(1, 3, 4, 64).to(torch.float16), randn(1, 3, 2, 64).to(torch.float16)
    spec = acf.Rope(torch.ones(12, device="cuda"))
    small = acf.KvBatch(b.dev[0][:, :1].contiguous(), *b.dev[1:], 3, 2, 40)
    bad = [(lambda: cache.attention(q[:, :3], b.h), "multiple"), (lambda: cache.attention(q, b.h, window=-1), "window"),
           (lambda: cache.attention(q, b.h, causal=False, window=3), "window"),
           (lambda: cache.attention(q, b.h, scale=float("inf")), "scale"),
           (lambda: cache.attention(q, b.h, out=q[:, :1].expand(3, 4, 64)), "overlap"),
           (lambda: cache.attention(q.float(), b.h), "dtype"), (lambda: cache.attention(q, small), "columns"),
           (lambda: cache.append(kv, kv, small), "columns"), (lambda: cache.append(kv, kv, b.h, rope=spec), "multiple of 16"),
           (lambda: cache.append(kv, kv, b.h, rope=acf.Rope(torch.ones(40, device="cuda"))), "rot")]
    for call, words in bad:
        with pytest.raises(acf.AcfunError, match=words):
            call()
    for call in (lambda: cache.attention(q[:2], b.h), lambda: cache.append(q, q, b.h), lambda: cache.append(kv, kv.float(), b.h),
                 lambda: cache.attention(q.transpose(1, 2), b.h), lambda: cache.attention(q, b.h, lse=torch.empty(3, device="cuda")),
                 lambda: acf.KvBatch(b.dev[0].long(), *b.dev[1:], 3, 2, 40), lambda: acf.rope(q, b.dev[2], spec)):
        with pytest.raises((ValueError, TypeError)):
            call()


def test_nothing_to_do(acf):
    cache = acf.KvCache8.empty(2, 1, 64, 16)
    i32 = dict(dtype=torch.int32, device="cuda")
    for seqs in (0, 2):
        h = acf.KvBatch(torch.zeros((seqs, 1), **i32), torch.zeros(seqs + 1, **i32), torch.zeros(seqs, **i32), 0, 0, 0)
        x = torch.empty((0, 1, 64), dtype=torch.float16, device="cuda")
        cache.append(x, x, h)
        assert cache.attention(x, h).shape == x.shape and cache.read(h, torch.float16)[0].shape == x.shape
    assert acf.rope(x, torch.empty(0, **i32), acf.Rope(torch.ones(4, device="cuda"))).shape == x.shape
    acf.synchronize()


# ------------------------------------------------------------------ all of them together
def test_decoder_example():
    """Prompt and decode steps through the example's block.  Its output differs from the 64-bit block's
    by the quantisation of keys and values (half a code of 127 per page maximum, about 2.5 standard
    deviations of what it scales: 0.5 / 127 * 2.5 / sqrt(3), near 0.6 % of a value) and by bf16
    activations (0.2 %); keys enter through scores of standard deviation near 1."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decoder_attention.py")
    spec = importlib.util.spec_from_file_location("decoder_attention", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    assert m.main() < 0.03

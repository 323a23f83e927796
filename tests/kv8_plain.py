"""Plain 64-bit implementations of the int8 cache's operators and of rotary positions, and the
batches that their tests share."""
import math

import torch

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # of rounding to the type, relative
SMALLEST = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}


def rope64(x, pos, freq, amp, interleaved):
    """x [tokens, heads, dim] float64 -> rotated, straight from the definition."""
    r = 2 * len(freq)
    a = pos.double()[:, None] * freq.double()[None, :]
    c, s = (amp * torch.cos(a))[:, None], (amp * torch.sin(a))[:, None]
    y = x.clone()
    i, j = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., j] * c + x[..., i] * s
    return y


class Batch:
    """Sequences with `new` tokens each, `length` tokens in the cache, pages in random order; the
    table has -1 where no page is needed."""

    def __init__(self, acf, new, length, page, seed=0, spare_cols=2, spare_pages=2):
        g = torch.Generator().manual_seed(seed)
        need = [-(-b // page) for b in length]
        self.pages = sum(need) + spare_pages
        order = torch.randperm(self.pages, generator=g)
        self.table = torch.full((len(new), max(need + [0]) + spare_cols), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n].int()
            at += n
        self.new, self.length, self.page = list(new), list(length), page
        self.start = [0]
        for n in new:
            self.start.append(self.start[-1] + n)
        self.tokens = self.start[-1]
        self.dev = [self.table.cuda(), torch.tensor(self.start, dtype=torch.int32, device="cuda"),
                    torch.tensor(self.length, dtype=torch.int32, device="cuda")]
        self.h = acf.KvBatch(*self.dev, self.tokens, max(self.new + [0]), max(self.length + [0]))

    def whole(self, codes, scale, i):
        """Values [length, heads, dim] (float64) of sequence i."""
        n = self.length[i]
        pg = self.table[i, : -(-n // self.page)].long().to(codes.device)
        v = codes[pg].double() * scale[pg].double()[:, :, None, None]
        return v.transpose(1, 2).reshape(-1, codes.shape[1], codes.shape[3])[:n]


def random_cache(acf, pages, heads, dim, page, seed, spread=1.0):
    """A cache of random codes; scales over `spread` powers of ten, keys and values of order one."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = [torch.randint(-127, 128, (pages, heads, page, dim), generator=g, device="cuda").to(torch.int8) for _ in range(2)]
    scales = [0.015 * 10 ** (spread * (torch.rand((pages, heads), generator=g, device="cuda") - 0.5)) for _ in range(2)]
    return acf.KvCache8(codes[0], codes[1], scales[0].float().contiguous(), scales[1].float().contiguous())


def attention64(cache, b, q, scale, causal, window):
    """(out, lse, mass, size, step) [tokens, q_heads(, dim)] in float64; mass = sum of p |v|, the
    scale of relative errors in p, size [tokens, q_heads] = the largest sum of |q k| * scale, that of
    errors in the scores, and step [tokens, q_heads] = keys * the largest p * (127 v_scale), that of
    absolute errors in weights p * v_scale."""
    heads, dim = cache.heads, cache.dim
    q = q.double()
    group = q.shape[1] // heads
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mass = torch.zeros_like(out)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(lse)
    step = torch.zeros_like(lse)
    for i in range(len(b.new)):
        n, L = b.new[i], b.length[i]
        if n == 0 or L == 0:
            continue
        k, v = b.whole(cache.k, cache.k_scale, i), b.whole(cache.v, cache.v_scale, i)
        k, v = (t.repeat_interleave(group, 1).transpose(0, 1) for t in (k, v))   # [q_heads, L, dim]
        rows = q[b.start[i]:b.start[i + 1]].transpose(0, 1)                       # [q_heads, n, dim]
        at = torch.arange(L - n, L, device=q.device)[:, None]
        key = torch.arange(L, device=q.device)[None, :]
        seen = (at >= 0).expand(n, L)
        if causal:
            seen = seen & (key <= at)
            if window:
                seen = seen & (key > at - window)
        z = (rows @ k.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
        e = torch.logsumexp(z, -1)
        p = torch.exp(z - torch.where(torch.isinf(e), torch.zeros_like(e), e)[..., None])
        s = slice(b.start[i], b.start[i + 1])
        out[s] = (p @ v).transpose(0, 1)
        mass[s] = (p @ v.abs()).transpose(0, 1)
        lse[s] = e.transpose(0, 1)
        reach = (rows.abs() @ k.abs().transpose(1, 2) * abs(scale)).masked_fill(~seen, 0.0)
        size[s] = reach.amax(-1).transpose(0, 1)
        unit = cache.v_scale[b.table[i, torch.arange(L) // b.page].long().to(q.device)].double()   # [L, heads]
        step[s] = (L * 127 * p * unit.t().repeat_interleave(group, 0)[:, None]).nan_to_num().amax(-1).transpose(0, 1)
    return out, lse, mass, size, step


def check_attention(got, lse, want, dtype):
    """Held to the rounding of the result, of the weights to fp16 (2^-11 of the mass; and half of
    fp16's smallest step, 2^-25, for every key where the largest weight is at least 2^7), and of the
    32-bit scores: dim products and sums of up to `size` each within 2^-20 of it, which moves p by
    that much."""
    out, e, mass, size, step = want
    tol = HALF_ULP[dtype] * out.abs() + SMALLEST[dtype] + mass * (2.0 ** -10.5 + 2.0 ** -18 + 2.0 ** -19 * size[..., None])
    tol = tol + 2.0 ** -32 * step[..., None]
    off = (got.double() - out).abs()
    assert torch.isfinite(got).all()
    assert (off <= tol).all(), f"worst {float((off / tol).max()):.3g} of the bound"
    assert (got[torch.isinf(e)] == 0).all()
    if lse is not None:
        assert torch.equal(torch.isinf(lse), torch.isinf(e))
        f = ~torch.isinf(e)
        # the 32-bit sum and logarithm, the scores' errors, and the maximum's own rounding
        assert ((lse.double() - e).abs()[f] <= (4e-6 * (1 + e.abs()) + 2.0 ** -20 * size)[f]).all()

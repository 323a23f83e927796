"""The attention half of a decoder block on this library: projections (acfun_gemm), rotary positions,
the int8 paged cache and attention over it, for prompts and then token by token.

    python examples/decoder_attention.py

Two sequences share one cache whose pages are handed out as they grow.  The same block in 64 bits
with keys and values that are not quantised is run beside it, and the largest relative difference
of the outputs is printed.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import acfun_b200 as acf  # noqa: E402

WIDTH, Q_HEADS, KV_HEADS, DIM, PAGE = 512, 8, 2, 64, 16


class Pages:
    """Page tables of some sequences over one pool."""

    def __init__(self, seqs, columns, pool):
        self.table = torch.full((seqs, columns), -1, dtype=torch.int32)
        self.free = list(range(pool))
        self.length = [0] * seqs

    def grow(self, new):
        """Makes room for new[i] tokens in sequence i: the batch of this step."""
        start = [0]
        for i, n in enumerate(new):
            for p in range(-(-self.length[i] // PAGE), -(-(self.length[i] + n) // PAGE)):
                self.table[i, p] = self.free.pop()
            self.length[i] += n
            start.append(start[-1] + n)
        i32 = dict(dtype=torch.int32, device="cuda")
        return acf.KvBatch(self.table.cuda(), torch.tensor(start, **i32), torch.tensor(self.length, **i32), start[-1],
                           max(new), max(self.length))


class Block:
    def __init__(self, cache, rope, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.w_in = (torch.randn((WIDTH, (Q_HEADS + 2 * KV_HEADS) * DIM), generator=g) / WIDTH ** 0.5).cuda()
        self.w_out = (torch.randn((Q_HEADS * DIM, WIDTH), generator=g) / WIDTH ** 0.5).cuda()
        self.cache, self.rope = cache, rope

    def __call__(self, x, positions, batch):
        """x [tokens, WIDTH] fp32 at their positions -> x + the block's output."""
        heads = acf.gemm(x, self.w_in).view(-1, Q_HEADS + 2 * KV_HEADS, DIM).to(torch.bfloat16)
        q, k, v = heads[:, :Q_HEADS], heads[:, Q_HEADS:-KV_HEADS], heads[:, -KV_HEADS:]
        self.cache.append(k, v, batch, rope=self.rope)           # keys are rotated on the way in
        acf.rope(q, positions, self.rope, out=q)
        o = self.cache.attention(q, batch)
        return x + acf.gemm(o.reshape(-1, Q_HEADS * DIM).float(), self.w_out)

    def plain(self, x):
        """The block over one whole sequence, in 64 bits and without a cache."""
        n = x.shape[0]
        heads = (x.double() @ self.w_in.double()).view(n, -1, DIM)
        angle = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * self.rope.freq.double()
        c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
        a, b = heads[:, :-KV_HEADS].chunk(2, -1)
        q, k = torch.cat([a * c - b * s, b * c + a * s], -1).split([Q_HEADS, KV_HEADS], 1)
        v = heads[:, -KV_HEADS:]
        k, v = (t.repeat_interleave(Q_HEADS // KV_HEADS, 1).transpose(0, 1) for t in (k, v))
        z = q.transpose(0, 1) @ k.transpose(1, 2) * DIM ** -0.5
        z = z.masked_fill(torch.ones((n, n), dtype=torch.bool, device="cuda").triu(1), float("-inf"))
        return x.double() + (torch.softmax(z, -1) @ v).transpose(0, 1).reshape(n, -1) @ self.w_out.double()


def main(prompts=(37, 90), steps=20):
    """The largest relative difference from the plain block."""
    freq, amplitude = acf.rope_frequencies(DIM)
    rope = acf.Rope(torch.from_numpy(freq).cuda(), amplitude=amplitude)
    columns = -(-(max(prompts) + steps) // PAGE)
    block = Block(acf.KvCache8.empty(len(prompts) * columns, KV_HEADS, DIM, PAGE), rope)
    pages = Pages(len(prompts), columns, len(prompts) * columns)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = [torch.randn((n + steps, WIDTH), generator=g, device="cuda") for n in prompts]
    out = [[] for _ in prompts]
    for step in range(steps + 1):
        new = list(prompts) if step == 0 else [1] * len(prompts)
        at = [n - k for n, k in zip((a + b for a, b in zip(pages.length, new)), new)]
        batch = pages.grow(new)
        rows = torch.cat([x[i][a:a + n] for i, (a, n) in enumerate(zip(at, new))])
        positions = torch.cat([torch.arange(a, a + n, dtype=torch.int32) for a, n in zip(at, new)]).cuda()
        for i, y in enumerate(block(rows, positions, batch).split(new)):
            out[i].append(y)
    acf.synchronize()
    worst = 0.0
    for i in range(len(prompts)):
        want, got = block.plain(x[i]), torch.cat(out[i])
        part, change = got.double() - want, want - x[i].double()
        worst = max(worst, float(part.norm() / change.norm()))
    return worst


if __name__ == "__main__":
    print(f"largest relative difference of the block's output from 64 bits without quantisation: {main():.4f}")

"""GPU: offsets that are out of range or decrease are reported, and the sequences whose own two offsets
are good come out as without them."""
import pytest
import torch

import kv8_plain as P

pytestmark = pytest.mark.gpu

NEW, LENGTH = [3, 40, 2, 35, 1], [90, 40, 300, 77, 1]
BAD = [  # entry of start, its value, the sequences that are not touched by it
    (2, 10 ** 6, [0, 3, 4]), (2, -5, [0, 3, 4]), (3, 10, [0, 1, 4]), (1, 82, [2, 3, 4]), (5, -2 ** 31, [0, 1, 2, 3]),
    (0, 2 ** 31 - 1, [1, 2, 3, 4]), (4, 0, [0, 1, 2])]


@pytest.mark.parametrize("hq", [1, 4, 40])       # streamed and tiled, tiled, more rows per token than are streamed
@pytest.mark.parametrize("dim", [64, 256])
def test_good_sequences_beside_bad_offsets(acf, hq, dim):
    b = P.Batch(acf, NEW, LENGTH, 16, seed=71)
    g = torch.Generator(device="cuda").manual_seed(72)
    q, k, v = (torch.randn((b.tokens, h, dim), generator=g, device="cuda").to(torch.float16) for h in (hq, 1, 1))
    cache = P.random_cache(acf, b.pages, 1, dim, 16, 73)
    state = (cache.k, cache.v, cache.k_scale, cache.v_scale)
    before = [t.clone() for t in state]
    start = b.dev[1].clone()

    def calls():
        out, lse = torch.full_like(q, 7.0), torch.full((b.tokens, hq), 7.0, device="cuda")
        cache.attention(q, b.h, out=out, lse=lse)
        yield [out, lse], ()
        yield list(cache.read(b.h, torch.float16)), ()
        cache.append(k, v, b.h)
        yield (), [t.clone() for t in state]

    def each():
        for rows, pages in calls():
            code = 0
            try:
                acf.synchronize()
            except acf.AcfunError as e:
                assert "argument check" in str(e)
                code = 1
            yield rows, pages, code
        for t, was in zip(state, before):
            t.copy_(was)

    want = list(each())
    assert [w[2] for w in want] == [0, 0, 0]
    for at, value, good in BAD:
        b.dev[1].copy_(start)
        b.dev[1][at] = value
        for (rows, pages, code), (w_rows, w_pages, _) in zip(each(), want):
            assert code == 1, (at, value)
            for i in good:
                for x, y in zip(rows, w_rows):
                    assert torch.equal(x[b.start[i]:b.start[i + 1]], y[b.start[i]:b.start[i + 1]]), (at, value, i)
                pid = b.table[i, : -(-LENGTH[i] // 16)].long().cuda()
                for x, y in zip(pages, w_pages):
                    assert torch.equal(x[pid], y[pid]), (at, value, i)

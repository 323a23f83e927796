"""GPU: a batch of more (sequence, head) pairs than the standing tickets, with a prompt in it: both kernels of
attention run, and the streamed one's tickets are zeroed between them."""
import pytest
import torch

import kv8_plain as P

pytestmark = pytest.mark.gpu


def test_a_prompt_beside_very_many_decode_steps(acf):
    n, heads = 2200, 32
    new = [1] * n
    new[700] = 300
    # 17000 keys pass the most pages of a chunk, so that the keys are divided
    b = P.Batch(acf, new, [max(k, 1 + i % 3) for i, k in enumerate(new[:-1])] + [17000], 16, seed=91)
    cache = P.random_cache(acf, b.pages, heads, 64, 16, 92)
    g = torch.Generator(device="cuda").manual_seed(93)
    q = (torch.randn((b.tokens, heads, 64), generator=g, device="cuda") * 0.3).to(torch.float16)
    outs = [cache.attention(q, b.h) for _ in range(3)]
    acf.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    some = [0, 699, 700, 701, n - 1]
    pick = P.Batch.__new__(P.Batch)
    pick.new, pick.length, pick.page = [new[i] for i in some], [b.length[i] for i in some], 16
    pick.table = b.table[some]
    pick.start = [0]
    for k in pick.new:
        pick.start.append(pick.start[-1] + k)
    rows = torch.cat([torch.arange(b.start[i], b.start[i + 1]) for i in some]).cuda()
    P.check_attention(outs[0][rows], None, P.attention64(cache, pick, q[rows], 64 ** -0.5, True, 0), "f16")

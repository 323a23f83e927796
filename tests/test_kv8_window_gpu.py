"""GPU: windows as long as an int holds, also where a sequence has more new tokens than cached ones
(their positions are negative)."""
import pytest
import torch

import kv8_plain as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 9, 2 ** 30, 500, 499])
@pytest.mark.parametrize("dtype,hq,heads,dim,new,length", [
    ("f16", 4, 2, 64, [9, 2], [4, 500]),            # streamed
    ("bf16", 4, 4, 256, [9], [4]),
    ("f16", 8, 2, 128, [99, 40], [90, 500]),        # tiled
    ("bf16", 48, 1, 64, [140, 129], [100, 129])])   # tiled, key tiles made before the kernel
def test_attention_with_the_longest_windows(acf, window, dtype, hq, heads, dim, new, length):
    b = P.Batch(acf, new, length, 32, seed=51)
    cache = P.random_cache(acf, b.pages, heads, dim, 32, 52)
    g = torch.Generator(device="cuda").manual_seed(53)
    q = (torch.randn((b.tokens, hq, dim), generator=g, device="cuda") * 0.3).to(P.DT[dtype])
    lse = torch.full((b.tokens, hq), 7.0, device="cuda")
    got = cache.attention(q, b.h, window=window, lse=lse)
    acf.synchronize()
    P.check_attention(got, lse, P.attention64(cache, b, q, dim ** -0.5, True, window), dtype)

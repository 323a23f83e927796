"""GPU: queries near both ends of bf16 under a scale that brings their scores back, in calls whose key
tiles are made before the kernel (many rows per cache head)."""
import pytest
import torch

import kv8_plain as P

pytestmark = pytest.mark.gpu

SHAPES = [(48, 1, 128, [130], [130], 0), (48, 1, 64, [131, 2], [700, 300], 0), (50, 1, 64, [125], [1000], 77)]


@pytest.mark.parametrize("factor", [1e34, 1e36, 1e-30, 1e-36])
@pytest.mark.parametrize("hq,heads,dim,new,length,window", SHAPES)
def test_attention_extreme_queries_of_many_rows(acf, factor, hq, heads, dim, new, length, window):
    b = P.Batch(acf, new, length, 32, seed=61)
    cache = P.random_cache(acf, b.pages, heads, dim, 32, 62)
    g = torch.Generator(device="cuda").manual_seed(63)
    q = (torch.randn((b.tokens, hq, dim), generator=g, device="cuda") * 0.5 * factor).to(torch.bfloat16)
    scale = 1.0 / factor * dim ** -0.5
    got = cache.attention(q, b.h, scale=scale, window=window)
    acf.synchronize()
    # the scale as the call gets it, in 32 bits
    P.check_attention(got, None, P.attention64(cache, b, q, float(torch.tensor(scale, dtype=torch.float32)), True, window), "bf16")


@pytest.mark.parametrize("hq,heads,dim,new,length,window", SHAPES)
def test_attention_large_queries_pick_one_key(acf, hq, heads, dim, new, length, window):
    """Scores beyond fp16's and near fp32's range under an ordinary scale: each row is the value of its
    best key, unless two scores are as close as their rounding."""
    b = P.Batch(acf, new, length, 32, seed=61)
    cache = P.random_cache(acf, b.pages, heads, dim, 32, 62)
    g = torch.Generator(device="cuda").manual_seed(64)
    q = (torch.randn((b.tokens, hq, dim), generator=g, device="cuda") * 1e36).to(torch.bfloat16)
    got = cache.attention(q, b.h, window=window)
    acf.synchronize()
    assert torch.isfinite(got).all()
    out, _, _, _, _ = P.attention64(cache, b, q, dim ** -0.5, True, window)
    # 64-bit scores that are not close give a one-hot softmax; of normal values nearly all rows do
    off = (got.double() - out).abs().amax(-1)
    assert (off <= P.HALF_ULP["bf16"] * out.abs().amax(-1) * 1.01).float().mean() > 0.99


@pytest.mark.parametrize("hq,heads,dim,new,length,window", SHAPES)
def test_attention_rows_of_different_size(acf, hq, heads, dim, new, length, window):
    """Rows whose sizes differ by many powers of two beside each other, and rows of zeros."""
    b = P.Batch(acf, new, length, 32, seed=61)
    cache = P.random_cache(acf, b.pages, heads, dim, 32, 62)
    g = torch.Generator(device="cuda").manual_seed(65)
    q = torch.randn((b.tokens, hq, dim), generator=g, device="cuda") * 0.5
    size = torch.randint(-120, 3, (b.tokens, hq, 1), generator=g, device="cuda").float()
    q = (q * torch.exp2(size)).to(torch.bfloat16)
    q[::5] = 0
    lse = torch.full((b.tokens, hq), 7.0, device="cuda")
    got = cache.attention(q, b.h, scale=0.3, window=window, lse=lse)
    acf.synchronize()
    P.check_attention(got, lse, P.attention64(cache, b, q, 0.3, True, window), "bf16")

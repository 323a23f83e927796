"""GPU: scores far beyond those whose powers of two a float holds, on every path of attention: the softmax
is the best key's alone unless two scores are as close as their rounding, and never an infinity or NaN."""
import pytest
import torch

import kv8_plain as P

pytestmark = pytest.mark.gpu

SHAPES = [(4, 2, 64, [1, 2], [300, 5000], 0), (10, 2, 256, [30], [333], 0),           # streamed
          (8, 2, 128, [200], [300], 0), (12, 4, 64, [77, 300], [400, 500], 100),      # tiled
          (6, 2, 128, [20], [6000], 0),                                               # tiled, keys divided
          (48, 1, 128, [130], [130], 0), (50, 1, 64, [125], [1000], 77)]              # key tiles made before


@pytest.mark.parametrize("dtype,factor,scale", [("bf16", 1e7, 0.1), ("bf16", 1e9, 0.1), ("bf16", 1e12, 0.1), ("bf16", 1e30, 0.01),
                                                ("f16", 1e3, 1e5), ("f16", 1.0, -1e12), ("bf16", 1.0, 1e25)])
@pytest.mark.parametrize("hq,heads,dim,new,length,window", SHAPES)
def test_attention_of_far_scores(acf, dtype, factor, scale, hq, heads, dim, new, length, window):
    b = P.Batch(acf, new, length, 32, seed=81)
    cache = P.random_cache(acf, b.pages, heads, dim, 32, 82)
    g = torch.Generator(device="cuda").manual_seed(83)
    q = (torch.randn((b.tokens, hq, dim), generator=g, device="cuda") * factor).to(P.DT[dtype])
    lse = torch.full((b.tokens, hq), 7.0, device="cuda")
    got = cache.attention(q, b.h, scale=scale, window=window, lse=lse)
    acf.synchronize()
    out, e, _, size, _ = P.attention64(cache, b, q, scale, True, window)
    assert torch.isfinite(got).all()
    off = (got.double() - out).abs().amax(-1)
    # a share of rows has two best scores that 2^-20 of `size` does not tell apart: their distance over
    # size is of order 0.1 and spread evenly near 0, so below 1 row in 10^4
    assert (off <= 1.01 * P.HALF_ULP[dtype] * out.abs().amax(-1)).float().mean() > 0.99
    assert ((lse.double() - e).abs() <= 4e-6 * (1 + e.abs()) + 2.0 ** -20 * size).all()


@pytest.mark.parametrize("hq,heads,dim,new,length,window", SHAPES)
def test_far_rows_beside_ordinary_ones(acf, hq, heads, dim, new, length, window):
    """Far rows and ordinary ones in the same tiles.  (The ordinary ones are not equal bit by bit to what they
    are alone: rows of a warp move their offsets together.)"""
    b = P.Batch(acf, new, length, 32, seed=81)
    cache = P.random_cache(acf, b.pages, heads, dim, 32, 82)
    g = torch.Generator(device="cuda").manual_seed(84)
    q = (torch.randn((b.tokens, hq, dim), generator=g, device="cuda") * 0.5).to(torch.bfloat16)
    far = torch.rand((b.tokens, hq), generator=g, device="cuda") < 0.1
    far[-1, -1] = True
    q = torch.where(far[..., None], q * 2.0 ** 60, q)
    got = cache.attention(q, b.h, window=window)
    acf.synchronize()
    want = P.attention64(cache, b, q, dim ** -0.5, True, window)
    P.check_attention(got[~far], None, [t[~far] for t in want], "bf16")
    assert torch.isfinite(got).all()
    off = (got.double() - want[0]).abs().amax(-1)
    assert (off <= 1.01 * P.HALF_ULP["bf16"] * want[0].abs().amax(-1))[far].float().mean() > 0.99

"""Rows of the 4-bit attention with all their weight on one token give that token's value, rounded
once: the dominant weight of a row is 1, so its product with a scale (8 bits) is exact in binary16.
Tolerance: the output's unit roundoff, and 2^-20 for the binary32 operations before it."""

from __future__ import annotations

import pytest
import torch

from oracle import serving as ref

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]
UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,heads", [(64, 8), (64, 32), (128, 4), (128, 16), (128, 24), (256, 2), (256, 16)])
def test_one_token_in_sight(dim, heads, dtype) -> None:
    from pck.cuda import kv4_append, kv4_attention, kv4_cache

    gen = torch.Generator().manual_seed(dim + heads)
    k, v = torch.randn(2, 96, 1, dim, generator=gen)
    cache = kv4_cache(6, 16, 1, dim)
    kv4_append(cache, k.cuda(), v.cuda(), torch.arange(96, device="cuda"))
    values = ref.cache_values(cache.cpu())[1].reshape(96, dim)
    table, lens = torch.arange(6, dtype=torch.int32).expand(4, 6).cuda(), torch.tensor([1, 17, 96, 50], dtype=torch.int32)
    q = torch.randn(4, 1, heads, dim, generator=gen).to(dtype)
    out = kv4_attention(q.cuda(), cache, table, lens.cuda(), window=1).cpu().double()[:, 0]
    want = values[lens.long() - 1][:, None].expand(4, heads, dim)
    assert bool(((out - want).abs() <= UNIT[dtype] * want.abs() + 2.0**-20).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_all_weight_on_one_token_of_many(dtype) -> None:
    """Scores apart by more than the exponential's range, the highest anywhere in the order of the tokens."""
    from pck.cuda import kv4_append, kv4_attention, kv4_cache

    gen = torch.Generator().manual_seed(1)
    for place in (0, 5, 40, 77, 159):
        v = torch.randn(160, 1, 64, generator=gen)
        level = -torch.rand(160, generator=gen)
        level[place] = 1.0
        k = level[:, None, None].expand(160, 1, 64)
        cache = kv4_cache(10, 16, 1, 64)
        kv4_append(cache, k.cuda(), v.cuda(), torch.arange(160, device="cuda"))
        q = torch.linspace(30, 90, 6)[None, :, None].expand(1, 6, 64).to(dtype)
        out = kv4_attention(q.cuda(), cache, torch.arange(10, dtype=torch.int32)[None].cuda(),
                            torch.tensor([160], dtype=torch.int32).cuda()).cpu().double()[0]  # fmt: skip
        want = ref.cache_values(cache.cpu())[1].reshape(160, 64)[place].expand(6, 64)
        assert bool(((out - want).abs() <= UNIT[dtype] * want.abs() + 2.0**-20).all())

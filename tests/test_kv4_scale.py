"""The attention at the ends of the softmax scale's range: a scale (or a scale times queries) that
binary32 cannot hold leaves scores of zero, the same weight for all tokens that a row sees, and
none for the others. Tolerance of tests/test_kv4_values.py."""

from __future__ import annotations

import pytest
import torch

from oracle import serving as ref

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]


@pytest.mark.parametrize("size,scale", [(1.0, 1e-50), (1.0, 1e-44), (1e-37, 1e-10), (1e-30, 1e-20), (1.0, 1e-30)])
@pytest.mark.parametrize("window", [0, 5])
def test_scores_too_small_for_binary32(size, scale, window) -> None:
    from pck.cuda import device_status, kv4_append, kv4_attention, kv4_cache

    gen = torch.Generator().manual_seed(1)
    k, v = torch.randn(2, 40, 2, 64, generator=gen)
    cache = kv4_cache(3, 16, 2, 64)
    kv4_append(cache, k.cuda(), v.cuda(), torch.arange(40, device="cuda"))
    q = (size * torch.randn(2, 6, 4, 64, generator=gen)).bfloat16()
    table, lens = torch.arange(3, dtype=torch.int32).expand(2, 3), torch.tensor([40, 4], dtype=torch.int32)
    out = kv4_attention(q.cuda(), cache, table.cuda(), lens.cuda(), scale=scale, window=window).cpu().double()
    want, largest = ref.attention(q, cache.cpu(), table, lens, scale, window)
    tol = 2.0**-8 * want.abs() + (2.0**-11 * 16 / 15 + 2.0**-16) * largest
    assert bool(((out - want).abs() <= tol).all()) and device_status() == 0
    assert not bool(out[1, :2].any())  # two of the six query tokens come before the request's first

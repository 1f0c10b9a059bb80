"""The scores of the 4-bit attention are as good as a binary32 dot product with the values that the
codes stand for. Two tokens with values 1 and -1 (constant, so exact) give tanh of half the
difference of their scores; queries nearly orthogonal to the difference of the two keys make that
small, so the output's rounding does not hide it.

Tolerance: dim 2^-24 times the sum of |q_c k_c| for each score, the bound of a binary32 sum of dim
products; 2^-10 of the difference for the output (binary16); 2^-20 for the exponentials and the
quotient."""

from __future__ import annotations

import pytest
import torch

from oracle import serving as ref

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]


@pytest.mark.parametrize("heads", [1, 16, 24, 32])
@pytest.mark.parametrize("kind", ["normal", "outliers", "offsets"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_the_difference_of_two_scores(dim, kind, heads) -> None:
    from pck.cuda import kv4_append, kv4_attention, kv4_cache

    n = 200
    gen = torch.Generator().manual_seed(dim + heads)
    k = torch.randn(n, 2, 1, dim, generator=gen)
    if kind != "normal":
        k[..., ::37] *= 6
    if kind == "offsets":
        k += 4 * torch.randn(dim, generator=gen)
    v = torch.ones(n, 2, 1, dim)
    v[:, 1] = -1
    cache = kv4_cache(n, 16, 1, dim)
    slots = (16 * torch.arange(n)[:, None] + torch.arange(2)).reshape(-1)
    kv4_append(cache, k.view(-1, 1, dim).cuda(), v.view(-1, 1, dim).cuda(), slots.cuda())
    keys = ref.cache_values(cache.cpu())[0][:, :2, 0]
    apart = keys[:, 0] - keys[:, 1]
    q = torch.randn(n, heads, dim, generator=gen, dtype=torch.float64)
    along = (q @ apart[..., None]) / apart.square().sum(-1)[:, None, None]
    q = (q - along * apart[:, None]).half()
    table, lens = torch.arange(n, dtype=torch.int32)[:, None], torch.full((n,), 2, dtype=torch.int32)
    out = kv4_attention(q.cuda(), cache, table.cuda(), lens.cuda()).cpu().double()[..., 0]
    want = (q.double() @ apart[..., None])[..., 0] * dim**-0.5
    size = (q.double().abs() @ keys.abs().sum(1)[..., None])[..., 0] * dim**-0.5  # of both scores
    tol = dim * 2.0**-24 * size + 2.0**-10 * want.abs() + 2.0**-20
    err = (2 * torch.atanh(out) - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ratio", [2.0**10, 2.0**20, 2.0**24])
def test_small_queries_that_meet_large_keys(ratio, dtype) -> None:
    """One group's queries are 1 / ratio of the other's and its keys ratio times as large: both count alike."""
    from pck.cuda import kv4_append, kv4_attention, kv4_cache

    n, dim = 200, 128
    gen = torch.Generator().manual_seed(9)
    k = torch.randn(n, 2, 1, dim, generator=gen) * 2.0**-10
    k[..., 64:] *= ratio
    v = torch.ones(n, 2, 1, dim)
    v[:, 1] = -1
    cache = kv4_cache(n, 16, 1, dim)
    slots = (16 * torch.arange(n)[:, None] + torch.arange(2)).reshape(-1)
    kv4_append(cache, k.view(-1, 1, dim).cuda(), v.view(-1, 1, dim).cuda(), slots.cuda())
    keys = ref.cache_values(cache.cpu())[0][:, :2, 0]
    q = torch.randn(n, 1, dim, generator=gen) * 2.0**10
    q[..., 64:] /= ratio
    q = q.to(dtype)
    table, lens = torch.arange(n, dtype=torch.int32)[:, None], torch.full((n,), 2, dtype=torch.int32)
    out = kv4_attention(q.cuda(), cache, table.cuda(), lens.cuda(), scale=2.0**-7).cpu().double()[..., 0]
    scores = torch.einsum("nhc,ntc->nht", q.double(), keys) * 2.0**-7
    size = torch.einsum("nhc,ntc->nh", q.double().abs(), keys.abs()) * 2.0**-7
    want = torch.tanh((scores[..., 0] - scores[..., 1]) / 2)
    # the difference's tolerance, halved by tanh's slope, and the rounding of the output and of the two values
    unit = 2.0**-8 if dtype is torch.bfloat16 else 2.0**-11
    tol = dim * 2.0**-24 * size / 2 + unit * want.abs() + 2.0**-20
    err = (out - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())

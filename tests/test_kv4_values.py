"""The 4-bit attention where the sizes of the values' scales differ between neighbouring tokens.

The keys of a token are one number, so its scale is 0 and its scores come out of a few binary32
operations. Tolerance, from the arithmetic: the output is rounded once (relative u), a weight times
a scale is rounded to binary16 (relative 2^-11) and multiplies a code less 8, at most 8 steps of a
range of 15, so at most 16/15 of the largest value of the group; beside these 2^-16 for the binary32
operations and the exponential:
|error| <= u |out| + (2^-11 * 16/15 + 2^-16) * sum over tokens of weight * max |v of the group|."""

from __future__ import annotations

import pytest
import torch

from oracle import serving as ref

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]
UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def check(levels, v, q, dtype=torch.float16, heads_see=None) -> None:
    """Attention of rows q (rows, dim) over tokens with keys levels[j] * (1, 1, ...) and values v (tokens, dim)."""
    from pck.cuda import device_status, kv4_append, kv4_attention, kv4_cache

    tokens, dim = v.shape
    pages = -(-tokens // 16)
    cache = kv4_cache(pages, 16, 1, dim)
    k = torch.as_tensor(levels, dtype=torch.float32)[:, None, None].expand(tokens, 1, dim)
    kv4_append(cache, k.cuda(), v[:, None].float().cuda(), torch.arange(tokens, device="cuda"))
    rows = q[None, None].to(dtype)  # one query token, a row a head
    table, lens = torch.arange(pages, dtype=torch.int32)[None], torch.tensor([tokens], dtype=torch.int32)
    out = kv4_attention(rows.cuda(), cache, table.cuda(), lens.cuda()).cpu().double()[0, 0]
    keys, values = (x.reshape(-1, dim)[:tokens] for x in ref.cache_values(cache.cpu()))
    w = torch.softmax(rows[0, 0].double() @ keys.T * dim**-0.5, dim=-1)
    want = w @ values
    largest = values.view(tokens, -1, 64).abs().amax(-1).repeat_interleave(64, dim=-1)
    tol = UNIT[dtype] * want.abs() + (2.0**-11 * 16 / 15 + 2.0**-16) * (w @ largest)
    tol += 2.0**-24 if dtype is torch.float16 else 0.0  # the spacing of the smallest binary16 numbers
    assert bool(torch.isfinite(out).all()) and device_status() == 0
    assert bool(((out - want).abs() <= tol).all()), float(((out - want).abs() / tol).max())


def rows_of(levels, dim):
    """Queries whose score against a key of ones is the level (natural logarithm)."""
    return torch.tensor(levels, dtype=torch.float32)[:, None].expand(len(levels), dim) * dim**-0.5


def normal(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads", [1, 12, 20, 30])
@pytest.mark.parametrize("ratio", [2.0**10, 2.0**18, 2.0**26, 2.0**60, 2.0**100])
def test_a_token_without_weight_beside_ones_that_have_it(ratio, heads, dim) -> None:
    """The neighbours' values are `ratio` times as large, their weights e^-200 or nothing."""
    v = normal(40, dim, seed=heads)
    v[[1, 8, 17, 30]] *= ratio
    levels = torch.full((40,), 4.0)
    levels[[1, 8, 17, 30]] = -4.0
    check(levels, v, rows_of([25.0] * heads, dim), torch.bfloat16)


@pytest.mark.parametrize("dim", [64, 128])
def test_rows_that_put_their_weight_on_different_tokens(dim) -> None:
    """Half of the rows take the tokens with small values, half those with large ones, a few both."""
    v = normal(100, dim, seed=1)
    v[::3] *= 2.0**40
    levels = torch.full((100,), 1.0)
    levels[::3] = -1.0
    q = rows_of([60.0 * (-1) ** i for i in range(20)], dim)
    check(levels, v, torch.cat([q, rows_of([0.0, 0.5, -0.5, 10.0], dim)]), torch.bfloat16)


def test_groups_of_a_token_of_different_sizes() -> None:
    v = normal(64, 256, seed=2)
    for g, size in enumerate((1.0, 2.0**-40, 2.0**30, 2.0**-90)):
        v[:, 64 * g : 64 * g + 64] *= size
        v[g::7, 64 * g : 64 * g + 64] *= 2.0**20
    check(torch.linspace(-1, 1, 64), v, rows_of([0.0, 1.0, -30.0], 256), torch.bfloat16)


@pytest.mark.parametrize("small", [1e-12, 1e-30, 1e-37])
@pytest.mark.parametrize("tokens", [64, 300])
def test_runs_of_small_values_after_large_ones_and_back(tokens, small) -> None:
    """Every warp meets tokens of ordinary size, a run of tiny ones, and (the longer case) ordinary ones again."""
    v = normal(tokens, 128, seed=3) * 8
    v[32:250] *= small
    levels = torch.zeros(tokens)
    check(levels, v, rows_of([0.0, 1.0], 128), torch.bfloat16)
    levels[:32] = -1.0  # and with nothing on the ordinary ones
    levels[250:] = -1.0
    check(levels, v, rows_of([0.0, 300.0, 60.0], 128), torch.bfloat16)


def test_scores_that_rise_while_values_shrink() -> None:
    """Each step of 32 tokens takes all the weight from the ones before it, with values 2^-12 their size."""
    v = normal(512, 64, seed=4)
    step = torch.arange(512) // 32
    v *= torch.exp2(-6.0 * step)[:, None]
    check(step.float(), v, rows_of([12.0, 3.0, 1.0, 40.0], 64), torch.bfloat16)
    check(-step.float(), v, rows_of([12.0, 3.0, 1.0, 40.0], 64), torch.bfloat16)


def test_scales_of_zero_and_the_largest_numbers() -> None:
    v = normal(48, 64, seed=5)
    v[::2] = 0.75  # constant: scale 0
    levels = torch.where(torch.arange(48) % 2 == 0, 1.0, -1.0)
    check(levels, v, rows_of([40.0, 3.0, -40.0, 0.0], 64))
    check(levels, normal(48, 64, seed=6) * 1e36, rows_of([0.0, 5.0], 64), torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_ordinary_values(dtype) -> None:
    v = normal(700, 128, seed=7)
    check(normal(700, seed=8), v, rows_of([0.0, 1.0, 5.0, -3.0, 20.0], 128), dtype)

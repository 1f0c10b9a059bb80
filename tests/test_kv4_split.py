"""Every token counted once, wherever the attention cuts the work: equal pieces of few items, and
many items on one line that is cut into parts.

Queries of zeros give all tokens that a row sees the same weight. The values of the tokens of tile i
are 15 in channel i % 64 of each group and 0 elsewhere, which 4 bits hold exactly (scale 1, zero 0),
so an output is 15 (tokens seen of such tiles) / (tokens seen). All weights are 1 before the
division, so the sums are whole numbers, exact in binary32; the zeros' sums and the codes less 8 add
up to them exactly too. What is left is the quotient and the output's rounding: 2^-8 relative in
bfloat16, with 2^-20 for the quotient and the joins. A tile left out or taken twice changes a
channel by more than a sixth of itself at the lengths below."""

from __future__ import annotations

import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]


def expected(lengths, queries: int, window: int) -> torch.Tensor:
    """(batch, queries, 64): 15 times the share of each class of tiles."""
    out = torch.zeros(len(lengths), queries, 64, dtype=torch.float64)
    for b, n in enumerate(lengths):
        for t in range(queries):
            last = n - queries + t
            first = max(0, last + 1 - window) if window else 0
            if last >= first:
                tokens = torch.arange(first, last + 1)
                out[b, t] = 15 * torch.bincount(tokens // 16 % 64, minlength=64).double() / tokens.numel()
    return out


def run(lengths, queries, heads, kv_heads, dim, page, window):
    """The attention's output over a cache whose pages are shared by all requests: place by place the
    same tiles, in pages of their own for every second request."""
    from pck.cuda import device_status, kv4_append, kv4_attention, kv4_cache

    most = max(lengths)
    per = -(-most // page)
    cache = kv4_cache(2 * per, page, kv_heads, dim)
    order = torch.randperm(2 * per, generator=torch.Generator().manual_seed(most))
    tokens = torch.arange(per * page)
    v = torch.zeros(per * page, kv_heads, dim // 64, 64)
    v[tokens, :, :, tokens // 16 % 64] = 15.0
    v = v.flatten(-2).cuda()
    for half in range(2):
        slots = order[half * per + tokens // page] * page + tokens % page
        kv4_append(cache, v, v, slots.cuda())
    table = torch.stack([order[(b % 2) * per : (b % 2) * per + per] for b in range(len(lengths))]).to(torch.int32)
    q = torch.zeros(len(lengths), queries, heads, dim, dtype=torch.bfloat16, device="cuda")
    out = kv4_attention(q, cache, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), window=window)
    assert device_status() == 0
    return out.cpu().double()


def on_a_line(lengths, queries, heads, kv_heads, dim) -> bool:
    """Whether the items are more than half of the most parts that any call has (CTAs that run at once)."""
    rows = queries * heads // kv_heads
    block = 8 if rows <= 8 else 16 if rows <= 16 or dim == 256 else 24 if dim == 128 else 32
    ctas = (4 if block <= 16 else 2) if dim == 64 else (3 if block <= 16 else 2) if dim == 128 else 2
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    filled = sum(n > 0 for n in lengths) * kv_heads * -(-rows // block)
    return 2 * filled > sms * ctas


def spread(count, most, seed):
    gen = torch.Generator().manual_seed(seed)
    return torch.exp(torch.rand(count, generator=gen) * torch.log(torch.tensor(float(most)))).long().tolist()


LINE = [
    # lengths, queries, heads, kv_heads, dim, page, window
    ([0, 1, 6000, 0, 2, *spread(60, 900, 1)], 1, 16, 8, 128, 16, 0),
    ([6111, 0, 3, *spread(70, 400, 2)], 1, 5, 5, 64, 48, 0),
    ([*spread(90, 300, 3), 5003], 1, 32, 8, 128, 64, 0),  # the long one at the line's end
    ([2500, 1, 0, 17, *spread(70, 700, 4)], 5, 12, 4, 128, 16, 0),  # queries, row blocks
    ([3000, 2, 5, *spread(60, 2000, 5)], 4, 24, 6, 64, 32, 300),  # and a window
    ([*spread(30, 600, 6), 4097], 3, 24, 8, 256, 16, 0),
    ([777] * 96, 1, 8, 4, 128, 16, 0),
    ([16] * 400, 1, 4, 2, 64, 16, 0),
    ([1, 15, 16, 17] * 80, 1, 2, 2, 64, 16, 0),
]
PIECES = [
    ([1027], 1, 32, 8, 128, 16, 0),
    ([6000, 1], 1, 8, 2, 64, 16, 0),
    ([5000, 0, 37], 4, 24, 4, 64, 32, 2048),
    ([2049, 900], 1, 16, 1, 256, 64, 0),
    ([129], 1, 1, 1, 64, 16, 0),
    ([3333, 3, 70], 7, 12, 2, 128, 112, 1500),
]


@pytest.mark.parametrize("case", range(len(LINE)))
def test_parts_of_the_line_of_many_items(case) -> None:
    lengths, queries, heads, kv_heads, dim, page, window = LINE[case]
    assert on_a_line(lengths, queries, heads, kv_heads, dim)
    compare(*LINE[case])


@pytest.mark.parametrize("case", range(len(PIECES)))
def test_equal_pieces_of_few_items(case) -> None:
    lengths, queries, heads, kv_heads, dim, page, window = PIECES[case]
    assert not on_a_line(lengths, queries, heads, kv_heads, dim)
    compare(*PIECES[case])


def compare(lengths, queries, heads, kv_heads, dim, page, window) -> None:
    out = run(lengths, queries, heads, kv_heads, dim, page, window)
    want = expected(lengths, queries, window)[:, :, None].repeat(1, 1, heads, dim // 64)
    bad = (out - want).abs() > (2.0**-8 + 2.0**-20) * want
    assert not bool(bad.any()), (bad.nonzero()[:4].tolist(), out[bad][:4].tolist(), want[bad][:4].tolist())

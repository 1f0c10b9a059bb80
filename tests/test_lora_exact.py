"""Rows that the adapters leave alone are y bit for bit: zeros keep their sign, NaN its payload."""

from __future__ import annotations

import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,m,rank", [(5, 64, 8), (40, 65, 16), (300, 64, 40), (300, 33, 100)])
def test_rows_without_an_adapter_or_of_rank_zero_are_y(tokens, m, rank, dtype) -> None:
    from pck.cuda import lora_add

    gen = torch.Generator().manual_seed(tokens)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    y = rand(tokens, m)
    y[:, ::5] = -0.0
    y[:, 1::7] = float("inf")
    y.view(torch.int32)[:, 3::11] = 0x7FC01234
    owner = torch.tensor([i % 3 - 1 for i in range(tokens)], dtype=torch.int32)
    ranks = torch.tensor([rank, 0], dtype=torch.int32)
    on = [t.cuda() for t in (rand(tokens, 64).to(dtype), y, rand(2, rank, 64).to(dtype), rand(2, m, rank).to(dtype), owner)]
    left = owner != 0
    for out in (None, on[1]):
        got = lora_add(*on, ranks=ranks.cuda(), out=out)
        assert torch.equal(got.cpu().view(torch.int32)[left], y.view(torch.int32)[left])

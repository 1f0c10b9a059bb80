"""The adapters' intermediate A x where its ranks differ in size or reach the ends of the types: a rank
scaled down in A and up in B by the same power of two is the same adapter. Tolerance of
tests/test_lora.py, whose bound goes by the terms' own size: 2^-23 (n + rank + 8) times the sum of
the absolute values of an output's terms."""

from __future__ import annotations

import pytest
import torch

from oracle import serving as ref

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,rank", [(3, 2), (3, 16), (40, 64), (3, 256), (300, 16), (300, 40), (300, 70)])
def test_ranks_of_different_sizes(tokens, rank, dtype) -> None:
    from pck.cuda import lora_add

    n, m = 8, 33
    gen = torch.Generator().manual_seed(rank)
    # what A takes away B gives back, up to 2^12 each way (binary16 holds both: elements of 2^-6 to 4)
    size = torch.exp2(torch.randint(-6, 7, (rank,), generator=gen).float() * 2)
    base = lambda *s: (torch.rand(*s, generator=gen) + 0.25) * torch.sign(torch.randn(*s, generator=gen))  # noqa: E731
    A = (base(1, rank, n) * size[:, None]).to(dtype)
    B = (base(1, m, rank) / size * 2.0**-6).to(dtype)
    x = base(tokens, n).to(dtype)
    y = torch.zeros(tokens, m)
    owner = torch.zeros(tokens, dtype=torch.int32)
    # columns that meet one rank only, the smallest and the largest among them
    for c, r in enumerate((int(size.argmin()), int(size.argmax()), 0, rank - 1)):
        B[0, c] = 0
        B[0, c, r] = 1.0
    got = lora_add(*[t.cuda() for t in (x, y, A, B, owner)]).cpu().double()
    want, terms = ref.lora(x, y, A, B, owner)
    bound = 2.0**-23 * (n + rank + 8) * terms
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("tokens", [2, 300])
def test_the_largest_finite_intermediate(tokens) -> None:
    """A x times the scale rounds up past bfloat16's largest number, but not past binary32's."""
    from pck.cuda import lora_add

    top = torch.finfo(torch.bfloat16).max
    x = torch.zeros(tokens, 8, dtype=torch.bfloat16)
    x[:, 0] = 1.0
    A = torch.zeros(1, 2, 8, dtype=torch.bfloat16)
    A[0, 0, 0], A[0, 1, 0] = top, -top
    B = torch.tensor([[1e-30, 0.0], [0.0, 1e-20], [1e-30, 1e-31]], dtype=torch.bfloat16)[None]
    args = (x, torch.zeros(tokens, 3), A, B, torch.zeros(tokens, dtype=torch.int32), torch.tensor([1.0035]))
    got = lora_add(*[t.cuda() for t in args]).cpu().double()
    want, terms = ref.lora(*args)
    assert bool(((got - want).abs() <= 2.0**-23 * 18 * terms).all())


@pytest.mark.parametrize("tokens", [2, 300])
def test_an_infinite_rank_beside_finite_ones(tokens) -> None:
    """One rank's product overflows with the scale; the others stay finite, so the sums are infinite, not NaN."""
    from pck.cuda import lora_add

    x = torch.zeros(tokens, 8, dtype=torch.float16)
    x[:, 0] = 1.0
    A = torch.zeros(1, 2, 8, dtype=torch.float16)
    A[0, 0, 0], A[0, 1, 0] = 6e4, 6e-5
    B = torch.tensor([[1.0, -1.0], [-1.0, 1.0], [1.0, 1.0]], dtype=torch.float16)[None]
    args = (x, torch.zeros(tokens, 3), A, B, torch.zeros(tokens, dtype=torch.int32), torch.tensor([1e35]))
    got = lora_add(*[t.cuda() for t in args]).cpu()
    assert torch.equal(got, torch.tensor([1.0, -1.0, 1.0]).mul(float("inf")).expand(tokens, 3))

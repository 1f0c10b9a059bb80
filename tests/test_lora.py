"""The low-rank adapters against binary64. Tolerance, from the arithmetic: sums of n products, then
of `rank`, then two more terms, all in binary32 in some order, each term rounded at most
n + rank + 8 times (2^-24 each, doubled for the tensor cores' truncation): |error| <=
2^-23 (n + rank + 8) * (sum of the absolute values of the terms)."""

from __future__ import annotations

import pytest
import torch

from oracle import serving as ref

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]


def problem(tokens, n, m, count, rank, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, n, generator=gen).to(dtype)
    y = torch.randn(tokens, m, generator=gen)
    A = (torch.randn(count, rank, n, generator=gen) * n**-0.5).to(dtype)
    B = (torch.randn(count, m, rank, generator=gen)).to(dtype)
    adapters = torch.randint(-1, count, (tokens,), generator=gen, dtype=torch.int32)
    scales = torch.rand(count, generator=gen) * 2 - 0.5
    ranks = torch.randint(0, rank + 1, (count,), generator=gen, dtype=torch.int32)
    ranks[0] = rank
    return x, y, A, B, adapters, scales, ranks


def check(got, args, n, rank) -> None:
    want, size = ref.lora(*args)
    bound = 2.0**-23 * (n + rank + 8) * size
    err = (got.cpu().double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound.clamp(min=1e-300)).max())


def test_the_library_rejects_bad_arguments() -> None:
    from pck.cuda import _lib

    lib = _lib.library()
    call = lambda fn, layout, args: fn(layout.pack(*(a or 0 for a in args)), None)  # noqa: E731
    ok = [16, 1, 3, 64, 64, 16, 32, 32, 16, 16, 2, 8, 16, None, None, 16, 32]
    for at, value, message in ((1, 0, "bfloat16"), (3, 0, "n >= 1"), (4, 63, "strides"), (7, 31, "strides"), (16, 31, "strides"),
                               (11, 0, "rank"), (11, 257, "rank"), (10, -1, "number"), (0, None, "NULL"), (8, None, "NULL"),
                               (15, None, "NULL")):  # fmt: skip
        args = list(ok)
        args[at] = value
        assert call(lib.pck_lora_add, _lib.LORA, args) == 1 and message in lib.pck_last_error().decode(), at
    for at in (2, 6):
        args = list(ok)
        args[at] = 0
        assert call(lib.pck_lora_add, _lib.LORA, args) == 0


class TestLora:
    pytestmark = gpu

    @pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
    @pytest.mark.parametrize("tokens,n,m,count,rank", [
        (1, 1, 1, 1, 1), (1, 4096, 512, 3, 16), (7, 72, 33, 2, 8), (16, 128, 128, 1, 64), (17, 520, 130, 5, 13),
        (33, 1000, 257, 40, 32), (64, 136, 64, 48, 128), (5, 64, 65, 2, 256), (70, 37, 50, 3, 5), (200, 256, 96, 4, 48),
        (300, 512, 200, 2, 24), (65, 2048, 1024, 3, 7),
        (270, 96, 70, 3, 68), (330, 160, 129, 2, 131), (260, 64, 96, 4, 256), (290, 100, 64, 3, 100)])  # fmt: skip
    def test_against_binary64(self, tokens, n, m, count, rank, dtype) -> None:
        from pck.cuda import device_status, lora_add

        args = problem(tokens, n, m, count, rank, dtype)
        on = [t.cuda() for t in args]
        check(lora_add(*on), args, n, rank)
        check(lora_add(*on[:5]), args[:5], n, rank)  # scales 1, full ranks
        assert device_status() == 0

    @pytest.mark.parametrize("tokens", [3, 40, 513])
    def test_runs_of_one_adapter_and_rows_without(self, tokens) -> None:
        """Prompts: long runs of one adapter whose ends fall inside a tile of rows."""
        from pck.cuda import lora_add

        x, y, A, B, _, scales, ranks = problem(tokens, 256, 192, 3, 16, torch.bfloat16)
        adapters = torch.tensor([(i // 37) % 4 - 1 for i in range(tokens)], dtype=torch.int32)
        args = (x, y, A, B, adapters, scales, ranks)
        got = lora_add(*[t.cuda() for t in args])
        check(got, args, 256, 16)
        assert torch.equal(got.cpu()[adapters < 0], y[adapters < 0])

    @pytest.mark.parametrize("m", [1, 31, 33, 257])
    @pytest.mark.parametrize("tokens", [40, 300])
    def test_rows_whose_outputs_are_not_aligned(self, tokens, m) -> None:
        """Single elements at the ends of the rows, and rows without an adapter beside them, in place too."""
        from pck.cuda import lora_add

        x, y, A, B, _, scales, ranks = problem(tokens, 128, m, 3, 40, torch.bfloat16)
        adapters = torch.tensor([(i // 23) % 4 - 1 for i in range(tokens)], dtype=torch.int32)
        args = (x, y, A, B, adapters, scales, ranks)
        on = [t.cuda() for t in args]
        got = lora_add(*on)
        check(got, args, 128, 40)
        assert torch.equal(got.cpu()[adapters < 0], y[adapters < 0])
        lora_add(*on, out=on[1])
        assert torch.equal(on[1], got)

    @pytest.mark.parametrize("tokens,rank", [(21, 16), (280, 96)])
    def test_strided_rows_in_place_and_unaligned(self, tokens, rank) -> None:
        from pck.cuda import lora_add

        for shift in (0, 1, 8):
            x, y, A, B, adapters, scales, ranks = problem(tokens, 264, 72, 4, rank, torch.bfloat16)
            wx = torch.zeros(tokens, 264 + 32, dtype=torch.bfloat16, device="cuda")
            wy = torch.full((tokens, 72 + 9), 7.0, device="cuda")
            xs, ys = wx[:, shift : shift + 264], wy[:, shift : shift + 72]
            xs.copy_(x)
            ys.copy_(y)
            rest = [t.cuda() for t in (A, B, adapters, scales, ranks)]
            fresh = lora_add(xs, ys, *rest)
            check(fresh, (x, y, A, B, adapters, scales, ranks), 264, rank)
            assert lora_add(xs, ys, *rest, out=ys) is ys
            assert torch.equal(ys, fresh)
            keep = torch.ones(81, dtype=torch.bool)
            keep[shift : shift + 72] = False
            assert bool((wy[:, keep.cuda()] == 7.0).all())

    def test_unaligned_adapters(self) -> None:
        from pck.cuda import lora_add

        x, y, A, B, adapters, scales, ranks = problem(9, 64, 40, 2, 8, torch.float16)
        for shift in (1, 4):
            flat = torch.zeros(A.numel() + B.numel() + 16, dtype=torch.float16, device="cuda")
            Ad = flat[shift : shift + A.numel()].view(A.shape)
            Bd = flat[-B.numel() - shift : -shift].view(B.shape)
            Ad.copy_(A)
            Bd.copy_(B)
            got = lora_add(x.cuda(), y.cuda(), Ad, Bd, adapters.cuda(), scales.cuda(), ranks.cuda())
            check(got, (x, y, A, B, adapters, scales, ranks), 64, 8)

    def test_unused_ranks_may_hold_anything(self) -> None:
        """NaN and infinities beyond an adapter's own rank, and in adapters no row names."""
        from pck.cuda import lora_add

        x, y, A, B, _, scales, ranks = problem(20, 128, 48, 3, 24, torch.bfloat16)
        ranks = torch.tensor([24, 5, 0], dtype=torch.int32)
        adapters = torch.tensor([i % 2 + 1 for i in range(20)], dtype=torch.int32)
        clean = (x, y, A.clone(), B.clone(), adapters, scales, ranks)
        A[0], B[0] = float("nan"), float("inf")
        A[1, 5:], B[1, :, 5:] = float("inf"), float("nan")
        A[2], B[2] = float("nan"), float("nan")
        got = lora_add(*[t.cuda() for t in (x, y, A, B, adapters, scales, ranks)])
        check(got, clean, 128, 24)

    def test_nan_stays_in_its_row(self) -> None:
        from pck.cuda import lora_add

        args = list(problem(40, 128, 48, 2, 8, torch.bfloat16))
        args[4] = torch.zeros(40, dtype=torch.int32)
        args[0][13, 7] = float("nan")
        got = lora_add(*[t.cuda() for t in args]).cpu()
        assert bool(got[13].isnan().all()) and not bool(got[:13].isnan().any()) and not bool(got[14:].isnan().any())

    def test_an_adapter_beyond_the_set_is_left_out_and_reported(self) -> None:
        from pck.cuda import device_status, lora_add

        x, y, A, B, _, scales, ranks = problem(18, 64, 32, 2, 8, torch.bfloat16)
        adapters = torch.full((18,), 2, dtype=torch.int32)
        device_status()
        got = lora_add(*[t.cuda() for t in (x, y, A, B, adapters, scales, ranks)])
        assert torch.equal(got.cpu(), y) and device_status() == 2 and device_status() == 0

    def test_same_bits_call_after_call(self) -> None:
        from pck.cuda import lora_add

        on = [t.cuda() for t in problem(50, 1024, 512, 9, 32, torch.bfloat16)]
        first = lora_add(*on)
        assert all(torch.equal(lora_add(*on), first) for _ in range(5))

    def test_refusals(self) -> None:
        from pck.cuda import lora_add

        x, y, A, B, adapters, scales, ranks = [t.cuda() for t in problem(6, 64, 32, 2, 8, torch.bfloat16)]
        good = dict(x=x, y=y, A=A, B=B, adapters=adapters, scales=scales, ranks=ranks)
        for change, message in ((dict(x=x.float()), "bfloat16 or all float16"), (dict(B=B.half()), "bfloat16 or all float16"),
                                (dict(A=A[:, :, :32]), "expected x"), (dict(y=y[:3]), "expected x"), (dict(y=y.bfloat16()), "y must be Float"),
                                (dict(adapters=adapters.long()), "adapters must be Int"), (dict(adapters=adapters[:2]), "adapters must have"),
                                (dict(ranks=ranks[:1]), "ranks must have"), (dict(scales=scales.double()), "scales must be Float"),
                                (dict(A=A.transpose(0, 1).contiguous().transpose(0, 1)), "A must be contiguous"),
                                (dict(x=x.t().contiguous().t()), "unit column stride"), (dict(out=y[:, 1:]), "out must be"),
                                (dict(out=torch.empty(6, 40, device="cuda")), "out must be Float"),
                                (dict(x=x.cpu()), "CUDA tensor")):  # fmt: skip
            with pytest.raises(RuntimeError, match=message):
                lora_add(**{**good, **change})
        assert lora_add(x[:0], y[:0], A, B, adapters[:0]).shape == (0, 32)

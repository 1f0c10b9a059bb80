"""Penalties, biases and grammar masks on logits, bit for bit against a restatement that applies
them one after another in binary32, a token at a time."""

from __future__ import annotations

import pytest
import torch

from oracle import serving as ref

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]


def problem(rows, vocab, history, bias, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, history + 1, (rows,), generator=gen, dtype=torch.int32)
    lens[0] = history
    per = torch.randint(0, bias + 1, (rows,), generator=gen)
    ids = torch.randint(0, vocab, (int(per.sum()),), generator=gen)
    return {
        "logits": (3 * torch.randn(rows, vocab, generator=gen)).to(dtype),
        "tokens": (torch.rand(rows, history, generator=gen) ** 3 * vocab).long().clamp(max=vocab - 1),
        "lengths": lens,
        "prompt_lengths": (lens * torch.rand(rows, generator=gen)).to(torch.int32),
        "repetition": 0.7 + torch.rand(rows, generator=gen),
        "frequency": torch.randn(rows, generator=gen),
        "presence": torch.randn(rows, generator=gen),
        "bias_starts": torch.cat([torch.zeros(1, dtype=torch.int64), per.cumsum(0)]).to(torch.int32),
        "bias_ids": ids,
        "bias_values": torch.randn(ids.numel(), generator=gen) * 5,
        "mask": torch.randint(-(2**31), 2**31, (rows, -(-vocab // 32)), generator=gen).to(torch.int32),
    }


def run(args, **more):
    from pck.cuda import process_logits

    on = {k: v.cuda() for k, v in args.items() if v is not None}
    return process_logits(on.pop("logits"), **on, **more)


def same(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Equal bits, any NaN equal to any other."""
    a, b = a.cpu(), b.cpu()
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(nan=0.0), b.nan_to_num(nan=0.0))


def test_the_library_rejects_bad_arguments() -> None:
    from pck.cuda import _lib

    lib = _lib.library()
    call = lambda fn, layout, args: fn(layout.pack(*(a or 0 for a in args)), None)  # noqa: E731
    ok = [16, 0, 2, 100, 100, 16, 8, 8, None, 16, 16, None, None, 16, 16, 16, 4, 16, 4, 16, 100]
    for at, value, message in ((1, 3, "dtype"), (3, 0, "vocab"), (4, 99, "strides"), (20, 99, "strides"), (9, None, "lengths"),
                               (6, 7, "whole rows"), (5, None, "need a history"), (14, None, "ids and values"),
                               (18, 3, "words"), (0, None, "NULL"), (19, None, "NULL")):  # fmt: skip
        args = list(ok)
        args[at] = value
        assert call(lib.pck_process_logits, _lib.LOGITS, args) == 1 and message in lib.pck_last_error().decode(), at
    args = list(ok)
    args[2] = 0
    assert call(lib.pck_process_logits, _lib.LOGITS, args) == 0


class TestLogits:
    pytestmark = gpu

    @pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
    @pytest.mark.parametrize("rows,vocab,history,bias", [(1, 1, 1, 1), (1, 50, 200, 9), (3, 4097, 300, 40), (5, 8191, 64, 0),
                                                         (2, 32003, 700, 300), (17, 1000, 5, 3), (1, 128256, 900, 20),
                                                         (150, 257, 40, 5)])  # fmt: skip
    def test_everything_at_once(self, rows, vocab, history, bias, dtype) -> None:
        args = problem(rows, vocab, history, bias, dtype)
        assert same(run(args), ref.process_logits(**args))

    @pytest.mark.parametrize("keep", [(), ("mask",), ("bias_starts", "bias_ids", "bias_values"), ("tokens", "lengths"),
                                      ("tokens", "lengths", "repetition"), ("tokens", "lengths", "prompt_lengths", "frequency"),
                                      ("tokens", "lengths", "prompt_lengths", "presence", "mask")])  # fmt: skip
    def test_each_part_alone(self, keep) -> None:
        args = {k: v for k, v in problem(4, 5003, 100, 30, torch.float32).items() if k in ("logits", *keep)}
        assert same(run(args), ref.process_logits(**args))

    def test_strides_in_place_and_no_write_outside(self) -> None:
        from pck.cuda import process_logits

        for shift in (0, 1, 3):
            args = problem(6, 1030, 50, 9, torch.float32)
            want = ref.process_logits(**args)
            wide = torch.full((6, 1040), 9.0, device="cuda")
            part = wide[:, shift : shift + 1030]
            part.copy_(args["logits"])
            on = {k: v.cuda() for k, v in args.items() if k != "logits"}
            for name in ("tokens", "mask"):
                on[name] = torch.cat([on[name], on[name]], dim=1)[:, : on[name].size(1)]
            assert process_logits(part, **on, out=part) is part
            assert same(part, want)
            outside = torch.ones(1040, dtype=torch.bool)
            outside[shift : shift + 1030] = False
            assert bool((wide[:, outside.cuda()] == 9.0).all())

    def test_half_logits_at_odd_places(self) -> None:
        args = problem(5, 1001, 30, 4, torch.bfloat16)
        wide = torch.zeros(5, 1011, dtype=torch.bfloat16)
        for shift in (0, 1, 2, 5):
            wide[:, shift : shift + 1001] = args["logits"]
            on = dict(args)
            on.pop("logits")
            from pck.cuda import process_logits

            got = process_logits(wide.cuda()[:, shift : shift + 1001], **{k: v.cuda() for k, v in on.items()})
            assert same(got, ref.process_logits(**args))

    def test_rows_without_history_and_padding_ids(self) -> None:
        args = problem(4, 300, 20, 6, torch.float32)
        args["lengths"] = torch.tensor([0, 20, -3, 10**6], dtype=torch.int32)
        args["prompt_lengths"] = torch.tensor([0, 30, 0, -1], dtype=torch.int32)
        args["tokens"][:, ::3] = torch.tensor([-1, 300, 2**40, -(2**40), 299, 0, 2**32]).tile(7)[: args["tokens"][:, ::3].size(1)]
        args["bias_ids"][::2] = 300
        assert same(run(args), ref.process_logits(**args))

    def test_repeated_bias_ids_the_last_counts(self) -> None:
        args = problem(2, 64, 3, 0, torch.float32)
        args["bias_starts"] = torch.tensor([0, 5, 9], dtype=torch.int32)
        args["bias_ids"] = torch.tensor([7, 9, 7, 7, 9, 1, 1, 63, 1])
        args["bias_values"] = torch.arange(9).float() + 0.5
        del args["mask"]
        assert same(run(args), ref.process_logits(**args))

    def test_bias_ranges_outside_the_list_are_cut(self) -> None:
        args = problem(3, 64, 3, 0, torch.float32)
        args["bias_starts"] = torch.tensor([-4, 2, 1, 10**6], dtype=torch.int32)
        args["bias_ids"] = torch.tensor([7, 9, 8])
        args["bias_values"] = torch.tensor([1.0, 2.0, 3.0])
        assert same(run(args), ref.process_logits(**args))

    def test_masks_hide_nan_and_infinities_and_may_leave_nothing(self) -> None:
        args = problem(4, 200, 10, 3, torch.float32)
        args["logits"][:, ::7] = float("nan")
        args["logits"][:, 1::7] = float("inf")
        args["logits"][:, 2::7] = -float("inf")
        args["logits"][:, 3::7] = torch.finfo(torch.float32).min
        args["mask"][1] = 0
        args["mask"][2] = -1
        got = run(args)
        assert same(got, ref.process_logits(**args)) and bool((got[1] == -float("inf")).all())
        del args["mask"]
        assert same(run(args), ref.process_logits(**args))

    def test_a_token_put_out_very_often(self) -> None:
        args = problem(1, 40, 70000, 0, torch.float32)
        args["tokens"][:] = 3
        args["lengths"][0], args["prompt_lengths"][0] = 70000, 1
        assert same(run(args), ref.process_logits(**args))

    def test_refusals(self) -> None:
        args = {k: v.cuda() for k, v in problem(3, 100, 8, 4, torch.float32).items()}
        from pck.cuda import process_logits

        for change, message in ((dict(logits=args["logits"].double()), "float32, bfloat16"), (dict(logits=args["logits"][0]), "rows, vocab"),
                                (dict(tokens=args["tokens"].int()), "tokens must be Long"), (dict(lengths=None), "need lengths"),
                                (dict(tokens=None), "need tokens"), (dict(repetition=args["repetition"][:2]), "repetition must have"),
                                (dict(frequency=args["frequency"].double()), "frequency must be Float"),
                                (dict(bias_starts=args["bias_starts"][:2]), "bias_starts must have"), (dict(bias_ids=None), "needs bias_ids"),
                                (dict(bias_starts=None), "biases need"), (dict(mask=args["mask"][:, :3]), "mask must be"),
                                (dict(mask=args["mask"].long()), "mask must be"), (dict(out=args["logits"][:, 1:]), "out must be Float"),
                                (dict(logits=args["logits"].cpu()), "CUDA tensor"),
                                (dict(logits=args["logits"].t().contiguous().t()), "unit column stride")):  # fmt: skip
            merged = {**args, **change}
            with pytest.raises(RuntimeError, match=message):
                process_logits(merged.pop("logits"), **merged)
        wide = torch.zeros(3, 101, device="cuda")
        with pytest.raises(RuntimeError, match="out must be the logits"):
            process_logits(wide[:, :100], out=wide[:, 1:])
        assert process_logits(args["logits"][:0]).shape == (0, 100)

"""The 4-bit key/value cache: the append against a byte-by-byte restatement (bit for bit), the
attention against binary64 over the values that the cache holds, and what both refuse.

Tolerance of the attention, from the arithmetic: the output is rounded once to its type (relative
u), and each weight may be rounded to 8 bits (2^-9 of its term) before the product with the values,
in a representation centred on the code range, whose terms are at most twice the largest value: so
|error| <= u |out| + 4 * 2^-9 max|v|, with 2^-16 max|v| for the binary32 sums."""

from __future__ import annotations

import ctypes

import pytest
import torch

from oracle import serving as ref

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]
UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def keys(shape, gen, dtype):
    x = torch.randn(shape, generator=gen)
    x[..., ::37] *= 6
    return x.to(dtype)


def filled_cache(pages: int, page: int, heads: int, dim: int, gen) -> torch.Tensor:
    """A cache of normal values on the CPU, every slot written by the restatement's formula."""
    cache = torch.zeros(pages, heads, page // 16, 18 * dim, dtype=torch.uint8)
    for side, (where, base) in enumerate(zip(ref.code_places(dim), (8 * dim, 17 * dim), strict=True)):
        x = keys((pages, heads, page // 16, 16, dim), gen, torch.float32) if side == 0 else torch.randn(
            pages, heads, page // 16, 16, dim, generator=gen)  # fmt: skip
        codes, pairs, _ = ref.quantise(x)
        flat = (codes[..., 0::2] | codes[..., 1::2] << 4).flatten(-2)
        cache[..., where[:, 0::2].flatten()] = flat
        cache[..., base : base + dim] = pairs.flatten(-3).contiguous().view(torch.uint8)
    return cache


# -- CPU ---------------------------------------------------------------------------------


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_every_code_of_a_tile_has_a_place_of_its_own(dim: int) -> None:
    key, value = ref.code_places(dim)
    assert sorted(key[:, 0::2].flatten().tolist()) == list(range(8 * dim))
    assert sorted(value[:, 0::2].flatten().tolist()) == list(range(9 * dim, 17 * dim))
    assert torch.equal(key[:, 0::2], key[:, 1::2]) and torch.equal(value[:, 0::2], value[:, 1::2])


def test_the_library_rejects_bad_arguments() -> None:
    from pck.cuda import _lib

    lib = _lib.library()
    call = lambda fn, layout, args: fn(layout.pack(*(a or 0 for a in args)), None)  # noqa: E731
    err = lambda: lib.pck_last_error().decode()  # noqa: E731
    ok = [16, 4, 2, 1, 128, 16, 16, 0, 3, 256, 128, 256, 128, 16, None, None]
    for at, value, message in ((4, 96, "dim"), (2, 0, "kv_heads"), (3, 0, "page_tiles"), (7, 3, "dtype"), (5, None, "NULL"),
                               (13, None, "NULL"), (0, 8, "aligned"), (14, 16, "together")):  # fmt: skip
        args = list(ok)
        args[at] = value
        assert call(lib.pck_kv4_append, _lib.KV4_APPEND, args) == 1 and message in err(), (at, err())
    args = list(ok)
    args[8] = 0
    assert call(lib.pck_kv4_append, _lib.KV4_APPEND, args) == 0  # nothing to write
    ok = [16, 1, 2, 1, 8, 128, 1024, 1024, 128, 16, 4, 2, 1, 16, 4, 4, 16, 0.1, 0, 16, None, 0]
    for at, value, message in ((5, 80, "dim"), (1, 0, "bfloat16"), (3, 0, "queries"), (4, 7, "multiple"), (12, 0, "page_tiles"),
                               (14, 3, "whole rows"), (18, -1, "window"), (17, 0.0, "scale"), (17, float("nan"), "scale"),
                               (0, None, "NULL"), (13, None, "NULL"), (9, 8, "aligned")):  # fmt: skip
        args = list(ok)
        args[at] = value
        assert call(lib.pck_kv4_attention, _lib.KV4_ATTENTION, args) == 1 and message in err(), (at, err())
    args = list(ok)
    args[2] = 0
    assert call(lib.pck_kv4_attention, _lib.KV4_ATTENTION, args) == 0
    assert lib.pck_kv4_attention_scratch(1, 0, 8, 8, 128, 64) == -1
    assert isinstance(ctypes.c_int64(lib.pck_kv4_attention_scratch(1, 1, 8, 8, 128, 64)).value, int)


def test_packed_descriptors_have_the_headers_fields() -> None:
    """Every field of a serving descriptor is 8 bytes, and the binding packs as many, doubles where they are."""
    import re
    from pathlib import Path

    from pck.cuda import _lib

    text = (Path(__file__).resolve().parents[1] / "include" / "pck_b200.h").read_text()
    for name, layout in (("kv4_append", _lib.KV4_APPEND), ("kv4_attention", _lib.KV4_ATTENTION), ("lora", _lib.LORA),
                         ("logits", _lib.LOGITS)):  # fmt: skip
        body = re.search(rf"typedef struct pck_{name}_desc {{(.*?)}}", text, re.S).group(1)
        kinds = ""
        for line in filter(None, (x.strip() for x in body.split(";"))):
            assert "*" in line or line.startswith(("int64_t", "double")), line
            kinds += ("d" if line.startswith("double") else "q") * len(line.split(","))
        want = "".join(k * int(n or 1) for n, k in re.findall(r"(\d*)([qd])", layout.format))
        assert kinds == want and layout.size == 8 * len(kinds), name


def test_cpu_tensors_and_bad_sizes_are_refused() -> None:
    from pck.cuda import kv4_append, kv4_attention, kv4_cache

    with pytest.raises(ValueError, match="multiple of 16"):
        kv4_cache(2, 24, 1, 64, device="cpu")
    with pytest.raises(ValueError, match="64, 128 or 256"):
        kv4_cache(2, 16, 1, 96, device="cpu")
    cache = kv4_cache(2, 16, 1, 64, device="cpu")
    assert cache.shape == (2, 1, 1, 1152)
    x = torch.zeros(3, 1, 64)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        kv4_append(cache, x, x, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        kv4_attention(x.bfloat16(), cache, torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))


# -- append ------------------------------------------------------------------------------


class TestAppend:
    pytestmark = gpu

    @pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
    @pytest.mark.parametrize("dim", [64, 128, 256])
    @pytest.mark.parametrize("tokens,heads,page", [(1, 1, 16), (5, 3, 48), (33, 8, 16), (71, 2, 64)])
    def test_bytes_and_values_equal_the_restatement(self, dtype, dim, tokens, heads, page) -> None:
        from pck.cuda import device_status, kv4_append

        gen = torch.Generator().manual_seed(dim + tokens)
        pages = -(-tokens // page) + 2
        cache = torch.randint(0, 256, (pages, heads, page // 16, 18 * dim), generator=gen, dtype=torch.uint8)
        # strided: keys and values side by side in a wider row, tokens two rows apart
        rows = keys((2 * tokens, 2 * heads + 1, dim), gen, dtype)
        if tokens > 4:
            rows[2, 0] = 0.375  # constant groups
            rows[4, 0, :64] = torch.linspace(0, 15, 64).to(dtype)
            rows[6, 0] *= 2.0**-14 if dtype is torch.float16 else 1e-37
        k, v = rows[::2, :heads], rows[::2, heads + 1 :]
        slots = torch.randperm(pages * page, generator=gen)[:tokens]
        slots[tokens // 2 :: 7] = -1
        on = rows.cuda()
        kd, vd = on[::2, :heads], on[::2, heads + 1 :]
        got = cache.cuda()
        k2, v2 = kv4_append(got, kd, vd, slots.cuda(), values=True)
        plain = cache.cuda()
        assert kv4_append(plain, kd, vd, slots.cuda()) is None
        want_k, want_v = ref.append(cache, k, v, slots)
        assert torch.equal(got.cpu(), cache) and torch.equal(plain.cpu(), cache)
        assert torch.equal(k2.cpu(), want_k) and torch.equal(v2.cpu(), want_v)
        assert device_status() == 0

    def test_stored_values_are_within_half_a_step(self) -> None:
        """|value - x| <= scale / 2 plus what rounding scale and zero to bfloat16 moves: 15 steps by
        2^-9 each, the zero by 2^-9 of itself, doubled for the binary32 rounding around them."""
        from pck.cuda import kv4_append, kv4_cache

        gen = torch.Generator().manual_seed(1)
        x = keys((64, 4, 128), gen, torch.float32) + 2
        cache = kv4_cache(4, 16, 4, 128)
        k, _ = kv4_append(cache, x.cuda(), x.cuda(), torch.arange(64, device="cuda"), values=True)
        g = x.view(64, 4, 2, 64)
        step = (g.amax(-1) - g.amin(-1)) / 15
        bound = step / 2 + 2 * (15 * step + g.amin(-1).abs()) * 2.0**-9
        err = (k.cpu().view(64, 4, 2, 64) - g).abs().amax(-1)
        assert bool((err <= bound).all())

    def test_not_finite_groups_are_stored_as_nan_and_only_they(self) -> None:
        from pck.cuda import kv4_append, kv4_cache

        gen = torch.Generator().manual_seed(2)
        x = torch.randn(8, 2, 128, generator=gen)
        x[1, 0, 3], x[2, 1, 100], x[3, 0, 127] = float("nan"), float("inf"), -float("inf")
        x[4, 0, 0], x[4, 0, 1] = 3e38, -3e38  # the range overflows
        cache = kv4_cache(1, 16, 2, 128)
        k, v = kv4_append(cache, x.cuda(), x.cuda(), torch.arange(8, device="cuda"), values=True)
        bad = torch.zeros(8, 2, 2, dtype=torch.bool)
        bad[1, 0, 0] = bad[2, 1, 1] = bad[3, 0, 1] = bad[4, 0, 0] = True
        for got in (k, v):
            assert torch.equal(got.cpu().view(8, 2, 2, 64).isnan().any(-1), bad)
            assert torch.equal(got.cpu().view(8, 2, 2, 64).isnan().all(-1), bad)
        want = torch.zeros(1, 2, 1, 18 * 128, dtype=torch.uint8)
        ref.append(want, x, x, torch.arange(8))
        assert torch.equal(cache.cpu(), want)

    def test_slots_beyond_the_cache_write_nothing_and_are_reported(self) -> None:
        from pck.cuda import device_status, kv4_append, kv4_cache

        device_status()
        cache = kv4_cache(2, 16, 1, 64)
        x = torch.randn(3, 1, 64, device="cuda")
        kv4_append(cache, x, x, torch.tensor([32, 2**40, -5], device="cuda"))
        assert not bool(cache.any()) and device_status() == 2 and device_status() == 0

    def test_refusals(self) -> None:
        from pck.cuda import kv4_append, kv4_cache

        cache = kv4_cache(2, 16, 2, 64)
        x = torch.zeros(3, 2, 64, device="cuda")
        slots = torch.arange(3, device="cuda")
        for args, message in (((cache, x.double(), x.double(), slots), "float32, bfloat16"),
                              ((cache, x, x.bfloat16(), slots), "both"), ((cache, x[:, :1], x[:, :1], slots), "shape"),
                              ((cache, x, x, slots.int()), "Long"), ((cache, x, x, slots[:2]), "shape"),
                              ((cache, x.transpose(1, 2).contiguous().transpose(1, 2), x, slots), "unit channel stride"),
                              ((cache[..., :1000], x, x, slots), "18"), ((cache.cpu(), x, x, slots), "contiguous on"),
                              ((cache, x, x, slots.cpu()), "must be on")):  # fmt: skip
            with pytest.raises(RuntimeError, match=message):
                kv4_append(*args)
        empty = x[:0]
        assert kv4_append(cache, empty, empty, slots[:0], values=True)[0].shape == (0, 2, 64)


# -- attention ---------------------------------------------------------------------------


def attend(batch, queries, heads, kv_heads, dim, page, dtype, lengths, window=0, scale=None, seed=0, poison=True, sharp=1.0):
    """(result, reference, tolerance) of one call over a cache whose unused places hold NaN scales."""
    from pck.cuda import kv4_attention

    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + 2
    cache = filled_cache(pages, page, kv_heads, dim, gen)
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    table = torch.full((batch, max([1, *need])), 2**31 - 1, dtype=torch.int32)  # never read past the length
    at = 0
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n]
        for i in range(n):
            used[order[at + i], : min(page, lengths[b] - i * page)] = True
        at += n
    if poison:
        flat = cache.view(pages, kv_heads, page // 16, 18 * dim)
        for base in (8 * dim, 17 * dim):
            pairs = flat[..., base : base + dim].view(pages, kv_heads, page // 16, 16, -1)
            mask = ~used.view(pages, 1, page // 16, 16, 1).expand(pairs.shape)
            pairs[mask] = 0xFF
    lens = torch.tensor(lengths, dtype=torch.int32)
    wide = (sharp * torch.randn(batch, queries + 1, heads + 2, dim, generator=gen)).to(dtype)
    q = wide[:, 1:, 1:-1]
    qd = wide.cuda()[:, 1:, 1:-1]
    out = kv4_attention(qd, cache.cuda(), table.cuda(), lens.cuda(), scale=scale, window=window)
    want, size = ref.attention(q, cache, table.clamp(max=pages - 1), lens, scale, window)
    tol = UNIT[dtype] * want.abs() + (4 * 2.0**-9 + 2.0**-16) * size
    return out.cpu(), want, tol


CASES = [
    # batch, queries, heads, kv_heads, dim, page, lengths, window
    (1, 1, 1, 1, 64, 16, [1], 0),
    (1, 1, 4, 1, 128, 16, [16], 0),
    (3, 1, 8, 2, 128, 16, [17, 0, 63], 0),
    (2, 1, 7, 7, 64, 48, [131, 48], 0),
    (2, 1, 32, 8, 128, 32, [1027, 5], 0),
    (2, 1, 16, 1, 256, 16, [70, 255], 0),
    (1, 1, 24, 1, 128, 64, [300], 0),
    (2, 1, 71, 1, 64, 16, [90, 33], 0),
    (3, 4, 8, 2, 64, 16, [2, 4, 130], 0),
    (2, 3, 12, 4, 128, 16, [50, 3], 7),
    (2, 5, 20, 4, 256, 32, [77, 1], 16),
    (2, 1, 8, 4, 128, 16, [500, 129], 100),
    (1, 9, 10, 2, 64, 16, [64], 1),
    (1, 130, 4, 2, 64, 16, [200], 0),
    (5, 2, 6, 3, 128, 112, [1, 2, 0, 113, 225], 3),
]


class TestAttention:
    pytestmark = gpu

    @pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
    @pytest.mark.parametrize("case", CASES)
    def test_against_binary64(self, case, dtype) -> None:
        from pck.cuda import device_status

        *head, lengths, window = case
        out, want, tol = attend(*head, dtype, lengths, window)
        assert out.dtype is dtype and bool(torch.isfinite(out).all())
        assert bool(((out.double() - want).abs() <= tol).all()), float(((out.double() - want).abs() - tol).max())
        assert device_status() == 0

    @pytest.mark.parametrize("sharp", [0.0, 30.0])
    def test_flat_and_sharp_weights(self, sharp) -> None:
        """All keys alike (the plain mean) and weights on one key (scores far beyond exp's range)."""
        out, want, tol = attend(2, 1, 8, 2, 128, 16, torch.bfloat16, [400, 33], sharp=sharp)
        assert bool(((out.double() - want).abs() <= tol).all())

    def test_many_requests_of_very_different_lengths(self) -> None:
        gen = torch.Generator().manual_seed(3)
        lengths = [0, 1, 2500, 0] + torch.randint(0, 200, (45,), generator=gen).tolist()
        out, want, tol = attend(49, 1, 4, 2, 64, 16, torch.bfloat16, lengths)
        assert bool(((out.double() - want).abs() <= tol).all())

    def test_rows_that_see_nothing_are_zero(self) -> None:
        out, _, _ = attend(2, 4, 4, 2, 64, 16, torch.bfloat16, [0, 2])
        assert not bool(out[0].any()) and not bool(out[1, :2].any()) and bool(out[1, 2:].any(-1).all())

    def test_three_dimensions_scale_out_and_streams(self) -> None:
        from pck.cuda import kv4_attention

        gen = torch.Generator().manual_seed(4)
        cache = filled_cache(6, 16, 2, 128, gen)
        q = torch.randn(2, 4, 128, generator=gen).bfloat16()
        table = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32)
        lens = torch.tensor([40, 48], dtype=torch.int32)
        want, size = ref.attention(q[:, None], cache, table, lens, 0.3)
        args = [t.cuda() for t in (q, cache, table, lens)]
        out = torch.empty_like(args[0])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            assert kv4_attention(*args, scale=0.3, out=out) is out
        side.synchronize()
        tol = UNIT[torch.bfloat16] * want.abs() + (4 * 2.0**-9 + 2.0**-16) * size
        assert bool(((out.cpu().double() - want[:, 0]).abs() <= tol[:, 0]).all())
        again = kv4_attention(*args, scale=0.3)
        assert torch.equal(again, out)  # same bits, call after call

    def test_lengths_beyond_the_table_are_cut_and_bad_pages_left_out(self) -> None:
        from pck.cuda import device_status, kv4_attention

        gen = torch.Generator().manual_seed(5)
        cache = filled_cache(3, 16, 1, 64, gen)
        q = torch.randn(1, 2, 64, generator=gen).bfloat16().cuda()
        table = torch.tensor([[2, 0]], dtype=torch.int32)
        device_status()
        full = kv4_attention(q, cache.cuda(), table.cuda(), torch.tensor([32], dtype=torch.int32).cuda())
        cut = kv4_attention(q, cache.cuda(), table.cuda(), torch.tensor([10**9], dtype=torch.int32).cuda())
        assert torch.equal(full, cut) and device_status() == 0
        none = kv4_attention(q, cache.cuda(), table.cuda(), torch.tensor([-3], dtype=torch.int32).cuda())
        assert not bool(none.any()) and device_status() == 0
        for bad in (3, -1):
            part = torch.tensor([[bad, 0]], dtype=torch.int32)
            got = kv4_attention(q, cache.cuda(), part.cuda(), torch.tensor([32], dtype=torch.int32).cuda())
            only, size = ref.attention(q.cpu()[:, None], cache, torch.tensor([[0]], dtype=torch.int32), torch.tensor([16], dtype=torch.int32))
            tol = UNIT[torch.bfloat16] * only.abs() + (4 * 2.0**-9 + 2.0**-16) * size
            assert bool(((got.cpu().double() - only[:, 0]).abs() <= tol[:, 0]).all())
            assert device_status() == 2

    def test_nan_reaches_the_rows_that_see_it_and_no_others(self) -> None:
        from pck.cuda import kv4_append, kv4_attention, kv4_cache

        gen = torch.Generator(device="cuda").manual_seed(6)
        x = torch.randn(40, 2, 64, generator=gen, device="cuda")
        for side in range(2):
            k, v = x.clone(), x.clone()
            (k, v)[side][20, 0, 5] = float("nan")
            cache = kv4_cache(3, 16, 2, 64)
            kv4_append(cache, k, v, torch.arange(40, device="cuda"))
            q = torch.randn(1, 25, 4, 64, generator=gen, device="cuda").half()
            out = kv4_attention(q, cache, torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda"),
                                torch.tensor([40], dtype=torch.int32, device="cuda"))  # fmt: skip
            seen = out.isnan().all(-1)
            assert torch.equal(out.isnan().any(-1), seen)
            assert not bool(seen[0, :, 2:].any()) and not bool(seen[0, :5, :2].any()) and bool(seen[0, 5:, :2].all())

    @pytest.mark.parametrize("size", [1e-12, 1.0, 1e12])
    def test_values_of_any_size_beside_a_nan(self, size) -> None:
        """Values far from 1 (binary16 holds neither), the last token's NaN: the earlier rows do not see it."""
        from pck.cuda import kv4_append, kv4_attention, kv4_cache

        gen = torch.Generator().manual_seed(7)
        k, v = torch.randn(2, 30, 1, 64, generator=gen)
        v *= size
        v[29, 0, 3] = float("nan")
        cache = kv4_cache(2, 16, 1, 64)
        kv4_append(cache, k.cuda(), v.cuda(), torch.arange(30, device="cuda"))
        q = torch.randn(1, 4, 2, 64, generator=gen).bfloat16()
        table, lens = torch.tensor([[0, 1]], dtype=torch.int32), torch.tensor([30], dtype=torch.int32)
        out = kv4_attention(q.cuda(), cache, table.cuda(), lens.cuda()).cpu()
        assert bool(out[0, 3].isnan().all())
        want, big = ref.attention(q[:, :3], cache.cpu(), table, torch.tensor([29], dtype=torch.int32))
        tol = UNIT[torch.bfloat16] * want.abs() + (4 * 2.0**-9 + 2.0**-16) * big
        assert bool(((out[:, :3].double() - want).abs() <= tol).all())

    def test_values_of_changing_size(self) -> None:
        """The values' scales rise and fall by 2^40 along the tokens, past what one power of two covers."""
        from pck.cuda import kv4_append, kv4_attention, kv4_cache

        gen = torch.Generator().manual_seed(8)
        k, v = torch.randn(2, 400, 1, 128, generator=gen)
        v *= torch.exp2(40 * torch.sin(torch.arange(400) / 20))[:, None, None]
        cache = kv4_cache(25, 16, 1, 128)
        kv4_append(cache, k.cuda(), v.cuda(), torch.arange(400, device="cuda"))
        q = torch.randn(1, 1, 5, 128, generator=gen).half()
        table, lens = torch.arange(25, dtype=torch.int32)[None], torch.tensor([400], dtype=torch.int32)
        out = kv4_attention(q.bfloat16().cuda(), cache, table.cuda(), lens.cuda()).cpu()
        want, big = ref.attention(q.bfloat16(), cache.cpu(), table, lens)
        tol = UNIT[torch.bfloat16] * want.abs() + (4 * 2.0**-9 + 2.0**-16) * big
        assert bool(((out.double() - want).abs() <= tol).all())

    def test_refusals(self) -> None:
        from pck.cuda import kv4_attention, kv4_cache

        cache = kv4_cache(2, 16, 2, 64)
        q = torch.zeros(1, 4, 64, dtype=torch.bfloat16, device="cuda")
        table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
        lens = torch.ones(1, dtype=torch.int32, device="cuda")
        for args, more, message in (((q.float(), cache, table, lens), {}, "bfloat16 or float16"),
                                    ((q[:, :3], cache, table, lens), {}, "multiple of 2"),
                                    ((q[..., :32], cache, table, lens), {}, "shape"),
                                    ((q, cache, table.long(), lens), {}, "page_table must be Int"),
                                    ((q, cache, table, lens.long()), {}, "lengths must be Int"),
                                    ((q, cache, table[:0], lens), {}, "page_table must have shape"),
                                    ((q, cache, table, lens), {"window": -1}, "window"),
                                    ((q, cache, table, lens), {"scale": 0.0}, "scale"),
                                    ((q, cache, table, lens), {"out": q}, "share memory"),
                                    ((q, cache, table, lens), {"out": torch.empty_like(q).half()}, "out must be"),
                                    ((q, cache.float(), table, lens), {}, "uint8")):  # fmt: skip
            with pytest.raises(RuntimeError, match=message):
                kv4_attention(*args, **more)
        assert kv4_attention(q[:0], cache, table[:0], lens[:0]).shape == (0, 4, 64)

"""Views as inputs of the serving operators: rows expanded without a copy (one grammar for a batch,
one page table for several samples of a prompt, one history, one x) reach the kernels with the
stride they have. What the functions hand to the library is read on the CPU; on the GPU an expanded
input gives the result of its contiguous copy."""

from __future__ import annotations

import pytest
import torch

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]


@pytest.fixture
def recorded(monkeypatch):
    """The descriptors of the calls, by entry point, instead of the calls; CPU tensors pass as the device's."""
    from pck.cuda import serving

    calls: dict[str, bytes] = {}
    monkeypatch.setattr(serving, "_index", lambda t, name: t.get_device())
    monkeypatch.setattr(serving, "_call", lambda name, index, descriptor: calls.__setitem__(name, descriptor))
    monkeypatch.setattr(serving, "_scratch_bytes", lambda *args: 0)
    return calls


def attention_args(batch=4, pages=3):
    q = torch.randn(batch, 2, 64).bfloat16()
    cache = torch.zeros(8, 1, 1, 1152, dtype=torch.uint8)
    table = torch.arange(batch * pages, dtype=torch.int32).view(batch, pages) % 8
    return q, cache, table, torch.tensor([40, 17, 1, 33][:batch], dtype=torch.int32)


def lora_args(tokens=4, n=64, m=32):
    gen = torch.Generator().manual_seed(tokens)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return (rand(tokens, n).bfloat16(), rand(tokens, m), rand(2, 8, n).bfloat16(), rand(2, m, 8).bfloat16(),
            torch.tensor([i % 3 - 1 for i in range(tokens)], dtype=torch.int32))  # fmt: skip


def logits_args(rows=4, vocab=1000, history=50):
    gen = torch.Generator().manual_seed(rows)
    return {"logits": torch.randn(rows, vocab, generator=gen), "tokens": torch.randint(0, vocab, (rows, history), generator=gen),
            "lengths": torch.tensor([50, 0, 7, 31], dtype=torch.int32), "repetition": torch.full((rows,), 1.5),
            "mask": torch.randint(-(2**31), 2**31, (rows, -(-vocab // 32)), generator=gen).to(torch.int32)}  # fmt: skip


def test_expanded_rows_go_to_the_library_with_their_stride(recorded) -> None:
    from pck.cuda import _lib, kv4_attention, lora_add, process_logits

    q, cache, table, lens = attention_args()
    kv4_attention(q, cache, table[:1].expand(4, 3), lens)
    assert _lib.KV4_ATTENTION.unpack(recorded["pck_kv4_attention"])[14:16] == (0, 3)  # table_stride, table_pages
    x, y, *rest = lora_args()
    lora_add(x[:1].expand(4, 64), y[:1].expand(4, 32), *rest)
    got = _lib.LORA.unpack(recorded["pck_lora_add"])
    assert (got[4], got[7], got[16]) == (0, 0, 32)  # x_stride, y_stride, out_stride
    a = logits_args()
    process_logits(a["logits"][:1].expand(4, 1000), tokens=a["tokens"][:1].expand(4, 50), lengths=a["lengths"],
                   mask=a["mask"][:1].expand(4, 32))  # fmt: skip
    got = _lib.LOGITS.unpack(recorded["pck_process_logits"])
    assert (got[4], got[6], got[18], got[20]) == (0, 0, 0, 1000)  # row, token, mask and out strides


def test_rows_that_overlap_in_part_go_with_their_stride_and_the_library_refuses_them(recorded) -> None:
    from pck.cuda import _lib, lora_add, process_logits

    lib = _lib.library()
    x, y, *rest = lora_args()
    lora_add(x.as_strided((4, 64), (8, 1)), y, *rest)
    assert lib.pck_lora_add(recorded["pck_lora_add"], None) == 1 and "strides" in lib.pck_last_error().decode()
    a = logits_args()
    process_logits(a["logits"].as_strided((4, 1000), (100, 1)))
    assert lib.pck_process_logits(recorded["pck_process_logits"], None) == 1 and "strides" in lib.pck_last_error().decode()


def test_a_single_row_may_have_any_stride(recorded) -> None:
    from pck.cuda import _lib, kv4_attention, lora_add, process_logits

    q, cache, table, lens = attention_args(batch=1)
    kv4_attention(q, cache, table.as_strided((1, 3), (1, 1)), lens)
    assert _lib.KV4_ATTENTION.unpack(recorded["pck_kv4_attention"])[14:16] == (3, 3)
    x, y, *rest = lora_args(tokens=1)
    lora_add(x.as_strided((1, 64), (1, 1)), y.as_strided((1, 32), (0, 1)), *rest)
    got = _lib.LORA.unpack(recorded["pck_lora_add"])
    assert (got[4], got[7]) == (64, 32)
    logits = torch.randn(1000)
    process_logits(logits.as_strided((1, 1000), (1, 1)))
    assert _lib.LOGITS.unpack(recorded["pck_process_logits"])[4] == 1000


def test_the_library_takes_one_row_for_all() -> None:
    """A row stride of 0 passes the checks: what is refused is the NULL that is checked after it."""
    from pck.cuda import _lib

    lib = _lib.library()
    for entry, layout, ok, strides, null in (
        (lib.pck_lora_add, _lib.LORA, [16, 1, 3, 64, 64, 16, 32, 32, 16, 16, 2, 8, 16, 0, 0, 16, 32], (4, 7), 0),
        (lib.pck_process_logits, _lib.LOGITS, [16, 0, 2, 100, 100, 16, 8, 8, 0, 16, 16, 0, 0, 16, 16, 16, 4, 16, 4, 16, 100], (4, 6, 18), 0),
        (lib.pck_kv4_attention, _lib.KV4_ATTENTION, [16, 1, 2, 1, 8, 128, 1024, 1024, 128, 16, 4, 2, 1, 16, 4, 4, 16, 0.1, 0, 16, 0, 0],
         (14,), 0)):  # fmt: skip
        args = list(ok)
        for at in strides:
            args[at] = 0
        args[null] = 0
        assert entry(layout.pack(*args), None) == 1 and "NULL" in lib.pck_last_error().decode()
        args[strides[0]] = -1
        assert entry(layout.pack(*args), None) == 1 and "whole rows" in lib.pck_last_error().decode()


class TestExpandedRows:
    pytestmark = gpu

    def test_attention_with_one_page_table(self) -> None:
        from pck.cuda import device_status, kv4_append, kv4_attention, kv4_cache

        gen = torch.Generator(device="cuda").manual_seed(1)
        cache = kv4_cache(4, 16, 1, 64)
        k, v = torch.randn(2, 64, 1, 64, generator=gen, device="cuda")
        kv4_append(cache, k, v, torch.arange(64, device="cuda"))
        q, _, _, lens = attention_args()
        table = torch.tensor([[2, 0, 3]], dtype=torch.int32, device="cuda").expand(4, 3)
        got = kv4_attention(q.cuda(), cache, table, lens.cuda())
        assert torch.equal(got, kv4_attention(q.cuda(), cache, table.contiguous(), lens.cuda())) and device_status() == 0

    @pytest.mark.parametrize("tokens,m", [(4, 32), (5, 33), (300, 32)])
    def test_adapters_with_one_x_and_one_y(self, tokens, m) -> None:
        from pck.cuda import lora_add

        x, y, *rest = [t.cuda() for t in lora_args(tokens=tokens, m=m)]
        xe, ye = x[:1].expand(tokens, 64), y[:1].expand(tokens, m)
        want = lora_add(xe.contiguous(), ye.contiguous(), *rest)
        assert torch.equal(lora_add(xe, y[:1].repeat(tokens, 1), *rest), want)
        assert torch.equal(lora_add(xe, ye, *rest), want)

    def test_logits_with_one_row_history_and_mask(self) -> None:
        from pck.cuda import process_logits

        a = {k: v.cuda() for k, v in logits_args().items()}
        for names in (("mask",), ("tokens",), ("logits",), ("logits", "tokens", "mask")):
            b = dict(a)
            for name in names:
                b[name] = a[name][:1].expand(a[name].shape)
            want = process_logits(**{k: v.contiguous() for k, v in b.items()})
            assert torch.equal(process_logits(**b), want)

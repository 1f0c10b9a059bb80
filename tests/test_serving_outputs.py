"""Where the outputs of the serving operators may lie: not on any input that the kernels still read,
and on the input itself where the call may work in place. The calls' descriptors are recorded
instead of run, so this needs no GPU."""

from __future__ import annotations

import pytest
import torch

from tests.test_serving_views import attention_args, logits_args, lora_args, recorded  # noqa: F401


def test_an_output_on_any_input_is_refused(recorded) -> None:  # noqa: F811
    from pck.cuda import kv4_attention, lora_add, process_logits

    shared = torch.zeros(4 * 1000 + 50)

    def on_shared(t):
        """A copy of a 4-byte tensor in the memory that the output will take."""
        view = shared.view(t.dtype) if t.dtype is not torch.float32 else shared
        return view[10 : 10 + t.numel()].view(t.shape).copy_(t)

    x, y, A, B, owner = lora_args()
    out = shared[: 4 * 32].view(4, 32)
    extra = {"scales": torch.ones(2), "ranks": torch.tensor([8, 3], dtype=torch.int32)}
    for name in extra:
        with pytest.raises(RuntimeError, match="out must be y itself or share no memory"):
            lora_add(x, y, A, B, owner, **{**extra, name: on_shared(extra[name])}, out=out)
    with pytest.raises(RuntimeError, match="out must be y itself or share no memory"):
        lora_add(x, y, A, B, on_shared(owner), out=out)
    a = logits_args()
    a.update(prompt_lengths=torch.zeros(4, dtype=torch.int32), frequency=torch.ones(4), presence=torch.ones(4),
             bias_starts=torch.tensor([0, 1, 1, 2, 2], dtype=torch.int32), bias_ids=torch.tensor([5, 6]), bias_values=torch.ones(2))  # fmt: skip
    out = shared[:4000].view(4, 1000)
    for name in ("lengths", "prompt_lengths", "repetition", "frequency", "presence", "bias_starts", "bias_values", "mask"):
        with pytest.raises(RuntimeError, match="out must be the logits themselves or share no memory"):
            process_logits(**{**a, name: on_shared(a[name])}, out=out)
    q, cache, table, lens = attention_args()
    wide = torch.zeros(q.numel() // 2, dtype=torch.int32)
    out = wide.view(torch.bfloat16).view(q.shape)
    for t, at in ((table, 2), (lens, 3)):
        args = [q, cache, table, lens]
        args[at] = wide[: t.numel()].view(t.shape).copy_(t)
        with pytest.raises(RuntimeError, match="out must not share memory"):
            kv4_attention(*args, out=out)
    assert not recorded


def test_one_row_in_place_whatever_its_stride(recorded) -> None:  # noqa: F811
    """The same memory as a single row, written with another stride of rows, is still the input itself."""
    from pck.cuda import _lib, lora_add, process_logits

    logits = torch.randn(1000)
    process_logits(logits.as_strided((1, 1000), (1200, 1)), out=logits.view(1, 1000))
    got = _lib.LOGITS.unpack(recorded["pck_process_logits"])
    assert got[0] == got[19] and got[4] == got[20] == 1000
    x, y, *rest = lora_args(tokens=1)
    lora_add(x, y.as_strided((1, 32), (40, 1)), *rest, out=y)
    got = _lib.LORA.unpack(recorded["pck_lora_add"])
    assert got[5] == got[15] and got[7] == got[16] == 32

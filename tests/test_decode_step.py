"""The decode-step example: the serving operators together with the checked projections, the sampler
and the membership check, a few steps of a small batch with requests of length zero and of several
pages. Every check passes, masked tokens are never drawn, and the attention of a step equals a
binary64 one over the values the cache then holds (tolerance of tests/test_kv4.py)."""

from __future__ import annotations

import importlib.util
import sys
from pathlib import Path

import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]

EXAMPLE = Path(__file__).resolve().parents[1] / "examples" / "decode_step.py"


def test_a_batch_of_different_requests_decodes_and_passes_its_checks() -> None:
    from oracle import serving as ref
    from pck.cuda import device_status

    spec = importlib.util.spec_from_file_location("decode_step", EXAMPLE)
    mod = importlib.util.module_from_spec(spec)
    sys.modules["decode_step"] = mod
    spec.loader.exec_module(mod)
    torch.manual_seed(3)
    shape = mod.Shape(hidden=512, heads=8, kv_heads=2, dim=64, vocab=2048, page=16, adapters=3, rank=8)
    lengths = [0, 1, 15, 16, 70]
    batch = mod.DecodeBatch(5, lengths, 80, shape)
    for step in range(4):
        got = batch.step()
        assert all(bool(got[name].all()) for name in ("qkv", "o", "head", "members"))
        assert batch.lengths.tolist() == [n + step + 1 for n in lengths]
        tokens = got["tokens"]
        assert bool((tokens[::4] % 2 == 0).all())  # the grammar's rows
        assert bool(torch.isfinite(got["logits"].gather(1, tokens[:, None])).all())
        want, size = ref.attention(got["q"].bfloat16().cpu()[:, None], batch.cache.cpu(), batch.table.cpu(), batch.lengths.cpu())
        tol = 2.0**-8 * want.abs() + (4 * 2.0**-9 + 2.0**-16) * size
        assert bool(((got["attended"].cpu().double() - want[:, 0]).abs() <= tol[:, 0]).all())
    assert device_status() == 0


def test_a_step_is_captured_in_a_graph() -> None:
    """The serving calls of a step replay from a CUDA graph with the results of the eager calls."""
    from pck.cuda import kv4_append, kv4_attention, kv4_cache, lora_add, process_logits

    gen = torch.Generator(device="cuda").manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x, y = rand(4, 256).bfloat16(), rand(4, 512)
    A, B = rand(2, 8, 256).bfloat16(), rand(2, 512, 8).bfloat16()
    owner = torch.tensor([0, 1, -1, 0], dtype=torch.int32, device="cuda")
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(4, 2)
    lens = torch.tensor([1, 17, 32, 5], dtype=torch.int32, device="cuda")
    mask = torch.randint(-(2**31), 2**31, (4, 32), generator=gen, device="cuda").to(torch.int32)
    history = torch.randint(0, 1000, (4, 40), generator=gen, device="cuda")
    penalty = torch.rand(4, generator=gen, device="cuda")

    def step(cache):
        out = lora_add(x, y, A, B, owner)
        q, k, v = out.view(4, 8, 64).split([4, 2, 2], dim=1)
        kv4_append(cache, k, v, table[:, 0].long() * 16 + 0)
        att = kv4_attention(q.half(), cache, table, lens)
        logits = process_logits(rand_logits, tokens=history, lengths=lens, frequency=penalty, mask=mask)
        return out, att, logits

    rand_logits = rand(4, 1000)
    caches = [kv4_cache(8, 16, 2, 64) for _ in range(2)]
    eager = [t.clone() for t in step(caches[0])]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = step(caches[1])
    caches[1].zero_()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(caches[0], caches[1])
    for a, b in zip(eager, replayed, strict=True):
        assert torch.equal(a, b)


def test_operators_trace_and_match_the_functions() -> None:
    from pck.cuda import kv4_attention, kv4_cache, lora_add, process_logits, serving

    gen = torch.Generator(device="cuda").manual_seed(6)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    cache = kv4_cache(4, 16, 2, 64)
    k = rand(20, 2, 64)
    slots = torch.arange(20, device="cuda")
    torch.ops.pck.kv4_append(cache, k, k, slots)
    q = rand(1, 3, 4, 64).bfloat16()
    table, lens = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), torch.tensor([20], dtype=torch.int32, device="cuda")
    assert torch.equal(torch.ops.pck.kv4_attention(q, cache, table, lens, None, 0), kv4_attention(q, cache, table, lens))
    x, y = rand(3, 64).bfloat16(), rand(3, 32)
    A, B = rand(2, 4, 64).bfloat16(), rand(2, 32, 4).bfloat16()
    owner = torch.tensor([1, 0, -1], dtype=torch.int32, device="cuda")
    assert torch.equal(torch.ops.pck.lora_add(x, y, A, B, owner), lora_add(x, y, A, B, owner))
    logits = rand(2, 100).bfloat16()
    mask = torch.zeros(2, 4, dtype=torch.int32, device="cuda") - 2
    assert torch.equal(torch.ops.pck.process_logits(logits, mask=mask), process_logits(logits, mask=mask))
    for name, args in (("kv4_attention", (q, cache, table, lens)), ("lora_add", (x, y, A, B, owner)), ("kv4_append", (cache, k, k, slots)),
                       ("process_logits", (logits,))):  # fmt: skip
        assert name in serving.OPS
        torch.library.opcheck(getattr(torch.ops.pck, name).default, args)

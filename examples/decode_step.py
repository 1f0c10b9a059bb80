"""One decode step of a batch of different requests with the serving operators between and beside the
checked projections: each request has its own adapter, cache length, penalties, biases and grammar.

    python examples/decode_step.py [--batch 32] [--steps 8]

A step is one attention block and the output layer: the checked q/k/v projection, the requests'
low-rank adapters on it, the append to the 4-bit cache, the attention over the cache, the checked o
projection, the checked LM head, the logits processing, the sampler, and the membership check of
every sampled token against the processed logits. Random weights; shapes of a Llama-3-8B layer by
default. Every launch goes to the current stream; the host only looks at the results.
"""

from __future__ import annotations

import argparse
import sys
from dataclasses import dataclass
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT / "proof-carrying-kernels_b200"))

import torch  # noqa: E402

from pck.cuda import (  # noqa: E402
    GpuBlockedChecker,
    device_status,
    gemv_tc,
    kv4_append,
    kv4_attention,
    kv4_cache,
    lora_add,
    process_logits,
    tc_height,
)
from pck.cuda.lm_head import CheckedLMHead, TopKTopPSampler, membership  # noqa: E402


@dataclass
class Shape:
    hidden: int = 4096
    heads: int = 32
    kv_heads: int = 8
    dim: int = 128
    vocab: int = 128256
    page: int = 16
    adapters: int = 16
    rank: int = 16


class DecodeBatch:
    """The weights, the cache and the per-request state of a batch."""

    def __init__(self, batch: int, lengths: list[int], most: int, shape: Shape | None = None, seed: int = 0) -> None:
        self.shape = s = shape or Shape()
        self.batch = batch
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.qkv_rows = (s.heads + 2 * s.kv_heads) * s.dim

        def weight(*size, scale=0.02):
            return (torch.randn(*size, generator=gen, device="cuda") * scale).bfloat16()

        self.qkv, self.o = weight(self.qkv_rows, s.hidden), weight(s.hidden, s.heads * s.dim)
        self.checks = [GpuBlockedChecker(w, 128, tc_height(w.size(1)), checks=1, generator=torch.Generator().manual_seed(i))
                       for i, w in enumerate((self.qkv, self.o))]  # fmt: skip
        self.embedding = weight(s.vocab, s.hidden, scale=1.0)
        self.x = torch.empty(batch, s.hidden, dtype=torch.bfloat16, device="cuda")
        self.head = CheckedLMHead(weight(s.vocab, s.hidden, scale=3.0 / s.hidden**0.5), self.x, s.vocab,
                                  generator=torch.Generator().manual_seed(9))  # fmt: skip
        # the adapters of all requests, and which request has which (-1: none)
        self.A, self.B = weight(s.adapters, s.rank, s.hidden), weight(s.adapters, self.qkv_rows, s.rank)
        self.owner = torch.tensor([i % (s.adapters + 1) - 1 for i in range(batch)], dtype=torch.int32, device="cuda")
        # pages of every request, in any order
        per = -(-most // s.page)
        self.cache = kv4_cache(batch * per, s.page, s.kv_heads, s.dim)
        self.table = torch.randperm(batch * per, generator=gen, device="cuda").to(torch.int32).view(batch, per)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        self.prompts = self.lengths.clone()
        self.tokens = torch.randint(0, s.vocab, (batch, most), generator=gen, device="cuda")
        for b, n in enumerate(lengths):  # the prompts' keys and values
            if n:
                kv = torch.randn(2, n, s.kv_heads, s.dim, generator=gen, device="cuda").bfloat16()
                kv4_append(self.cache, kv[0], kv[1], self.slots(b, torch.arange(n, device="cuda")))
        # what each request asks of its logits
        self.repetition = torch.full((batch,), 1.1, device="cuda")
        self.frequency = torch.linspace(0, 0.5, batch, device="cuda")
        self.presence = torch.full((batch,), 0.2, device="cuda")
        self.bias_starts = torch.arange(0, 2 * batch + 1, 2, dtype=torch.int32, device="cuda")
        self.bias_ids = torch.randint(0, s.vocab, (2 * batch,), generator=gen, device="cuda")
        self.bias_values = torch.randn(2 * batch, generator=gen, device="cuda")
        self.mask = torch.full((batch, -(-s.vocab // 32)), -1, dtype=torch.int32, device="cuda")
        self.mask[::4] = 0x55555555  # a grammar that allows every other token
        self.sampler = TopKTopPSampler(batch, s.vocab, k=50, p=0.9, temperature=1.0, device=self.head.device)
        self.last = torch.randint(0, s.vocab, (batch,), generator=gen, device="cuda")

    def slots(self, b, at: torch.Tensor) -> torch.Tensor:
        """Cache slots of places ``at`` of request(s) ``b``."""
        return self.table[b, at // self.shape.page].long() * self.shape.page + at % self.shape.page

    def step(self) -> dict[str, torch.Tensor]:
        """Takes every request one token further; returns the step's tokens and verdicts."""
        s, n = self.shape, self.batch
        x = self.embedding[self.last]
        qkv, passed_qkv = gemv_tc(self.qkv, x, self.checks[0])
        qkv = lora_add(x, qkv, self.A, self.B, self.owner)  # a new tensor: the checked output stays as it was
        q, k, v = qkv.view(n, -1, s.dim).split([s.heads, s.kv_heads, s.kv_heads], dim=1)
        rows = torch.arange(n, device="cuda")
        kv4_append(self.cache, k, v, self.slots(rows, self.lengths.long()))
        self.tokens[rows, self.lengths.long()] = self.last
        self.lengths += 1
        attended = kv4_attention(q.bfloat16(), self.cache, self.table, self.lengths)
        o, passed_o = gemv_tc(self.o, attended.view(n, -1), self.checks[1])
        hidden = x.float() + o
        self.x.copy_(hidden * torch.rsqrt(hidden.square().mean(-1, keepdim=True) + 1e-5))
        self.head.forward()
        logits = process_logits(self.head.logits, tokens=self.tokens, prompt_lengths=self.prompts, lengths=self.lengths,
                                repetition=self.repetition, frequency=self.frequency, presence=self.presence,
                                bias_starts=self.bias_starts, bias_ids=self.bias_ids, bias_values=self.bias_values,
                                mask=self.mask)  # fmt: skip
        self.last = self.sampler(logits).clone()
        verdict = membership(logits, self.sampler)
        return {"tokens": self.last, "members": verdict["ok"], "logits": logits, "attended": attended, "q": q,
                "qkv": passed_qkv.passed, "o": passed_o.passed, "head": self.head.passed}  # fmt: skip


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=32)
    ap.add_argument("--steps", type=int, default=8)
    args = ap.parse_args()
    lengths = [(37 * i * i) % 2000 for i in range(args.batch)]
    batch = DecodeBatch(args.batch, lengths, max(lengths) + args.steps + 1)
    for i in range(args.steps):
        got = batch.step()
        checks = {name: bool(got[name].all()) for name in ("qkv", "o", "head", "members")}
        print(f"step {i}: tokens {got['tokens'][:6].tolist()} ..., checks {checks}")
    print("device status", device_status())


if __name__ == "__main__":
    main()

"""The serving operators of a decode step as measured cases: the append to a key/value cache held
in 4 bits, the attention that reads it, the low-rank adapters of many requests beside a shared
projection, and the penalties, biases and grammar masks on the logits.

`run` computes a pass in plain torch operations in binary32, or, where `own` is true, with the
framework's operators on the same inputs. `exact` computes it in binary64.
"""

from __future__ import annotations

import functools
import math
import random
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
TILE = 16  # tokens of a cache tile
GROUP = 64  # channels that share a scale and a zero
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ESIZE = {"f32": 4, "bf16": 2, "f16": 2}


@functools.cache
def _pck():
    root = str(Path(__file__).resolve().parents[1] / "proof-carrying-kernels_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import pck.cuda

    return pck.cuda


# -- cases -----------------------------------------------------------------------------


def listed() -> list[dict]:
    return [
        # the new token of 16 requests, binary32 keys and values as the k and v projections give them
        {"name": "append decode", "op": "append", "tokens": 16, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "f32"},
        # the prompts of a few requests, an odd number of tokens, through pages of 64
        {"name": "append prompts", "op": "append", "tokens": 16381, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # one request of ordinary length: latency
        {"name": "attend one", "op": "attend", "batch": 1, "queries": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "dtype": "bf16", "shortest": 1027, "longest": 1027, "window": 0},
        # a decode batch of very different lengths, some requests just admitted and still empty
        {"name": "attend batch", "op": "attend", "batch": 64, "queries": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "dtype": "bf16", "shortest": 300, "longest": 16384, "window": 0},
        # two requests over very long documents: the largest
        {"name": "attend long", "op": "attend", "batch": 2, "queries": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "dtype": "bf16", "shortest": 262143, "longest": 262143, "window": 0},
        # four drafted tokens a request, verified in one pass, with a sliding window
        {"name": "attend drafts", "op": "attend", "batch": 24, "queries": 4, "heads": 24, "kv_heads": 4, "dim": 64, "page": 32,
         "dtype": "f16", "shortest": 5, "longest": 8191, "window": 2048},
        # one request with an adapter beside a 4096 x 4096 projection: latency
        {"name": "adapters one", "op": "adapters", "tokens": 1, "n": 4096, "m": 4096, "adapters": 8, "rank": 16, "run": 1,
         "dtype": "bf16"},
        # a decode batch, nearly every request with an adapter of its own, beside the q, k and v rows
        {"name": "adapters batch", "op": "adapters", "tokens": 64, "n": 4096, "m": 6144, "adapters": 48, "rank": 64, "run": 1,
         "dtype": "bf16"},
        # the rows of a few prompts, each prompt one adapter, beside the down projection
        {"name": "adapters prompts", "op": "adapters", "tokens": 4099, "n": 14336, "m": 4096, "adapters": 8, "rank": 32, "run": 911,
         "dtype": "bf16"},
        # one request's logits with penalties over a short history: latency
        {"name": "logits one", "op": "logits", "rows": 1, "vocab": 128256, "history": 700, "bias": 20, "grammar": 0, "dtype": "f32"},
        # a decode batch with long histories, biases and a grammar on some rows
        {"name": "logits batch", "op": "logits", "rows": 64, "vocab": 128256, "history": 9000, "bias": 300, "grammar": 1, "dtype": "f32"},
        # a wide batch over a small odd vocabulary, logits in half precision
        {"name": "logits wide", "op": "logits", "rows": 256, "vocab": 32003, "history": 2100, "bias": 9, "grammar": 1, "dtype": "bf16"},
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(["append", "attend", "attend", "adapters", "logits"])
    half = rng.choice(["bf16", "f16"])
    if op == "append":
        kv_heads, dim = rng.randint(1, 16), rng.choice([64, 128, 256])
        most = max(1, min(16384, 16384 * 8 * 128 // (kv_heads * dim)))
        return {"op": op, "tokens": _log(rng, 1, most), "kv_heads": kv_heads, "dim": dim, "page": 16 * rng.randint(1, 8),
                "dtype": rng.choice(["f32", "bf16", "f16"])}
    if op == "attend":
        kv_heads, dim, queries = rng.randint(1, 8), rng.choice([64, 128, 128, 256]), rng.choice([1, 1, 1, 2, 3, 5])
        batch = _log(rng, 1, 64)
        most = min(262143, 2 * 262143 * 8 * 128 // (batch * queries * kv_heads * dim))
        longest = _log(rng, 1, most)
        return {"op": op, "batch": batch, "queries": queries, "heads": kv_heads * rng.randint(1, 8), "kv_heads": kv_heads, "dim": dim,
                "page": 16 * rng.choice([1, 1, 2, 3, 4, 8]), "dtype": half, "shortest": _log(rng, 1, longest), "longest": longest,
                "window": rng.choice([0, 0, 0, _log(rng, 16, 4096)])}
    if op == "adapters":
        n, m, rank = 8 * _log(rng, 32, 1792), _log(rng, 128, 14336), _log(rng, 1, 128)
        tokens = _log(rng, 1, 4099)
        tokens = max(1, min(tokens, 4099 * (14336 + 2 * 4096) * 32 // ((n + 2 * m) * max(32, rank))))
        return {"op": op, "tokens": tokens, "n": n, "m": m, "adapters": rng.randint(1, 48 if tokens <= 256 else 8), "rank": rank,
                "run": 1 if tokens <= 256 else rng.randint(100, 1500), "dtype": half}
    rows, vocab = _log(rng, 1, 256), _log(rng, 1000, 200000)
    rows = max(1, min(rows, 64 * 128256 // vocab))
    return {"op": op, "rows": rows, "vocab": vocab, "history": _log(rng, 1, 9000), "bias": rng.randint(0, 300),
            "grammar": rng.randint(0, 1), "dtype": rng.choice(["f32", "bf16", "f16"])}


def _spread(case: dict, count: int, lo: int, hi: int) -> list[int]:
    """`count` lengths in [lo, hi], spread over their logarithm: the same for a case whatever the seed."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    return [_log(rng, lo, hi) for _ in range(count)]


def _lengths(case: dict) -> list[int]:
    got = _spread(case, case["batch"], case["shortest"], case["longest"])
    got[0] = case["longest"]
    if case["batch"] >= 16:  # requests that were just admitted hold nothing yet
        got[1] = 0
        got[2] = 1
    return got


def _histories(case: dict) -> list[int]:
    got = _spread(case, case["rows"], max(1, case["history"] // 20), case["history"])
    got[0] = case["history"]
    if case["rows"] >= 4:
        got[1] = 0
    return got


def _ranks(case: dict) -> list[int]:
    got = _spread(case, case["adapters"], max(1, case["rank"] // 4), case["rank"])
    got[0] = case["rank"]
    return got


def _owners(case: dict) -> list[int]:
    """The adapter of each row (-1: none): runs of `run` rows, an adapter each."""
    rng = random.Random(7 + case["tokens"])
    runs = -(-case["tokens"] // case["run"])
    per = [rng.randrange(case["adapters"]) if rng.random() < 0.9 else -1 for _ in range(runs)]
    per[0] = 0
    return [per[i // case["run"]] for i in range(case["tokens"])]


# -- the packed cache ------------------------------------------------------------------
# A tile holds 16 tokens of one head in 18 * dim bytes: key codes, key scales, value codes, value
# scales. A byte holds two codes, the lower one in its low four bits; scales are (scale, zero)
# pairs of bfloat16 for each token and group. With planes of up to two groups, key bytes go by
# (plane, token, quarter of 16 channels, group, byte) and value bytes by (plane, token / 8, channel
# / 8, token / 2, group, half of 4 channels, token parity, byte).


def _planes(dim: int) -> tuple[int, int]:
    groups = dim // GROUP
    return max(1, groups // 2), min(groups, 2)


def _pack(kc, km, vc, vm):
    """(..., 16, dim) codes and (..., 16, groups, 2) scales of keys and values -> (..., 18 * dim) bytes."""
    lead, dim = kc.shape[:-2], kc.shape[-1]
    p, w = _planes(dim)
    n = len(lead)
    k = kc.view(*lead, 16, p, w, 4, 8, 2)
    k = (k[..., 0] | (k[..., 1] << 4)).permute(*range(n), n + 1, n, n + 3, n + 2, n + 4).reshape(*lead, 8 * dim)
    v = vc.view(*lead, 2, 4, 2, p, w, 8, 2, 2, 2)
    v = v[..., 0] | (v[..., 1] << 4)  # j, t, parity, p, w, g, half, byte
    v = v.permute(*range(n), n + 3, n, n + 5, n + 1, n + 4, n + 6, n + 2, n + 7).reshape(*lead, 8 * dim)
    km = km.contiguous().view(torch.uint8).reshape(*lead, dim)
    vm = vm.contiguous().view(torch.uint8).reshape(*lead, dim)
    return torch.cat([k, km, v, vm], dim=-1)


def _unpack(tiles):
    """(..., 18 * dim) bytes -> key and value values (..., 16, dim) in binary32."""
    lead, dim = tiles.shape[:-1], tiles.shape[-1] // 18
    p, w = _planes(dim)
    n, groups = len(lead), dim // GROUP
    kb, km, vb, vm = tiles.split([8 * dim, dim, 8 * dim, dim], dim=-1)
    k = kb.reshape(*lead, p, 16, 4, w, 8).permute(*range(n), n + 1, n, n + 3, n + 2, n + 4)
    k = torch.stack([k & 15, k >> 4], dim=-1).reshape(*lead, 16, groups, GROUP)
    v = vb.reshape(*lead, p, 2, 8, 4, w, 2, 2, 2)  # p, j, g, t, w, half, parity, byte
    v = v.permute(*range(n), n + 1, n + 3, n + 6, n, n + 4, n + 2, n + 5, n + 7)
    v = torch.stack([v & 15, v >> 4], dim=-1).reshape(*lead, 16, groups, GROUP)
    got = []
    for codes, meta in ((k, km), (v, vm)):
        meta = meta.contiguous().view(torch.bfloat16).reshape(*lead, 16, groups, 2).float()
        got.append((codes.float() * meta[..., :1] + meta[..., 1:]).reshape(*lead, 16, dim))
    return got


def _quantise(x):
    """(..., dim) binary32 -> codes (..., dim) uint8, scales (..., groups, 2) bfloat16, values (..., dim)."""
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    low, high = g.amin(-1), g.amax(-1)
    scale = ((high - low) * torch.full_like(low, 1 / 15)).bfloat16().float()
    zero = low.bfloat16().float()
    fine = torch.isfinite(scale) & torch.isfinite(zero)
    scale, zero = scale.where(fine, math.nan), zero.where(fine, math.nan)
    inv = torch.where(scale >= 2.0**-126, torch.ones_like(scale) / scale, torch.zeros_like(scale))
    codes = torch.nan_to_num(torch.round((g - zero[..., None]) * inv[..., None]), nan=0.0).clamp(0, 15)
    values = codes * scale[..., None] + zero[..., None]
    return codes.to(torch.uint8).reshape(x.shape), torch.stack([scale, zero], dim=-1).bfloat16(), values.reshape(x.shape)


# -- inputs ----------------------------------------------------------------------------


def _keys(shape, gen):
    """Normal values whose channels differ in size, a few of them much larger, as keys have."""
    x = torch.randn(shape, generator=gen, device=DEV)
    size = torch.exp(0.4 * torch.randn(shape[-1], generator=gen, device=DEV))
    size[:: max(1, shape[-1] // 3)] *= 5
    return x * size


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = random.Random(seed)
    s = {"case": case}
    if case["op"] == "append":
        tokens, heads, dim, page = case["tokens"], case["kv_heads"], case["dim"], case["page"]
        pages = -(-tokens // page) * 2 + 1
        dt = DTYPES[case["dtype"]]
        # both as they lie in the rows of the fused projection's output
        both = torch.cat([_keys((tokens, heads, dim), gen), torch.randn(tokens, heads, dim, generator=gen, device=DEV)], dim=1).to(dt)
        s["k"], s["v"] = both[:, :heads], both[:, heads:]
        s["cache"] = torch.zeros(pages, heads, page // TILE, 18 * dim, dtype=torch.uint8, device=DEV)
        if tokens < 64:  # one token each of many requests: any slot
            slots = torch.randperm(pages * page, generator=gen, device=DEV)[:tokens]
        else:  # prompts: whole pages in any order, a few rows of padding between them
            order = torch.randperm(pages, generator=gen, device=DEV)[: -(-tokens // page)]
            slots = (order[:, None] * page + torch.arange(page, device=DEV)).reshape(-1)[:tokens].clone()
            slots[37::997] = -1
        s["slots"] = slots
    elif case["op"] == "attend":
        batch, queries, kv_heads, dim, page = (case[k] for k in ("batch", "queries", "kv_heads", "dim", "page"))
        dt = DTYPES[case["dtype"]]
        lens = _lengths(case)
        rng.shuffle(lens)
        need = [-(-n // page) for n in lens]
        pages, tiles = sum(need) + 1, page // TILE
        codes = []
        for x in (_keys((pages, kv_heads, tiles, 16, dim), gen), torch.randn(pages, kv_heads, tiles, 16, dim, generator=gen, device=DEV)):
            codes += list(_quantise(x)[:2])
        s["cache"] = _pack(*codes)
        order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
        table = torch.zeros(batch, max(1, max(need)), dtype=torch.int32, device=DEV)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at : at + n]
            at += n
        s["page_table"] = table
        s["lengths"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["q"] = torch.randn(batch, queries, case["heads"], dim, generator=gen, device=DEV).to(dt)
    elif case["op"] == "adapters":
        tokens, n, m, count, rank = (case[k] for k in ("tokens", "n", "m", "adapters", "rank"))
        dt = DTYPES[case["dtype"]]
        s["x"] = torch.randn(tokens, n, generator=gen, device=DEV).to(dt)
        s["y"] = torch.randn(tokens, m, generator=gen, device=DEV)
        s["A"] = (torch.randn(count, rank, n, generator=gen, device=DEV) * n**-0.5).to(dt)
        s["B"] = (torch.randn(count, m, rank, generator=gen, device=DEV) * 0.1).to(dt)
        s["adapters"] = torch.tensor(_owners(case), dtype=torch.int32, device=DEV)
        s["ranks"] = torch.tensor(_ranks(case), dtype=torch.int32, device=DEV)
        s["scales"] = 0.5 + torch.rand(count, generator=gen, device=DEV)
    else:
        rows, vocab = case["rows"], case["vocab"]
        s["logits"] = (3 * torch.randn(rows, vocab, generator=gen, device=DEV)).to(DTYPES[case["dtype"]])
        hist = _histories(case)
        rng.shuffle(hist)
        lens = torch.tensor(hist, dtype=torch.int32, device=DEV)
        # words repeat: ids go by a power law
        u = torch.rand(rows, case["history"], generator=gen, device=DEV)
        s["tokens"] = (vocab ** u - 1).long().clamp(0, vocab - 1) * 7919 % vocab
        s["lengths"] = lens
        s["prompt_lengths"] = (lens * torch.rand(rows, generator=gen, device=DEV)).to(torch.int32)
        s["repetition"] = 1 + 0.3 * torch.rand(rows, generator=gen, device=DEV)
        s["frequency"] = torch.rand(rows, generator=gen, device=DEV)
        s["presence"] = torch.rand(rows, generator=gen, device=DEV)
        per = [rng.randint(0, case["bias"]) for _ in range(rows)]
        starts = torch.tensor([0] + per).cumsum(0)
        s["bias_starts"] = starts.to(torch.int32).to(DEV)
        ids = [rng.sample(range(vocab), k) for k in per]
        s["bias_ids"] = torch.tensor([i for row in ids for i in row], dtype=torch.int64, device=DEV)
        s["bias_values"] = 4 * torch.randn(sum(per), generator=gen, device=DEV)
        s["mask"] = None
        if case["grammar"]:  # a third of the rows unconstrained, a third nearly so, a third to a few tokens
            words = -(-vocab // 32)
            bits = torch.randint(0, 2**31, (2, rows, words), generator=gen, device=DEV)
            few = bits[0] & (bits[1] >> 3) & (bits[0] >> 7) & (bits[1] >> 11)
            kind = torch.arange(rows, device=DEV)[:, None] % 3
            s["mask"] = torch.where(kind == 0, -1, torch.where(kind == 1, bits[0] | bits[1], few)).to(torch.int32)
    return s


# -- one pass --------------------------------------------------------------------------


def _append(cache, k, v, slots):
    pages, heads, tiles, size = cache.shape
    dim = size // 18
    p, w = _planes(dim)
    got = [_quantise(x.float()) for x in (k, v)]
    flat = cache.view(-1)
    keep = slots >= 0
    slot = slots[keep]
    token = slot % TILE
    page, tile = slot // (tiles * TILE), slot % (tiles * TILE) // TILE
    head = torch.arange(heads, device=DEV)
    base = ((page[:, None] * heads + head) * tiles + tile[:, None]) * size  # (tokens, heads)
    row = 32 * w
    # each side's bytes in channel order within the token, and where they go
    kb = got[0][0][keep].view(-1, heads, p, w, 4, 8, 2)
    kb = (kb[..., 0] | (kb[..., 1] << 4)).permute(0, 1, 2, 4, 3, 5).reshape(-1, heads, 8 * dim // 16)
    at = (torch.arange(p, device=DEV)[:, None] * 16 * row + torch.arange(row, device=DEV)).reshape(-1)
    flat[(base[..., None] + at + token[:, None, None] * row)] = kb
    vb = got[1][0][keep].view(-1, heads, p, w, 8, 2, 2, 2)
    vb = (vb[..., 0] | (vb[..., 1] << 4)).permute(0, 1, 2, 4, 3, 5, 6).reshape(-1, heads, 8 * dim // 16)
    steps = [16 * row, 32 * w, 8, 4, 1]  # plane, eighth of the channels, group, half, byte
    at = torch.zeros((), dtype=torch.int64, device=DEV)
    for count, step in zip((p, 8, w, 2, 2), steps):
        at = at[..., None] + torch.arange(count, device=DEV) * step
    inside = token // 8 * 256 * w + token % 8 // 2 * 8 * w + token % 2 * 2
    flat[(base[..., None] + 9 * dim + at.reshape(-1) + inside[:, None, None])] = vb
    meta = torch.arange(dim // 16, device=DEV)
    for offset, (_, scales, _) in zip((8 * dim, 17 * dim), got):
        b = scales[keep].contiguous().view(torch.uint8).reshape(-1, heads, dim // 16)
        flat[(base[..., None] + offset + token[:, None, None] * (dim // 16) + meta)] = b
    return {"cache": cache, "k": got[0][2].to(k.dtype), "v": got[1][2].to(v.dtype)}


def _attend(q, cache, page_table, lengths, window):
    batch, queries, heads, dim = q.shape
    kv_heads, tiles = cache.shape[1], cache.shape[2]
    most = page_table.shape[1] * tiles * TILE
    k, v = (x.permute(0, 2, 1, 3, 4, 5).reshape(batch, kv_heads, most, dim) for x in _unpack(cache[page_table.long()]))
    rows = q.float().view(batch, queries, kv_heads, heads // kv_heads, dim).permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, -1, dim)
    scores = (rows @ k.transpose(-1, -2)).view(batch, kv_heads, queries, heads // kv_heads, most) * dim**-0.5
    at = torch.arange(most, device=DEV)
    last = lengths.long()[:, None] - queries + torch.arange(queries, device=DEV)  # each row's own position
    seen = at <= last[..., None]
    if window:
        seen &= at > last[..., None] - window
    seen = seen[:, None, :, None]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - top.where(torch.isfinite(top), 0.0))
    total = e.sum(-1, keepdim=True)
    weights = e / total.where(total > 0, 1.0)
    out = weights.reshape(batch, kv_heads, -1, most) @ v
    out = out.view(batch, kv_heads, queries, -1, dim).permute(0, 2, 1, 3, 4).reshape(batch, queries, heads, dim)
    return out.to(q.dtype)


def _adapt(x, y, A, B, adapters, scales, ranks):
    count, rank, n = A.shape
    lane = torch.arange(rank, device=DEV)
    on = (adapters[:, None] == torch.arange(count, device=DEV)).float() * scales  # (tokens, adapters)
    h = (x.float() @ A.float().view(count * rank, n).T).view(-1, count, rank)
    h = h * on[..., None] * (lane < ranks[:, None])
    return y + h.view(-1, count * rank) @ B.float().permute(0, 2, 1).reshape(count * rank, -1)


def _logits(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    at = torch.arange(s["tokens"].shape[1], device=DEV)
    there = (at < s["lengths"][:, None]).float()
    said = there * (at >= s["prompt_lengths"][:, None])
    seen = torch.zeros(rows, vocab, device=DEV).scatter_add_(1, s["tokens"], there) > 0
    count = torch.zeros(rows, vocab, device=DEV).scatter_add_(1, s["tokens"], said)
    rep = s["repetition"][:, None].expand_as(x)
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count
    x = x - s["presence"][:, None] * (count > 0)
    starts = s["bias_starts"].long()
    row = torch.searchsorted(starts[1:], torch.arange(s["bias_ids"].numel(), device=DEV), right=True)
    x = x.index_put((row, s["bias_ids"]), s["bias_values"], accumulate=True)
    if s["mask"] is not None:
        bit = torch.arange(vocab, device=DEV)
        x = x.masked_fill((s["mask"][:, bit // 32] >> (bit % 32)) & 1 == 0, -math.inf)
    return x


def run(s: dict):
    op = s["case"]["op"]
    if op == "append":
        if own:
            k, v = _pck().kv4_append(s["cache"], s["k"], s["v"], s["slots"], values=True)
            return {"cache": s["cache"], "k": k, "v": v}
        return _append(s["cache"], s["k"], s["v"], s["slots"])
    if op == "attend":
        window = s["case"]["window"]
        if own:
            return _pck().kv4_attention(s["q"], s["cache"], s["page_table"], s["lengths"], window=window)
        return _attend(s["q"], s["cache"], s["page_table"], s["lengths"], window)
    if op == "adapters":
        args = (s["x"], s["y"], s["A"], s["B"], s["adapters"], s["scales"], s["ranks"])
        return _pck().lora_add(*args) if own else _adapt(*args)
    if own:
        return _pck().process_logits(s["logits"], tokens=s["tokens"], prompt_lengths=s["prompt_lengths"], lengths=s["lengths"],
                                     repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                                     bias_starts=s["bias_starts"], bias_ids=s["bias_ids"], bias_values=s["bias_values"], mask=s["mask"])
    return _logits(s)


def work(case: dict) -> dict:
    if case["op"] == "append":
        values = 2 * case["tokens"] * case["kv_heads"] * case["dim"]
        return {"bytes": values * (2 * ESIZE[case["dtype"]] + 9 / 16) + 8 * case["tokens"], "flops": 6 * values}
    if case["op"] == "attend":
        tokens = [min(n, case["window"] + case["queries"] - 1) if case["window"] else n for n in _lengths(case)]
        rows = case["batch"] * case["queries"] * case["heads"]
        nbytes = sum(tokens) * case["kv_heads"] * case["dim"] * 9 / 8 + 4 * rows * case["dim"] + 4 * case["batch"]
        nbytes += 4 * sum(-(-n // case["page"]) for n in tokens)
        return {"bytes": nbytes, "flops": 4 * case["queries"] * case["heads"] * case["dim"] * sum(tokens)}
    if case["op"] == "adapters":
        owners, ranks = _owners(case), _ranks(case)
        used = sum(ranks[a] for a in set(owners) if a >= 0)
        nbytes = case["tokens"] * (2 * case["n"] + 8 * case["m"] + 4) + used * 2 * (case["n"] + case["m"])
        return {"bytes": nbytes, "flops": 2 * (case["n"] + case["m"]) * sum(ranks[a] for a in owners if a >= 0)}
    size = case["rows"] * case["vocab"]
    nbytes = size * (4 + ESIZE[case["dtype"]]) + 8 * sum(_histories(case)) + 6 * case["rows"] * case["bias"]
    return {"bytes": nbytes + (size / 8 if case["grammar"] else 0), "flops": 4 * size}


# -- the same in 64 bits ---------------------------------------------------------------


def _read(tiles, dim: int):
    """Keys and values (heads, tokens, dim) in binary64 of (heads, tiles, 18 * dim) bytes, each code looked up where it lies."""
    token = torch.arange(TILE, device=DEV)[:, None]
    c = torch.arange(dim, device=DEV)
    width = min(2, dim // GROUP)  # groups of a plane
    plane, group, inner = c // (GROUP * width), c // GROUP % width, c % GROUP
    key = plane * 512 * width + token * 32 * width + inner // 16 * 8 * width + group * 8 + inner % 16 // 2
    value = plane * 512 * width + token // 8 * 256 * width + inner // 8 * 32 * width + token % 8 // 2 * 8 * width
    value = value + group * 8 + inner % 8 // 4 * 4 + token % 2 * 2 + inner % 4 // 2
    got = []
    for at, where in ((0, key), (9 * dim, value)):
        codes = (tiles[..., at + where] >> (4 * (c % 2))) & 15
        pair = tiles[..., at + 8 * dim : at + 9 * dim].contiguous().view(torch.bfloat16).double()
        pair = pair.view(*tiles.shape[:-1], TILE, dim // GROUP, 2)[..., c // GROUP, :]
        got.append((codes * pair[..., 0] + pair[..., 1]).flatten(-3, -2))
    return got


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "append":
        got = {"cache": None}
        for name in ("k", "v"):
            x = s[name].double()
            g = x.unflatten(-1, (-1, GROUP))
            low = g.min(-1, keepdim=True).values
            step = ((g.max(-1, keepdim=True).values - low) / 15).bfloat16().double()
            low = low.bfloat16().double()
            codes = ((g - low) / step.clamp(min=2.0**-126)).round().clamp(0, 15)
            got[name] = (low + step * codes).flatten(-2)
        return got
    if case["op"] == "attend":
        q, cache, table, window = s["q"].double(), s["cache"], s["page_table"].long(), case["window"]
        kv_heads, dim, queries = case["kv_heads"], case["dim"], case["queries"]
        out = torch.zeros_like(q)
        share = case["heads"] // kv_heads
        for b, n in enumerate(s["lengths"].tolist()):
            tiles = cache[table[b, : -(-n // case["page"])]].transpose(0, 1).reshape(kv_heads, -1, 18 * dim)
            for h in range(kv_heads if n else 0):
                k, v = _read(tiles[h], dim)
                for i in range(queries):
                    last = n - queries + i
                    first = max(0, last + 1 - window) if window else 0
                    if last >= first:
                        scores = k[first : last + 1] @ q[b, i, h * share : (h + 1) * share].T / math.sqrt(dim)
                        out[b, i, h * share : (h + 1) * share] = torch.softmax(scores, dim=0).T @ v[first : last + 1]
        return out
    if case["op"] == "adapters":
        out = s["y"].double()
        for a, (rank, scale) in enumerate(zip(s["ranks"].tolist(), s["scales"].tolist())):
            rows = (s["adapters"] == a).nonzero()[:, 0]
            if len(rows):
                low = s["x"][rows].double() @ s["A"][a, :rank].double().T
                out[rows] += scale * (low @ s["B"][a, :, :rank].double().T)
        return out
    x = s["logits"].double()
    starts = s["bias_starts"].tolist()
    for b, (n, p) in enumerate(zip(s["lengths"].tolist(), s["prompt_lengths"].tolist())):
        seen = s["tokens"][b, :n].unique()
        r = s["repetition"][b].double()
        x[b, seen] = torch.where(x[b, seen] > 0, x[b, seen] / r, x[b, seen] * r)
        seen, count = s["tokens"][b, p:n].unique(return_counts=True)
        x[b, seen] -= s["frequency"][b].double() * count + s["presence"][b].double()
        x[b, s["bias_ids"][starts[b] : starts[b + 1]]] += s["bias_values"][starts[b] : starts[b + 1]].double()
        if s["mask"] is not None:
            bits = (s["mask"][b, :, None] >> torch.arange(32, device=DEV)) & 1
            x[b, bits.flatten()[: case["vocab"]] == 0] = -math.inf
    return x

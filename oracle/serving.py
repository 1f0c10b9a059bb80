"""Plain statements of the serving operators (test side): the 4-bit cache's layout and formula, and
attention, adapters and logits in binary64. The reference has no counterpart; the definitions are
those of include/pck_b200.h."""

from __future__ import annotations

import math

import torch

TILE = 16
GROUP = 64


def code_places(dim: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Byte of a tile that holds each (token, channel) of the keys and of the values."""
    t = torch.arange(TILE)[:, None]
    c = torch.arange(dim)
    w = min(2, dim // GROUP)
    plane, group, i = c // (GROUP * w), c // GROUP % w, c % GROUP
    # mixed-radix numbers: (plane, token, quarter, group, byte) and (plane, j, g, t, group, half, parity, byte)
    key = (((plane * 16 + t) * 4 + i // 16) * w + group) * 8 + i % 16 // 2
    value = (((((plane * 2 + t // 8) * 8 + i // 8) * 4 + t % 8 // 2) * w + group) * 2 + i % 8 // 4) * 4 + t % 2 * 2 + i % 4 // 2
    return key, 9 * dim + value


def quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Codes (..., dim) uint8, (scale, zero) (..., groups, 2) bfloat16 and values (..., dim) binary32,
    by binary32 operations one at a time."""
    g = x.float().reshape(*x.shape[:-1], -1, GROUP)
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((high - low) * torch.tensor(1 / 15, dtype=torch.float32)).bfloat16().float()
    zero = low.bfloat16().float()
    bad = ~(torch.isfinite(scale) & torch.isfinite(zero))
    scale[bad] = math.nan
    zero[bad] = math.nan
    inv = torch.where(scale >= 2.0**-126, 1 / scale, torch.zeros_like(scale))
    codes = torch.round((g - zero) * inv)
    codes = torch.where(codes.isnan(), torch.zeros_like(codes), codes).clamp(0, 15)
    values = codes * scale + zero
    pairs = torch.cat([scale, zero], dim=-1).bfloat16()
    pairs.view(torch.int16)[pairs.isnan()] = 0x7FC0  # one NaN, whatever the conversion makes of it
    return codes.to(torch.uint8).reshape(x.shape), pairs, values.reshape(x.shape)


def cache_values(cache: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values (pages, page tokens, kv_heads, dim) in binary64 that a cache (on the CPU) holds."""
    pages, heads, tiles, size = cache.shape
    dim = size // 18
    out = []
    for where, scales in zip(code_places(dim), (8 * dim, 17 * dim), strict=True):
        codes = (cache[..., where] >> (4 * (torch.arange(dim) % 2))) & 15
        pair = cache[..., scales : scales + dim].contiguous().view(torch.bfloat16).double()
        pair = pair.view(pages, heads, tiles, TILE, dim // GROUP, 2).repeat_interleave(GROUP, dim=4)
        x = codes.double() * pair[..., 0] + pair[..., 1]
        out.append(x.permute(0, 2, 3, 1, 4).reshape(pages, tiles * TILE, heads, dim))
    return out[0], out[1]


def append(cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Writes tokens to a cache on the CPU, one byte after another; returns the values stored."""
    pages, heads, tiles, size = cache.shape
    dim = size // 18
    places = code_places(dim)
    out = []
    for side, x in enumerate((k, v)):
        codes, pairs, values = quantise(x)
        out.append(values.to(x.dtype))
        for n, slot in enumerate(slots.tolist()):
            if slot < 0:
                continue
            page, tile, t = slot // (tiles * TILE), slot % (tiles * TILE) // TILE, slot % TILE
            to = cache[page, :, tile]
            to[:, places[side][t, 0::2]] = codes[n, :, 0::2] | codes[n, :, 1::2] << 4
            per = dim // GROUP * 4
            base = (8 * dim, 17 * dim)[side] + t * per
            to[:, base : base + per] = pairs[n].reshape(heads, -1).view(torch.uint8)
    return out[0], out[1]


def attention(q: torch.Tensor, cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, scale: float | None = None,
              window: int = 0) -> tuple[torch.Tensor, torch.Tensor]:  # fmt: skip
    """(out, largest |value| that each output's row sees), both (batch, queries, heads, dim), in binary64."""
    batch, queries, heads, dim = q.shape
    keys, values = cache_values(cache)
    kv_heads, page = cache.size(1), cache.size(2) * TILE
    share = heads // kv_heads
    scale = dim**-0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    size = torch.zeros(q.shape, dtype=torch.float64)
    for b in range(batch):
        n = min(max(int(lengths[b]), 0), page_table.size(1) * page)
        rows = page_table[b, : -(-n // page)].long()
        k, v = keys[rows].reshape(-1, kv_heads, dim)[:n], values[rows].reshape(-1, kv_heads, dim)[:n]
        for t in range(queries):
            last = n - queries + t
            first = max(0, last + 1 - window) if window else 0
            if last < first:
                continue
            for h in range(heads):
                s = k[first : last + 1, h // share] @ q[b, t, h].double() * scale
                vv = v[first : last + 1, h // share]
                out[b, t, h] = torch.softmax(s, 0) @ vv
                size[b, t, h] = vv.abs().amax()
    return out, size


def lora(x, y, A, B, adapters, scales=None, ranks=None) -> tuple[torch.Tensor, torch.Tensor]:
    """(out, sum of the absolute values of all terms of each output) in binary64."""
    out, size = y.double(), y.double().abs()
    for t, a in enumerate(adapters.tolist()):
        if a < 0:
            continue
        r = A.size(1) if ranks is None else int(ranks[a])
        s = 1.0 if scales is None else float(scales[a])
        Ad, Bd, xd = A[a, :r].double(), B[a, :, :r].double(), x[t].double()
        out[t] += s * (Bd @ (Ad @ xd))
        size[t] += abs(s) * (Bd.abs() @ (Ad.abs() @ xd.abs()))
    return out, size


def process_logits(logits, tokens=None, prompt_lengths=None, lengths=None, repetition=None, frequency=None, presence=None,
                   bias_starts=None, bias_ids=None, bias_values=None, mask=None) -> torch.Tensor:  # fmt: skip
    """By binary32 operations one at a time, a token after another."""
    out = logits.float().clone()
    rows, vocab = out.shape
    one = lambda t, b, d: torch.tensor(d) if t is None else t[b]  # noqa: E731
    for b in range(rows):
        l = out[b]
        if tokens is not None:
            ids = tokens[b, : max(0, min(int(lengths[b]), tokens.size(1)))].tolist()
            p = 0 if prompt_lengths is None else int(prompt_lengths[b])
            said: dict[int, int] = {}
            for i, t in enumerate(ids):
                if 0 <= t < vocab:
                    said[t] = said.get(t, 0) + (i >= p)
            rep, freq, pres = one(repetition, b, 1.0), one(frequency, b, 0.0), one(presence, b, 0.0)
            for t, n in said.items():
                l[t] = l[t] / rep if l[t] > 0 else l[t] * rep
                if n:
                    l[t] = l[t] - freq * torch.tensor(float(n)) - pres
        if bias_starts is not None:
            last = {}
            for i in range(max(0, int(bias_starts[b])), min(int(bias_starts[b + 1]), bias_ids.numel())):
                last[int(bias_ids[i])] = bias_values[i]
            for t, value in last.items():
                if 0 <= t < vocab:
                    l[t] = l[t] + value
        if mask is not None:
            bits = (mask[b][:, None] >> torch.arange(32)) & 1
            l[bits.reshape(-1)[:vocab] == 0] = -math.inf
    return out

"""Serving operators of a decode step, between and beside the checked projections: a key/value
cache held in 4 bits and the attention that reads it, the low-rank adapters of many requests
beside a shared projection, and the penalties, biases and grammar masks that a batch's logits go
through before the sampler. The reference has no counterpart; nothing here is part of the trusted
path (the projections' checks and the membership check stay what they are).

Every function makes one call of the C ABI on the current stream, without synchronizing, and can
be captured in a CUDA graph. It calls the library directly, as the launch objects of
`pck.cuda.plan` do, to keep the host cost of a decode step low; the same calls are registered as
`torch.ops.pck.kv4_append`, `kv4_attention`, `lora_add` and `process_logits` for tracing. Shapes,
types and strides are checked here, indices in device memory by the kernels (`device_status`, bit 1).
"""

from __future__ import annotations

import functools

import torch

from pck.cuda import _lib
from pck.cuda._ext import on_device, type_name

KV4_TILE = 16
"""Tokens of a cache tile; a page holds a whole number of them."""
KV4_GROUP = 64
"""Channels of a token that share a scale and a zero."""

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # PCK_LOGITS_*
_HALF = {torch.bfloat16: 1, torch.float16: 2}


def _tensor(t: torch.Tensor, name: str, dtype: torch.dtype, device: torch.device) -> int:
    """Pointer of a contiguous tensor of the given type on the device."""
    if t.dtype is not dtype:
        raise RuntimeError(f"{name} must be {type_name(dtype)}, got {type_name(t.dtype)}")
    if t.device != device:
        raise RuntimeError(f"{name} must be on {device}")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")
    return t.data_ptr()


def _cuda(t: torch.Tensor, name: str) -> torch.device:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    return t.device


def _call(fn: str, device: torch.device, *args) -> None:
    lib = _lib.library()
    with on_device(device):
        rc = getattr(lib, fn)(*args, torch._C._cuda_getCurrentRawStream(device.index))
    if rc:
        _lib.check(rc, fn)


def _overlaps(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory spans of two tensors meet."""

    def span(t):
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride(), strict=True))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()

    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


# -- 4-bit key/value cache -------------------------------------------------------------


def kv4_cache(pages: int, page_size: int, kv_heads: int, head_dim: int, device: torch.device | str = "cuda") -> torch.Tensor:
    """An empty cache of ``pages`` pages of ``page_size`` tokens (a multiple of 16): uint8
    (pages, kv_heads, page_size / 16, 18 * head_dim), 1.125 bytes for a key and value element.
    ``head_dim`` is 64, 128 or 256. include/pck_b200.h gives the layout."""
    if page_size < KV4_TILE or page_size % KV4_TILE:
        raise ValueError(f"page_size must be a positive multiple of {KV4_TILE}, got {page_size}")
    if head_dim not in (64, 128, 256):
        raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
    if pages < 1 or kv_heads < 1:
        raise ValueError("need pages >= 1 and kv_heads >= 1")
    return torch.zeros(pages, kv_heads, page_size // KV4_TILE, 18 * head_dim, dtype=torch.uint8, device=device)


def _cache(cache: torch.Tensor, device: torch.device) -> tuple[int, int, int, int]:
    """(pages, kv_heads, tiles of a page, dim) of a cache."""
    if cache.dim() != 4 or cache.dtype is not torch.uint8 or cache.size(3) not in (1152, 2304, 4608):
        raise RuntimeError("cache must be uint8 (pages, kv_heads, page_size / 16, 18 * dim) with dim 64, 128 or 256")
    if cache.device != device or not cache.is_contiguous():
        raise RuntimeError(f"cache must be contiguous on {device}")
    pages, heads, tiles, size = cache.shape
    return pages, heads, tiles, size // 18


def kv4_append(cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
               values: bool = False) -> tuple[torch.Tensor, torch.Tensor] | None:  # fmt: skip
    """Quantise the keys and values ``k``, ``v`` (tokens, kv_heads, dim; float32, bfloat16 or
    float16, any token and head strides, e.g. views of a fused projection's output) to 4 bits and
    write them to their ``slots`` (tokens,) int64 of the ``cache``: page * page_size + place in the
    page, each slot once, negative to leave a token out.

    Each group of 64 channels keeps a bfloat16 scale and zero (its range over 15, its minimum). A
    group that holds a NaN or an infinity is stored, and read back, as NaN. With ``values`` the
    call returns (k, v) as the cache holds them, in the input's type, left-out tokens included: an
    attention over the fresh prompt with these sees what later decode steps will see."""
    device = _cuda(k, "k")
    pages, heads, tiles, dim = _cache(cache, device)
    code = _TYPES.get(k.dtype)
    if code is None or v.dtype is not k.dtype:
        raise RuntimeError("k and v must both be float32, bfloat16 or float16")
    if k.dim() != 3 or k.shape != v.shape or k.size(1) != heads or k.size(2) != dim:
        raise RuntimeError(f"expected k and v of shape (tokens, {heads}, {dim}), got {list(k.shape)} and {list(v.shape)}")
    if v.device != device or k.stride(2) != 1 or v.stride(2) != 1:
        raise RuntimeError(f"k and v must be on {device} with unit channel stride")
    tokens = k.size(0)
    if slots.dim() != 1 or slots.size(0) != tokens:
        raise RuntimeError(f"slots must have shape ({tokens},)")
    out = (torch.empty(k.shape, dtype=k.dtype, device=device), torch.empty(k.shape, dtype=k.dtype, device=device)) if values else None
    _call("pck_kv4_append", device, cache.data_ptr(), pages, heads, tiles, dim, k.data_ptr(), v.data_ptr(), code, tokens,
          k.stride(0), k.stride(1), v.stride(0), v.stride(1), _tensor(slots, "slots", torch.int64, device),
          out[0].data_ptr() if out else None, out[1].data_ptr() if out else None)  # fmt: skip
    return out


@functools.lru_cache(maxsize=4096)
def _scratch_bytes(device: int, batch: int, queries: int, heads: int, kv_heads: int, dim: int, max_tokens: int) -> int:
    with on_device(torch.device("cuda", device)):
        return _lib.library().pck_kv4_attention_scratch(batch, queries, heads, kv_heads, dim, max_tokens)


def kv4_attention(q: torch.Tensor, cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                  scale: float | None = None, window: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:  # fmt: skip
    """softmax(scale * q k^T) v of the query tokens ``q`` (batch, queries, heads, dim), or (batch,
    heads, dim) for one token a request, bfloat16 or float16, over a 4-bit ``cache``; the result
    has q's shape and type.

    Request b holds ``lengths[b]`` (int32) tokens, its query tokens the last of them (append them
    first), in the pages ``page_table[b, 0], page_table[b, 1], ...`` (int32; entries past the
    length are not read). Query token t sees tokens up to its own; with ``window`` > 0 the last
    ``window`` of those. One that sees nothing (an empty request) gives zeros. heads is a multiple
    of the cache's kv_heads; ``scale`` is dim**-0.5 by default."""
    device = _cuda(q, "q")
    pages, kv_heads, tiles, dim = _cache(cache, device)
    code = _HALF.get(q.dtype)
    if code is None:
        raise RuntimeError(f"q must be bfloat16 or float16, got {type_name(q.dtype)}")
    shape = q.shape
    if q.dim() == 3:
        q = q.unsqueeze(1)
    if q.dim() != 4 or q.size(3) != dim or q.size(2) % kv_heads or q.size(2) == 0 or q.size(1) == 0:
        raise RuntimeError(f"expected q of shape (batch, queries, heads, {dim}) with heads a multiple of {kv_heads}, got {list(shape)}")
    if q.stride(3) != 1:
        raise RuntimeError("q must have unit channel stride")
    batch, queries, heads = q.size(0), q.size(1), q.size(2)
    if page_table.dim() != 2 or page_table.size(0) != batch or lengths.dim() != 1 or lengths.size(0) != batch:
        raise RuntimeError(f"page_table must have shape ({batch}, pages) and lengths ({batch},)")
    if page_table.dtype is not torch.int32 or page_table.device != device or (page_table.size(1) > 1 and page_table.stride(1) != 1):
        raise RuntimeError(f"page_table must be Int on {device} with unit column stride")
    if window < 0:
        raise RuntimeError("window must be 0 (none) or positive")
    table_pages = page_table.size(1)
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=device)
    elif out.shape != shape:
        raise RuntimeError(f"out must have shape {list(shape)}")
    elif _overlaps(out, q) or _overlaps(out, cache):
        raise RuntimeError("out must not share memory with q or the cache")
    bytes_ = _scratch_bytes(device.index, batch, queries, heads, kv_heads, dim, table_pages * tiles * KV4_TILE)
    scratch = torch.empty(bytes_, dtype=torch.uint8, device=device) if bytes_ > 0 else None
    _call("pck_kv4_attention", device, q.data_ptr(), code, batch, queries, heads, dim, q.stride(0), q.stride(1), q.stride(2),
          cache.data_ptr(), pages, kv_heads, tiles, page_table.data_ptr(), max(page_table.stride(0), table_pages), table_pages,
          _tensor(lengths, "lengths", torch.int32, device), dim**-0.5 if scale is None else float(scale), window,
          _tensor(out, "out", q.dtype, device), scratch.data_ptr() if scratch is not None else None, bytes_)  # fmt: skip
    return out


# -- low-rank adapters -----------------------------------------------------------------


def lora_add(x: torch.Tensor, y: torch.Tensor, A: torch.Tensor, B: torch.Tensor, adapters: torch.Tensor,
             scales: torch.Tensor | None = None, ranks: torch.Tensor | None = None,
             out: torch.Tensor | None = None) -> torch.Tensor:  # fmt: skip
    """y + s_a B_a (A_a x) for every row, each with an adapter of its own: the adapters of many
    requests beside the shared projection y = W x (`gemv_tc`, `gemv_coalesced`).

    ``x`` (tokens, n) bfloat16 or float16 is the projection's input, ``y`` (tokens, m) float32 its
    output, ``A`` (count, rank, n) and ``B`` (count, m, rank) the adapters in x's type, ``adapters``
    (tokens,) int32 each row's adapter (negative: none, the row is y). ``scales`` (count,) float32
    (default 1) multiplies, ``ranks`` (count,) int32 gives an adapter's own rank (at most the
    stored one; the rest is not used). rank is at most 256. The result is ``out`` (float32; may be
    y) or a new tensor. A checked y must have been decided before it is overwritten."""
    device = _cuda(x, "x")
    code = _HALF.get(x.dtype)
    if code is None or A.dtype is not x.dtype or B.dtype is not x.dtype:
        raise RuntimeError("x, A and B must all be bfloat16 or all float16")
    if x.dim() != 2 or y.dim() != 2 or A.dim() != 3 or B.dim() != 3:
        raise RuntimeError("expected x (tokens, n), y (tokens, m), A (count, rank, n) and B (count, m, rank)")
    tokens, n = x.shape
    m = y.size(1)
    count, rank = A.size(0), A.size(1)
    if y.size(0) != tokens or A.size(2) != n or tuple(B.shape) != (count, m, rank):
        raise RuntimeError(f"expected x (tokens, n), y (tokens, m), A (count, rank, n) and B (count, m, rank), got {list(x.shape)}, "
                           f"{list(y.shape)}, {list(A.shape)} and {list(B.shape)}")  # fmt: skip
    if y.dtype is not torch.float32 or y.device != device:
        raise RuntimeError(f"y must be Float on {device}")
    if (n > 1 and x.stride(1) != 1) or (m > 1 and y.stride(1) != 1):
        raise RuntimeError("x and y must have unit column stride")
    if tuple(adapters.shape) != (tokens,):
        raise RuntimeError(f"adapters must have shape ({tokens},)")
    for t, name in ((scales, "scales"), (ranks, "ranks")):
        if t is not None and tuple(t.shape) != (count,):
            raise RuntimeError(f"{name} must have shape ({count},)")
    if out is None:
        out = torch.empty((tokens, m), dtype=torch.float32, device=device)
    else:
        if tuple(out.shape) != (tokens, m) or out.dtype is not torch.float32 or out.device != device or (m > 1 and out.stride(1) != 1):
            raise RuntimeError(f"out must be Float ({tokens}, {m}) on {device} with unit column stride")
        if tokens > 1 and out.stride(0) < m:
            raise RuntimeError("out must not overlap itself")
        same = out.data_ptr() == y.data_ptr() and out.stride() == y.stride()
        if (not same and _overlaps(out, y)) or any(_overlaps(out, t) for t in (x, A, B, adapters)):
            raise RuntimeError("out must be y itself or share no memory with the inputs")
    _call("pck_lora_add", device, x.data_ptr(), code, tokens, n, max(x.stride(0), n), y.data_ptr(), m, max(y.stride(0), m),
          _tensor(A, "A", x.dtype, device), _tensor(B, "B", x.dtype, device), count, rank,
          _tensor(adapters, "adapters", torch.int32, device),
          None if scales is None else _tensor(scales, "scales", torch.float32, device),
          None if ranks is None else _tensor(ranks, "ranks", torch.int32, device), out.data_ptr(), max(out.stride(0), m))  # fmt: skip
    return out


# -- logits ----------------------------------------------------------------------------


def process_logits(logits: torch.Tensor, *, tokens: torch.Tensor | None = None, prompt_lengths: torch.Tensor | None = None,
                   lengths: torch.Tensor | None = None, repetition: torch.Tensor | None = None,
                   frequency: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                   bias_starts: torch.Tensor | None = None, bias_ids: torch.Tensor | None = None,
                   bias_values: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:  # fmt: skip
    """The logits (rows, vocab; float32, bfloat16 or float16) that a batch's sampler and membership
    check take, in float32: penalties for repeated tokens, then biases, then the grammar mask.

    ``tokens`` (rows, max_tokens) int64 with ``lengths`` (rows,) int32 is each row's history, the
    first ``prompt_lengths`` (rows,) int32 of it the prompt (default none), the rest put out by the
    model. ``repetition`` (rows,) float32 divides positive and multiplies other logits of every
    token of the history, ``frequency`` is subtracted for every time a token was put out,
    ``presence`` once. ``bias_starts`` (rows + 1,) int32 gives each row's range of ``bias_ids``
    (int64) and ``bias_values`` (float32), added to those tokens; of entries that name one token
    twice the last counts. ``mask`` (rows, ceil(vocab / 32)) int32: a token whose bit is 0 becomes
    -inf, whatever its logit was. Ids outside the vocabulary are skipped. ``out`` may be the logits
    themselves (float32)."""
    device = _cuda(logits, "logits")
    code = _TYPES.get(logits.dtype)
    if code is None:
        raise RuntimeError(f"logits must be float32, bfloat16 or float16, got {type_name(logits.dtype)}")
    if logits.dim() != 2 or logits.size(1) == 0:
        raise RuntimeError("expected logits of shape (rows, vocab)")
    rows, vocab = logits.shape
    if vocab > 1 and logits.stride(1) != 1:
        raise RuntimeError("logits must have unit column stride")
    history = [None, 0, 0]
    if tokens is not None:
        if tokens.dim() != 2 or tokens.size(0) != rows or tokens.dtype is not torch.int64 or tokens.device != device:
            raise RuntimeError(f"tokens must be Long ({rows}, max_tokens) on {device}")
        if tokens.size(1) > 1 and tokens.stride(1) != 1:
            raise RuntimeError("tokens must have unit column stride")
        if lengths is None:
            raise RuntimeError("tokens need lengths")
        history = [tokens.data_ptr() if tokens.numel() else None, max(tokens.stride(0), tokens.size(1)), tokens.size(1)]
    elif any(t is not None for t in (lengths, prompt_lengths, repetition, frequency, presence)):
        raise RuntimeError("lengths and penalties need tokens")
    per_row = []
    for t, name, dtype in ((prompt_lengths, "prompt_lengths", torch.int32), (lengths, "lengths", torch.int32),
                           (repetition, "repetition", torch.float32), (frequency, "frequency", torch.float32),
                           (presence, "presence", torch.float32)):  # fmt: skip
        if t is None or history[0] is None:
            per_row.append(None)
            continue
        if tuple(t.shape) != (rows,):
            raise RuntimeError(f"{name} must have shape ({rows},)")
        per_row.append(_tensor(t, name, dtype, device))
    bias = [None, None, None, 0]
    if bias_starts is not None:
        if bias_ids is None or bias_values is None:
            raise RuntimeError("bias_starts needs bias_ids and bias_values")
        if tuple(bias_starts.shape) != (rows + 1,) or bias_ids.dim() != 1 or bias_ids.shape != bias_values.shape:
            raise RuntimeError(f"bias_starts must have shape ({rows + 1},), bias_ids and bias_values one length")
        bias = [_tensor(bias_starts, "bias_starts", torch.int32, device), _tensor(bias_ids, "bias_ids", torch.int64, device),
                _tensor(bias_values, "bias_values", torch.float32, device), bias_ids.numel()]  # fmt: skip
        if bias[3] == 0:
            bias = [None, None, None, 0]
    elif bias_ids is not None or bias_values is not None:
        raise RuntimeError("biases need bias_starts")
    words = -(-vocab // 32)
    mask_ptr, mask_stride = None, 0
    if mask is not None:
        if tuple(mask.shape) != (rows, words) or mask.dtype is not torch.int32 or mask.device != device:
            raise RuntimeError(f"mask must be Int ({rows}, {words}) on {device}")
        if words > 1 and mask.stride(1) != 1:
            raise RuntimeError("mask must have unit column stride")
        mask_ptr, mask_stride = mask.data_ptr(), max(mask.stride(0), words)
    if out is None:
        out = torch.empty((rows, vocab), dtype=torch.float32, device=device)
    else:
        if tuple(out.shape) != (rows, vocab) or out.dtype is not torch.float32 or out.device != device:
            raise RuntimeError(f"out must be Float ({rows}, {vocab}) on {device}")
        if (vocab > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < vocab):
            raise RuntimeError("out must have unit column stride and rows of their own")
        same = out.data_ptr() == logits.data_ptr() and out.stride() == logits.stride() and out.dtype is logits.dtype
        inputs = [t for t in (tokens, bias_ids, bias_values, mask) if t is not None]
        if (not same and _overlaps(out, logits)) or any(_overlaps(out, t) for t in inputs):
            raise RuntimeError("out must be the logits themselves or share no memory with the inputs")
    _call("pck_process_logits", device, logits.data_ptr(), code, rows, vocab, max(logits.stride(0), vocab), *history, *per_row,
          *bias, mask_ptr, mask_stride, out.data_ptr(), max(out.stride(0), vocab))  # fmt: skip
    return out


# -- the same calls as PyTorch operators -----------------------------------------------


@torch.library.custom_op("pck::kv4_append", mutates_args=("cache",))
def _kv4_append_op(cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    kv4_append(cache, k, v, slots)


@_kv4_append_op.register_fake
def _(cache, k, v, slots):
    return None


@torch.library.custom_op("pck::kv4_attention", mutates_args=())
def _kv4_attention_op(q: torch.Tensor, cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                      scale: float | None = None, window: int = 0) -> torch.Tensor:  # fmt: skip
    return kv4_attention(q, cache, page_table, lengths, scale, window)


@_kv4_attention_op.register_fake
def _(q, cache, page_table, lengths, scale=None, window=0):
    return q.new_empty(q.shape)


@torch.library.custom_op("pck::lora_add", mutates_args=())
def _lora_add_op(x: torch.Tensor, y: torch.Tensor, A: torch.Tensor, B: torch.Tensor, adapters: torch.Tensor,
                 scales: torch.Tensor | None = None, ranks: torch.Tensor | None = None) -> torch.Tensor:  # fmt: skip
    return lora_add(x, y, A, B, adapters, scales, ranks)


@_lora_add_op.register_fake
def _(x, y, A, B, adapters, scales=None, ranks=None):
    return y.new_empty(y.shape)


@torch.library.custom_op("pck::process_logits", mutates_args=())
def _process_logits_op(logits: torch.Tensor, tokens: torch.Tensor | None = None, prompt_lengths: torch.Tensor | None = None,
                       lengths: torch.Tensor | None = None, repetition: torch.Tensor | None = None,
                       frequency: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                       bias_starts: torch.Tensor | None = None, bias_ids: torch.Tensor | None = None,
                       bias_values: torch.Tensor | None = None, mask: torch.Tensor | None = None) -> torch.Tensor:  # fmt: skip
    return process_logits(logits, tokens=tokens, prompt_lengths=prompt_lengths, lengths=lengths, repetition=repetition,
                          frequency=frequency, presence=presence, bias_starts=bias_starts, bias_ids=bias_ids,
                          bias_values=bias_values, mask=mask)  # fmt: skip


@_process_logits_op.register_fake
def _(logits, tokens=None, prompt_lengths=None, lengths=None, repetition=None, frequency=None, presence=None, bias_starts=None,
      bias_ids=None, bias_values=None, mask=None):  # fmt: skip
    return logits.new_empty(logits.shape, dtype=torch.float32)


OPS = ("kv4_append", "kv4_attention", "lora_add", "process_logits")

"""Serving operators of a decode step, between and beside the checked projections: a key/value
cache held in 4 bits and the attention that reads it, the low-rank adapters of many requests
beside a shared projection, and the penalties, biases and grammar masks that a batch's logits go
through before the sampler. The reference has no counterpart; nothing here is part of the trusted
path (the projections' checks and the membership check stay what they are).

Every function makes one call of the C ABI on the current stream, without synchronizing, and can
be captured in a CUDA graph. It calls the library directly, as the launch objects of
`pck.cuda.plan` do, to keep the host cost of a decode step low. For tracing, `torch.ops.pck.kv4_append`,
`kv4_attention`, `lora_add` and `process_logits` are the same operators without `out`, and the append
without `values`. Shapes, types and strides are checked here, indices in device memory by the kernels
(`device_status`, bit 1).
"""

from __future__ import annotations

import functools

import torch

from pck.cuda import _lib
from pck.cuda._ext import type_name

KV4_TILE = 16
"""Tokens of a cache tile; a page holds a whole number of them."""
KV4_GROUP = 64
"""Channels of a token that share a scale and a zero."""

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # PCK_LOGITS_*
_HALF = {torch.bfloat16: 1, torch.float16: 2}
_CONTIGUOUS = torch.contiguous_format

# A decode step makes many of these calls, each shorter on the GPU than a dozen Python calls, so the
# checks use the cheapest accessors and the arguments travel as one packed descriptor.


def _tensor(t: torch.Tensor, name: str, dtype: torch.dtype, index: int) -> int:
    """Pointer of a contiguous tensor of the given type on CUDA device `index`."""
    if t.dtype is not dtype:
        raise RuntimeError(f"{name} must be {type_name(dtype)}, got {type_name(t.dtype)}")
    if t.get_device() != index:
        raise RuntimeError(f"{name} must be on cuda:{index}")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")
    return t.data_ptr()


def _per_row(t: torch.Tensor | None, name: str, dtype: torch.dtype, index: int, count: int) -> int:
    """Pointer of one value per row (0 for none)."""
    if t is None:
        return 0
    if t.shape != (count,):
        raise RuntimeError(f"{name} must have shape ({count},)")
    return _tensor(t, name, dtype, index)


def _row_stride(stride: int, rows: int, width: int) -> int:
    """What the library is told of a row stride: the tensor's own (0 for expanded rows, which the kernels
    read as they are; it refuses rows that overlap in part), but a whole row where there is only one."""
    return stride if rows > 1 else width


def _index(t: torch.Tensor, name: str) -> int:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    return t.get_device()


@functools.cache
def _entry(name: str):
    return getattr(_lib.library(), name)


def _call(name: str, index: int, descriptor: bytes) -> None:
    if torch._C._cuda_getDevice() == index:
        rc = _entry(name)(descriptor, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = _entry(name)(descriptor, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc, name)


def _overlaps(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory spans of two tensors meet."""

    def span(t):
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride(), strict=True))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()

    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _same_rows(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two matrices of one shape are the same memory, row for row."""
    return a.data_ptr() == b.data_ptr() and a.dtype is b.dtype and (a.shape[0] <= 1 or a.stride() == b.stride())


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


def _cache(cache: torch.Tensor, index: int) -> tuple[int, int, int, int]:
    """(pages, kv_heads, tiles of a page, dim) of a cache."""
    shape = cache.shape
    if len(shape) != 4 or cache.dtype is not torch.uint8 or shape[3] not in (1152, 2304, 4608):
        raise RuntimeError("cache must be uint8 (pages, kv_heads, page_size / 16, 18 * dim) with dim 64, 128 or 256")
    if cache.get_device() != index or not cache.is_contiguous():
        raise RuntimeError(f"cache must be contiguous on cuda:{index}")
    pages, heads, tiles, size = shape
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
    index = _index(k, "k")
    pages, heads, tiles, dim = _cache(cache, index)
    code = _TYPES.get(k.dtype)
    if code is None or v.dtype is not k.dtype:
        raise RuntimeError("k and v must both be float32, bfloat16 or float16")
    shape = k.shape
    if len(shape) != 3 or v.shape != shape or shape[1] != heads or shape[2] != dim:
        raise RuntimeError(f"expected k and v of shape (tokens, {heads}, {dim}), got {list(shape)} and {list(v.shape)}")
    (kt, kh, kc), (vt, vh, vc) = k.stride(), v.stride()
    if v.get_device() != index or kc != 1 or vc != 1:
        raise RuntimeError(f"k and v must be on cuda:{index} with unit channel stride")
    tokens = shape[0]
    slot_ptr = _per_row(slots, "slots", torch.int64, index, tokens)
    out = None
    k_ptr = v_ptr = 0
    if values:
        out = (torch.empty_like(k, memory_format=_CONTIGUOUS), torch.empty_like(v, memory_format=_CONTIGUOUS))
        k_ptr, v_ptr = out[0].data_ptr(), out[1].data_ptr()
    _call("pck_kv4_append", index, _lib.KV4_APPEND.pack(
        cache.data_ptr(), pages, heads, tiles, dim, k.data_ptr(), v.data_ptr(), code, tokens, kt, kh, vt, vh, slot_ptr, k_ptr,
        v_ptr))  # fmt: skip
    return out


@functools.lru_cache(maxsize=4096)
def _scratch_bytes(index: int, batch: int, queries: int, heads: int, kv_heads: int, dim: int, max_tokens: int) -> int:
    with torch.cuda.device(index):
        return _entry("pck_kv4_attention_scratch")(batch, queries, heads, kv_heads, dim, max_tokens)


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
    index = _index(q, "q")
    pages, kv_heads, tiles, dim = _cache(cache, index)
    dtype = q.dtype
    code = _HALF.get(dtype)
    if code is None:
        raise RuntimeError(f"q must be bfloat16 or float16, got {type_name(dtype)}")
    shape, strides = q.shape, q.stride()
    if len(shape) == 4:
        batch, queries, heads, channels = shape
        qb, qt, qh, qc = strides
    elif len(shape) == 3:
        batch, heads, channels = shape
        queries = 1
        qb, qh, qc = strides
        qt = 0
    else:
        heads = channels = 0
    if channels != dim or heads == 0 or heads % kv_heads or queries == 0:
        raise RuntimeError(f"expected q of shape (batch, queries, heads, {dim}) with heads a multiple of {kv_heads}, got {list(shape)}")
    if qc != 1:
        raise RuntimeError("q must have unit channel stride")
    table_shape = page_table.shape
    if len(table_shape) != 2 or table_shape[0] != batch or lengths.shape != (batch,):
        raise RuntimeError(f"page_table must have shape ({batch}, pages) and lengths ({batch},)")
    table_pages = table_shape[1]
    table_stride, column = page_table.stride()
    if page_table.dtype is not torch.int32 or page_table.get_device() != index or (table_pages > 1 and column != 1):
        raise RuntimeError(f"page_table must be Int on cuda:{index} with unit column stride")
    if window < 0:
        raise RuntimeError("window must be 0 (none) or positive")
    if out is None:
        out = torch.empty_like(q, memory_format=_CONTIGUOUS)
    elif out.shape != shape:
        raise RuntimeError(f"out must have shape {list(shape)}")
    elif any(_overlaps(out, t) for t in (q, cache, page_table, lengths)):
        raise RuntimeError("out must not share memory with the inputs")
    size = _scratch_bytes(index, batch, queries, heads, kv_heads, dim, table_pages * tiles * KV4_TILE)
    scratch = cache.new_empty((size,)) if size > 0 else None
    _call("pck_kv4_attention", index, _lib.KV4_ATTENTION.pack(
        q.data_ptr(), code, batch, queries, heads, dim, qb, qt, qh, cache.data_ptr(), pages, kv_heads, tiles,
        page_table.data_ptr(), _row_stride(table_stride, batch, table_pages), table_pages,
        _tensor(lengths, "lengths", torch.int32, index), dim**-0.5 if scale is None else scale, window,
        _tensor(out, "out", dtype, index), 0 if scratch is None else scratch.data_ptr(), size))  # fmt: skip
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
    index = _index(x, "x")
    dtype = x.dtype
    code = _HALF.get(dtype)
    if code is None or A.dtype is not dtype or B.dtype is not dtype:
        raise RuntimeError("x, A and B must all be bfloat16 or all float16")
    x_shape, y_shape, a_shape = x.shape, y.shape, A.shape
    if len(x_shape) != 2 or len(y_shape) != 2 or len(a_shape) != 3:
        raise RuntimeError("expected x (tokens, n), y (tokens, m), A (count, rank, n) and B (count, m, rank)")
    tokens, n = x_shape
    m = y_shape[1]
    count, rank, _ = a_shape
    if y_shape[0] != tokens or a_shape[2] != n or B.shape != (count, m, rank):
        raise RuntimeError(f"expected x (tokens, n), y (tokens, m), A (count, rank, n) and B (count, m, rank), got {list(x_shape)}, "
                           f"{list(y_shape)}, {list(a_shape)} and {list(B.shape)}")  # fmt: skip
    if y.dtype is not torch.float32 or y.get_device() != index:
        raise RuntimeError(f"y must be Float on cuda:{index}")
    (x_stride, x_column), (y_stride, y_column) = x.stride(), y.stride()
    if (n > 1 and x_column != 1) or (m > 1 and y_column != 1):
        raise RuntimeError("x and y must have unit column stride")
    if out is None:
        out = torch.empty_like(y, memory_format=_CONTIGUOUS)
        out_stride = m
    else:
        if out.shape != y_shape or out.dtype is not torch.float32 or out.get_device() != index or (m > 1 and out.stride(1) != 1):
            raise RuntimeError(f"out must be Float ({tokens}, {m}) on cuda:{index} with unit column stride")
        out_stride = out.stride(0)
        if tokens > 1 and out_stride < m:
            raise RuntimeError("out must not overlap itself")
        same = _same_rows(out, y)
        inputs = [t for t in (x, A, B, adapters, scales, ranks) if t is not None]
        if (not same and _overlaps(out, y)) or any(_overlaps(out, t) for t in inputs):
            raise RuntimeError("out must be y itself or share no memory with the inputs")
    _call("pck_lora_add", index, _lib.LORA.pack(
        x.data_ptr(), code, tokens, n, _row_stride(x_stride, tokens, n), y.data_ptr(), m, _row_stride(y_stride, tokens, m),
        _tensor(A, "A", dtype, index), _tensor(B, "B", dtype, index), count, rank,
        _per_row(adapters, "adapters", torch.int32, index, tokens), _per_row(scales, "scales", torch.float32, index, count),
        _per_row(ranks, "ranks", torch.int32, index, count), out.data_ptr(), _row_stride(out_stride, tokens, m)))  # fmt: skip
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
    index = _index(logits, "logits")
    code = _TYPES.get(logits.dtype)
    if code is None:
        raise RuntimeError(f"logits must be float32, bfloat16 or float16, got {type_name(logits.dtype)}")
    shape = logits.shape
    if len(shape) != 2 or shape[1] == 0:
        raise RuntimeError("expected logits of shape (rows, vocab)")
    rows, vocab = shape
    stride, column = logits.stride()
    if vocab > 1 and column != 1:
        raise RuntimeError("logits must have unit column stride")
    history = history_stride = most = prompts = counts = rep = freq = pres = 0
    if tokens is not None:
        t_shape = tokens.shape
        if len(t_shape) != 2 or t_shape[0] != rows or tokens.dtype is not torch.int64 or tokens.get_device() != index:
            raise RuntimeError(f"tokens must be Long ({rows}, max_tokens) on cuda:{index}")
        most = t_shape[1]
        history_stride, column = tokens.stride()
        if most > 1 and column != 1:
            raise RuntimeError("tokens must have unit column stride")
        if lengths is None:
            raise RuntimeError("tokens need lengths")
        history_stride = _row_stride(history_stride, rows, most)
        prompts = _per_row(prompt_lengths, "prompt_lengths", torch.int32, index, rows)
        counts = _per_row(lengths, "lengths", torch.int32, index, rows)
        rep = _per_row(repetition, "repetition", torch.float32, index, rows)
        freq = _per_row(frequency, "frequency", torch.float32, index, rows)
        pres = _per_row(presence, "presence", torch.float32, index, rows)
        if most:
            history = tokens.data_ptr()
        else:
            prompts = counts = rep = freq = pres = 0
    elif lengths is not None or prompt_lengths is not None or repetition is not None or frequency is not None or presence is not None:
        raise RuntimeError("lengths and penalties need tokens")
    starts = ids = amounts = biases = 0
    if bias_starts is not None:
        if bias_ids is None or bias_values is None:
            raise RuntimeError("bias_starts needs bias_ids and bias_values")
        b_shape = bias_ids.shape
        if bias_starts.shape != (rows + 1,) or len(b_shape) != 1 or bias_values.shape != b_shape:
            raise RuntimeError(f"bias_starts must have shape ({rows + 1},), bias_ids and bias_values one length")
        starts = _tensor(bias_starts, "bias_starts", torch.int32, index)
        ids = _tensor(bias_ids, "bias_ids", torch.int64, index)
        amounts = _tensor(bias_values, "bias_values", torch.float32, index)
        biases = b_shape[0]
        if biases == 0:
            starts = 0
    elif bias_ids is not None or bias_values is not None:
        raise RuntimeError("biases need bias_starts")
    mask_ptr = mask_stride = 0
    if mask is not None:
        words = -(-vocab // 32)
        if mask.shape != (rows, words) or mask.dtype is not torch.int32 or mask.get_device() != index:
            raise RuntimeError(f"mask must be Int ({rows}, {words}) on cuda:{index}")
        mask_stride, column = mask.stride()
        if words > 1 and column != 1:
            raise RuntimeError("mask must have unit column stride")
        mask_ptr, mask_stride = mask.data_ptr(), _row_stride(mask_stride, rows, words)
    if out is None:
        out = torch.empty_like(logits, dtype=torch.float32, memory_format=_CONTIGUOUS)
        out_stride = vocab
    else:
        if out.shape != shape or out.dtype is not torch.float32 or out.get_device() != index:
            raise RuntimeError(f"out must be Float ({rows}, {vocab}) on cuda:{index}")
        out_stride, column = out.stride()
        if (vocab > 1 and column != 1) or (rows > 1 and out_stride < vocab):
            raise RuntimeError("out must have unit column stride and rows of their own")
        same = _same_rows(out, logits)
        inputs = [t for t in (tokens, prompt_lengths, lengths, repetition, frequency, presence, bias_starts, bias_ids, bias_values,
                              mask) if t is not None]  # fmt: skip
        if (not same and _overlaps(out, logits)) or any(_overlaps(out, t) for t in inputs):
            raise RuntimeError("out must be the logits themselves or share no memory with the inputs")
        out_stride = _row_stride(out_stride, rows, vocab)
    _call("pck_process_logits", index, _lib.LOGITS.pack(
        logits.data_ptr(), code, rows, vocab, _row_stride(stride, rows, vocab), history, history_stride, most, prompts, counts,
        rep, freq, pres, starts, ids, amounts, biases, mask_ptr, mask_stride, out.data_ptr(), out_stride))  # fmt: skip
    return out


# -- the operators as PyTorch custom operators (no `out`, no `values`) -------------------


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

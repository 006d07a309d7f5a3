"""The INT8 prefix cache of one layer and the attention that reads it.

The reference keeps the prefix's K/V in bf16 (QwenImage21KVLayerCache,
transformer_qwenimage21.py:56-74). Here a cached row (one token of one head)
is 128 INT8 codes and an fp32 scale: half the memory, and half the bytes an
attention over it streams. `cached_attention` multiplies the codes as f16 rows,
exact or scaled by powers of two; `kv_cache_read` gives bf16 rows to an attention
of another kind.
"""
from __future__ import annotations

import struct

import torch

from .. import _lib

HEAD_DIM = 128
# stride arguments (int64[]) as bytes
_strides6 = struct.Struct("6q").pack
_strides12 = struct.Struct("12q").pack
_NO_ROWS = (0,) * 6


class _Held:
    """What the host knows of a cache's requests: per request, the most tokens
    that it may hold and whether it holds just that; `changes` counts updates."""

    def __init__(self, extent: int, batch: int):
        self.counts, self.changes = [(extent, False)] * batch, 0


class QuantizedKV:
    """K and V of up to `capacity` tokens of each of `batch` requests.

    k_codes, v_codes: int8 [batch, kv_heads, capacity, 128]; k_scales,
    v_scales: float32 [batch, kv_heads, capacity]; lengths: int32 [batch] on
    the device, the tokens each request holds. The host counts them too, in one
    list that a cache shares with its parts (select), so that a write through any
    of them is known to all; `extent` is the longest request's count (the key
    columns of a mask). What the host cannot count is set: `cache.extent = n`
    says that each of its requests holds up to n tokens, e.g. the most that
    replays of a captured append may reach."""

    def __init__(self, batch: int, kv_heads: int, capacity: int, device="cuda"):
        dev = torch.device(device)
        shape = (batch, kv_heads, capacity)
        self._bind(torch.zeros(*shape, HEAD_DIM, dtype=torch.int8, device=dev),
                   torch.zeros(*shape, HEAD_DIM, dtype=torch.int8, device=dev),
                   torch.zeros(shape, dtype=torch.float32, device=dev),
                   torch.zeros(shape, dtype=torch.float32, device=dev),
                   torch.zeros(batch, dtype=torch.int32, device=dev),
                   torch.zeros(batch, dtype=torch.int32, device=dev), 0)
        self._count(0)

    @classmethod
    def from_tensors(cls, k_codes, v_codes, k_scales, v_scales, lengths, extent: int) -> "QuantizedKV":
        """A cache around tensors of the class's layout (contiguous); no
        entry of `lengths` may exceed `extent`."""
        self = cls.__new__(cls)
        self._bind(k_codes, v_codes, k_scales, v_scales, lengths, torch.zeros_like(lengths), int(extent))
        return self

    def _bind(self, k_codes, v_codes, k_scales, v_scales, lengths, tickets, extent, held=None, first=0):
        _lib.require_cuda(k_codes, v_codes, k_scales, v_scales, lengths)
        if k_codes.ndim != 4 or k_codes.shape[-1] != HEAD_DIM:
            raise ValueError(f"QuantizedKV: codes must be [batch, kv_heads, capacity, 128], got {tuple(k_codes.shape)}")
        batch, heads, capacity, _ = k_codes.shape
        for t, shape, dtype in ((k_codes, k_codes.shape, torch.int8), (v_codes, k_codes.shape, torch.int8),
                                (k_scales, k_codes.shape[:3], torch.float32),
                                (v_scales, k_codes.shape[:3], torch.float32), (lengths, (batch,), torch.int32)):
            if t.shape != shape or t.dtype != dtype or not t.is_contiguous() or t.device != k_codes.device:
                raise ValueError(f"QuantizedKV: expected a contiguous {dtype} {tuple(shape)}, got {t.dtype} "
                                 f"{tuple(t.shape)}")
        if not 0 <= extent <= capacity:
            raise ValueError(f"QuantizedKV: extent {extent} of capacity {capacity}")
        self.k_codes, self.v_codes, self.k_scales, self.v_scales = k_codes, v_codes, k_scales, v_scales
        self.lengths, self._tickets = lengths, tickets
        self.batch, self.kv_heads, self.capacity = batch, heads, capacity
        self._held, self._first = _Held(extent, batch) if held is None else held, first
        self._seen, self._extent = -1, 0
        self.device, self._index = k_codes.device, k_codes.get_device()
        # the buffers' addresses, for the calls below
        self._buffers = tuple(t.data_ptr() for t in (k_codes, v_codes, k_scales, v_scales, lengths))
        self._ticket = tickets.data_ptr()
        self._rows = torch.empty(0, dtype=torch.bfloat16, device=self.device)   # the type of rows read back

    def select(self, first: int, count: int = 1) -> "QuantizedKV":
        """Requests [first, first + count) of this cache, sharing its memory
        (prefixes of different lengths are written one request at a time). Its
        extent is that of the requests it covers."""
        if first < 0 or count <= 0 or first + count > self.batch:
            raise ValueError(f"QuantizedKV.select: requests {first}+{count} of {self.batch}")
        part = QuantizedKV.__new__(QuantizedKV)
        s = slice(first, first + count)
        part._bind(self.k_codes[s], self.v_codes[s], self.k_scales[s], self.v_scales[s], self.lengths[s],
                   self._tickets[s], 0, self._held, self._first + first)
        return part

    @property
    def extent(self) -> int:
        held = self._held
        if self._seen != held.changes:
            self._extent = max(held.counts[self._first:self._first + self.batch], default=(0, True))[0]
            self._seen = held.changes
        return self._extent

    @extent.setter
    def extent(self, tokens: int) -> None:
        self._hold([(tokens, False)] * self.batch)

    def _hold(self, counts: list) -> None:
        self._held.counts[self._first:self._first + self.batch] = counts
        self._held.changes += 1

    @property
    def uniform(self) -> bool:
        """Whether every request is known to hold `extent` tokens, as after one
        write to all of them (not after `extent` was set, from_tensors included)."""
        held = set(self._held.counts[self._first:self._first + self.batch])
        return len(held) <= 1 and all(known for _, known in held)

    def _count(self, tokens: int, behind: bool = False) -> None:
        """Each request holds `tokens` tokens, or that many more (how often a
        captured append will be replayed is not known)."""
        if behind:
            known = not (torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing())
            counts = self._held.counts[self._first:self._first + self.batch]
            self._hold([(n + tokens, k and known) for n, k in counts])
        else:
            self._hold([(tokens, True)] * self.batch)


def _strides(a: torch.Tensor, b: torch.Tensor) -> tuple:
    """Batch, sequence and head strides of a, then of b."""
    i, j, k, _ = a.stride()
    m, n, o, _ = b.stride()
    if (i | j | k | m | n | o) & 7:
        return tuple(_lib.used_strides((i, j, k, m, n, o), a.shape[:3], b.shape[:3]))
    return i, j, k, m, n, o


def _check_rows(who: str, cache: QuantizedKV, k: torch.Tensor, v: torch.Tensor) -> None:
    _lib.require_cuda(k, v)
    shape = k.shape
    if k.ndim != 4 or shape[0] != cache.batch or shape[2] != cache.kv_heads or shape[3] != HEAD_DIM or v.shape != shape:
        raise ValueError(f"{who}: k and v must be [{cache.batch}, seq, {cache.kv_heads}, {HEAD_DIM}], got "
                         f"{tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16 or k.stride(3) != 1 or v.stride(3) != 1:
        raise NotImplementedError(f"{who}: k and v must be bf16 with contiguous rows")
    if k.get_device() != cache._index or v.get_device() != cache._index:
        raise ValueError(f"{who}: k, v and the cache are on different devices")


def _check_output(who: str, out: torch.Tensor) -> None:
    strides = out.stride()
    if 0 in strides and any(n > 1 and not s for n, s in zip(out.shape, strides)):
        raise ValueError(f"{who}: several elements of an output share memory")


def kv_cache_write(cache: QuantizedKV, k: torch.Tensor, v: torch.Tensor, start: int = 0) -> None:
    """Quantise k, v [batch, seq, kv_heads, 128] bf16 (any strides that are
    multiples of 8, rows contiguous) into tokens [start, start + seq) of every
    request, which then holds start + seq tokens."""
    _check_rows("kv_cache_write", cache, k, v)
    seq = k.shape[1]
    if start < 0 or start + seq > cache.capacity:
        raise ValueError(f"kv_cache_write: tokens {start}+{seq} of capacity {cache.capacity}")
    _write(cache, k, v, seq, start)
    cache._count(start + seq)


def kv_cache_append(cache: QuantizedKV, k: torch.Tensor, v: torch.Tensor) -> None:
    """kv_cache_write behind the tokens that each request holds (lengths read
    on the device, so a captured append replays)."""
    _check_rows("kv_cache_append", cache, k, v)
    seq = k.shape[1]
    extent = cache.extent
    if extent + seq > cache.capacity:
        raise ValueError(f"kv_cache_append: {seq} tokens behind {extent} of capacity {cache.capacity}")
    _write(cache, k, v, seq, -1)
    cache._count(seq, behind=True)


def _write(cache, k, v, seq, start):
    kc, vc, ks, vs, lengths = cache._buffers
    _lib.call("qia_kv_cache_write", k.data_ptr(), v.data_ptr(), kc, vc, ks, vs, lengths, cache.batch, seq,
              cache.kv_heads, HEAD_DIM, cache.capacity, start, _strides6(*_strides(k, v)),
              cache._ticket, _lib.raw_stream(cache._index))


def kv_cache_read(cache: QuantizedKV, first: int = 0, tokens: int | None = None, out_k: torch.Tensor | None = None,
                  out_v: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Cached tokens [first, first + tokens) (default: up to the extent) as
    bf16 rows [batch, tokens, kv_heads, 128], into out_k / out_v when given
    (e.g. the head of a joint K/V buffer); rows past a request's length are
    zeros."""
    if tokens is None:
        tokens = cache.extent - first
    if first < 0 or tokens < 0 or first + tokens > cache.capacity:
        raise ValueError(f"kv_cache_read: tokens {first}+{tokens} of capacity {cache.capacity}")
    shape = (cache.batch, tokens, cache.kv_heads, HEAD_DIM)
    given = out_k is not None or out_v is not None
    if out_k is None:
        out_k = cache._rows.new_empty(shape)
    if out_v is None:
        out_v = cache._rows.new_empty(shape) if given else torch.empty_like(out_k)
    if given:
        _check_rows("kv_cache_read", cache, out_k, out_v)
        if out_k.shape != shape:
            raise ValueError(f"kv_cache_read: the outputs must be {shape}, got {tuple(out_k.shape)}")
        _check_output("kv_cache_read", out_k)
        _check_output("kv_cache_read", out_v)
        if _lib.overlaps(out_k, out_v):
            raise ValueError("kv_cache_read: the outputs overlap")
    _lib.call("qia_kv_cache_read", *cache._buffers, out_k.data_ptr(), out_v.data_ptr(), cache.batch, first, tokens,
              cache.kv_heads, HEAD_DIM, cache.capacity, _strides6(*_strides(out_k, out_v)),
              _lib.raw_stream(cache._index))
    return out_k, out_v


def cached_attention(q: torch.Tensor, cache: QuantizedKV, k: torch.Tensor | None = None,
                     v: torch.Tensor | None = None, key_valid: torch.Tensor | None = None,
                     scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q K^T) V over [cached prefix, fresh k / v], unmasked but
    for key_valid (no causal limit: a query sees every fresh key).

    q: bf16 [batch, seq, heads, 128], heads a multiple of the cache's K/V
    heads (query head h reads K/V head h // (heads // kv_heads)); k, v: bf16
    [batch, fresh, kv_heads, 128] or None; key_valid: bool [batch, cache.extent
    + fresh], False where a key takes no part (whatever it holds). Cached
    tokens past a request's length never take part. A query without any key
    gives zeros. scale defaults to 1/sqrt(128). Returns bf16 like q, or `out`,
    which may be q itself."""
    who = "cached_attention"
    _lib.require_cuda(q, key_valid)
    shape = q.shape
    if len(shape) != 4 or shape[0] != cache.batch or shape[3] != HEAD_DIM or shape[2] % cache.kv_heads:
        raise ValueError(f"{who}: q must be [{cache.batch}, seq, a multiple of {cache.kv_heads}, {HEAD_DIM}], got "
                         f"{tuple(shape)}")
    if q.dtype != torch.bfloat16 or q.stride(3) != 1:
        raise NotImplementedError(f"{who}: q must be bf16 with contiguous rows")
    if q.get_device() != cache._index:
        raise ValueError(f"{who}: q and the cache are on different devices")
    if scale is not None and not scale > 0:
        raise ValueError(f"{who}: scale={scale} must be positive")
    if (k is None) != (v is None):
        raise ValueError(f"{who}: k and v come together")
    extent, fresh, rows = cache.extent, 0, _NO_ROWS
    if k is not None:
        _check_rows(who, cache, k, v)
        fresh, rows = k.shape[1], _strides(k, v)
    mask_stride = 0
    if key_valid is not None:
        if key_valid.shape != (cache.batch, extent + fresh) or key_valid.dtype != torch.bool:
            raise ValueError(f"{who}: key_valid must be bool [{cache.batch}, {extent + fresh}], got "
                             f"{key_valid.dtype} {tuple(key_valid.shape)}")
        if key_valid.stride(1) != 1 and key_valid.shape[1] > 1 or key_valid.get_device() != cache._index:
            raise NotImplementedError(f"{who}: key_valid must have contiguous rows on the cache's device")
        mask_stride = key_valid.stride(0)
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != shape or out.dtype != torch.bfloat16 or out.stride(3) != 1 or out.get_device() != cache._index:
        raise ValueError(f"{who}: out must be like q")
    else:
        _check_output(who, out)
        if (out.data_ptr() != q.data_ptr() or out.stride() != q.stride()) and _lib.overlaps(out, q) or (
                fresh and (_lib.overlaps(out, k) or _lib.overlaps(out, v))):
            raise ValueError(f"{who}: out may be q, not overlap it, k or v")
    if not out.numel():
        return out
    size = 0
    if shape[1] * shape[2] > 16 * cache.kv_heads:       # (up to 16 rows per K/V head need none)
        size = _lib.load().qia_cached_attention_workspace_bytes(cache.batch, shape[1], fresh, shape[2], cache.kv_heads,
                                                                extent)
    ws = q.new_empty(size >> 1) if size else None       # (bf16 elements)
    outer = _strides(q, out)
    _lib.call("qia_cached_attention", q.data_ptr(), k.data_ptr() if fresh else None, v.data_ptr() if fresh else None,
              *cache._buffers, None if key_valid is None else key_valid.data_ptr(), out.data_ptr(), cache.batch,
              shape[1], fresh, shape[2], cache.kv_heads, HEAD_DIM, cache.capacity, extent,
              _strides12(*outer[:3], *rows, *outer[3:]), mask_stride, 0.0 if scale is None else float(scale),
              None if ws is None else ws.data_ptr(), _lib.raw_stream(cache._index))
    return out

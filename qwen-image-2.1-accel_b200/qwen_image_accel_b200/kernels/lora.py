"""Low-rank adapters of many requests beside a shared projection.

Requests of one batch share the projection's weights but bring adapters of
their own (or none): y[b] = base[b] + scale_i B_i (A_i x[b]) with i = ids[b].
The base output comes from whatever computes the shared projection (a bf16
linear or an MXFP8Linear).
"""
from __future__ import annotations

import struct

import torch

from .. import _lib

MAX_RANK = 128
_strides6 = struct.Struct("6q").pack      # stride arguments (int64[]) as bytes


class LoraWeights:
    """The adapters of one projection, laid out once: `adapters` is a list of
    (A [rank, in], B [out, rank], scale), ranks to 128 in any mix (rank 0: an
    adapter that adds nothing).

    a: bf16 [n, r_pad, in], b: bf16 [n, out, r_pad], zero-padded to the
    largest rank (a multiple of 8); ranks int32 [n], scales float32 [n]."""

    def __init__(self, adapters, device="cuda"):
        if not adapters:
            raise ValueError("LoraWeights: no adapters")
        dev = torch.device(device)
        (_, self.in_features), self.out_features = adapters[0][0].shape, adapters[0][1].shape[0]
        ranks = [a.shape[0] for a, _, _ in adapters]
        for (a, b, _), r in zip(adapters, ranks):
            if a.ndim != 2 or b.ndim != 2 or a.shape[1] != self.in_features or b.shape != (self.out_features, r):
                raise ValueError(f"LoraWeights: A {tuple(a.shape)} and B {tuple(b.shape)} do not fit a "
                                 f"{self.in_features} -> {self.out_features} projection")
        if self.in_features % 8 or self.out_features % 8 or max(ranks) > MAX_RANK:
            raise NotImplementedError(f"LoraWeights: {self.in_features} -> {self.out_features}, ranks {min(ranks)} to "
                                      f"{max(ranks)} (features in multiples of 8, ranks to {MAX_RANK})")
        self.count = len(adapters)
        self.r_pad = max(8, (max(ranks) + 7) // 8 * 8)
        self.a = torch.zeros(self.count, self.r_pad, self.in_features, dtype=torch.bfloat16, device=dev)
        self.b = torch.zeros(self.count, self.out_features, self.r_pad, dtype=torch.bfloat16, device=dev)
        for i, ((a, b, _), r) in enumerate(zip(adapters, ranks)):
            self.a[i, :r] = a.to(dev, torch.bfloat16)
            self.b[i, :, :r] = b.to(dev, torch.bfloat16)
        self.ranks = torch.tensor(ranks, dtype=torch.int32, device=dev)
        self.scales = torch.tensor([float(s) for _, _, s in adapters], dtype=torch.float32, device=dev)
        _lib.require_cuda(self.a)
        self.device, self._index = self.a.device, self.a.get_device()
        self._buffers = tuple(t.data_ptr() for t in (self.a, self.b, self.ranks, self.scales))


def lora_add(x: torch.Tensor, base: torch.Tensor, weights: LoraWeights, ids: torch.Tensor,
             out: torch.Tensor | None = None) -> torch.Tensor:
    """base [batch, seq, out] plus each request's adapter applied to x [batch,
    seq, in], both bf16 with contiguous rows; ids: int32 [batch] on the device,
    -1 for a request without an adapter. Returns a new bf16 tensor, or `out`,
    which may be `base` itself but may not share memory with x or lie otherwise
    over base.

    Sums are fp32. Up to 8 tokens per request the scaled A x is kept to 2^-17,
    beyond that to one bf16 rounding (2^-8) wherever the form for many tokens is
    the faster one. That depends on all sizes, the batch's too, so a request's
    last bits may differ with the number of requests beside it."""
    who = "lora_add"
    _lib.require_cuda(x, base, ids, out)
    shape = x.shape
    if len(shape) != 3 or shape[2] != weights.in_features or base.shape != (shape[0], shape[1], weights.out_features):
        raise ValueError(f"{who}: x {tuple(x.shape)} and base {tuple(base.shape)} do not fit a "
                         f"{weights.in_features} -> {weights.out_features} projection")
    batch, seq, _ = shape
    x_batch, x_row, x_unit = x.stride()
    base_batch, base_row, base_unit = base.stride()
    if x.dtype != torch.bfloat16 or base.dtype != torch.bfloat16 or x_unit != 1 or base_unit != 1:
        raise NotImplementedError(f"{who}: x and base must be bf16 with contiguous rows")
    if ids.shape != (batch,) or ids.dtype != torch.int32 or not ids.is_contiguous():
        raise ValueError(f"{who}: ids must be int32 [{batch}], got {ids.dtype} {tuple(ids.shape)}")
    given = out is not None
    if not given:
        out = torch.empty_like(base)
    elif out.shape != base.shape or out.dtype != torch.bfloat16:
        raise ValueError(f"{who}: out must be like base")
    if not out.numel():
        return out
    out_batch, out_row, out_unit = strides = out.stride()
    if given:
        if 0 in strides and any(n > 1 and not s for n, s in zip(out.shape, strides)):
            raise ValueError(f"{who}: several elements of out share memory")
        if _lib.overlaps(out, x):
            raise ValueError(f"{who}: out may be base, not x or a part of it")
        if out is not base and (out.data_ptr() != base.data_ptr() or strides != base.stride()) and \
                _lib.overlaps(out, base):
            raise ValueError(f"{who}: out may be base, not overlap it")
    if out_unit != 1:
        raise NotImplementedError(f"{who}: out must have contiguous rows")
    index = weights._index
    if x.get_device() != index or base.get_device() != index or ids.get_device() != index or out.get_device() != index:
        raise ValueError(f"{who}: the adapters are on {weights.device}, x, base, ids or out are not")
    # (up to eight tokens per request need none)
    size = _lib.load().qia_lora_workspace_bytes(batch, seq, weights.r_pad) if seq > 8 else 0
    ws = x.new_empty(size >> 1) if size else None       # (bf16 elements)
    rows = x_batch, x_row, base_batch, base_row, out_batch, out_row
    if (x_batch | x_row | base_batch | base_row | out_batch | out_row) & 7:
        rows = _lib.used_strides(rows, shape[:2], shape[:2], shape[:2])
    _lib.call("qia_lora_add", x.data_ptr(), base.data_ptr(), out.data_ptr(), *weights._buffers, ids.data_ptr(), batch,
              seq, weights.in_features, weights.out_features, weights.count, weights.r_pad,
              _strides6(*rows), None if ws is None else ws.data_ptr(),
              _lib.raw_stream(index))
    return out

"""Low-rank adapters of many requests beside a shared projection.

Requests of one batch share the projection's weights but bring adapters of
their own (or none): y[b] = base[b] + scale_i B_i (A_i x[b]) with i = ids[b].
The base output comes from whatever computes the shared projection (a bf16
linear or an MXFP8Linear).
"""
from __future__ import annotations

import ctypes

import torch

from .. import _lib

MAX_RANK = 128
_Strides6 = ctypes.c_int64 * 6


class LoraWeights:
    """The adapters of one projection, laid out once: `adapters` is a list of
    (A [rank, in], B [out, rank], scale), ranks 1 to 128 in any mix.

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
        if self.in_features % 8 or self.out_features % 8 or not 1 <= min(ranks) <= max(ranks) <= MAX_RANK:
            raise NotImplementedError(f"LoraWeights: {self.in_features} -> {self.out_features}, ranks {min(ranks)} to "
                                      f"{max(ranks)} (features in multiples of 8, ranks 1 to {MAX_RANK})")
        self.count = len(adapters)
        self.r_pad = (max(ranks) + 7) // 8 * 8
        self.a = torch.zeros(self.count, self.r_pad, self.in_features, dtype=torch.bfloat16, device=dev)
        self.b = torch.zeros(self.count, self.out_features, self.r_pad, dtype=torch.bfloat16, device=dev)
        for i, ((a, b, _), r) in enumerate(zip(adapters, ranks)):
            self.a[i, :r] = a.to(dev, torch.bfloat16)
            self.b[i, :, :r] = b.to(dev, torch.bfloat16)
        self.ranks = torch.tensor(ranks, dtype=torch.int32, device=dev)
        self.scales = torch.tensor([float(s) for _, _, s in adapters], dtype=torch.float32, device=dev)
        _lib.require_cuda(self.a)
        self.device = self.a.device
        self._buffers = tuple(_lib.ptr(t) for t in (self.a, self.b, self.ranks, self.scales))


def lora_add(x: torch.Tensor, base: torch.Tensor, weights: LoraWeights, ids: torch.Tensor,
             out: torch.Tensor | None = None) -> torch.Tensor:
    """base [batch, seq, out] plus each request's adapter applied to x [batch,
    seq, in], both bf16 with contiguous rows; ids: int32 [batch] on the device,
    -1 for a request without an adapter. Returns a new bf16 tensor, or `out`,
    which may be `base` itself."""
    who = "lora_add"
    _lib.require_cuda(x, base, ids, out)
    if x.ndim != 3 or x.shape[2] != weights.in_features or base.shape != (*x.shape[:2], weights.out_features):
        raise ValueError(f"{who}: x {tuple(x.shape)} and base {tuple(base.shape)} do not fit a "
                         f"{weights.in_features} -> {weights.out_features} projection")
    if x.dtype != torch.bfloat16 or base.dtype != torch.bfloat16 or x.stride(2) != 1 or base.stride(2) != 1:
        raise NotImplementedError(f"{who}: x and base must be bf16 with contiguous rows")
    batch, seq, _ = x.shape
    if ids.shape != (batch,) or ids.dtype != torch.int32 or not ids.is_contiguous():
        raise ValueError(f"{who}: ids must be int32 [{batch}], got {ids.dtype} {tuple(ids.shape)}")
    if out is None:
        out = torch.empty(base.shape, dtype=torch.bfloat16, device=x.device)
    elif out.shape != base.shape or out.dtype != torch.bfloat16 or out.stride(2) != 1:
        raise ValueError(f"{who}: out must be like base")
    for t in (base, ids, out):
        if t.device != x.device:
            raise ValueError(f"{who}: tensors on different devices")
    if x.device != weights.device:
        raise ValueError(f"{who}: the adapters are on {weights.device}, x on {x.device}")
    if not out.numel():
        return out
    size = _lib.load().qia_lora_workspace_bytes(batch, seq, weights.r_pad)
    ws = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
    a, b, ranks, scales = weights._buffers
    _lib.call("qia_lora_add", x.data_ptr(), base.data_ptr(), out.data_ptr(), a, b, ranks, scales, ids.data_ptr(),
              batch, seq, weights.in_features, weights.out_features, weights.count, weights.r_pad,
              _Strides6(*x.stride()[:2], *base.stride()[:2], *out.stride()[:2]), _lib.ptr(ws), _lib.stream(x.device))
    return out

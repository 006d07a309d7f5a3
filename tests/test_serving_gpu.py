"""Requests served together by Qwen21Transformer: an INT8 prefix cache and one
low-rank adapter per request, against the bf16 cache and against models with
the adapters merged into their weights.

Gates: an INT8 row's rounding noise is max/127/sqrt(12), about 0.0065 of a
Gaussian row's rms (44 dB below it), and the attention averages it, so the
outputs stay above 40 dB PSNR of the bf16 cache's. Merged weights differ from
adapters by one bf16 rounding of each weight (2^-9 relative, 54 dB below the
products): 45 dB after two blocks. The MXFP8 profiles quantise merged and
unmerged weights differently (about 2^-5 per element, 30 dB): 30 dB."""
from pathlib import Path

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
GOLD = Path(__file__).resolve().parent / "golden"
LINEARS = {"attn.to_q": 16, "attn.to_v": 8, "attn.to_out.0": 3, "img_mlp.gate_layer": 16, "img_mlp.proj": 5,
           "img_mlp.out": 24}


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def t_bf16(a):
    return torch.from_numpy(np.ascontiguousarray(a).view(np.int16)).view(torch.bfloat16)


def psnr(a, ref):
    a, ref = a.double(), ref.double()
    peak = ref.max() - ref.min()
    return (10 * torch.log10(peak * peak / (a - ref).pow(2).mean())).item()


def build(profile, merged=None):
    from qwen_image_accel_b200.mmdit import init_parameter
    from qwen_image_accel_b200.qwen21 import Block21Config
    from qwen_image_accel_b200.qwen21_model import Qwen21Transformer, model21_parameter_shapes
    cfg = Block21Config(dim=512, heads=4)
    shapes = model21_parameter_shapes(2, cfg, context_in_dim=256)

    def param(n):
        w = init_parameter(n, shapes[n], seed=13)
        key = n.removesuffix(".weight")
        if merged and key in merged:
            a, b, s = merged[key]
            w = (w.float() + s * (b.float() @ a.float()).to(w.device)).to(torch.bfloat16)
        return w

    return Qwen21Transformer(param, num_layers=2, cfg=cfg, context_in_dim=256, device="cuda", profile=profile), shapes


def adapter(shapes, seed, skip=()):
    g = torch.Generator().manual_seed(seed)
    out = {}
    for i in range(2):
        for n, r in LINEARS.items():
            if n in skip:
                continue
            o, w = shapes[f"transformer_blocks.{i}.{n}.weight"]
            out[f"transformer_blocks.{i}.{n}"] = (
                (torch.randn(r, w, generator=g) / w ** 0.5).to(torch.bfloat16),
                (torch.randn(o, r, generator=g) * 0.3 / r ** 0.5).to(torch.bfloat16), 0.5)
    return out


def two_steps(model, quantized, ids=None, rows=slice(None), mask=False):
    from qwen_image_accel_b200.qwen21 import KVCache
    g = np.load(GOLD / "model21_tiny.npz")
    lat, lat2, enc = (t_bf16(g[n]).cuda().repeat(3, 1, 1) for n in ("lat", "lat2", "enc"))
    lat, lat2 = lat * torch.tensor([1.0, 0.9, 0.8], device="cuda", dtype=torch.bfloat16)[:, None, None], lat2
    lat, lat2, enc = lat[rows], lat2[rows], enc[rows]
    img_mask = torch.from_numpy(g["img_mask"]).cuda()
    img_shapes = [[tuple(int(v) for v in s) for s in g["shapes"]]]
    n = lat.shape[0]
    img_mask = img_mask.expand(n, -1)
    enc_mask = None
    if mask:
        enc_mask = torch.ones(enc.shape[:2], dtype=torch.bool, device="cuda")
        enc_mask[:, :3] = False
    cache = KVCache(2, quantized=quantized)
    pre = model.forward(lat, enc, torch.full((n,), 0.8, device="cuda"), img_shapes, img_mask, enc_mask,
                        kv_cache=cache, kv_cache_mode="extract", adapter_ids=ids)
    dec = model.forward(lat2, enc, torch.full((n,), 0.6, device="cuda"), img_shapes, img_mask, enc_mask,
                        kv_cache=cache, kv_cache_mode="cached", adapter_ids=ids)
    return pre.float(), dec.float()


@pytest.mark.parametrize("profile", ["fused", "fused_sage", "mxfp8_sage"])
@pytest.mark.parametrize("mask", [False, True])
def test_quantized_cache_against_the_bf16_cache(profile, mask):
    model, _ = build(profile)
    pre, dec = two_steps(model, False, mask=mask)
    qpre, qdec = two_steps(model, True, mask=mask)
    assert torch.equal(pre, qpre)                     # the prefill only writes the cache
    p = psnr(qdec, dec)
    print(profile, mask, round(p, 1))
    assert torch.isfinite(qdec).all() and p >= 40


@pytest.mark.parametrize("profile,gate", [("fused", 45), ("mxfp8_sage", 30)])
@pytest.mark.parametrize("quantized", [False, True])
def test_adapters_per_request_against_merged_weights(profile, gate, quantized):
    model, shapes = build(profile)
    items = [adapter(shapes, 1), adapter(shapes, 2, skip=("attn.to_v", "img_mlp.out"))]
    plain = two_steps(model, quantized)
    model.load_adapters(items)
    got = two_steps(model, quantized, ids=torch.tensor([1, -1, 0], dtype=torch.int32, device="cuda"))
    for row, which in ((0, 1), (2, 0)):
        ref = two_steps(build(profile, merged=items[which])[0], quantized, rows=slice(row, row + 1))
        for name, a, r, base in zip(("prefill", "cached"), got, ref, plain):
            p, moved = psnr(a[row:row + 1], r), psnr(base[row:row + 1], r)
            print(profile, quantized, name, which, round(p, 1), "without adapter", round(moved, 1))
            assert p >= gate and p > moved + 6
    for a, base in zip(got, plain):
        assert psnr(a[1:2], base[1:2]) >= gate        # the request without an adapter


def test_unknown_linears_are_refused():
    model, _ = build("fused")
    with pytest.raises(ValueError, match="unknown"):
        model.load_adapters([{"transformer_blocks.0.attn.norm_q": (torch.zeros(1, 8), torch.zeros(8, 1), 1.0)}])
    from qwen_image_accel_b200.qwen21 import QuantizedKVLayerCache
    with pytest.raises(RuntimeError, match="populated"):
        QuantizedKVLayerCache().get()

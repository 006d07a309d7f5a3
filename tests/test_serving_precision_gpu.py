"""What the serving operators keep of their operands, against plain 64-bit code.

Half an ulp, relative: 2^-8 for bf16 (eight bits), 2^-11 for f16 (eleven).
"""
import pytest
import torch

from test_kv_cache_gpu import gen, make_cache, rows
from test_lora_gpu import adapters, lora64, rand

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


# Adapters: one rounding of y (2^-8 |y|); the scaled A x as an operand, 2^-17 of each
# term where it is two bf16 numbers and 2^-8 where it is one; fp32 sums of at most 64
# steps of at most 2^-23 each, beside their exact products: 2^-17 of the magnitudes. The
# base output cancels the adapter's, so that y's own rounding does not hide the rest.
@pytest.mark.parametrize("b,s,width,out,ranks,kept", [
    (1, 1, 64, 256, [8], -17), (3, 1, 512, 264, [16, 40], -17), (2, 5, 136, 1000, [64], -17),
    (4, 8, 256, 512, [128, 3], -17), (2, 1000, 256, 512, [64], -8), (1, 3000, 136, 264, [16], -8),
])
def test_adapters_keep_what_their_form_says(b, s, width, out, ranks, kept):
    from qwen_image_accel_b200.kernels.lora import LoraWeights, lora_add
    g = gen(s + width)
    items = adapters(g, width, out, ranks)
    ids = [i % len(ranks) for i in range(b)]
    x = rand(g, b, s, width)
    base = (-lora64(x, torch.zeros(b, s, out, device=DEV), items, ids)[0]).to(torch.bfloat16)
    got = lora_add(x, base, LoraWeights(items), torch.tensor(ids, dtype=torch.int32, device=DEV))
    y, mag, deep = lora64(x, base, items, ids)
    bound = 2.0 ** -8 * y.abs() + 2.0 ** kept * mag + 2.0 ** -17 * deep + 1e-30
    worst = ((got.double() - y).abs() / bound).max().item()
    assert worst <= 1.0, f"off by {worst:.3f} of the bound"


# Attention. A score is off by at most
#   d_j = c (eps_k sum |q_d k_jd| + 2^-24 (sum |q| max |k_j| + max |q| sum |k_j|)) + 2^-21 (65 + |c q.k_j|),
# eps_k = 2^-18 for fp32 products and sums of 128 exact terms, plus, in the forms for more
# than 16 rows, where a cached key is code x a factor of 15 bits, rounded to f16,
# 2^-11 + 2^-15; elements too small for f16 lose 2^-25 of their row's largest; the last
# term is the exponent's own arithmetic (log2 of a V scale among it). Weights are f16
# (2^-11), V likewise rounded in the larger forms (eps_v); weights too small for f16 lose
# at most 2^-33 of the largest; fp32 sums over up to 6000 keys 2^-15; one rounding of the
# output (2^-8):
#   |err| <= 2^-8 |o| + (2^-11 + eps_v + 2^-15) sum p|v| + sum p d|v| + |o| sum p d
#            + 2^-24 sum p max|v| + 2^-33 max p sum|v|
FORMS = [  # batch, queries, heads, kv_heads, lengths, fresh, more than 16 rows
    (2, 1, 8, 8, [900, 300], 1, False), (1, 16, 4, 4, [700], 16, False), (2, 4, 8, 2, [333, 64], 4, False),
    (3, 77, 40, 40, [400, 1, 257], 77, True), (1, 40, 32, 8, [5200], 40, True),
    (1, 40, 4, 4, [700], 40, True), (1, 300, 3, 3, [500], 300, True), (2, 257, 14, 2, [640, 12], 257, True),
]


def check(got, q, cache, k, v, lengths, rounded):
    h, kvh = q.shape[2], cache.kv_heads
    c, share = 128 ** -0.5, h // kvh
    eps_k = 2.0 ** -18 + (2.0 ** -11 + 2.0 ** -15 if rounded else 0.0)
    eps_v = 2.0 ** -11 + 2.0 ** -15 if rounded else 0.0
    for i, n in enumerate(lengths):
        for j in range(kvh):
            kj, vj = (torch.cat([getattr(cache, t + "_codes")[i, j, :n].double() *
                                 getattr(cache, t + "_scales")[i, j, :n].double()[:, None], f[i, :, j].double()])
                      for t, f in (("k", k), ("v", v)))
            qj = q[i, :, j * share:(j + 1) * share].double().flatten(0, 1)
            s = qj @ kj.T * c
            p, av = torch.softmax(s, dim=-1), vj.abs()
            o = p @ vj
            d = c * (eps_k * (qj.abs() @ kj.abs().T) +
                     2.0 ** -24 * (qj.abs().sum(-1, keepdim=True) * kj.abs().amax(-1) +
                                   qj.abs().amax(-1, keepdim=True) * kj.abs().sum(-1))) + 2.0 ** -21 * (65 + s.abs())
            bound = (2.0 ** -8 * o.abs() + (2.0 ** -11 + eps_v + 2.0 ** -15) * (p @ av) + (p * d) @ av +
                     o.abs() * (p * d).sum(-1, keepdim=True) + 2.0 ** -24 * (p @ av.amax(-1, keepdim=True)) +
                     2.0 ** -33 * p.amax(-1, keepdim=True) * av.sum(0))
            off = (got[i, :, j * share:(j + 1) * share].double().flatten(0, 1) - o).abs()
            worst = (off / bound).max().item()
            assert worst <= 1.0, f"off by {worst:.3f} of the bound"


@pytest.mark.parametrize("b,sq,h,kvh,lengths,fresh,tiled", FORMS)
@pytest.mark.parametrize("std", [1.0, 12.0, 60.0])
def test_attention_keeps_what_its_form_says(b, sq, h, kvh, lengths, fresh, tiled, std):
    """Keys that differ, scores of standard deviation about `std`."""
    from qwen_image_accel_b200.kernels.kv_cache import cached_attention
    g = gen(sq * 31 + h)
    cache = make_cache(g, b, kvh, max(lengths) + 13, lengths)
    q = rows(g, b, sq, h, 128, std=std / 1.5)
    k, v = rows(g, b, fresh, kvh, 128, std=1.5), rows(g, b, fresh, kvh, 128)
    check(cached_attention(q, cache, k, v), q, cache, k, v, lengths, tiled)


@pytest.mark.parametrize("sq,kvh", [(16, 8), (100, 8), (200, 170), (600, 4)])
def test_attention_weights_of_keys_that_cancel(sq, kvh):
    """Two keys of opposite V, scales that are powers of two (every row is exact
    in f16): the output is small, and the weights' rounding, an eighth of
    bf16's, is what is left."""
    from qwen_image_accel_b200.kernels.kv_cache import cached_attention
    g = gen(41)
    cache = make_cache(g, 1, kvh, 2, [2])
    cache.v_codes[:, :, 1] = -cache.v_codes[:, :, 0]
    for x in (cache.k_scales, cache.v_scales):
        x.fill_(2.0 ** -6)
    q, none = rows(g, 1, sq, kvh, 128, std=0.05), rows(g, 1, 0, kvh, 128)
    check(cached_attention(q, cache), q, cache, none, none, [2], False)

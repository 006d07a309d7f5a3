"""The cached attention and the adapters at the sizes that choose the forms for
many keys and for many tokens, against plain 64-bit code.

Attention: as for smaller calls, one bf16 rounding of the output and of each
softmax weight (u = 2^-8) and 2^-11 sum p|v| for fp32 scores below 2^6. Adapters:
one rounding of y, one of each scaled A x, fp32 sums (2^-13 of the magnitudes).
"""
import pytest
import torch

from test_kv_cache_gpu import assert_attention, attention64, gen, make_cache, rows
from test_lora_gpu import adapters, check, lora64, rand

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


# more than 320 key tiles in all, at most two query tiles a K/V head
SHAPES = [  # batch, queries, heads, kv_heads, lengths, fresh
    (3, 77, 40, 40, [400, 1, 257], 77), (1, 77, 8, 8, [5300], 0), (1, 40, 32, 8, [5200], 40),
    (2, 129, 100, 100, [200, 130], 1), (1, 20, 4, 4, [1], 10500), (1, 100, 2, 1, [41000], 3),
    (5, 17, 64, 64, [128, 0, 127, 129, 64], 130), (2, 256, 90, 90, [0, 140], 129), (2, 30, 112, 16, [1300, 9], 33),
]


@pytest.mark.parametrize("b,sq,h,kvh,lengths,fresh", SHAPES)
@pytest.mark.parametrize("masked", [False, True])
def test_many_keys_vs_64_bits(b, sq, h, kvh, lengths, fresh, masked):
    from qwen_image_accel_b200.kernels.kv_cache import cached_attention
    g = gen(sq * 31 + h)
    cache = make_cache(g, b, kvh, max(lengths) + 13, lengths)
    q = rows(g, b, sq, h, 128)
    k, v = (rows(g, b, fresh, kvh, 128) for _ in range(2)) if fresh else (None, None)
    valid = None
    if masked:
        valid = torch.rand(b, cache.extent + fresh, device=DEV, generator=g) < 0.7
    got = cached_attention(q, cache, k, v, key_valid=valid)
    assert_attention(got, *attention64(q, cache, k, v, valid))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = cached_attention(q, cache, k, v, key_valid=valid)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, got)                              # the same bits on another stream


@pytest.mark.parametrize("sq", [20, 200])
def test_many_keys_masked_garbage_and_no_keys(sq):
    """Masked keys hold NaN, infinities and the type's largest values; requests
    without a key give zeros."""
    from qwen_image_accel_b200.kernels.kv_cache import cached_attention
    g = gen(21)
    cache = make_cache(g, 3, 40, 330, [300, 140, 0])
    q = rows(g, 3, sq, 40, 128)
    k, v = (rows(g, 3, 50, 40, 128) for _ in range(2))
    valid = torch.rand(3, 300 + 50, device=DEV, generator=g) < 0.5
    valid[1] = False
    valid[2, 300:] = False
    valid[0, :128] = False
    clean = attention64(q, cache, k, v, valid)
    bad = torch.tensor([float("nan"), float("inf"), float("-inf"), 3e38, -3e38], device=DEV)
    for x in (k, v):
        junk = bad[torch.randint(0, 5, x.shape, device=DEV, generator=g)].to(torch.bfloat16)
        x.copy_(torch.where(valid[:, 300:, None, None], x, junk))
    for x in (cache.k_scales, cache.v_scales):
        junk = bad[torch.randint(0, 5, x.shape, device=DEV, generator=g)]
        held = torch.zeros(3, 330, dtype=torch.bool, device=DEV)
        held[:, :300] = valid[:, :300]
        held &= torch.arange(330, device=DEV) < cache.lengths[:, None]
        x.copy_(torch.where(held[:, None], x, junk))
    got = cached_attention(q, cache, k, v, key_valid=valid)
    assert_attention(got, *clean)
    assert not got[1].any() and not got[2].any()


@pytest.mark.parametrize("sq", [60, 150])
def test_many_keys_extreme_scores_and_nan(sq):
    from qwen_image_accel_b200.kernels.kv_cache import cached_attention
    g = gen(22)
    cache = make_cache(g, 1, 60, 700, [700])
    cache.k_scales.mul_(torch.linspace(0.01, 3, 700, device=DEV))
    cache.v_scales.copy_(10.0 ** (torch.rand(1, 60, 700, device=DEV, generator=g) * 12 - 8))
    cache.v_codes[:, :, 40:60] = 0
    cache.v_scales[:, :, 40:60] = 0
    q = rows(g, 1, sq, 60, 128, std=0.3)
    q[0, 0] = 0
    assert_attention(cached_attention(q, cache), *attention64(q, cache, None, None, None))
    cache.v_scales[0, 1, 650] = float("nan")
    out = cached_attention(q, cache)
    assert torch.isfinite(out[:, :, 0]).all() and out[:, :, 1].isnan().all()


def test_many_keys_strides_and_broadcasts():
    from qwen_image_accel_b200.kernels.kv_cache import cached_attention
    g = gen(23)
    for sq in (33, 144):
        cache = make_cache(g, 2, 64, 399, [399, 150])
        q = rows(g, 2, 64, sq + 2, 128).transpose(1, 2)[:, 2:]                # head-major memory
        k, v = rows(g, 1, 30, 64, 128).expand(2, -1, -1, -1), rows(g, 2, 30, 1, 136)[..., :128].expand(-1, -1, 64, -1)
        out = torch.full((2, sq + 1, 64, 256), 7.0, device=DEV, dtype=torch.bfloat16)
        mask = (torch.rand(2, 440, device=DEV, generator=g) < 0.8)[:, 3:432]
        got = cached_attention(q, cache, k, v, key_valid=mask, out=out[:, :sq, :, :128])
        assert_attention(got, *attention64(q, cache, k, v, mask))
        assert (out[:, sq:] == 7).all() and (out[..., 128:] == 7).all()


# weights that every eight tokens would read again, or outputs that several clusters share
CASES = [  # batch, tokens, in, out, ranks, ids
    (2, 300, 1024, 1000, [100, 128], [1, 0]), (1, 333, 4096, 4096, [64], [0]), (3, 200, 520, 4104, [128, 40], [0, 1, -1]),
    (2, 140, 12288, 72, [120], [0, 0]), (40, 77, 520, 264, [128, 64], [i % 3 - 1 for i in range(40)]),
    (2, 1000, 2056, 2056, [33, 64], [1, 0]), (1, 1, 4096, 12288, [128], [0]), (2, 5, 264, 20000, [9, 72], [1, 0]),
    (9, 1, 64, 12296, [64], [0, 0, -1, 0, 0, 0, 0, 0, 0]), (1, 60, 136, 9000, [24], [0]),
]


@pytest.mark.parametrize("b,s,width,out,ranks,ids", CASES)
def test_adapter_forms_vs_64_bits(b, s, width, out, ranks, ids):
    from qwen_image_accel_b200.kernels.lora import LoraWeights, lora_add
    g = gen(s + width)
    items = adapters(g, width, out, ranks)
    x, base = rand(g, b, s, width), rand(g, b, s, out)
    idt = torch.tensor(ids, dtype=torch.int32, device=DEV)
    w = LoraWeights(items)
    got = lora_add(x, base, w, idt)
    check(got, lora64(x, base, items, ids))
    for i, a in enumerate(ids):
        if a < 0:
            assert torch.equal(got[i], base[i])
    again = base.clone()
    assert lora_add(x, again, w, idt, out=again) is again       # in place, the same bits
    assert torch.equal(again, got)


@pytest.mark.parametrize("sign", [-1.0, 1.0])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("sq,kvh,length,fresh", [(1, 2, 40, 3), (12, 2, 0, 1), (50, 2, 1, 1), (300, 2, 150, 70),
                                                 (40, 64, 700, 5), (150, 64, 700, 0)])
def test_scores_of_one_sign_far_from_zero(sq, kvh, length, fresh, masked, sign):
    """Every key scores the same, some 900 below or above zero: the output is
    the mean of V, and no power of two of a maximum may reach the sums."""
    from qwen_image_accel_b200.kernels.kv_cache import cached_attention
    g = gen(24)
    cache = make_cache(g, 2, kvh, max(length, 1) + 3, [length, 0 if fresh else length])
    cache.k_codes.fill_(-127 if sign < 0 else 127)
    cache.k_scales.fill_(40.0 / 127)
    q = torch.full((2, sq, kvh, 128), 2.0, dtype=torch.bfloat16, device=DEV)
    k, v = (torch.full((2, fresh, kvh, 128), sign * 40.0, dtype=torch.bfloat16, device=DEV),
            rows(g, 2, fresh, kvh, 128)) if fresh else (None, None)
    valid = None
    if masked:
        valid = torch.rand(2, cache.extent + fresh, device=DEV, generator=g) < 0.5
        valid[:, -1] = True
    assert_attention(cached_attention(q, cache, k, v, key_valid=valid), *attention64(q, cache, k, v, valid))

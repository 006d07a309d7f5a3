"""The INT8 prefix cache and the attention over it, against plain 64-bit code.

Bounds, with u = 2^-8 the relative half ulp of bf16:
* codes and scales follow from fp32 operations that torch runs identically:
  equal; a value read back is bf16(code * scale): equal, and within half a
  step of what was stored (plus the fp32 rounding of x * 127 / max);
* attention: one bf16 rounding of the output (u |o|) and of each softmax weight
  (u sum p|v|); fp32 scores of magnitude below 2^6 with 128-term sums add less
  than 2^-11 sum p|v|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -8


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rows(g, *shape, std=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * std).to(torch.bfloat16)


def quantised(x):
    """codes [.., 128] int32 and scales [..] of bf16 rows, in torch's fp32."""
    f = x.float()
    amax = f.abs().amax(-1)
    inv = torch.where(amax > 0, torch.full_like(amax, 127.0) / amax, torch.zeros_like(amax))
    return (f * inv[..., None]).round().clamp(-127, 127).to(torch.int32), amax / torch.full_like(amax, 127.0)


def make_cache(g, batch, kvh, capacity, lengths):
    from qwen_image_accel_b200.kernels.kv_cache import QuantizedKV
    shape = (batch, kvh, capacity)
    codes = [torch.randint(-127, 128, (*shape, 128), device=DEV, generator=g).to(torch.int8) for _ in range(2)]
    scales = [0.01 + 0.02 * torch.rand(shape, device=DEV, generator=g) for _ in range(2)]
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    return QuantizedKV.from_tensors(*codes, *scales, n, max(lengths))


def attention64(q, cache, k, v, key_valid, scale=None):
    """(o, sum p|v|) in 64 bits; queries without keys give zeros."""
    b, sq, h, d = q.shape
    share = h // cache.kv_heads
    scale = 1 / math.sqrt(d) if scale is None else scale
    out = torch.zeros(b, sq, h, d, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    for i in range(b):
        n = int(cache.lengths[i])
        keep = torch.ones(n + (0 if k is None else k.shape[1]), dtype=torch.bool, device=q.device)
        if key_valid is not None:
            keep = torch.cat([key_valid[i, :n], key_valid[i, cache.extent:]])
        for j in range(h):
            kj = cache.k_codes[i, j // share, :n].double() * cache.k_scales[i, j // share, :n].double()[:, None]
            vj = cache.v_codes[i, j // share, :n].double() * cache.v_scales[i, j // share, :n].double()[:, None]
            if k is not None:
                kj = torch.cat([kj, k[i, :, j // share].double()])
                vj = torch.cat([vj, v[i, :, j // share].double()])
            kj, vj = kj[keep], vj[keep]
            if kj.shape[0] == 0:
                continue
            p = torch.softmax(q[i, :, j].double() @ kj.T * scale, dim=-1)
            out[i, :, j] = p @ vj
            mag[i, :, j] = p @ vj.abs()
    return out, mag


def assert_attention(got, ref, mag):
    assert got.dtype == torch.bfloat16 and torch.isfinite(got).all()
    bound = U * ref.abs() + (U + 2.0 ** -11) * mag + 1e-30
    worst = ((got.double() - ref).abs() / bound).max().item()
    assert worst <= 1.0, f"off by {worst:.3f} of the bound"


# ------------------------------------------------------------------ write / read
@pytest.mark.parametrize("b,s,h,start,cap", [(1, 1, 1, 0, 1), (2, 1, 32, 7, 9), (1, 16, 4, 0, 16), (3, 17, 5, 2, 40),
                                             (2, 333, 24, 0, 333), (1, 1000, 32, 129, 1201)])
def test_write_codes_scales_and_read_back(b, s, h, start, cap):
    from qwen_image_accel_b200.kernels.kv_cache import QuantizedKV, kv_cache_read, kv_cache_write
    g = gen(s)
    joint = [rows(g, b, s + 3, h, 128, std=3.0) for _ in range(2)]
    k, v = (x[:, 1:s + 1] for x in joint)                     # rows of a longer sequence
    k[0, 0, 0] = 0                                            # an all-zero row
    v[0, -1, -1, 5] = 3e38                                    # a channel at the type's end
    cache = QuantizedKV(b, h, cap)
    kv_cache_write(cache, k, v, start=start)
    for x, codes, scales in ((k, cache.k_codes, cache.k_scales), (v, cache.v_codes, cache.v_scales)):
        qc, qs = quantised(x)
        assert torch.equal(codes[:, :, start:start + s].transpose(1, 2).to(torch.int32), qc)
        assert torch.equal(scales[:, :, start:start + s].transpose(1, 2), qs)
        assert not codes[:, :, :start].any() and not codes[:, :, start + s:].any()
    assert cache.lengths.tolist() == [start + s] * b and cache.extent == start + s
    rk, rv = kv_cache_read(cache, first=start, tokens=s)
    for x, r in ((k, rk), (v, rv)):
        qc, qs = quantised(x)
        assert torch.equal(r, (qc.float() * qs[..., None]).to(torch.bfloat16))
        step = x.double().abs().amax(-1, keepdim=True) / 127
        assert ((qc.double() * qs[..., None].double() - x.double()).abs() <= step * (0.5 + 1e-4)).all()


def test_rows_with_nan_infinity_and_tiny_values():
    from qwen_image_accel_b200.kernels.kv_cache import QuantizedKV, kv_cache_read, kv_cache_write
    x = torch.ones(1, 5, 1, 128, device=DEV, dtype=torch.bfloat16)
    x[0, 0, 0, 3] = float("nan")
    x[0, 1, 0, 4] = float("-inf")
    x[0, 2] = 0
    x[0, 3] = 2.0 ** -130
    x[0, 3, 0, 1] = 0
    x[0, 4] = -2.0
    cache = QuantizedKV(1, 1, 5)
    kv_cache_write(cache, x, x)
    r, _ = kv_cache_read(cache)
    assert r[0, 0].isnan().all() and r[0, 1].isnan().all()
    assert not r[0, 2].any() and r[0, 3, 0, 1] == 0
    assert torch.equal(r[0, 4], x[0, 4])
    assert (r[0, 3].abs() <= 2.0 ** -129).all()


def test_append_follows_each_request_and_read_zeroes_what_is_not_held():
    from qwen_image_accel_b200.kernels.kv_cache import QuantizedKV, kv_cache_append, kv_cache_read, kv_cache_write
    g = gen(5)
    cache = QuantizedKV(3, 4, 64)
    prefix = [rows(g, 1, n, 4, 128) for n in (40, 1, 17)]
    for i, x in enumerate(prefix):
        kv_cache_write(cache.select(i), x, -x)
    assert cache.extent == 40 and cache.lengths.tolist() == [40, 1, 17]
    new = [rows(g, 3, s, 4, 128) for s in (1, 5)]
    for x in new:
        kv_cache_append(cache, x, -x)
    assert cache.extent == 46 and cache.lengths.tolist() == [46, 7, 23]
    rk, rv = kv_cache_read(cache)
    assert torch.equal(rk, -rv)
    for i, x in enumerate(prefix):
        full = torch.cat([x[0], new[0][i], new[1][i]])
        qc, qs = quantised(full)
        n = full.shape[0]
        assert torch.equal(rk[i, :n], (qc.float() * qs[..., None]).to(torch.bfloat16))
        assert not rk[i, n:].any()


def test_append_past_the_capacity_is_dropped_and_recorded():
    from qwen_image_accel_b200 import _lib
    from qwen_image_accel_b200.kernels.kv_cache import QuantizedKV, kv_cache_append, kv_cache_write
    g = gen(6)
    cache = QuantizedKV(1, 2, 8)
    kv_cache_write(cache, *(rows(g, 1, 7, 2, 128) for _ in range(2)))
    cache.extent = 0                       # a host that lost count (a replayed graph): the device still knows
    before = cache.k_codes.clone()
    kv_cache_append(cache, *(rows(g, 1, 3, 2, 128) for _ in range(2)))
    torch.cuda.synchronize()
    assert _lib.device_error() == 1
    assert cache.lengths.tolist() == [8] and torch.equal(cache.k_codes[:, :, :7], before[:, :, :7])
    assert _lib.device_error() == 0


def test_offsets_past_32_bits():
    from qwen_image_accel_b200.kernels.kv_cache import QuantizedKV, cached_attention, kv_cache_read, kv_cache_write
    g = gen(7)
    cap = (1 << 31) // 128 // 4 + 1000      # the last head's codes start past 2^31 - 2^29 and end past 2^31
    cache = QuantizedKV(1, 4, cap)
    k, v = (rows(g, 1, 300, 4, 128) for _ in range(2))
    kv_cache_write(cache, k, v, start=cap - 300)
    rk, _ = kv_cache_read(cache, first=cap - 300)
    qc, qs = quantised(k)
    assert torch.equal(rk, (qc.float() * qs[..., None]).to(torch.bfloat16))
    valid = torch.zeros(1, cap, dtype=torch.bool, device=DEV)
    valid[:, -300:] = True
    for sq in (1, 130):
        q = rows(g, 1, sq, 4, 128)
        tail = make_cache(g, 1, 4, 300, [300])
        tail.k_codes.copy_(cache.k_codes[:, :, -300:])
        tail.v_codes.copy_(cache.v_codes[:, :, -300:])
        tail.k_scales.copy_(cache.k_scales[:, :, -300:])
        tail.v_scales.copy_(cache.v_scales[:, :, -300:])
        assert_attention(cached_attention(q, cache, key_valid=valid), *attention64(q, tail, None, None, None))


# ------------------------------------------------------------------ attention
SHAPES = [  # batch, queries, heads, kv_heads, lengths, fresh
    (1, 1, 1, 1, [1], 0), (1, 1, 4, 4, [0], 1), (2, 1, 32, 32, [515, 3], 1), (3, 1, 32, 8, [100, 1, 2049], 1),
    (1, 1, 8, 1, [8193], 0), (2, 3, 12, 4, [65, 64], 3), (1, 16, 4, 4, [127], 16), (2, 17, 4, 2, [129, 16], 17),
    (1, 77, 6, 2, [300], 77), (2, 128, 2, 2, [256, 255], 0), (1, 129, 2, 1, [1], 129), (1, 300, 3, 3, [0], 300),
    (2, 257, 14, 2, [640, 12], 257), (1, 1000, 2, 2, [777], 1000), (1, 40, 5, 1, [2000], 7), (1, 513, 1, 1, [64], 1),
    (1, 5, 100, 1, [200], 5), (2, 90, 9, 3, [70, 2], 0), (1, 700, 16, 1, [1, ], 33),
]


@pytest.mark.parametrize("b,sq,h,kvh,lengths,fresh", SHAPES)
@pytest.mark.parametrize("masked", [False, True])
def test_attention_vs_64_bits(b, sq, h, kvh, lengths, fresh, masked):
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


@pytest.mark.parametrize("sq", [1, 20, 200])
def test_rows_without_keys_and_masked_garbage(sq):
    """Masked keys hold NaN, infinities and the type's largest values; one
    request has no key at all."""
    from qwen_image_accel_b200.kernels.kv_cache import cached_attention
    g = gen(11)
    cache = make_cache(g, 3, 2, 200, [150, 40, 0])
    q = rows(g, 3, sq, 4, 128)
    k, v = (rows(g, 3, 50, 2, 128) for _ in range(2))
    valid = torch.rand(3, 150 + 50, device=DEV, generator=g) < 0.5
    valid[1] = False
    valid[2, 150:] = False
    valid[0, -1] = True
    clean = attention64(q, cache, k, v, valid)
    bad = torch.tensor([float("nan"), float("inf"), float("-inf"), 3e38, -3e38], device=DEV)
    for x, part in ((k, valid[:, 150:]), (v, valid[:, 150:])):
        junk = bad[torch.randint(0, 5, x.shape, device=DEV, generator=g)].to(torch.bfloat16)
        x.copy_(torch.where(part[:, :, None, None], x, junk))
    for x in (cache.k_scales, cache.v_scales):
        junk = bad[torch.randint(0, 5, x.shape, device=DEV, generator=g)]
        held = torch.zeros(3, 200, dtype=torch.bool, device=DEV)
        held[:, :150] = valid[:, :150]
        held &= torch.arange(200, device=DEV) < cache.lengths[:, None]
        x.copy_(torch.where(held[:, None], x, junk))
    got = cached_attention(q, cache, k, v, key_valid=valid)
    assert_attention(got, *clean)
    assert not got[1].any() and not got[2].any()


@pytest.mark.parametrize("sq", [1, 150])
def test_extreme_scores_and_values(sq):
    """Scores far apart, scores that grow along the keys, V rows whose scales
    differ by many orders, all-zero rows."""
    from qwen_image_accel_b200.kernels.kv_cache import cached_attention
    g = gen(12)
    cache = make_cache(g, 1, 2, 700, [700])
    cache.k_scales.mul_(torch.linspace(0.01, 3, 700, device=DEV))
    cache.v_scales.copy_(10.0 ** (torch.rand(1, 2, 700, device=DEV, generator=g) * 12 - 8))
    cache.v_codes[:, :, 40:60] = 0
    cache.v_scales[:, :, 40:60] = 0
    q = rows(g, 1, sq, 2, 128, std=0.3)
    q[0, 0] = 0
    assert_attention(cached_attention(q, cache), *attention64(q, cache, None, None, None))
    q = rows(g, 1, sq, 2, 128, std=0.3) * 1e-3
    assert_attention(cached_attention(q, cache, scale=2.5), *attention64(q, cache, None, None, None, scale=2.5))


def test_nan_of_a_key_that_takes_part_reaches_the_output():
    from qwen_image_accel_b200.kernels.kv_cache import cached_attention
    g = gen(13)
    for sq in (1, 140):
        cache = make_cache(g, 1, 2, 100, [100])
        cache.v_scales[0, 1, 50] = float("nan")
        out = cached_attention(rows(g, 1, sq, 2, 128), cache)
        assert torch.isfinite(out[:, :, 0]).all() and out[:, :, 1].isnan().all()


def test_strided_inputs_head_major_views_and_out():
    from qwen_image_accel_b200.kernels.kv_cache import cached_attention
    g = gen(14)
    for sq in (1, 5, 144):
        cache = make_cache(g, 2, 4, 99, [99, 50])
        q = rows(g, 2, 8, sq + 2, 128).transpose(1, 2)[:, 2:]                 # head-major memory
        kv = rows(g, 2, 30, 2 * 4 * 128 + 8)                                  # k | v columns of one projection
        k, v = (kv[..., i * 512:(i + 1) * 512].view(2, 30, 4, 128) for i in range(2))
        out = torch.full((2, sq + 1, 8, 256), 7.0, device=DEV, dtype=torch.bfloat16)
        mask = (torch.rand(2, 140, device=DEV, generator=g) < 0.8)[:, 3:132]
        got = cached_attention(q, cache, k, v, key_valid=mask, out=out[:, :sq, :, :128])
        assert_attention(got, *attention64(q, cache, k, v, mask))
        assert (out[:, sq:] == 7).all() and (out[..., 128:] == 7).all()


def test_broadcast_keys():
    """Fresh rows shared by all requests, or by all heads: zero strides."""
    from qwen_image_accel_b200.kernels.kv_cache import cached_attention, kv_cache_read, kv_cache_write
    g = gen(19)
    for sq in (2, 50, 300):
        cache = make_cache(g, 3, 4, 64, [64, 9, 30])
        k, v = rows(g, 1, 40, 4, 128).expand(3, -1, -1, -1), rows(g, 3, 40, 1, 128).expand(-1, -1, 4, -1)
        q = rows(g, 3, sq, 4, 128)
        assert_attention(cached_attention(q, cache, k, v), *attention64(q, cache, k, v, None))
        kv_cache_write(cache, k, v)
        rk, rv = kv_cache_read(cache)
        assert torch.equal(rk[0], rk[1]) and torch.equal(rv[:, :, 0], rv[:, :, 3])


def test_same_bits_twice_and_on_another_stream():
    from qwen_image_accel_b200.kernels.kv_cache import cached_attention
    g = gen(15)
    for sq in (1, 70, 400):
        cache = make_cache(g, 2, 4, 1500, [1500, 900])
        q, k, v = rows(g, 2, sq, 8, 128), rows(g, 2, sq, 4, 128), rows(g, 2, sq, 4, 128)
        first = cached_attention(q, cache, k, v)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            second = cached_attention(q, cache, k, v)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(first, second)


def test_append_and_attend_replay_in_a_graph():
    from qwen_image_accel_b200.kernels.kv_cache import QuantizedKV, cached_attention, kv_cache_append, kv_cache_write
    g = gen(16)
    cache = QuantizedKV(2, 2, 64)
    base = rows(g, 2, 10, 2, 128)
    kv_cache_write(cache, base, base)
    q, k, v = (rows(g, 2, 1, 2, 128) for _ in range(3))
    cache.extent = cache.capacity - 1           # the longest that the replays may reach
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cached_attention(q, cache, k, v)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    extent = cache.extent
    with torch.cuda.graph(graph):
        out = cached_attention(q, cache, k, v)
        kv_cache_append(cache, k, v)
    cache.extent = extent
    for i in range(3):
        assert cache.lengths.tolist() == [10 + i] * 2
        ref = attention64(q, cache, k, v, None)
        graph.replay()
        assert_attention(out, *ref)
        for t in (q, k, v):
            t.copy_(rows(g, 2, 1, 2, 128))


# ------------------------------------------------------------------ refusals
def test_refusals():
    from qwen_image_accel_b200 import _lib
    from qwen_image_accel_b200.kernels.kv_cache import (QuantizedKV, cached_attention, kv_cache_append, kv_cache_read,
                                                        kv_cache_write)
    g = gen(17)
    cache = QuantizedKV(2, 4, 16)
    x = rows(g, 2, 8, 4, 128)
    with pytest.raises(ValueError, match="capacity"):
        kv_cache_write(cache, x, x, start=9)
    with pytest.raises(ValueError, match="must be"):
        kv_cache_write(cache, x[:, :, :3], x[:, :, :3])
    with pytest.raises(NotImplementedError, match="bf16"):
        kv_cache_write(cache, x.float(), x.float())
    kv_cache_write(cache, x, x)
    kv_cache_append(cache, x, x)
    with pytest.raises(ValueError, match="behind 16"):
        kv_cache_append(cache, x, x)
    with pytest.raises(ValueError, match="capacity"):
        kv_cache_read(cache, first=10, tokens=7)
    q = rows(g, 2, 3, 8, 128)
    with pytest.raises(ValueError, match="multiple of 4"):
        cached_attention(q[:, :, :6], cache)
    with pytest.raises(ValueError, match="key_valid"):
        cached_attention(q, cache, key_valid=torch.ones(2, 15, dtype=torch.bool, device=DEV))
    with pytest.raises(ValueError, match="together"):
        cached_attention(q, cache, x)
    with pytest.raises(ValueError, match="positive"):
        cached_attention(q, cache, scale=0.0)
    with pytest.raises(ValueError, match="CUDA"):
        cached_attention(q.cpu(), cache)
    with pytest.raises(_lib.QiaError, match="multiple of 8"):
        cached_attention(rows(g, 2, 3, 8 * 128 + 4)[..., :1024].view(2, 3, 8, 128), cache)
    with pytest.raises(ValueError, match="requests"):
        cache.select(1, 2)
    with pytest.raises(ValueError, match="extent"):
        QuantizedKV.from_tensors(cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales, cache.lengths, 17)
    assert cached_attention(q[:, :0], cache).shape == (2, 0, 8, 128)


def test_empty_write_sets_the_lengths():
    from qwen_image_accel_b200.kernels.kv_cache import QuantizedKV, cached_attention, kv_cache_read, kv_cache_write
    g = gen(18)
    cache = QuantizedKV(2, 4, 16)
    x = rows(g, 2, 8, 4, 128)
    kv_cache_write(cache, x, x)
    kv_cache_write(cache, x[:, :0], x[:, :0], start=3)
    assert cache.lengths.tolist() == [3, 3] and cache.extent == 3
    assert kv_cache_read(cache)[0].shape == (2, 3, 4, 128)
    kv_cache_write(cache, x[:, :0], x[:, :0])
    assert kv_cache_read(cache)[0].shape == (2, 0, 4, 128)
    assert not cached_attention(rows(g, 2, 3, 8, 128), cache).any()

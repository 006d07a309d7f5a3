"""Calls of the serving operators that once answered wrongly, against plain
64-bit code (bounds as in the operators' own tests unless stated)."""
import pytest
import torch

from test_kv_cache_gpu import assert_attention, attention64, gen, make_cache, rows

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


# ------------------------------------------------------------- widened keys, more than one wave
@pytest.mark.parametrize("b,h,lengths,sq,fresh", [
    (20, 4, [0] * 19 + [5000], 300, 0),           # the whole first wave has no key at all
    (20, 4, [0] * 18 + [1, 5000], 300, 0),
    (1, 80, [900], 300, 0), (5, 16, [700, 0, 3, 129, 1300], 500, 40),
])
def test_the_groups_left_over_see_widened_keys(b, h, lengths, sq, fresh):
    """160 groups of query tiles: a full wave, and twelve whose keys are split
    in a launch of their own. The workspace holds NaN before each call."""
    from qwen_image_accel_b200.kernels.kv_cache import cached_attention
    g = gen(31)
    cache = make_cache(g, b, h, max(lengths) + 3, lengths)
    q = rows(g, b, sq, h, 128)
    k, v = (rows(g, b, fresh, h, 128) for _ in range(2)) if fresh else (None, None)
    ref = attention64(q, cache, k, v, None)
    for _ in range(3):
        junk = torch.full((1 << 28,), float("nan"), dtype=torch.bfloat16, device=DEV)
        del junk                                  # (the allocator hands its memory to the workspace)
        assert_attention(cached_attention(q, cache, k, v), *ref)


# ------------------------------------------------------------- parts of a cache held across writes
@pytest.mark.parametrize("sq", [1, 30, 300])
def test_a_held_part_sees_writes_through_its_parent_and_through_other_parts(sq):
    from qwen_image_accel_b200.kernels.kv_cache import (QuantizedKV, cached_attention, kv_cache_append, kv_cache_read,
                                                        kv_cache_write)
    g = gen(32)
    cache = QuantizedKV(3, 2, 200)
    part, other = cache.select(1), cache.select(1, 2)
    kv_cache_write(cache, rows(g, 3, 90, 2, 128), rows(g, 3, 90, 2, 128))
    kv_cache_append(other, rows(g, 2, 45, 2, 128), rows(g, 2, 45, 2, 128))
    assert part.lengths.tolist() == [135] and kv_cache_read(part)[0].shape[1] == 135
    q = rows(g, 1, sq, 2, 128)
    assert_attention(cached_attention(q, part), *attention64(q, part, None, None, None))
    kv_cache_append(part, rows(g, 1, 1, 2, 128), rows(g, 1, 1, 2, 128))
    q = rows(g, 2, sq, 2, 128)
    assert other.lengths.tolist() == [136, 135]
    assert_attention(cached_attention(q, other), *attention64(q, other, None, None, None))


# ------------------------------------------------------------- zero V rows beside very small or large ones
@pytest.mark.parametrize("sq", [1, 4, 16, 60, 300])
@pytest.mark.parametrize("power", [-70, -40, -24, 0, 40, 46])
def test_zero_rows_leave_the_weights_of_small_rows_alone(sq, power):
    """A zero row has no scale of its own, so nothing may depend on the scales
    of the rows around it."""
    from qwen_image_accel_b200.kernels.kv_cache import cached_attention
    g = gen(33)
    cache = make_cache(g, 1, 2, 150, [150])
    k, v = rows(g, 1, 20, 2, 128), rows(g, 1, 20, 2, 128) * 2.0 ** power
    cache.v_scales.mul_(2.0 ** power)
    zero = torch.arange(150, device=DEV) % 3 == 0
    cache.v_codes[:, :, zero] = 0
    cache.v_scales[:, :, zero] = 0
    v[:, ::4] = 0
    q = rows(g, 1, sq, 2, 128)
    assert_attention(cached_attention(q, cache), *attention64(q, cache, None, None, None))
    assert_attention(cached_attention(q, cache, k, v), *attention64(q, cache, k, v, None))


# ------------------------------------------------------------- one prefix for several samples
@pytest.mark.parametrize("profile", ["fused", "fused_sage"])
@pytest.mark.parametrize("masked", [False, True])
def test_attention_cached_takes_one_prefix_for_all_samples(profile, masked):
    """A bf16 prefix of batch 1 serves a batch, like one that is stored once per sample."""
    from test_block21_gpu import build, t_bf16
    from qwen_image_accel_b200.qwen21 import KVLayerCache
    blk, gold = build(profile)
    ht = t_bf16(gold["h_target"]).cuda().repeat(2, 1, 1)
    freqs = torch.view_as_complex(torch.from_numpy(gold["rope"]).contiguous()).cuda()[int(gold["prefix_len"]):]
    k, v = t_bf16(gold["cached_k"]).cuda(), t_bf16(gold["cached_v"]).cuda()
    valid = None
    if masked:
        valid = torch.ones(2, k.shape[1] + ht.shape[1], dtype=torch.bool, device=DEV)
        valid[1, :3] = False
    one, each = KVLayerCache(), KVLayerCache()
    one.store(k, v)
    each.store(k.repeat(2, 1, 1, 1), v.repeat(2, 1, 1, 1))
    got = blk.attention_cached(ht, freqs.contiguous(), one, key_valid=valid)
    assert torch.equal(got, blk.attention_cached(ht, freqs.contiguous(), each, key_valid=valid))


# ------------------------------------------------------------- adapters of rank 0
@pytest.mark.parametrize("b,s", [(2, 1), (2, 8), (1, 60), (2, 300), (3, 1000)])
@pytest.mark.parametrize("rank", [0, -1])
def test_an_adapter_of_rank_zero_adds_nothing(b, s, rank):
    """As a caller of the C entry may lay it out: zero rows and columns only."""
    from qwen_image_accel_b200.kernels.lora import LoraWeights, lora_add
    from test_lora_gpu import adapters, check, lora64, rand
    g = gen(34)
    items = adapters(g, 512, 1024, [40, 64])
    w = LoraWeights(items)
    x, base = rand(g, b, s, 512), rand(g, b, s, 1024)
    ids = [i % 2 for i in range(b)]
    idt = torch.tensor(ids, dtype=torch.int32, device=DEV)
    used = lora_add(x, base, w, idt)                # (leaves its sums in the accumulators)
    check(used, lora64(x, base, items, ids))
    w.a[0], w.b[0], w.ranks[0] = 0, 0, rank
    got = lora_add(x, base, w, idt)
    for i, a in enumerate(ids):
        assert torch.equal(got[i], used[i] if a else base[i])


@pytest.mark.parametrize("s", [1, 300])
def test_an_adapter_that_leaves_a_linear_out_does_nothing_there(s):
    """Whatever the activations hold: infinities and NaN too."""
    from qwen_image_accel_b200.kernels.lora import LoraWeights, lora_add
    from test_lora_gpu import adapters, rand
    from test_serving_gpu import adapter, build
    model, shapes = build("fused")
    model.load_adapters([adapter(shapes, 1), adapter(shapes, 2, skip=("attn.to_v",))])
    w = model.blocks[0].adapters["attn.to_v"]
    assert (w.in_features, w.out_features, w.count) == (512, 512, 2)
    g = gen(35)
    x, base = rand(g, 2, s, 512), rand(g, 2, s, 512)
    x[1, 0, 7], x[1, s - 1, 9] = float("inf"), float("nan")
    got = lora_add(x, base, w, torch.tensor([0, 1], dtype=torch.int32, device=DEV))
    assert torch.equal(got[1], base[1]) and not torch.equal(got[0], base[0])
    alone = LoraWeights([(torch.zeros(0, 512), torch.zeros(512, 0), 1.0)])
    assert torch.equal(lora_add(x, base, alone, torch.zeros(2, dtype=torch.int32, device=DEV)), base)
    with pytest.raises(ValueError, match="do not fit"):
        LoraWeights(adapters(g, 512, 512, [8]) + [(torch.zeros(0, 512), torch.zeros(512, 1), 1.0)])


# ------------------------------------------------------------- strides that nothing is apart by
def odd(t, *dims):
    """t with an odd stride in dimensions of size 1."""
    strides = [13 if i in dims else s for i, s in enumerate(t.stride())]
    assert all(t.shape[i] == 1 for i in dims)
    return t.as_strided(t.shape, strides)


@pytest.mark.parametrize("sq", [1, 40, 300])
def test_odd_strides_of_dimensions_of_size_one(sq):
    from qwen_image_accel_b200.kernels.kv_cache import QuantizedKV, cached_attention, kv_cache_read, kv_cache_write
    from qwen_image_accel_b200.kernels.lora import LoraWeights, lora_add
    from test_lora_gpu import adapters, check, lora64, rand
    g = gen(36)
    cache = QuantizedKV(1, 1, 1)
    k, v = rows(g, 1, 1, 1, 128), rows(g, 1, 1, 1, 128)
    kv_cache_write(cache, odd(k, 0, 1, 2), odd(v, 0, 1, 2))
    ok, ov = torch.empty_like(k), torch.empty_like(v)
    kv_cache_read(cache, out_k=odd(ok, 0, 1, 2), out_v=odd(ov, 0, 1))
    assert all(torch.equal(a, b) for a, b in zip((ok, ov), kv_cache_read(cache)))
    q = rows(g, 1, sq, 1, 128)
    out = torch.empty_like(q)
    cached_attention(odd(q, 0, 2), cache, odd(k, 0, 1, 2), odd(v, 0, 2), out=odd(out, 0, 2))
    assert_attention(out, *attention64(q, cache, k, v, None))
    mask = torch.ones(1, 2, dtype=torch.bool, device=DEV)[:, ::2]             # one column, stride 2
    got = cached_attention(q, cache, key_valid=mask)
    assert_attention(got, *attention64(q, cache, None, None, mask))
    items = adapters(g, 64, 128, [8])
    x, base = rand(g, 1, sq, 64), rand(g, 1, sq, 128)
    ids = torch.zeros(1, dtype=torch.int32, device=DEV)
    dims = (0, 1) if sq == 1 else (0,)
    got = lora_add(odd(x, *dims), odd(base, *dims), LoraWeights(items), ids)
    check(got, lora64(x, base, items, [0]))


@pytest.mark.parametrize("b,sq,h,kvh,n,fresh", [(2, 1, 8, 4, 700, 1), (1, 16, 4, 4, 300, 0), (2, 60, 4, 2, 300, 60),
                                                (2, 60, 90, 90, 300, 60), (2, 700, 4, 4, 300, 90)])
def test_attention_written_over_its_queries(b, sq, h, kvh, n, fresh):
    from qwen_image_accel_b200.kernels.kv_cache import cached_attention
    g = gen(37)
    cache = make_cache(g, b, kvh, n, [n] * b)
    q = rows(g, b, sq, h, 128)
    k, v = (rows(g, b, fresh, kvh, 128) for _ in range(2)) if fresh else (None, None)
    want = cached_attention(q, cache, k, v)
    assert cached_attention(q, cache, k, v, out=q) is q and torch.equal(q, want)


# ------------------------------------------------------------- prefixes of different lengths
@pytest.mark.parametrize("profile", ["fused", "fused_sage", "mxfp8_sage"])
def test_a_block_leaves_out_what_a_shorter_request_does_not_hold(profile):
    """Without a mask, the requests' lengths are the mask (the Sage attention
    took the rows past them as keys of zeros)."""
    from test_block21_gpu import build, t_bf16
    from qwen_image_accel_b200.kernels.kv_cache import QuantizedKV, kv_cache_write
    from qwen_image_accel_b200.qwen21 import QuantizedKVLayerCache, modulation_values
    blk, gold = build(profile)
    ht = t_bf16(gold["h_target"]).cuda().repeat(2, 1, 1)
    mod = t_bf16(gold["modulation"]).cuda()
    vals = modulation_values(torch.cat([mod[:1], mod[:1], mod[1:]]))
    p = int(gold["prefix_len"])
    freqs = torch.view_as_complex(torch.from_numpy(gold["rope"]).contiguous()).cuda()[p:].contiguous()
    k, v = t_bf16(gold["cached_k"]).cuda(), t_bf16(gold["cached_v"]).cuda()
    layer = QuantizedKVLayerCache()
    layer.quantized = QuantizedKV(2, k.shape[2], p)
    kv_cache_write(layer.quantized.select(0), k, v)
    kv_cache_write(layer.quantized.select(1), k[:, :p // 3], v[:, :p // 3])
    valid = torch.ones(2, p + ht.shape[1], dtype=torch.bool, device=DEV)
    valid[1, p // 3:p] = False
    assert torch.equal(blk.forward_cached(ht, vals, freqs, layer), blk.forward_cached(ht, vals, freqs, layer, valid))
    assert torch.equal(blk.attention_cached(ht, freqs, layer), blk.attention_cached(ht, freqs, layer, valid))


def test_a_captured_store_and_decode_equal_the_eager_ones():
    """A store inside the graph keeps the block on the Sage attention; a
    captured append leaves it (the host cannot count its replays)."""
    from test_block21_gpu import build, t_bf16
    from qwen_image_accel_b200.kernels.kv_cache import kv_cache_append
    from qwen_image_accel_b200.qwen21 import QuantizedKVLayerCache, modulation_values
    blk, gold = build("fused_sage")
    ht, mod = t_bf16(gold["h_target"]).cuda(), t_bf16(gold["modulation"]).cuda()
    vals, p = modulation_values(mod), int(gold["prefix_len"])
    freqs = torch.view_as_complex(torch.from_numpy(gold["rope"]).contiguous()).cuda()[p:].contiguous()
    k, v = t_bf16(gold["cached_k"]).cuda(), t_bf16(gold["cached_v"]).cuda()
    layer = QuantizedKVLayerCache()

    def step():
        layer.store(k, v)
        return blk.forward_cached(ht, vals, freqs, layer)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    assert torch.equal(got, want) and layer.quantized.uniform
    layer.quantized.extent = p - 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv_cache_append(layer.quantized, k[:, :1], v[:, :1])
    assert layer.quantized.extent == p and not layer.quantized.uniform


# ------------------------------------------------------------- launch accounting
def test_launches_are_counted_by_form():
    from qwen_image_accel_b200 import _lib
    from qwen_image_accel_b200.kernels.kv_cache import (QuantizedKV, cached_attention, kv_cache_append, kv_cache_read,
                                                        kv_cache_write)
    from qwen_image_accel_b200.kernels.lora import LoraWeights, lora_add
    from test_lora_gpu import adapters, rand
    g = gen(38)

    def kernels(call):
        before = _lib.launch_count
        call()
        return _lib.launch_count - before

    small = QuantizedKV(1, 2, 64)
    x = rows(g, 1, 8, 2, 128)
    assert kernels(lambda: kv_cache_write(small, x, x)) == 1
    assert kernels(lambda: kv_cache_append(small, x[:, :0], x[:, :0])) == 0
    assert kernels(lambda: kv_cache_read(small)) == 1

    def attend(b, h, n, sq):
        cache, q = make_cache(g, b, h, n, [n] * b), rows(g, b, sq, h, 128)
        return kernels(lambda: cached_attention(q, cache))

    assert attend(1, 2, 64, 4) == 1               # one 16-row tile
    assert attend(3, 40, 500, 77) == 1            # converted in place
    assert attend(1, 2, 64, 77) == 2              # widened, attended
    assert attend(1, 80, 900, 300) == 3           # and a remainder of twelve groups
    w = LoraWeights(adapters(g, 512, 1024, [64]))

    def adapt(b, s):
        x, base = rand(g, b, s, 512), rand(g, b, s, 1024)
        ids = torch.zeros(b, dtype=torch.int32, device=DEV)
        return kernels(lambda: lora_add(x, base, w, ids))

    assert adapt(2, 1) == 1 and adapt(2, 1000) == 2


# ------------------------------------------------------------- no keys at all
@pytest.mark.parametrize("sq", [1, 16, 17, 100, 300])
def test_attention_over_an_empty_cache_and_no_fresh_keys(sq):
    from qwen_image_accel_b200 import _lib
    from qwen_image_accel_b200.kernels.kv_cache import QuantizedKV, cached_attention
    g = gen(39)
    cache = QuantizedKV(3, 60, 40)
    q = rows(g, 3, sq, 60, 128)
    out = torch.full_like(q, float("nan"))
    assert not cached_attention(q, cache, out=out).any()
    none, mask = q[:, :0], torch.zeros(3, 0, dtype=torch.bool, device=DEV)
    assert not cached_attention(q, cache, none, none, key_valid=mask).any()
    assert _lib.device_error() == 0


@pytest.mark.parametrize("profile", ["fused", "fused_sage"])
def test_an_empty_prefix_is_stored_and_decoded_like_a_bf16_one(profile):
    from test_block21_gpu import build, psnr, t_bf16
    from qwen_image_accel_b200.qwen21 import KVLayerCache, QuantizedKVLayerCache, modulation_values
    blk, gold = build(profile)
    ht, mod = t_bf16(gold["h_target"]).cuda(), t_bf16(gold["modulation"]).cuda()
    freqs = torch.view_as_complex(torch.from_numpy(gold["rope"]).contiguous()).cuda()[int(gold["prefix_len"]):]
    k = t_bf16(gold["cached_k"]).cuda()[:, :0]
    outs = []
    for layer in (KVLayerCache(), QuantizedKVLayerCache()):
        layer.store(k, k)
        assert layer.get()[0].shape == k.shape
        outs.append(blk.forward_cached(ht, modulation_values(mod), freqs.contiguous(), layer))
    # no cached row, so nothing of INT8: the same attention (Sage), or two roundings to bf16 of one (the weights, 40 dB at least)
    assert torch.equal(*outs) if profile == "fused_sage" else psnr(*outs) >= 40


# ------------------------------------------------------------- codes in flight for two teams
@pytest.mark.parametrize("b,h,n,sq", [(3, 40, 600, 77), (2, 80, 900, 200), (1, 8, 5300, 60), (1, 8, 5300, 256)])
def test_many_calls_with_cold_codes_give_the_same_bits(b, h, n, sq):
    """Copies of K and V that land late and in another order: L2 holds other
    data before each call."""
    from qwen_image_accel_b200 import _lib
    from qwen_image_accel_b200.kernels.kv_cache import cached_attention
    g = gen(40)
    cache = make_cache(g, b, h, n, [n] * b)
    q = rows(g, b, sq, h, 128)
    flush = torch.empty(1 << 27, dtype=torch.int16, device=DEV)
    want = cached_attention(q, cache)
    assert_attention(want, *attention64(q, cache, None, None, None))
    for i in range(100):
        flush.fill_(i)
        assert torch.equal(cached_attention(q, cache), want)
    assert _lib.device_error() == 0

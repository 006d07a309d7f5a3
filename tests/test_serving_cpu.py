"""Host logic of the serving operators (no GPU: the launches are stubbed)."""
import pytest
import torch


@pytest.fixture
def host(monkeypatch):
    """kernels.kv_cache with CPU tensors and launches that do nothing."""
    from qwen_image_accel_b200 import _lib
    from qwen_image_accel_b200.kernels import kv_cache
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: None)
    monkeypatch.setattr(_lib, "raw_stream", lambda index: 0)
    monkeypatch.setattr(_lib, "call", lambda name, *args: None)
    return kv_cache


def rows(batch, seq):
    return torch.zeros(batch, seq, 2, 128, dtype=torch.bfloat16)


def test_extent_is_shared_by_a_cache_and_its_parts(host):
    cache = host.QuantizedKV(3, 2, 32, device="cpu")
    first, pair, again = cache.select(0), cache.select(1, 2), cache.select(1, 2).select(0)
    host.kv_cache_write(cache, rows(3, 10), rows(3, 10))
    assert [c.extent for c in (cache, first, pair, again)] == [10, 10, 10, 10]
    host.kv_cache_append(pair, rows(2, 5), rows(2, 5))
    assert [c.extent for c in (cache, first, pair, again)] == [15, 10, 15, 15]
    host.kv_cache_append(again, rows(1, 2), rows(1, 2))
    assert [c.extent for c in (cache, first, pair, again, cache.select(2))] == [17, 10, 17, 17, 15]
    with pytest.raises(ValueError, match="behind 17"):
        host.kv_cache_append(cache, rows(3, 16), rows(3, 16))


def test_extent_falls_when_every_longer_request_is_written_again(host):
    cache = host.QuantizedKV(2, 2, 32, device="cpu")
    host.kv_cache_write(cache, rows(2, 30), rows(2, 30))
    for i, n in enumerate((4, 6)):
        host.kv_cache_write(cache.select(i), rows(1, n), rows(1, n))
    assert cache.extent == 6
    host.kv_cache_append(cache, rows(2, 26), rows(2, 26))           # there is room
    assert cache.extent == 32 and cache.select(0).extent == 30


def test_extent_can_be_set_for_what_the_host_does_not_count(host):
    cache = host.QuantizedKV(2, 2, 32, device="cpu")
    part = cache.select(1)
    cache.extent = 20
    assert part.extent == 20
    part.extent = 3
    assert cache.extent == 20 and part.extent == 3


def test_token_positions_that_overflow_are_refused():
    """The C entries, called past the Python checks: position + count beyond 64 bits."""
    import ctypes
    from qwen_image_accel_b200 import _lib
    lib = _lib.load()
    at, top = ctypes.c_void_p(4096), 2 ** 63 - 1
    strides = (ctypes.c_int64 * 6)(*([1024] * 6))
    rc = lib.qia_kv_cache_write(at, at, at, at, at, at, at, 1, 4, 1, 128, 8, top - 1, strides, None, None)
    assert rc == 1 and b"capacity 8" in lib.qia_last_error_string()
    rc = lib.qia_kv_cache_read(at, at, at, at, at, at, at, 1, top - 1, 4, 1, 128, 8, strides, None)
    assert rc == 1 and b"capacity 8" in lib.qia_last_error_string()


def test_overlaps_of_views():
    """Views of one buffer, against the sets of their elements."""
    import random
    from qwen_image_accel_b200 import _lib
    rng, buf = random.Random(1), torch.arange(400, dtype=torch.int16)

    def view():
        while True:
            dims = rng.randint(1, 4)
            shape = [rng.choice([1, 1, 2, 3, 5]) for _ in range(dims)]
            stride = [rng.choice([0, 1, 2, 3, 4, 7, 8, 16, 30]) for _ in range(dims)]
            first = rng.randint(0, 150)
            if first + sum((n - 1) * s for n, s in zip(shape, stride)) < 400:
                return buf.as_strided(shape, stride, first)

    seen = set()
    for _ in range(4000):
        a, b = view(), view()
        want = bool(set(a.flatten().tolist()) & set(b.flatten().tolist()))
        assert _lib.overlaps(a, b) == want
        seen.add(want)
    assert seen == {True, False}
    wide = torch.empty(4, 4096, 12288, dtype=torch.bfloat16, device="meta")
    assert not _lib.overlaps(wide[:0], wide)


def test_adapters_refuse_outputs_over_their_inputs(monkeypatch):
    from qwen_image_accel_b200 import _lib
    from qwen_image_accel_b200.kernels import lora
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: None)
    monkeypatch.setattr(_lib, "raw_stream", lambda index: 0)
    monkeypatch.setattr(_lib, "call", lambda name, *args: None)
    w = lora.LoraWeights([(torch.zeros(8, 64), torch.zeros(64, 8), 1.0)], device="cpu")
    ids = torch.zeros(2, dtype=torch.int32)
    buf = torch.zeros(2, 20, 256, dtype=torch.bfloat16)
    x, base = buf[:, :9, :64], buf[:, :9, 64:128]
    assert lora.lora_add(x, base, w, ids, out=base) is base                   # columns beside x
    for out in (buf[:, 1:10, :64], buf[:, :9, 8:72], x):
        with pytest.raises(ValueError, match="not x"):
            lora.lora_add(x, base, w, ids, out=out)
    for out in (buf[:, 1:10, 64:128], buf[:, :9, 72:136]):
        with pytest.raises(ValueError, match="not overlap"):
            lora.lora_add(x, base, w, ids, out=out)
    shared = torch.zeros(1, 9, 64, dtype=torch.bfloat16).expand(2, -1, -1)
    with pytest.raises(ValueError, match="share memory"):
        lora.lora_add(x, shared, w, ids, out=shared)
    assert lora.lora_add(x, shared, w, ids).shape == (2, 9, 64)


def test_attention_and_read_back_refuse_outputs_over_their_inputs(host, monkeypatch):
    from qwen_image_accel_b200 import _lib
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: None)
    cache = host.QuantizedKV(2, 2, 32, device="cpu")
    host.kv_cache_write(cache, rows(2, 8), rows(2, 8))
    buf = torch.zeros(2, 12, 2, 4 * 128, dtype=torch.bfloat16)
    q, k, v = (buf[:, :5, :, 128 * i:128 * (i + 1)] for i in range(3))
    assert host.cached_attention(q, cache, k, v, out=q) is q
    assert host.cached_attention(q, cache, k, v, out=buf[:, :5, :, 384:]).shape == q.shape
    for out in (k, v, buf[:, 1:6, :, 128:256], buf[:, 1:6, :, :128], buf[:, :5, :, 8:136]):
        with pytest.raises(ValueError, match="not overlap"):
            host.cached_attention(q, cache, k, v, out=out)
    one = rows(2, 1).expand(-1, 5, -1, -1)
    with pytest.raises(ValueError, match="share memory"):
        host.cached_attention(q, cache, k, v, out=one)
    with pytest.raises(ValueError, match="share memory"):
        host.kv_cache_read(cache, tokens=5, out_k=one, out_v=rows(2, 5))
    with pytest.raises(ValueError, match="overlap"):
        host.kv_cache_read(cache, tokens=5, out_k=k, out_v=buf[:, 2:7, :, 128:256])
    host.kv_cache_read(cache, tokens=5, out_k=k, out_v=v)


def test_step_graph_refuses_an_int8_cache():
    from qwen_image_accel_b200.optimizations import cuda_graph, decode
    from qwen_image_accel_b200.qwen21 import KVCache

    class Block(torch.nn.Module):
        def forward(self, hidden_states, **kwargs):
            return hidden_states

    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.transformer_blocks = [Block(), Block()]

        def forward(self, kv_cache=None, **kwargs):
            return self.transformer_blocks[0].forward(**kwargs)

    model = Model()
    setattr(model, decode._STATE, {"bound": [None, None]})
    cuda_graph.install_cuda_graph(model)
    h = torch.zeros(1, 4, 8)
    step = {"hidden_states": h, "modulation": h, "rotary_emb": h, "kv_cache_mode": "cached"}
    with pytest.raises(NotImplementedError, match="INT8"):
        model(kv_cache=KVCache(2, quantized=True), **step)


def test_the_package_imports_in_a_torch_without_cuda():
    import subprocess
    import sys
    from pathlib import Path
    code = ("import torch\ndel torch._C._cuda_getCurrentRawStream\n"
            "import qwen_image_accel_b200.kernels.lora, qwen_image_accel_b200.qwen21_model\n")
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True,
                          cwd=Path(__file__).resolve().parents[1] / "qwen-image-2.1-accel_b200")
    assert done.returncode == 0, done.stderr[-500:]


def test_uniform_lengths_are_those_the_host_counted(host):
    cache = host.QuantizedKV(2, 2, 32, device="cpu")
    part = cache.select(1)
    assert cache.uniform
    host.kv_cache_write(cache, rows(2, 10), rows(2, 10))
    host.kv_cache_append(cache, rows(2, 1), rows(2, 1))
    assert cache.uniform and part.uniform
    host.kv_cache_append(part, rows(1, 1), rows(1, 1))
    assert not cache.uniform and part.uniform
    host.kv_cache_append(cache.select(0), rows(1, 1), rows(1, 1))
    assert cache.uniform
    part.extent = 12
    assert not cache.uniform and not part.uniform and cache.extent == 12
    host.kv_cache_write(cache, rows(2, 3), rows(2, 3))
    assert cache.uniform
    same = host.QuantizedKV.from_tensors(cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales, cache.lengths, 3)
    assert not same.uniform and same.extent == 3

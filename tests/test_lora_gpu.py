"""Per-request low-rank adapters, against plain 64-bit code.

With u = 2^-8 the relative half ulp of bf16: one rounding of y (u |y|), one of
each scaled A x where it feeds the tensor cores (u sum |s t_r B_or|), and fp32
sums over up to 12288 terms (below 2^-13 of the sums of magnitudes).
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


def rand(g, *shape, std=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * std).to(torch.bfloat16)


def adapters(g, width, out, ranks):
    return [(rand(g, r, width, std=1 / math.sqrt(width)), rand(g, out, r, std=0.3), 0.5 + 0.3 * i)
            for i, r in enumerate(ranks)]


def lora64(x, base, items, ids):
    y = base.double().clone()
    mag = torch.zeros_like(y)
    deep = torch.zeros_like(y)
    for b, i in enumerate(ids):
        if i < 0 or i >= len(items):
            continue
        a, w, s = items[i]
        s = float(torch.tensor(s, dtype=torch.float32))
        t = s * (x[b].double() @ a.double().T)
        y[b] += t @ w.double().T
        mag[b] = t.abs() @ w.double().abs().T
        deep[b] = s * ((x[b].double().abs() @ a.double().abs().T) @ w.double().abs().T)
    return y, mag, deep


def check(got, ref):
    y, mag, deep = ref
    bound = U * y.abs() + (U * mag + 2.0 ** -13 * deep) + 1e-30
    worst = ((got.double() - y).abs() / bound).max().item()
    assert got.dtype == torch.bfloat16 and worst <= 1.0, f"off by {worst:.3f} of the bound"


CASES = [  # batch, tokens, in, out, ranks, ids
    (1, 1, 64, 64, [8], [0]), (1, 1, 4096, 4096, [64], [0]), (5, 1, 1000, 2056, [3, 16, 128], [2, -1, 0, 1, 2]),
    (3, 2, 4096, 64, [1, 64], [1, 0, 1]), (2, 7, 64, 4096, [9], [0, 0]), (2, 9, 520, 264, [17, 40], [1, 0]),
    (4, 77, 256, 512, [16, 8, 4], [0, 1, 2, -1]), (1, 128, 136, 128, [32], [0]), (2, 129, 192, 136, [64, 33], [0, 1]),
    (3, 300, 1024, 1000, [100, 128], [1, -1, 0]), (1, 1000, 8, 8, [5], [0]), (2, 260, 4096, 392, [24], [0, 0]),
    (2, 64, 12288, 72, [12], [0, -1]), (65, 1, 128, 256, [48, 7], [i % 3 - 1 for i in range(65)]),
]


@pytest.mark.parametrize("b,s,width,out,ranks,ids", CASES)
def test_lora_add_vs_64_bits(b, s, width, out, ranks, ids):
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
    assert torch.equal(lora_add(x, base, w, idt), got)          # the same bits again
    again = base.clone()
    assert lora_add(x, again, w, idt, out=again) is again       # in place
    assert torch.equal(again, got)


@pytest.mark.parametrize("s", [1, 5, 200])
def test_strides_and_streams(s):
    from qwen_image_accel_b200.kernels.lora import LoraWeights, lora_add
    g = gen(s)
    items = adapters(g, 256, 384, [16, 64])
    w = LoraWeights(items)
    x = rand(g, 2, s + 3, 512)[:, 1:s + 1, 128:384]
    both = rand(g, 2, s, 384 * 2)                    # one half of a stacked projection's output
    want = lora64(x, both[..., 384:], items, [1, 0])
    left = both[..., :384].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lora_add(x, both[..., 384:], w, torch.tensor([1, 0], dtype=torch.int32, device=DEV), out=both[..., 384:])
    torch.cuda.current_stream().wait_stream(side)
    check(both[..., 384:], want)
    assert torch.equal(both[..., :384], left)


@pytest.mark.parametrize("s", [3, 40])
def test_broadcast_inputs(s):
    """One activation, and one base row, for all requests: zero strides."""
    from qwen_image_accel_b200.kernels.lora import LoraWeights, lora_add
    g = gen(s)
    items = adapters(g, 128, 256, [16, 8])
    x, base = rand(g, 1, s, 128).expand(3, -1, -1), rand(g, 3, 1, 256).expand(-1, s, -1)
    ids = [1, 0, -1]
    out = torch.empty(3, s, 256, dtype=torch.bfloat16, device=DEV)
    got = lora_add(x, base, LoraWeights(items), torch.tensor(ids, dtype=torch.int32, device=DEV), out=out)
    check(got, lora64(x, base, items, ids))


@pytest.mark.parametrize("s", [1, 150])
def test_padding_of_smaller_ranks_is_not_read_and_unused_adapters_do_not_matter(s):
    from qwen_image_accel_b200.kernels.lora import LoraWeights, lora_add
    g = gen(3)
    items = adapters(g, 512, 256, [5, 64, 16])
    w = LoraWeights(items)
    x, base = rand(g, 2, s, 512), rand(g, 2, s, 256)
    ids = torch.tensor([0, 2], dtype=torch.int32, device=DEV)
    clean = lora_add(x, base, w, ids)
    w.a[1] = float("nan")                            # an adapter that no request uses
    w.b[1] = float("inf")
    assert torch.equal(lora_add(x, base, w, ids), clean)
    x[1] = float("nan")                              # a request does not reach another
    assert torch.equal(lora_add(x, base, w, ids)[0], clean[0])


def test_an_id_past_the_table_is_recorded():
    from qwen_image_accel_b200 import _lib
    from qwen_image_accel_b200.kernels.lora import LoraWeights, lora_add
    g = gen(4)
    w = LoraWeights(adapters(g, 64, 64, [8]))
    for s in (1, 140):
        x, base = rand(g, 2, s, 64), rand(g, 2, s, 64)
        got = lora_add(x, base, w, torch.tensor([1, 7], dtype=torch.int32, device=DEV))
        assert torch.equal(got, base)
        assert _lib.device_error() == 1
    assert _lib.device_error() == 0


def test_refusals():
    from qwen_image_accel_b200 import _lib
    from qwen_image_accel_b200.kernels.lora import LoraWeights, lora_add
    g = gen(5)
    with pytest.raises(ValueError, match="no adapters"):
        LoraWeights([])
    with pytest.raises(ValueError, match="do not fit"):
        LoraWeights([(rand(g, 8, 64), rand(g, 64, 4), 1.0)])
    with pytest.raises(NotImplementedError, match="ranks"):
        LoraWeights(adapters(g, 64, 64, [129]))
    with pytest.raises(NotImplementedError, match="multiples of 8"):
        LoraWeights(adapters(g, 60, 64, [4]))
    w = LoraWeights(adapters(g, 64, 64, [8]))
    x, base = rand(g, 2, 3, 64), rand(g, 2, 3, 64)
    ids = torch.zeros(2, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="do not fit"):
        lora_add(x[..., :56], base, w, ids)
    with pytest.raises(ValueError, match="ids"):
        lora_add(x, base, w, ids.long())
    with pytest.raises(NotImplementedError, match="bf16"):
        lora_add(x.float(), base, w, ids)
    with pytest.raises(ValueError, match="CUDA"):
        lora_add(x.cpu(), base.cpu(), w, ids)
    with pytest.raises(ValueError, match="not x"):
        lora_add(x, base, w, ids, out=x)
    with pytest.raises(_lib.QiaError, match="multiple of 8"):
        lora_add(rand(g, 2, 3, 68)[..., :64], base, w, ids)
    assert lora_add(x[:, :0], base[:, :0], w, ids).shape == (2, 0, 64)

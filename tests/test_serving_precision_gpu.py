"""What the serving operators keep of their operands, against plain 64-bit code.

Half an ulp, relative: 2^-9 for bf16 (eight bits), 2^-12 for f16 (eleven), taken
as 2^-11 to cover truncation.
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


# Adapters: one rounding of y (2^-9 |y|); the scaled A x as an operand, 2^-17 of each
# term where it is two bf16 numbers and 2^-9 where it is one; fp32 sums of at most 64
# steps of at most 2^-23 each, beside their exact products: 2^-17 of the magnitudes. The
# base output cancels the adapter's, so that y's own rounding does not hide the rest.
@pytest.mark.parametrize("b,s,width,out,ranks,kept", [
    (1, 1, 64, 256, [8], -17), (3, 1, 512, 264, [16, 40], -17), (2, 5, 136, 1000, [64], -17),
    (4, 8, 256, 512, [128, 3], -17), (2, 1000, 256, 512, [64], -9), (1, 3000, 136, 264, [16], -9),
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
    bound = 2.0 ** -9 * y.abs() + 2.0 ** kept * mag + 2.0 ** -17 * deep + 1e-30
    worst = ((got.double() - y).abs() / bound).max().item()
    assert worst <= 1.0, f"off by {worst:.3f} of the bound"

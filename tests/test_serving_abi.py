"""The serving entry points (INT8 cache, attention over it, adapters) check
their arguments on the host: status codes and messages, without a GPU."""
import ctypes

import pytest

P, I, F = ctypes.c_void_p, ctypes.c_int64, ctypes.c_float
D = P(4096)
S6 = (ctypes.c_int64 * 6)(*([1024] * 6))
S12 = (ctypes.c_int64 * 12)(*([1024] * 12))


@pytest.fixture(scope="module")
def lib():
    import qwen_image_accel_b200._lib as L
    return L.load()


def refused(lib, rc, code, text):
    assert rc == code and text in lib.qia_last_error_string(), (rc, lib.qia_last_error_string())


def write(lib, k=D, codes=D, batch=1, seq=1, heads=1, dim=128, cap=8, start=0, strides=S6, ticket=D):
    return lib.qia_kv_cache_write(k, D, codes, D, D, D, D, I(batch), I(seq), I(heads), I(dim), I(cap), I(start), strides,
                                  ticket, None)


def test_cache_write_and_read(lib):
    refused(lib, write(lib, codes=None), 1, b"null")
    refused(lib, write(lib, k=None), 1, b"null")
    refused(lib, write(lib, dim=64), 2, b"head_dim=64")
    refused(lib, write(lib, seq=9), 1, b"capacity 8")
    refused(lib, write(lib, start=-1, ticket=None), 1, b"ticket")
    refused(lib, write(lib, k=P(4104)), 3, b"misaligned")
    refused(lib, write(lib, strides=(ctypes.c_int64 * 6)(1024, 1024, 100, 1024, 1024, 1024)), 3, b"multiple of 8")
    refused(lib, write(lib, batch=0), 1, b"batch=0")
    rc = lib.qia_kv_cache_read(D, D, D, D, D, D, D, I(1), I(4), I(5), I(1), I(128), I(8), S6, None)
    refused(lib, rc, 1, b"capacity 8")


def attend(lib, q=D, k=D, seq_q=1, seq_k=1, heads=4, kv=2, dim=128, cap=8, extent=8, strides=S12, ws=None):
    return lib.qia_cached_attention(q, k, D, D, D, D, D, D, None, D, I(1), I(seq_q), I(seq_k), I(heads), I(kv), I(dim),
                                    I(cap), I(extent), strides, I(0), F(0.0), ws, None)


def test_attention(lib):
    refused(lib, attend(lib, q=None), 1, b"null")
    refused(lib, attend(lib, k=None), 1, b"without k and v")
    refused(lib, attend(lib, dim=64), 2, b"head_dim=64")
    refused(lib, attend(lib, heads=5), 1, b"not a multiple")
    refused(lib, attend(lib, heads=258, kv=2), 2, b"258/2")
    refused(lib, attend(lib, extent=9), 1, b"extent=9 of 8")
    refused(lib, attend(lib, strides=(ctypes.c_int64 * 12)(*([1024] * 11 + [12]))), 3, b"multiple of 8")
    assert attend(lib, seq_q=0) == 0
    size = lib.qia_cached_attention_workspace_bytes
    assert size(I(1), I(8), I(8), I(4), I(2), I(1000)) == 0          # one 16-row tile
    assert size(I(1), I(128), I(8), I(4), I(2), I(30000)) == 0       # two tiles of 64 tokens x 2 heads, many keys
    # f16 rows of 8 + 1 key tiles of two heads, K and V, and 32 bytes a tile: few keys, or three query tiles
    assert size(I(1), I(128), I(8), I(4), I(2), I(1000)) == 2 * 9 * (2 * 128 * 128 * 2 + 32)
    assert size(I(1), I(129), I(8), I(4), I(2), I(30000)) == 2 * 236 * (2 * 128 * 128 * 2 + 32)


def lora(lib, x=D, width=64, out=64, r=8, strides=S6, ws=D, seq=1):
    return lib.qia_lora_add(x, D, D, D, D, D, D, D, I(1), I(seq), I(width), I(out), I(1), I(r), strides, ws, None)


def test_adapters(lib):
    refused(lib, lora(lib, x=None), 1, b"null")
    refused(lib, lora(lib, width=60), 2, b"in=60")
    refused(lib, lora(lib, r=136), 2, b"r_pad=136")
    refused(lib, lora(lib, x=P(4100)), 3, b"misaligned")
    refused(lib, lora(lib, strides=(ctypes.c_int64 * 6)(64, 64, 64, 64, 64, 60)), 3, b"multiple of 8")
    refused(lib, lora(lib, seq=40, ws=None), 1, b"workspace")
    assert lora(lib, seq=0) == 0
    size = lib.qia_lora_workspace_bytes
    assert size(I(4), I(8), I(64)) == 0 and size(I(4), I(9), I(64)) == 4 * 9 * 64 * 2

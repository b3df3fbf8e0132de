"""The 8-bit operators without a GPU: what they refuse before anything is launched, and the plain forms the GPU tests compare with."""
import copy
import ctypes as C
import math

import pytest
import torch

from tests import q8_ref as ref
from whisperjav_amd import q8


def test_host_tensors_are_refused():
    x, w = torch.zeros(2, 8), torch.ones(8)
    c, s = torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2)
    for call in (lambda: q8.rmsnorm(x, w), lambda: q8.quantize(x), lambda: q8.dequantize(c, s), lambda: q8.gemm(c, s, c, s)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    cache = q8.KV8Cache.empty(1, 1, 4, 64, torch.device("cpu"))
    with pytest.raises(ValueError, match="GPU"):
        q8.kv_attention(torch.zeros(1, 1, 64), cache, q8.Batch(*(torch.zeros(n, dtype=torch.int32) for n in (1, 2, 1)), 1, 1))


@pytest.mark.parametrize("call", [
    lambda: q8.quantize(torch.zeros(8)),
    lambda: q8.quantize(torch.zeros(2, 8, dtype=torch.float64)),
    lambda: q8.quantize(torch.zeros(2, 8, dtype=torch.int32)),
    lambda: q8.dequantize(torch.zeros(2, 8), torch.zeros(2)),
    lambda: q8.gemm(torch.zeros(2, 8), torch.zeros(2), torch.zeros(2, 8), torch.zeros(2)),
    lambda: q8.kv_write(q8.KV8Cache(*(torch.zeros(2, 2) for _ in range(4))), torch.zeros(1, 1, 64), torch.zeros(1, 1, 64), None),
])
def test_wrong_types_and_shapes_are_refused(call):
    with pytest.raises(ValueError):
        call()


def test_null_arguments_are_refused_at_the_c_entries(hip):
    assert hip.wj_q8_rmsnorm(None, 0, None, 0, 0, None, 0, None, 1e-6, None, 0, None, 0, None, 1, 8, None) == -1
    assert hip.wj_q8_quantize(None, 0, None, 0, 0, None, 0, None, 1, 8, None) == -1
    assert hip.wj_q8_dequantize(None, None, 0, None, 0, None, 0, 1, 8, None) == -1
    assert hip.wj_q8_gemm(None, None, 0, None, None, 0, None, None, 0, None, 0, 1, 1, 1, None, 0, None) == -1
    assert hip.wj_kv8_write(None, None, None, 0, None, 0, None, 0, None) == -1
    assert hip.wj_kv8_read(None, None, None, 0, None, 0, None, 0, None) == -1
    assert hip.wj_kv8_attention(None, None, None, 0, None, 0, None, 0, 1, 1.0, 1, None, 0, None) == -1
    assert b"NULL" in hip.wj_last_error()


def test_struct_layouts():
    assert C.sizeof(q8.Kv8C) == 48 and C.sizeof(q8.Kv8BatchC) == 40


def test_copies_describe_their_own_tensors():
    """a cache and a batch that were used hold addresses: a copy must not take them over"""
    cache = q8.KV8Cache.empty(1, 1, 4, 64, torch.device("cpu"))
    batch = q8.Batch(*(torch.zeros(n, dtype=torch.int32) for n in (1, 2, 1)), 1, 1)
    cache.__dict__["_c"], batch.__dict__["_c"] = q8.Kv8C(), (1, 0, q8.Kv8BatchC())
    for used in (cache, batch):
        for other in (copy.deepcopy(used), copy.copy(used), used._replace()):
            assert type(other) is type(used) and "_c" not in other.__dict__ and len(other) == len(used)
    assert copy.deepcopy(cache).k.data_ptr() != cache.k.data_ptr()


def test_plain_quantiser():
    y = torch.tensor([[1.0, -2.0, 0.5, 127.0], [0, 0, 0, 0], [math.nan, 1, 2, 3], [1.5, 2.5, -0.5, 127.0]])
    codes, scale = ref.quantize(y)
    assert codes[0].tolist() == [1, -2, 0, 127] and codes[3].tolist() == [2, 2, 0, 127]      # ties to even
    assert scale[0] == 1 and scale[1] == 0 and math.isnan(scale[2]) and codes[2].tolist() == [0, 0, 0, 0]


def test_plain_attention_against_a_sum_written_out():
    g = torch.Generator().manual_seed(1)
    q = torch.randn(3, 2, 4, generator=g, dtype=torch.float64)
    k, v = (torch.randn(2, 1, 5, 4, generator=g, dtype=torch.float64) for _ in range(2))
    got = ref.attention(q, k, v, [1, -1], [0, 2, 3], [3, 3], True, 0.5)
    for t, pos in ((0, 1), (1, 2)):
        for h in range(2):
            w = [math.exp(0.5 * float((q[t, h] * k[1, 0, j]).sum())) for j in range(pos + 1)]
            want = sum(wi * v[1, 0, j] for j, wi in enumerate(w)) / sum(w)
            assert torch.allclose(got[t, h], want, atol=1e-12)
    assert bool((got[2] == 0).all())


def meta(*shape, dtype=torch.int8):
    return torch.empty(*shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("call", [
    lambda: q8.quantize(meta(1, 2 ** 32 + 8, dtype=torch.float16)),
    lambda: q8.rmsnorm(meta(1, 2 ** 32 + 8, dtype=torch.float16), meta(2 ** 32 + 8, dtype=torch.float32)),
    lambda: q8.dequantize(meta(1, 2 ** 32 + 8), meta(1, dtype=torch.float32)),
    lambda: q8.gemm(meta(1, 2 ** 32 + 8), meta(1, dtype=torch.float32), meta(1, 2 ** 32 + 8), meta(1, dtype=torch.float32)),
    lambda: q8._batch(q8.Batch(*(torch.zeros(n, dtype=torch.int32) for n in (1, 2, 1)), 1, 1), 2 ** 32 + 1, 0),
])
def test_sizes_past_32_bits_are_refused(call):
    """ctypes would hand the library their low 32 bits: 8 columns, 1 row"""
    with pytest.raises(ValueError, match=r"at most 2\^31 - 1"):
        call()


def test_products_wider_than_a_grid_are_refused(hip):
    nobody = C.create_string_buffer(1 << 16)                 # a context of zeros: nothing of it is read before the checks
    one = C.c_void_p(64)
    assert hip.wj_q8_gemm(nobody, one, 16, one, one, 16, one, None, 0, one, 1 << 28, 1, 1 << 27, 16, None, 0, None) == -1
    assert b"2^27 - 16" in hip.wj_last_error()

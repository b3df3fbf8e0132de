"""Calls of the 8-bit operators that their arguments' checks cannot see through, and what they leave alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


@pytest.fixture(scope="module")
def q8():
    from whisperjav_amd import q8
    assert torch.cuda.is_available()
    return q8


@pytest.mark.parametrize("starts,lens", [([0, 3, -2 ** 31], [5, 5]), ([0, 3, 1], [5, 5]), ([0, 3, 3], [5, -2 ** 31]), ([0, 3, 2 ** 31 - 1], [5, -7])])
def test_arrays_that_are_no_spans(q8, starts, lens):
    """the second sequence's entries make no sense: it owns no rows, or rows before position 0"""
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(6, 2, 64, generator=g).cuda() for _ in range(2))
    q = torch.randn(6, 4, 64, generator=g).cuda()
    cache, good = q8.KV8Cache.empty(3, 2, 16, 64), q8.KV8Cache.empty(3, 2, 16, 64)
    batch = q8.Batch(ints([1, 2]), ints(starts), ints(lens), 3, 5)
    one = q8.Batch(ints([1]), ints([0, 3]), ints([5]), 3, 5)
    rows = min(max(starts[-1], 3), 6)                                                       # of both sequences together
    out, want = torch.full((6, 4, 64), 9.0).cuda(), torch.full((6, 4, 64), 9.0).cuda()
    q8.kv_write(cache, k, v, batch)
    q8.kv_write(good, k, v, one)
    for a, b in zip(cache, good):
        assert torch.equal(a, b)
    for causal in (True, False):
        q8.kv_attention(q, cache, batch, causal=causal, out=out)
        q8.kv_attention(q, good, one, causal=causal, out=want)
        assert torch.equal(out[:3], want[:3]) and bool((out[3:rows] == 0).all()) and bool((out[rows:] == 9).all())
    back = q8.kv_read(cache, batch, 6, torch.float32)
    assert torch.equal(back[0][:3], q8.kv_read(good, one, 6, torch.float32)[0][:3]) and bool((back[0][3:rows] == 0).all())

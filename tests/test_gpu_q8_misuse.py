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


def layer_inputs(q8):
    g = torch.Generator().manual_seed(2)
    x, d = torch.randn(4, 64, generator=g).cuda(), torch.randn(4, 64, generator=g).cuda()
    codes, scale = q8.quantize(x)
    cache = q8.KV8Cache.empty(1, 1, 8, 64)
    return x, d, codes, scale, cache, q8.Batch(ints([0]), ints([0, 4]), ints([4]), 4, 4), torch.ones(64).cuda()


def writers(q8):
    """name -> (the tensor that is written, the call)"""
    x, d, codes, scale, cache, batch, w = layer_inputs(q8)
    rows, res, out, att = x.view(4, 1, 64), torch.zeros_like(x), torch.zeros(4, 4).cuda(), torch.zeros(4, 1, 64).cuda()
    return {
        "rmsnorm in place": (x, lambda: q8.rmsnorm(x, w, delta=d)),
        "rmsnorm residual": (res, lambda: q8.rmsnorm(x, w, residual=res)),
        "gemm out": (out, lambda: q8.gemm(codes, scale, codes, scale, out=out)),
        "attention out": (att, lambda: q8.kv_attention(rows, cache, batch, out=att)),
        "cache k": (cache.k_scale, lambda: q8.kv_write(cache, rows, rows, batch)),
        "cache v": (cache.v_scale, lambda: q8.kv_write(cache, rows, rows, batch)),
    }


@pytest.mark.parametrize("name", ["rmsnorm in place", "rmsnorm residual", "gemm out", "attention out", "cache k", "cache v"])
def test_a_backward_that_saved_what_is_written_raises(q8, name):
    written, call = writers(q8)[name]
    p = torch.ones(written.shape, device="cuda", requires_grad=True)
    loss = (written * p).sum()                               # saves `written` for p's gradient
    call()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_what_is_only_read_keeps_its_version(q8):
    x, d, codes, scale, cache, batch, w = layer_inputs(q8)
    read = [x, d, codes, scale, w, *cache, *batch[:3]]
    before = [t._version for t in read]
    q8.rmsnorm(x, w)
    q8.rmsnorm(x, w, delta=d, residual=torch.empty_like(x))
    q8.dequantize(*q8.quantize(x))
    q8.gemm(codes, scale, codes, scale)
    q8.kv_attention(x.view(4, 1, 64), cache, batch)
    q8.kv_read(cache, batch, 4)
    assert [t._version for t in read] == before


def test_tensors_of_inference_mode_are_served(q8):
    with torch.inference_mode():
        calls = writers(q8)
        for _, call in calls.values():
            call()
    for _, call in calls.values():
        call()


def test_tangents_and_gradients_are_refused(q8):
    import torch.autograd.forward_ad as forward
    x, d, codes, scale, cache, batch, w = layer_inputs(q8)
    rows = x.view(4, 1, 64)

    def calls(wrap):
        return [lambda: q8.quantize(wrap(x)), lambda: q8.rmsnorm(wrap(x), w), lambda: q8.rmsnorm(x, wrap(w)), lambda: q8.rmsnorm(x, w, delta=wrap(d)),
                lambda: q8.rmsnorm(x, w, residual=wrap(d)), lambda: q8.dequantize(codes, wrap(scale)), lambda: q8.gemm(codes, wrap(scale), codes, scale),
                lambda: q8.gemm(codes, scale, codes, scale, bias=wrap(scale)), lambda: q8.kv_write(cache, wrap(rows), rows, batch),
                lambda: q8.kv_write(cache, rows, wrap(rows), batch), lambda: q8.kv_attention(wrap(rows), cache, batch),
                lambda: q8.kv_attention(rows, cache._replace(v_scale=wrap(cache.v_scale)), batch),
                lambda: q8.kv_read(cache._replace(k_scale=wrap(cache.k_scale)), batch, 4)]
    with forward.dual_level():
        for call in calls(lambda t: forward.make_dual(t, torch.ones_like(t))):
            with pytest.raises(ValueError, match="tangent"):
                call()
        q8.rmsnorm(x, w)                                     # tensors without one go on
    for call in calls(lambda t: t.clone().requires_grad_()):
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad():
            call()
    used = cache._replace(v_scale=cache.v_scale.clone())
    q8.kv_attention(rows, used, batch)
    used.v_scale.requires_grad_()                            # ... after its first use too
    with pytest.raises(ValueError, match="gradient"):
        q8.kv_attention(rows, used, batch)


def test_arrays_and_caches_whose_memory_moved(q8):
    """a used batch or cache whose tensors were given other memory: the new memory counts, and is checked (what was there before may be freed)"""
    x, d, codes, scale, cache, batch, w = layer_inputs(q8)
    rows = x.view(4, 1, 64)
    q8.kv_write(cache, rows, rows, batch)
    q8.kv_attention(rows, cache, batch)
    batch.lens.data = ints([2])                              # two of the four rows lie before position 0 now
    want = q8.kv_attention(rows, cache, q8.Batch(ints([0]), ints([0, 4]), ints([2]), 4, 4))
    assert torch.equal(q8.kv_attention(rows, cache, batch), want)
    other = q8.KV8Cache.empty(1, 1, 8, 64)
    q8.kv_write(other, d.view(4, 1, 64), rows, batch)
    cache.k.data, cache.k_scale.data, cache.v.data, cache.v_scale.data = (t.clone() for t in other)
    assert torch.equal(q8.kv_attention(rows, cache, batch), q8.kv_attention(rows, other, batch))
    q8.kv_write(cache, rows, rows, batch)                    # goes to the new memory, not to the other cache's
    assert not torch.equal(cache.k, other.k)
    batch.lens.data = ints([2, 3])
    with pytest.raises(ValueError, match="lens"):
        q8.kv_attention(rows, cache, batch)
    batch.lens.data = ints([2])
    cache.v_scale.data = torch.zeros(1, 1, 7).cuda()
    with pytest.raises(ValueError, match="scales"):
        q8.kv_attention(rows, cache, batch)

"""8-bit operators whose calls use workspaces: captured and replayed, and two at once on two streams."""
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


def random_cache(q8, g, slots, heads, ctx, dim):
    def codes():
        return torch.randint(-127, 128, (slots, heads, ctx, dim), generator=g).to(torch.int8).cuda()

    def scale():
        return ((0.5 + torch.rand(slots, heads, ctx, generator=g)) * (2 / 127)).cuda()
    return q8.KV8Cache(codes(), scale(), codes(), scale())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_parts_and_slices_replayed_while_lengths_change(q8, dim, causal):
    """attention over parts of the positions, then a product over slices of k, as one graph: lengths from none to all of the cache"""
    g = torch.Generator().manual_seed(dim)
    cache = random_cache(q8, g, 3, 1, 2500, dim)
    w, ws = q8.quantize(torch.randn(140, 9000, generator=g).cuda())
    a, sa = q8.quantize(torch.randn(70, 9000, generator=g).cuda())
    q = torch.randn(4, 4, dim, generator=g).half().cuda()
    out, prod = torch.zeros(4, 4, dim, dtype=torch.float16).cuda(), torch.zeros(70, 140).cuda()
    batch = q8.Batch(ints([2, 0]), ints([0, 1, 4]), ints([1000, 1200]), 3, 2500)

    def step(o, p):
        q8.kv_attention(q, cache, batch, causal=causal, out=o)
        q8.gemm(a, sa, w, ws, out=p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(out, prod)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out, prod)
    eager_out, eager_prod = torch.empty_like(out), torch.empty_like(prod)
    for lens in ([2500, 2500], [1, 3], [0, 2], [300, 2499], [2500, 0], [1000, 1200], [357, 358], [2600, 700]):
        batch.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(torch.randn(4, 4, dim, generator=g).half())
        sa.copy_(torch.rand(70, generator=g))
        out.fill_(3)
        prod.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        step(eager_out, eager_prod)
        assert torch.equal(out, eager_out) and torch.equal(prod, eager_prod), lens
        for b, first, last in ((0, 0, 1), (1, 1, 4)):
            for t in range(first, last):
                seen = (lens[b] - (last - first) + t - first + 1) if causal else lens[b]
                assert bool((out[t] == 0).all()) == (seen <= 0), (lens, t)


def test_two_streams_at_once(q8):
    """each call has its own workspace: what runs beside it does not change a result"""
    g = torch.Generator().manual_seed(3)
    cache = random_cache(q8, g, 4, 1, 2500, 128)
    jobs = []
    for n in range(2):
        w, ws = q8.quantize(torch.randn(140, 9000, generator=g).cuda())
        a, sa = q8.quantize(torch.randn(70, 9000, generator=g).cuda())
        q = torch.randn(2, 4, 128, generator=g).half().cuda()
        batch = q8.Batch(ints([2 * n, 2 * n + 1]), ints([0, 1, 2]), ints([2400 - 300 * n, 2100]), 1, 2500)
        jobs.append(lambda a=a, sa=sa, w=w, ws=ws, q=q, batch=batch: (q8.gemm(a, sa, w, ws, dtype=torch.float32), q8.kv_attention(q, cache, batch)))
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[], []]
    for _ in range(20):
        for n, (stream, job) in enumerate(zip(streams, jobs)):
            with torch.cuda.stream(stream):
                got[n].append(job())
    torch.cuda.synchronize()
    for n in range(2):
        for product, attended in got[n]:
            assert torch.equal(product, want[n][0]) and torch.equal(attended, want[n][1])

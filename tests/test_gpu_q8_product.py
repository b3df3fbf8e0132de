"""Every kernel of the int8 product (whisperjav_amd/q8.py), with enough steps of k to use its buffers again, against the formula in every row."""
import pytest
import torch

from tests.q8_cases import PRODUCT_PAST_THE_CACHES, PRODUCTS

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.float32: E, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


@pytest.fixture(scope="module")
def q8():
    from whisperjav_amd import q8
    assert torch.cuda.is_available()
    return q8


def rows(g, count, k):
    """codes of the whole range in rows that start at multiples of 16 bytes, with codes behind k that must not count"""
    pad = k + -k % 16
    return torch.randint(-128, 128, (count, pad), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)[:, :k]


def check(q8, m, n, k, dtype, bias):
    g = torch.Generator(device="cuda")
    g.manual_seed(m + n + k)
    a, w = rows(g, m, k), rows(g, n, k)
    sa, sw = (torch.rand(c, generator=g, device="cuda") * s + 1e-4 for c, s in ((m, 0.02), (n, 0.02 / k ** 0.5)))
    b = torch.randn(n, generator=g, device="cuda") if bias else None
    # the sum of at most 131071 products of 14 bits is exact in 64-bit floating point; the epilogue rounds a scale product, the sum's
    # conversion, their product and the addition: 4 E, then the type
    prod = torch.matmul(a.double(), w.double().t().contiguous()).mul_(sa.double()[:, None]).mul_(sw.double())
    lim = prod.abs().mul_(4 * E)
    want = prod if b is None else prod.add_(b.double())
    lim.add_(want.abs(), alpha=U[dtype] + E).add_(TINY[dtype])
    room = torch.full((m, n + 3), 7.0, dtype=dtype, device="cuda")
    q8.gemm(a, sa, w, sw, bias=b, out=room[:, :n])
    off = (room[:, :n].double() - want).abs_()
    assert bool((off <= lim).all()), float((off / lim).max())
    assert bool((room[:, n:] == 7).all())
    assert torch.equal(q8.gemm(a, sa, w, sw, bias=b, dtype=dtype), room[:, :n])


@pytest.mark.parametrize("kernel,slices,m,n,k", PRODUCTS)
@pytest.mark.parametrize("dtype,bias", [(torch.float32, True), (torch.float16, True), (torch.bfloat16, True), (torch.float16, False)])
def test_product(q8, kernel, slices, m, n, k, dtype, bias):
    check(q8, m, n, k, dtype, bias)


@pytest.mark.parametrize("bias", [False, True])
def test_product_past_the_caches(q8, bias):
    check(q8, *PRODUCT_PAST_THE_CACHES, torch.float32, bias)


@pytest.mark.parametrize("m,n,k", [(129, 515, 4500), (385, 4900, 1285), (2050, 8301, 640)])
def test_product_of_one_input_is_the_same_bits_in_another_layout(q8, m, n, k):
    """the kernel for any layout sums the same integers"""
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    a, w = rows(g, m, k), rows(g, n, k)
    one = torch.ones(max(m, n), device="cuda")
    odd = [torch.empty(t.shape[0], k + 1 + -k % 16, dtype=torch.int8, device="cuda")[:, :k].copy_(t) for t in (a, w)]
    assert odd[0].stride(0) % 16
    assert torch.equal(q8.gemm(a, one[:m], w, one[:n], dtype=torch.float32), q8.gemm(odd[0], one[:m], odd[1], one[:n], dtype=torch.float32))

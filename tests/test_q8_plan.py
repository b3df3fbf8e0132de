"""The plain arithmetic of the 8-bit operators (whisperjav_amd/csrc/q8_plan.hpp), compiled for the host and run here."""
import ctypes as C
import itertools
import shutil
import subprocess

import pytest

from tests.q8_cases import ATTENTION, PRODUCT_PAST_THE_CACHES, PRODUCTS
from whisperjav_amd import build

CXX = shutil.which("g++") or shutil.which("clang++")
pytestmark = pytest.mark.skipif(CXX is None, reason="no host C++ compiler")

ENTRIES = """
#include "%s"
extern "C" void span(const int* in, int* out) {
  const wj::Span s = wj::span_from(in[0], in[1], in[2], in[3], in[4], in[5]);
  out[0] = s.slot; out[1] = s.first; out[2] = s.n; out[3] = s.len; out[4] = s.pos0;
}
extern "C" void gemm(int64_t m, int n, int k, int* out) {
  const wj::GemmPlan p = wj::plan_gemm(m, n, k);
  out[0] = p.kind; out[1] = p.ksplit;
}
extern "C" void attention(const int* in, int* out) {
  const wj::AttnPlan p = wj::plan_attention(in[0], in[1], in[2], in[3], wj::most_new(in[4], in[5]), in[6], in[7]);
  out[0] = p.rt; out[1] = p.waves; out[2] = p.nsplit; out[3] = p.chunk;
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("plan")
    (tmp / "plan.cpp").write_text(ENTRIES % (build.CSRC / "q8_plan.hpp"))
    subprocess.run([CXX, "-std=c++17", "-O1", "-shared", "-fPIC", str(tmp / "plan.cpp"), "-o", str(tmp / "plan.so")], check=True)
    return C.CDLL(str(tmp / "plan.so"))


def span(plan, *args):
    out = (C.c_int * 5)()
    plan.span((C.c_int * 6)(*args), out)
    return tuple(out)


def test_spans_of_documented_arrays(plan):
    assert span(plan, 2, 4, 9, 30, 3, 20) == (2, 4, 5, 30, 25)
    assert span(plan, -1, 0, 2, 2, 3, 20) == (-1, 0, 2, 2, 0)
    assert span(plan, 3, 0, 2, 2, 3, 20)[0] == -1
    assert span(plan, 0, 5, 5, 7, 3, 20)[2:] == (0, 7, 7)                     # no new rows
    assert span(plan, 0, 18, 25, 7, 3, 20)[1:] == (18, 2, 7, 5)               # rows behind the arrays' end are nobody's
    assert span(plan, 0, 2, 6, 1, 3, 20)[1:] == (2, 4, 1, -3)                 # rows before position 0


def test_no_array_leads_out_of_the_rows(plan):
    """a starts entry far below the one before it: their difference leaves 32 bits (-2^31 - 3 is 2147483645 there)"""
    ends = [-2 ** 31, -2 ** 31 + 1, -5, -1, 0, 1, 3, 19, 20, 21, 2 ** 31 - 1]
    for first, last, length, rows in itertools.product(ends, ends, ends, (1, 20, 2 ** 31 - 1)):
        _, f, n, positions, pos0 = span(plan, 0, first, last, length, 1, rows)
        assert n >= 0 and (n == 0 or (0 <= f and f + n <= rows and f == first and f + n == min(last, rows)))
        assert positions == max(0, length) and pos0 == positions - n and -2 ** 31 < pos0 and pos0 + n == positions


@pytest.mark.parametrize("kernel,slices,m,n,k", PRODUCTS + [("big", 1, *PRODUCT_PAST_THE_CACHES)])
def test_sizes_still_reach_their_product_kernel(plan, kernel, slices, m, n, k):
    out = (C.c_int * 2)()
    plan.gemm(C.c_int64(m), n, k, out)
    assert (["rows", "big", "tile", "tile128"][out[0]], out[1]) == (kernel, slices)


@pytest.mark.parametrize("name", sorted(ATTENTION))
@pytest.mark.parametrize("dim", [64, 128])
def test_sizes_still_reach_their_attention_kernel(plan, name, dim):
    (seqs, new, length, heads, per), want = ATTENTION[name]
    out = (C.c_int * 4)()
    plan.attention((C.c_int * 8)(heads, length, dim, seqs, new, seqs * new, length, heads * per), out)
    assert tuple(out)[:3] == want
    if want[2] > 1:
        assert out[3] * (want[2] - 1) < length <= out[3] * want[2]


def test_every_product_has_a_kernel_and_slices_that_hold_steps(plan):
    out = (C.c_int * 2)()
    for m, n, k in itertools.product((1, 16, 17, 64, 65, 300, 5000, 4194240), (1, 130, 5000, 2 ** 27 - 16), (1, 127, 2049, 131071)):
        plan.gemm(C.c_int64(m), n, k, out)
        assert 0 <= out[0] <= 3 and 1 <= out[1] <= 8 and (out[1] == 1 or (out[0] == 2 and (k + 127) // 128 >= out[1]))

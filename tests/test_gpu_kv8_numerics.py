"""The arithmetic of the attention over the 8-bit cache (whisperjav_amd/q8.py): what its precision is, not only that it is right.

Every kernel that a call can take is reached, with both head dimensions."""
import pytest
import torch

from tests import q8_ref as ref
from tests.q8_cases import ATTENTION

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]

CASES = [(name, *sizes, dim) for name, (sizes, _) in ATTENTION.items() for dim in (64, 128)]
IDS = [f"{c[0]}-{c[6]}" for c in CASES]


def rng(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def ints(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def make(q8, g, case, dtype, scales=None):
    """(queries, cache tensors on the host, sequences' starts and lengths): every sequence has the same size, slots in another order"""
    _, seqs, new, length, heads, per, dim = case
    codes = [torch.randint(-127, 128, (seqs, heads, length, dim), generator=g).to(torch.int8) for _ in range(2)]
    ks = (0.5 + torch.rand(seqs, heads, length, generator=g)) * (2 / 127)
    vs = (0.5 + torch.rand(seqs, heads, length, generator=g)) * (2 / 127) if scales is None else scales
    q = torch.randn(seqs * new, heads * per, dim, generator=g).to(dtype)
    return q, [codes[0], ks, codes[1], vs], [new * b for b in range(seqs + 1)], [length] * seqs


def attend(q8, q, host, starts, lens, causal=True):
    """(the operator's output, the 64-bit one, the 64-bit sum of weight x |value|)"""
    seqs = len(lens)
    slots = list(range(seqs))[::-1]
    cache = q8.KV8Cache(*(t.cuda() for t in host))
    batch = q8.Batch(ints(slots), ints(starts), ints(lens), max(b - a for a, b in zip(starts, starts[1:])), max(lens))
    got = q8.kv_attention(q.cuda(), cache, batch, causal=causal).cpu()
    k, v = (host[i].double() * host[i + 1].double()[..., None] for i in (0, 2))
    scale = q.shape[2] ** -0.5
    return got, ref.attention(q, k, v, slots, starts, lens, causal, scale), ref.attention(q, k, v.abs(), slots, starts, lens, causal, scale)


@pytest.fixture(scope="module")
def q8():
    from whisperjav_amd import q8
    assert torch.cuda.is_available()
    return q8


@pytest.mark.parametrize("case", CASES, ids=IDS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_sixteen_bit_outputs_are_the_nearest_ones(q8, case, dtype):
    """Before its last rounding a result is off by about 2^-18 of its row (scores below 16 in units of log2, their queries and sums good to
    2^-22, numerators to 2^-21): it rounds to another value than the exact result does where that lies as near to a border between
    two values.  A step between values is at least 2^-p of the value itself (p = 10, 8 - 1), so of normally distributed results the share is at most
    2^(p - 17) (0.8 ln 2^(17 - p) + 0.3): 3.3 % for float16, 0.6 % for bfloat16.  One half per weight makes it 8 % for bfloat16."""
    q, host, starts, lens = make(q8, rng(case[3] + case[6]), case, dtype)
    got, want, _ = attend(q8, q, host, starts, lens)
    off = float((got != want.to(dtype)).double().mean())
    assert off <= {torch.float16: 0.04, torch.bfloat16: 0.01}[dtype], off


def value_scales(kind, g, shape):
    """float32 value scales [sequence][head][position]"""
    length, near = shape[2], (0.5 + torch.rand(shape, generator=g, dtype=torch.float64))
    along = torch.arange(length, dtype=torch.float64) / max(1, length - 1)
    if kind == "huge":                                       # rows of up to 3.4e38: the largest scales that a finite row has
        return (near / 1.5 * 2.67e36).float()
    if kind == "tiny":
        return (near * 2.0 ** -105).float()
    if kind == "one_huge":                                   # a single position of them among ordinary ones
        s = near * 0.016
        s[:, :, length // 2] = 2.0e36
        return s.float()
    if kind == "growing":
        return (near * 2.0 ** (-60 + 170 * along)).float()
    if kind == "shrinking":
        return (near * 2.0 ** (110 - 170 * along)).float()
    if kind == "spread":
        return (near * 2.0 ** (torch.rand(shape, generator=g, dtype=torch.float64) * 80 - 40)).float()
    if kind == "spread_16":                                  # ... within float16's own range
        return (near * 2.0 ** (torch.rand(shape, generator=g, dtype=torch.float64) * 24 - 20)).float()
    assert kind == "zeros"
    return torch.where(torch.rand(shape, generator=g) < 0.5, torch.zeros(()), near.float() * 0.016)


@pytest.mark.parametrize("case", CASES, ids=IDS)
@pytest.mark.parametrize("dtype,kind", [(t, k) for t in (torch.float32, torch.bfloat16) for k in ("huge", "tiny", "one_huge", "growing", "shrinking", "spread", "zeros")]
                         + [(torch.float16, "spread_16"), (torch.float16, "zeros")])
def test_value_scales_of_any_size(q8, case, dtype, kind):
    """A row's output against 64 bits, relative to its sum of weight x |value|.  A weight is off by 2^-18 at most: scores stay below 16 in units of log2
    (checked) and are good to 2^-22 of that (2^-18 ln 2), numerators to 2^-21; the sums of a few thousand float32 terms add about 2^-20.  Numerators
    lose 2^-24 of at least 2^10 a position besides, times a code of 127 against one of 64 (what a row's largest code here exceeds): 2^-33 each."""
    name, seqs, new, length, heads, per, dim = case
    g = rng(length + dim + len(kind))
    q, host, starts, lens = make(q8, g, case, dtype, value_scales(kind, g, (seqs, heads, length)))
    k = host[0].double() * host[1].double()[..., None]
    most = max(float((k[s, h] @ q[:, h * per:(h + 1) * per].double().reshape(-1, dim).t()).abs().max()) for s in range(seqs) for h in range(heads))
    assert most * dim ** -0.5 * 1.4427 < 16
    if kind == "zeros":                                       # the position with the highest score of each (sequence, head) has nothing to give
        for s in range(seqs):
            for h in range(heads):
                rows = q[(seqs - 1 - s) * new:(seqs - s) * new, h * per:(h + 1) * per].double().reshape(-1, dim)
                host[3][s, h, int((k[s, h] @ rows.t()).amax(1).argmax())] = 0
    got, want, spread = attend(q8, q, host, starts, lens)
    assert bool(torch.isfinite(got).all())
    off = (got.double() - want).norm(dim=-1)
    step = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    lim = (2.0 ** -17 + length * 2.0 ** -33) * spread.norm(dim=-1) + step * want.norm(dim=-1) + 2.0 ** -126 * dim
    assert bool((off <= lim).all()), float((off / lim).max())


@pytest.mark.parametrize("case", CASES, ids=IDS)
@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_all_zero(q8, case, dtype):
    _, seqs, _, length, heads, _, _ = case
    q, host, starts, lens = make(q8, rng(5), case, dtype, torch.zeros(seqs, heads, length))
    got, _, _ = attend(q8, q, host, starts, lens)
    assert bool((got == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("positions", [1, 5, 40])
def test_largest_rows_written_and_read_by_attention(q8, dtype, positions):
    """alike rows come back as they were, one code's step off at most"""
    v = torch.full((positions, 2, 64), 3e38).to(dtype)
    v[:, :, 3] = 0
    v[:, :, 5] = -1e37
    cache, batch = q8.KV8Cache.empty(1, 2, 64, 64), q8.Batch(ints([0]), ints([0, positions]), ints([positions]), positions, positions)
    q8.kv_write(cache, torch.zeros_like(v).cuda(), v.cuda(), batch)
    got = q8.kv_attention(torch.ones(positions, 2, 64).to(dtype).cuda(), cache, batch).cpu().double()
    held = cache.v[0, :, 0].cpu().double() * cache.v_scale[0, :, 0].cpu().double()[:, None]
    assert bool(((got - held).abs() <= (2.0 ** -17 + {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}[dtype]) * held.abs()).all())


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_float32_outputs_are_good_to_18_bits(q8, case):
    """Weights are off by 2^-18 at most (see the value scales' test), each for itself: so is the sum of weight x value against its own norm.  Queries of
    one half would make it 2^-12 / sqrt(3) of a score of about 1.7 (in units of log2), 1.7e-4; numerators of one half 2^-12 / sqrt(3), 1.4e-4."""
    q, host, starts, lens = make(q8, rng(case[3] + case[6]), case, torch.float32)
    got, want, _ = attend(q8, q, host, starts, lens)
    assert float((got.double() - want).norm() / want.norm()) <= 2.0 ** -18


@pytest.mark.parametrize("case", CASES, ids=IDS)
@pytest.mark.parametrize("dtype,power", [(torch.float16, -18), (torch.float16, 9), (torch.bfloat16, -100), (torch.bfloat16, 100), (torch.float32, -100), (torch.float32, 100)])
def test_queries_of_any_size(q8, case, dtype, power):
    """queries 2^power times as large under a scale 2^-power times as large (float16 ones below 2^-14 have fewer bits: those they have count)"""
    q, host, starts, lens = make(q8, rng(case[3] + case[6]), case, torch.float32)
    q = (q.double() * 2.0 ** power).to(dtype)
    seqs, scale = len(lens), q.shape[2] ** -0.5 * 2.0 ** -power
    slots = list(range(seqs))
    cache = q8.KV8Cache(*(t.cuda() for t in host))
    batch = q8.Batch(ints(slots), ints(starts), ints(lens), max(b - a for a, b in zip(starts, starts[1:])), max(lens))
    got = q8.kv_attention(q.cuda(), cache, batch, scale=scale).cpu()
    k, v = (host[i].double() * host[i + 1].double()[..., None] for i in (0, 2))
    want = ref.attention(q, k, v, slots, starts, lens, True, scale)
    if dtype == torch.float32:
        assert float((got.double() - want).norm() / want.norm()) <= 2.0 ** -18
    else:
        off = float((got != want.to(dtype)).double().mean())
        assert off <= {torch.float16: 0.04, torch.bfloat16: 0.01}[dtype], off

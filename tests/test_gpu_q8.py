"""The 8-bit decoder operators (whisperjav_amd/q8.py) against plain 64-bit forms, at the sizes, strides and masks where they can go wrong.

Tolerances count roundings: a value rounded to a type is off by at most U[type] relative to itself; a float32 sum of n terms in any order by
n * 2^-24 of the sum of magnitudes; a code by half a step plus the float32 error of the value it stands for."""
import math

import pytest
import torch

from tests import q8_ref as ref

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}     # half a step of the smallest values
E = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def q8():
    from whisperjav_amd import q8
    assert torch.cuda.is_available()
    return q8


def rng(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def strided(t, pad, offset=0):
    """The same rows on the GPU in storage whose rows are `pad` elements longer, starting `offset` elements in."""
    rows, cols = t.shape
    room = torch.full((rows * (cols + pad) + offset + 1,), 7, dtype=t.dtype).cuda()
    view = room[offset: offset + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    view.copy_(t.cuda())
    return view


def check_rows(codes, scale, y, e):
    """Codes and scale stand for the float64 rows y, known to a relative `e`."""
    want_codes, want = ref.quantize(y)
    codes, scale = codes.cpu(), scale.cpu().double()
    assert codes.dtype == torch.int8 and int(codes.int().abs().max() if codes.numel() else 0) <= 127
    bad = torch.isnan(want)
    assert torch.equal(torch.isnan(scale), bad)
    assert bool((codes[bad] == 0).all())
    ok = ~bad
    assert bool(((scale[ok] - want[ok]).abs() <= (e + 2 * E) * want[ok] + 2.0 ** -149).all())
    off = (codes[ok].double() * want[ok][:, None] - y.double()[ok]).abs()
    lim = want[ok][:, None] * (0.5 + 127 * (2 * e + 4 * E)) + 2.0 ** -149
    assert bool((off <= lim).all()), float((off / lim.clamp_min(1e-300)).max())


# ---- rows -------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 2048), (3, 17), (5, 64), (2, 255), (7, 256), (4, 1000), (9, 1280), (3, 2040), (130, 2048), (2, 4097),
                                       (3, 6144), (2, 8192), (1, 20000), (1, 32768)])
@pytest.mark.parametrize("dtype,delta", [(torch.float32, torch.float16), (torch.float16, torch.float16), (torch.bfloat16, torch.float32),
                                         (torch.float32, None), (torch.bfloat16, None), (torch.float32, torch.bfloat16)])
def test_rmsnorm(q8, rows, cols, dtype, delta):
    g = rng(rows * 7 + cols)
    x = torch.randn(rows, cols, generator=g).to(dtype)
    d = torch.randn(rows, cols, generator=g).to(delta) if delta else None
    w = 1 + 0.2 * torch.randn(cols, generator=g)
    for pad, offset in ((0, 0), (3, 1), (8, 8)):
        xd, dd = strided(x, pad, offset), None if d is None else strided(d, pad + 1, offset)
        res = strided(torch.zeros_like(x), pad, offset)
        codes, scale = q8.rmsnorm(xd, w.cuda(), 1e-5, delta=dd, residual=res)
        r, y = ref.rmsnorm(x, w, 1e-5, d)
        # sum of squares: cols * E, halved by the root; the sum x + delta, the root, two products: 6 E
        check_rows(codes, scale, y, (cols / 2 + 8) * E)
        assert bool(((res.cpu().double() - r).abs() <= (U[dtype] + E) * r.abs() + TINY[dtype]).all())
        assert torch.equal(xd.cpu(), x)
        # in place: the same codes, and x holds the sum
        again, scale2 = q8.rmsnorm(xd, w.cuda(), 1e-5, delta=dd)
        assert torch.equal(again, codes) and torch.equal(scale2, scale)
        assert torch.equal(xd, res if d is not None else xd)


@pytest.mark.parametrize("cols", [40, 2048, 5000])
def test_rows_that_are_empty_or_not_finite(q8, cols):
    g = rng(cols)
    x = torch.randn(8, cols, generator=g)
    x[1] = 0
    x[2, cols // 2] = math.inf
    x[3, cols - 1] = math.nan
    x[4, 0] = -math.inf
    x[5] *= 1e-38                     # maximum near the smallest normal numbers
    x[6] = 0
    x[6, 3] = 1e-44
    codes, scale = q8.quantize(x.cuda())
    check_rows(codes, scale, x, 0.0)
    codes, scale = q8.rmsnorm(x[:5].cuda(), torch.ones(cols).cuda(), 1e-6)
    assert torch.isnan(scale.cpu()).tolist() == [False, False, True, True, True]
    assert bool((codes[1] == 0).all()) and float(scale[1]) == 0.0
    values = q8.dequantize(codes, scale)
    assert bool(torch.isnan(values[2:]).all()) and bool(torch.isfinite(values[:2]).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_ties_go_to_the_even_code(q8, dtype):
    """127 x / max that lies half way between two codes, exactly: maxima whose 127th part is no float32"""
    tops = torch.tensor([1 + i / 32 for i in range(32)], dtype=torch.float64)
    parts = torch.tensor([1.0, -0.5, 0.5, -0.0, 1 / 256, 3 / 256], dtype=torch.float64)                 # of the maximum, exact in both types
    x = (tops[:, None] * parts).to(dtype)
    codes, scale = q8.quantize(x.cuda())
    exact = 127 * x.double() / tops[:, None]                                                           # multiples of 127 / 256: exact
    assert torch.equal(codes.cpu().double(), torch.round(exact) + 0.0)
    assert torch.equal(scale.cpu(), (tops / 127).float())
    k = x.repeat(1, 11)[:, :64].reshape(32, 1, 64).cuda()
    cache = q8.KV8Cache.empty(1, 1, 32, 64)
    q8.kv_write(cache, k, -k, make_batch(q8, [0], [0, 32], [32]))
    want = torch.round(exact).repeat(1, 11)[:, :64]
    assert torch.equal(cache.k[0, 0].cpu().double(), want + 0.0) and torch.equal(cache.v[0, 0].cpu().double(), 0.0 - want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_the_largest_values(q8, dtype):
    x = torch.randn(3, 300, generator=rng(1)).double()
    x = (x / x.abs().max() * torch.tensor([3.38e38, 2e30, 1e37], dtype=torch.float64)[:, None]).to(dtype)
    codes, scale = q8.quantize(x.cuda())
    check_rows(codes, scale, x, 0.0)


@pytest.mark.parametrize("rows,cols,block", [(1, 16, 16), (3, 48, 16), (24, 6144, 16), (5, 640, 640), (2, 33, 33), (4, 96, 8), (3, 6, 2), (2, 10000, 16), (1, 32768, 32768)])
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_swiglu(q8, rows, cols, block, dtype):
    x = (torch.randn(rows, 2 * cols, generator=rng(cols)) * 3).to(dtype)
    x[0, 0] = -200.0                   # exp overflows: silu is a zero
    for pad, offset in ((0, 0), (5, 3), (16, 16)):
        codes, scale = q8.quantize(strided(x, pad, offset), swiglu_block=block)
        check_rows(codes, scale, ref.swiglu(x, block), 16 * E)      # exponential 4 E, sum, quotient, product


@pytest.mark.parametrize("rows,cols", [(1, 1), (2, 15), (3, 16), (5, 2040), (300, 2048), (2, 12000)])
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_and_read_back(q8, rows, cols, dtype):
    x = torch.randn(rows, cols, generator=rng(rows + cols)).to(dtype)
    for pad, offset in ((0, 0), (1, 1), (32, 16)):
        codes, scale = q8.quantize(strided(x, pad, offset))
        assert codes.stride(0) % 16 == 0 and codes.shape == (rows, cols)
        check_rows(codes, scale, x, 0.0)
        for out in TYPES:
            assert torch.equal(q8.dequantize(codes, scale, out).cpu(), (codes.cpu().float() * scale.cpu()[:, None]).to(out))
            assert torch.equal(q8.dequantize(strided(codes.cpu(), pad, offset), scale, out).cpu(), (codes.cpu().float() * scale.cpu()[:, None]).to(out))


# ---- product ------------------------------------------------------------------------------------------------------------------------

def int8(g, rows, cols):
    return torch.randint(-128, 128, (rows, cols), generator=g).to(torch.int8)


def check_gemm(q8, g, m, n, k, dtype, bias, pads=((0, 0),)):
    a, w = int8(g, m, k), int8(g, n, k)
    sa, sw = torch.rand(m, generator=g) * 0.02, torch.rand(n, generator=g) * (0.02 / max(1, k) ** 0.5)
    b = torch.randn(n, generator=g) if bias else None
    want, prod = ref.gemm(a, sa, w, sw, b), ref.gemm(a, sa, w, sw).abs()
    for pad, offset in pads:
        out = strided(torch.zeros(m, n, dtype=dtype), 3, 1)
        got = q8.gemm(strided(a, pad, offset), sa.cuda(), strided(w, pad, offset), sw.cuda(), bias=None if b is None else b.cuda(), dtype=dtype)
        q8.gemm(strided(a, pad, offset), sa.cuda(), strided(w, pad, offset), sw.cuda(), bias=None if b is None else b.cuda(), out=out)
        assert torch.equal(out, got)
        lim = 4 * E * prod + (U[dtype] + E) * want.abs() + TINY[dtype]
        off = (got.cpu().double() - want).abs()
        assert bool((off <= lim).all()), (m, n, k, pad, float((off / lim.clamp_min(1e-300)).max()))


def pads_for(k):
    up = -k % 16
    return ((up, 0), (up + 16, 32), (up + 1, 0), (up, 3))       # rows at multiples of 16 bytes twice, then odd strides and an odd base


@pytest.mark.parametrize("m", [1, 2, 7, 16, 17, 33, 64, 65, 100, 129, 256, 300])
@pytest.mark.parametrize("n,k", [(1, 1), (16, 64), (33, 65), (100, 127), (130, 129), (257, 512), (64, 1285)])
def test_gemm_sizes(q8, m, n, k):
    check_gemm(q8, rng(m * 1000 + n + k), m, n, k, torch.float32, True, pads_for(k))


@pytest.mark.parametrize("m,n,k", [(1, 4096, 2048), (24, 2048, 6144), (240, 1280, 5120), (513, 1030, 1000), (1000, 520, 384), (770, 2304, 640)])
@pytest.mark.parametrize("dtype,bias", [(torch.float16, False), (torch.bfloat16, True), (torch.float32, True)])
def test_gemm_layers(q8, m, n, k, dtype, bias):
    check_gemm(q8, rng(m + n + k), m, n, k, dtype, bias, ((-k % 16, 0),))


@pytest.mark.parametrize("dtype,m,n", [(torch.float32, 8200, 8301), (torch.bfloat16, 16397, 8301)])
def test_gemm_output_beyond_the_caches(q8, dtype, m, n):
    """an output of more than 256 MiB takes other stores: the same bits as its parts computed alone, and the formula's values"""
    k, g = 130, rng(m)
    a, w = strided(int8(g, m, k), 14), strided(int8(g, n, k), 14)
    sa, sw = torch.rand(m, generator=g) * 0.02, torch.rand(n, generator=g) * 0.02
    got = q8.gemm(a, sa.cuda(), w, sw.cuda(), dtype=dtype)
    for lo in range(0, m, 2050):
        part = slice(lo, min(m, lo + 2050))
        assert torch.equal(got[part], q8.gemm(a[part], sa[part].cuda(), w, sw.cuda(), dtype=dtype)), lo
    rows = torch.tensor([0, 1, 255, 256, m // 2, m - 2, m - 1])
    want = ref.gemm(a[rows.cuda()].cpu(), sa[rows], w.cpu(), sw)
    assert bool(((got[rows.cuda()].cpu().double() - want).abs() <= 4 * E * want.abs() + (U[dtype] + E) * want.abs() + TINY[dtype]).all())


def test_gemm_largest_sum_is_exact(q8):
    k = 131071
    a = torch.full((3, k), -128, dtype=torch.int8)
    a[1] = 127
    w = torch.full((20, k), -128, dtype=torch.int8)
    one = torch.ones(20).cuda()
    for up in (-k % 16, -k % 16 + 1):
        got = q8.gemm(strided(a, up), one[:3], strided(w, up), one, dtype=torch.float32).cpu()
        assert torch.equal(got[0], torch.full((20,), float(128 * 128 * k))) and torch.equal(got[1], torch.full((20,), -float(127 * 128 * k)))


def test_gemm_empty(q8):
    z = torch.zeros
    one = torch.ones(5).cuda()
    assert q8.gemm(z(0, 8, dtype=torch.int8).cuda(), one[:0], z(5, 8, dtype=torch.int8).cuda(), one).shape == (0, 5)
    assert q8.gemm(z(5, 8, dtype=torch.int8).cuda(), one, z(0, 8, dtype=torch.int8).cuda(), one[:0]).shape == (5, 0)
    bias = torch.arange(4.0).cuda()
    got = q8.gemm(z(5, 0, dtype=torch.int8).cuda(), one, z(4, 0, dtype=torch.int8).cuda(), one[:4], bias=bias, dtype=torch.float32)
    assert torch.equal(got, bias.expand(5, 4))
    assert q8.rmsnorm(z(0, 8).cuda(), torch.ones(8).cuda())[0].shape == (0, 8)
    assert q8.quantize(z(0, 8).cuda())[1].shape == (0,)
    assert q8.dequantize(z(0, 8, dtype=torch.int8).cuda(), one[:0]).shape == (0, 8)


def test_gemm_row_of_nan_scale_stays_a_row(q8):
    g = rng(4)
    a, w = int8(g, 70, 256).cuda(), int8(g, 96, 256).cuda()
    sa = torch.ones(70).cuda()
    sa[13] = math.nan
    got = q8.gemm(a, sa, w, torch.ones(96).cuda(), dtype=torch.float32)
    assert bool(torch.isnan(got[13]).all()) and not bool(torch.isnan(got[torch.arange(70) != 13]).any())


# ---- cache ----------------------------------------------------------------------------------------------------------------------------

def make_batch(q8, slots, starts, lens, max_new=None, max_len=None):
    def ints(v):
        return torch.tensor(v, dtype=torch.int32).cuda()
    news = [b - a for a, b in zip(starts, starts[1:])]
    return q8.Batch(ints(slots), ints(starts), ints(lens), max(news + [0]) if max_new is None else max_new, max(lens + [0]) if max_len is None else max_len)


@pytest.mark.parametrize("dim,heads", [(64, 1), (64, 20), (128, 2), (128, 8)])
@pytest.mark.parametrize("dtype", TYPES)
def test_kv_write_and_read(q8, dim, heads, dtype):
    g, ctx, n_slots = rng(dim + heads), 45, 6
    slots, starts, lens = [4, -1, 0, 2, 9, 5, 1], [0, 3, 5, 5, 25, 27, 28, 33], [7, 2, 5, 20, 4, 45, 47]        # slots 4, 0, 2, 5, 1; 1 runs past the end
    rows = starts[-1] + 2                                                                                       # two rows that nobody owns
    k, v = (torch.randn(rows, heads, dim, generator=g).to(dtype) for _ in range(2))
    k[6, 0, 3] = math.nan
    v[7] = 0
    fused = torch.cat([torch.zeros(rows, 5, dtype=dtype), k.reshape(rows, -1), v.reshape(rows, -1)], 1).cuda()   # k and v as views of one matrix
    n = heads * dim
    cache = q8.KV8Cache.empty(n_slots, heads, ctx, dim)
    for t in cache:
        t.fill_(3)
    for hint in (None, 1, 100):
        batch = make_batch(q8, slots, starts, lens, max_new=hint)
        q8.kv_write(cache, fused[:, 5: 5 + n].view(rows, heads, dim), fused[:, 5 + n:].view(rows, heads, dim), batch)
        owned = {}
        for b, t, pos in ref.spans(starts, lens, rows):
            if 0 <= slots[b] < n_slots and 0 <= pos < ctx:
                owned[(slots[b], pos)] = t
        host = [t.cpu() for t in cache]
        for codes, scale, x in ((host[0], host[1], k), (host[2], host[3], v)):
            for s in range(n_slots):
                for p in range(ctx):
                    if (s, p) in owned:
                        check_rows(codes[s, :, p], scale[s, :, p], x[owned[(s, p)]], 0.0)
                    else:
                        assert bool((codes[s, :, p] == 3).all()) and bool((scale[s, :, p] == 3).all())
        for out in TYPES:
            rk, rv = q8.kv_read(cache, batch, rows, out)
            for b, t, pos in ref.spans(starts, lens, rows):
                there = 0 <= slots[b] < n_slots and 0 <= pos < ctx
                for got, codes, scale in ((rk, host[0], host[1]), (rv, host[2], host[3])):
                    want = (codes[slots[b], :, pos].float() * scale[slots[b], :, pos, None]).to(out) if there else torch.zeros(heads, dim, dtype=out)
                    assert torch.equal(torch.nan_to_num(got[t].cpu(), 11.0), torch.nan_to_num(want, 11.0)), (b, t, pos)


def test_kv_rows_behind_are_left(q8):
    cache = q8.KV8Cache.empty(2, 1, 8, 64)
    batch = make_batch(q8, [0, 1], [0, 2, 3], [2, 1])
    k = torch.randn(6, 1, 64).cuda()
    q8.kv_write(cache, k, k, batch)
    out = torch.full((6, 2, 64), 5.0, device="cuda")
    q8.kv_attention(torch.randn(6, 2, 64).cuda(), cache, batch, out=out)
    assert bool((out[3:] == 5).all()) and not bool((out[:3] == 5).any())


# ---- attention --------------------------------------------------------------------------------------------------------------------------

def filled_cache(q8, g, n_slots, heads, ctx, dim):
    codes = [torch.randint(-127, 128, (n_slots, heads, ctx, dim), generator=g).to(torch.int8) for _ in range(2)]
    scales = [(0.5 + torch.rand(n_slots, heads, ctx, generator=g)) * (2 / 127) for _ in range(2)]
    values = [c.double() * s.double()[..., None] for c, s in zip(codes, scales)]
    return [codes[0], scales[0], codes[1], scales[1]], values


def poison_behind(host, slots, lens, causal):
    """Whatever lies behind the last visible position: scales of NaN and infinity, codes of both ends."""
    for s in range(host[0].shape[0]):
        n = max([min(l, host[0].shape[2]) for b, l in zip(slots, lens) if b == s] + [0])
        for codes, scale in ((host[0], host[1]), (host[2], host[3])):
            codes[s, :, n:] = -128
            scale[s, :, n:] = math.nan
            scale[s, :, n + 1::2] = math.inf


def check_attention(got, q, values, slots, starts, lens, causal, scale, dtype):
    k, v = values
    want = ref.attention(q, k, v, slots, starts, lens, causal, scale)
    spread = ref.attention(q, k, v.abs(), slots, starts, lens, causal, scale)          # sum of weight x |value|
    dim, per = q.shape[2], q.shape[1] // k.shape[1]
    # a score: dim products and sums in float32, scales and 22-bit operands: (dim + 16) E of the sum of magnitudes, which is at most
    # dim * max |q| * max |k|; two scores make a weight.  exp, running sums and the merge of parts: (keys / 8 + 64) E.
    top = q.double().abs().amax(-1) * k.abs().amax() * dim ** 0.5 * abs(scale) * dim ** 0.5
    keys = max(lens + [1])
    e = 2 * (dim + 16) * E * top.clamp_max(1e6) + (keys / 8 + 64) * E
    if dtype != torch.float32:
        e = e + 2.0 ** -10                                                                # a weight carried in 16 bits, and their sum
    # A numerator is carried in halves, whose step is 2^-24 at least: off by 2^-25, times a code of at most 128.  The largest numerator is kept
    # above 2^10 = 2^11 * (its value scale / that scale's next power of two), so the denominator is above 2^10 / vs for some vs: per position
    # the output is off by 2^-25 * 128 vs / 2^10 = 2^-35 * 128 vs, whatever the small weights are, and 64 vs < max |v| here.
    floor = keys * 2.0 ** -34 * v.abs().amax()
    lim = e[..., None] * spread + (U[dtype] + E) * want.abs() + TINY[dtype] + floor
    got = got.cpu().double()
    owned = torch.zeros(q.shape[0], dtype=torch.bool)
    for _, t, _ in ref.spans(starts, lens, q.shape[0]):
        owned[t] = True
    off = (got - want).abs()[owned]
    assert bool(torch.isfinite(got[owned]).all())
    assert bool((off <= lim[owned]).all()), float((off / lim[owned].clamp_min(1e-300)).max())


LAYOUTS = {
    # slots, starts, lens: the rows are the last positions
    "one": ([1], [0, 1], [1]),
    "steps": ([3, 0, 1, 2], [0, 1, 2, 3, 4], [1, 64, 65, 200]),
    "ragged": ([2, 0, -1, 3, 1, 7], [0, 5, 5, 8, 24, 41, 42], [70, 3, 9, 16, 130, 4]),
    "hundreds": ([4, 0], [0, 1, 4], [199, 180]),
    "short": ([0, 1, 2], [0, 4, 8, 20], [2, 0, 12]),                    # rows before position 0; an empty cache
    "past": ([0, 1], [0, 2, 5], [201, 260]),                             # lengths beyond the cache's 200 positions
    "prompt": ([1, 0, 3], [0, 150, 151, 351], [150, 1, 200]),
}


@pytest.mark.parametrize("layout", sorted(LAYOUTS))
@pytest.mark.parametrize("dim,heads,per", [(64, 1, 1), (64, 2, 5), (128, 1, 2), (128, 2, 4), (128, 1, 16), (64, 3, 1)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_attention(q8, layout, dim, heads, per, dtype, causal):
    slots, starts, lens = LAYOUTS[layout]
    g, ctx, n_slots = rng(dim + heads + per), 200, 5
    host, values = filled_cache(q8, g, n_slots, heads, ctx, dim)
    poison_behind(host, slots, lens, causal)
    cache = q8.KV8Cache(*(t.cuda() for t in host))
    rows = starts[-1] + 1
    q = (torch.randn(rows, heads * per, dim, generator=g) * 1.5).to(dtype)
    wide = torch.zeros(rows, heads * per * dim + 8, dtype=dtype).cuda()
    wide[:, 8:] = q.reshape(rows, -1).cuda()
    out = torch.zeros(rows, heads * per + 1, dim, dtype=dtype).cuda()
    for hint_new, hint_len in ((None, None), (1, 1)):
        batch = make_batch(q8, slots, starts, lens, hint_new, hint_len)
        got = q8.kv_attention(wide[:, 8:].view(rows, heads * per, dim), cache, batch, causal=causal, out=out[:, : heads * per])
        check_attention(got, q, values, slots, starts, lens, causal, dim ** -0.5, dtype)
        assert bool((out[:, heads * per] == 0).all()) and bool((out[-1] == 0).all())


@pytest.mark.parametrize("dim,heads,per", [(64, 4, 1), (64, 2, 3), (128, 3, 2), (128, 2, 4), (64, 8, 1), (128, 8, 1), (64, 1, 16)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_attention_of_many_prompts(q8, dim, heads, per, dtype, causal):
    """whole prompts and later parts of them, enough of them for the kernel that takes 128 rows at a time"""
    g, ctx, n_slots = rng(dim * heads + per), 210, 30
    slots = torch.randperm(n_slots, generator=g).tolist()[:26]
    slots[3], slots[9] = -1, n_slots
    starts, lens = [0], []
    for b in range(26):
        n = int(torch.randint(0, 60, (1,), generator=g)) * (3 if b % 4 == 0 else 1)
        starts.append(starts[-1] + n)
        lens.append(n if b % 3 else min(ctx, n + 37))
    lens[5], lens[6] = max(0, lens[5] - 7), 64                              # rows before position 0; whole 64s
    host, values = filled_cache(q8, g, n_slots, heads, ctx, dim)
    poison_behind(host, slots, lens, causal)
    cache = q8.KV8Cache(*(t.cuda() for t in host))
    rows = starts[-1] + 3
    q = (torch.randn(rows, heads * per, dim, generator=g) * 1.5).to(dtype)
    out = torch.zeros(rows, heads * per + 1, dim, dtype=dtype).cuda()
    for hint in (None, 150):
        batch = make_batch(q8, slots, starts, lens, hint)
        got = q8.kv_attention(q.cuda(), cache, batch, causal=causal, out=out[:, : heads * per])
        check_attention(got, q, values, slots, starts, lens, causal, dim ** -0.5, dtype)
        assert bool((out[:, heads * per] == 0).all()) and bool((out[starts[-1]:] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,length", [(1, 5000), (3, 4099), (20, 3001), (70, 2500), (1, 1000), (13, 777)])
def test_attention_over_a_long_cache(q8, dtype, new, length):
    """few rows, many positions: the work is split over the positions and joined"""
    g = rng(length)
    host, values = filled_cache(q8, g, 2, 1, length + 3, 128)
    slots, starts, lens = [1, 0], [0, new, new + 1], [length, 129]
    poison_behind(host, slots, lens, True)
    q = (torch.randn(new + 1, 2, 128, generator=g) * 1.5).to(dtype)
    cache, batch = q8.KV8Cache(*(t.cuda() for t in host)), make_batch(q8, slots, starts, lens)
    got = q8.kv_attention(q.cuda(), cache, batch)
    check_attention(got, q, values, slots, starts, lens, True, 128 ** -0.5, dtype)
    assert torch.equal(got, q8.kv_attention(q.cuda(), cache, batch))            # the same bits again


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_peaked_and_flat(q8, dtype):
    """scores far apart (one weight is all), all alike (every weight the same), and a scale of zero"""
    g = rng(3)
    host, values = filled_cache(q8, g, 1, 2, 300, 128)
    cache = q8.KV8Cache(*(t.cuda() for t in host))
    q = torch.randn(3, 4, 128, generator=g)
    q[0] *= 60
    q[1] = 0
    q = q.to(dtype)
    batch = make_batch(q8, [0], [0, 3], [300])
    for scale in (128 ** -0.5, 0.0, -1.0 / 128):
        check_attention(q8.kv_attention(q.cuda(), cache, batch, scale=scale), q, values, [0], [0, 3], [300], True, scale, dtype)


@pytest.mark.parametrize("new", [1, 40])
def test_attention_of_a_row_that_is_not_finite(q8, new):
    """a cached row that was not finite makes NaN of the rows that see it, and of no other; so does a query"""
    g = rng(new)
    host, _ = filled_cache(q8, g, 2, 1, 120, 64)
    host[1][0, 0, 90] = math.nan
    cache = q8.KV8Cache(*(t.cuda() for t in host))
    starts, lens = [0, new, 2 * new], [100, 100]
    q = torch.randn(2 * new, 2, 64, generator=g)
    q[new, 1, 5] = math.inf
    got = q8.kv_attention(q.cuda(), cache, make_batch(q8, [0, 1], starts, lens)).cpu()
    for t in range(new):
        sees = 100 - new + t >= 90
        assert bool(torch.isnan(got[t]).all()) == sees and bool(torch.isfinite(got[t]).all()) != sees
    assert bool(torch.isnan(got[new, 1]).all()) and bool(torch.isfinite(got[new, 0]).all()) and bool(torch.isfinite(got[new + 1:]).all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", TYPES)
def test_many_prompts_with_rows_that_are_not_finite_or_peaked(q8, dim, dtype):
    """in the kernel for many rows: NaN stays with the rows that see it; scores far apart, all alike, and none at all"""
    g, seqs, heads, new, length = rng(dim), 52, 4, 70, 100
    host, values = filled_cache(q8, g, seqs, heads, 110, dim)
    slots, starts, lens = list(range(seqs)), [new * b for b in range(seqs + 1)], [length] * seqs
    poison_behind(host, slots, lens, True)
    q = torch.randn(seqs * new, 2 * heads, dim, generator=g)
    q[2 * new] *= 60
    q[2 * new + 1] = 0
    q = q.to(dtype)
    cache = q8.KV8Cache(*(t.cuda() for t in host))
    batch = make_batch(q8, slots, starts, lens)
    for scale in (dim ** -0.5, 0.0):
        check_attention(q8.kv_attention(q.cuda(), cache, batch, scale=scale), q, values, slots, starts, lens, True, scale, dtype)
    host[1][0, 1, 90] = math.nan                                              # a key of head 1 of sequence 0
    bad = q.clone()
    bad[new + 7, 5, dim - 1] = math.inf                                       # a query of sequence 1
    cache = q8.KV8Cache(*(t.cuda() for t in host))
    clean = q8.kv_attention(q.cuda(), q8.KV8Cache(*(t.cuda() for t in [host[0], host[1].nan_to_num(0.01), host[2], host[3]])), batch).cpu()
    got = q8.kv_attention(bad.cuda(), cache, batch).cpu()
    want = torch.zeros(seqs * new, 2 * heads, dtype=torch.bool)
    want[90 - (length - new):new, 2:4] = True
    want[new + 7, 5] = True
    assert torch.equal(torch.isnan(got).all(-1), want) and torch.equal(torch.isnan(got).any(-1), want)
    assert torch.equal(got[~want], clean[~want])


# ---- together ---------------------------------------------------------------------------------------------------------------------------

class Layer:
    """One decoder layer (no rotary embedding: it is not an operator of this set) over the 8-bit operators."""

    def __init__(self, q8, g, hidden=256, heads=4, kv=2, dim=64, ffn=320, slots=3, ctx=96):
        self.q8, self.heads, self.kv, self.dim = q8, heads, kv, dim
        rows = lambda n, k: q8.quantize((torch.randn(n, k, generator=g) / k ** 0.5).cuda())      # noqa: E731
        self.qkv, self.o, self.gu, self.down = rows((heads + 2 * kv) * dim, hidden), rows(hidden, heads * dim), rows(2 * ffn, hidden), rows(hidden, ffn)
        self.ln1, self.ln2 = ((1 + 0.1 * torch.randn(hidden, generator=g)).cuda() for _ in range(2))
        self.cache = q8.KV8Cache.empty(slots, kv, ctx, dim)

    def __call__(self, x, delta, batch):
        q8, n, steps = self.q8, x.shape[0], {}
        a = q8.rmsnorm(x, self.ln1, 1e-6, delta=delta)
        qkv = q8.gemm(*a, *self.qkv)
        q, k, v = (t.view(n, -1, self.dim) for t in qkv.split([self.heads * self.dim, self.kv * self.dim, self.kv * self.dim], 1))
        q8.kv_write(self.cache, k, v, batch)
        o = q8.kv_attention(q, self.cache, batch)
        ao = q8.gemm(*q8.quantize(o.view(n, -1)), *self.o)
        b = q8.rmsnorm(x, self.ln2, 1e-6, delta=ao)
        gu = q8.gemm(*b, *self.gu)
        out = q8.gemm(*q8.quantize(gu, swiglu_block=16), *self.down)
        steps.update(qkv=qkv, o=o, ao=ao, gu=gu, out=out, x=x)
        return steps

    def reference(self, x, delta, batch, steps):
        """Every step in 64 bits from the step before it as the device holds it."""
        f = lambda t: t.cpu().double()                                   # noqa: E731
        w = {n: f(c) * f(s)[:, None] for n, (c, s) in (("qkv", self.qkv), ("o", self.o), ("gu", self.gu), ("down", self.down))}

        def product(y, name):
            codes, scale = ref.quantize(y)
            return (codes * scale[:, None]) @ w[name].t(), scale, w[name].abs().sum(1)
        r1, y1 = ref.rmsnorm(x, self.ln1.cpu(), 1e-6, delta)
        r2, y2 = ref.rmsnorm(r1, self.ln2.cpu(), 1e-6, f(steps["ao"]))
        return {"qkv": product(y1, "qkv"), "ao": product(f(steps["o"]).view(x.shape[0], -1), "o"), "gu": product(y2, "gu"),
                "out": product(ref.swiglu(f(steps["gu"]), 16), "down"), "x": r2}


def test_a_layer_prompt_then_steps(q8):
    g = rng(11)
    layer = Layer(q8, g)
    slots, starts, lens = [2, 0, 1], [0, 40, 41, 75], [40, 1, 34]
    for step in range(3):
        n = starts[-1]
        x, delta = torch.randn(n, 256, generator=g), torch.randn(n, 256, generator=g).half()
        batch = make_batch(q8, slots, starts, lens)
        xd = x.cuda()
        got = layer(xd, delta.cuda(), batch)
        want = layer.reference(x, delta, batch, got)
        for name in ("qkv", "ao", "gu", "out"):
            value, scale, weight = want[name]
            # a code next to a border may fall to the other side of it (one step, on at most one code in a hundred: here at most three of
            # a row's 256 or 320, each times the row's largest weight); the rest is the epilogue's rounding to float16
            step_off = 3 * scale[:, None] * (weight / 256 * 4)[None, :]
            lim = step_off + (U[torch.float16] + 8 * E) * value.abs() + 1e-5
            off = (got[name].cpu().double() - value).abs()
            assert bool((off <= lim).all()), (step, name, float((off / lim).max()))
        assert bool(((xd.cpu().double() - want["x"]).abs() <= 4 * E * want["x"].abs() + 4 * E).all())
        values = [layer.cache[i].cpu().double() * layer.cache[i + 1].cpu().double()[..., None] for i in (0, 2)]
        q = got["qkv"][:, :256].cpu().view(n, 4, 64)
        check_attention(got["o"], q, values, slots, starts, lens, True, 0.125, torch.float16)
        # the next token of every sequence
        starts, lens = [0, 1, 2, 3], [l + 1 for l in lens]


def test_a_layer_captured_and_replayed(q8):
    """one captured decode step, replayed while the batch's arrays change underneath, against the same calls made eagerly"""
    g = rng(12)
    eager, captured = Layer(q8, rng(5)), Layer(q8, rng(5))
    slots, starts, lens = [2, 0, 1], [0, 30, 31, 60], [30, 1, 29]
    x, delta = torch.randn(60, 256, generator=g).cuda(), torch.randn(60, 256, generator=g).half().cuda()
    for layer in (eager, captured):
        layer(x.clone(), delta, make_batch(q8, slots, starts, lens))
    xs, ds = torch.zeros(3, 256).cuda(), torch.zeros(3, 256).half().cuda()
    batch = make_batch(q8, slots, [0, 1, 2, 3], [31, 2, 30], max_new=1, max_len=96)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        captured(xs.clone(), ds, batch)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        steps = captured(xs, ds, batch)
    for step in range(5):
        x, delta = torch.randn(3, 256, generator=g), torch.randn(3, 256, generator=g).half()
        now = [l + 1 + step for l in lens]
        xe = x.cuda()
        want = eager(xe, delta.cuda(), make_batch(q8, slots, [0, 1, 2, 3], now, max_new=1, max_len=96))
        xs.copy_(x)
        ds.copy_(delta)
        batch.lens.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for name in want:
            assert torch.equal(steps[name], want[name]), (step, name)
        for a, b in zip(eager.cache, captured.cache):
            assert torch.equal(a, b)


def test_another_stream(q8):
    """calls made on a side stream run there, behind the work that fills their inputs"""
    g = rng(6)
    a, w = int8(g, 300, 512), int8(g, 256, 512)
    want = ref.gemm(a, torch.ones(300), w, torch.ones(256)).float()
    side = torch.cuda.Stream()
    one = torch.ones(300).cuda()
    aw = torch.zeros(300, 512, dtype=torch.int8).cuda(), torch.zeros(256, 512, dtype=torch.int8).cuda()
    big = torch.randn(4096, 4096).cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(4):
            big = big @ big * 1e-3
        aw[0].copy_(a.cuda(), non_blocking=True)
        aw[1].copy_(w.cuda(), non_blocking=True)
        got = q8.gemm(aw[0], one, aw[1], one[:256], dtype=torch.float32)
    side.synchronize()
    assert torch.equal(got.cpu(), want)


# ---- refusals ---------------------------------------------------------------------------------------------------------------------------

def test_refusals_on_the_device(q8):
    from whisperjav_amd.hipbind import WjError
    x = torch.zeros(4, 64).cuda()
    w = torch.ones(64).cuda()
    codes, scale = q8.quantize(x)
    with pytest.raises(ValueError):
        q8.quantize(x.t())
    with pytest.raises(ValueError):
        q8.rmsnorm(x, w[:32])
    with pytest.raises(ValueError):
        q8.rmsnorm(x, w, delta=torch.zeros(4, 64))                        # on the host
    with pytest.raises(ValueError):
        q8.rmsnorm(x, w, residual=x.half())
    with pytest.raises(ValueError):
        q8.rmsnorm(x, w, residual=x[:1].expand(4, 64))                    # rows overlap
    with pytest.raises(ValueError):
        q8.quantize(x, swiglu_block=5)
    with pytest.raises(WjError):
        q8.rmsnorm(x, w, -1.0)
    grad = torch.zeros(4, 64, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        q8.quantize(grad)
    with pytest.raises(ValueError, match="gradient"):
        q8.rmsnorm(x, w.clone().requires_grad_())
    with pytest.raises(ValueError, match="gradient"):
        q8.gemm(codes, scale, codes, scale, bias=torch.zeros(4, device="cuda", requires_grad=True))
    with torch.no_grad():
        q8.quantize(grad)
        q8.rmsnorm(x, w.clone().requires_grad_())
    with pytest.raises(WjError):
        q8.quantize(torch.zeros(1, 32769).cuda())
    with pytest.raises(ValueError):
        q8.gemm(codes, scale, codes[:, :32], scale)
    with pytest.raises(ValueError):
        q8.gemm(codes, scale, codes, scale, bias=w)
    with pytest.raises(ValueError):
        q8.gemm(codes, scale[:3], codes, scale)
    with pytest.raises(ValueError):
        q8.gemm(codes, scale, codes, scale, dtype=torch.float64)
    with pytest.raises(WjError):
        q8.gemm(torch.zeros(1, 131072, dtype=torch.int8).cuda(), scale[:1], torch.zeros(1, 131072, dtype=torch.int8).cuda(), scale[:1])
    cache = q8.KV8Cache.empty(2, 2, 8, 64)
    batch = make_batch(q8, [0], [0, 1], [1])
    k = torch.zeros(1, 2, 64).cuda()
    with pytest.raises(ValueError):
        q8.kv_write(cache, k, k.half(), batch)
    with pytest.raises(ValueError):
        q8.kv_write(cache, k[:, :1], k[:, :1], batch)
    with pytest.raises(ValueError):
        q8.kv_attention(torch.zeros(1, 2, 128).cuda(), cache, batch)
    with pytest.raises(WjError):
        q8.kv_attention(torch.zeros(1, 3, 64).cuda(), cache, batch)       # 3 query heads on 2
    with pytest.raises(WjError):
        q8.kv_attention(torch.zeros(1, 34, 64).cuda(), cache, batch)      # 17 each
    with pytest.raises(WjError):
        q8.kv_write(q8.KV8Cache.empty(2, 2, 8, 96), torch.zeros(1, 2, 96).cuda(), torch.zeros(1, 2, 96).cuda(), batch)
    with pytest.raises(ValueError):
        q8.kv_attention(k, q8.KV8Cache(cache.k, cache.k_scale, cache.v, cache.v_scale[:1]), batch)
    with pytest.raises(ValueError):
        q8.kv_attention(k, cache, batch._replace(lens=batch.lens.long()))
    with pytest.raises(ValueError):
        q8.kv_attention(k, cache, batch._replace(starts=batch.starts[:1]))
    with pytest.raises(ValueError):
        q8.kv_attention(k, cache, batch._replace(slots=batch.slots.cpu()))

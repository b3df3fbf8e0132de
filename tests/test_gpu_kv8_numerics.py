"""The arithmetic of the attention over the 8-bit cache (whisperjav_amd/q8.py): what its precision is, not only that it is right.

Every kernel that a call can take is reached: PLANS names them by what sends a call there."""
import math

import pytest
import torch

from tests import q8_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]

# sequences, new rows, positions, heads, queries per head, dim
PLANS = {
    "four_waves": (3, 1, 120, 2, 2, 128),                # 16 rows, up to 128 positions
    "eight_waves": (3, 2, 700, 2, 2, 128),               # 16 rows, more of them
    "parts": (2, 1, 2500, 1, 4, 128),                    # positions split over workgroups and joined
    "two_blocks": (2, 20, 300, 2, 1, 128),               # 32 rows
    "two_blocks_parts": (2, 20, 1300, 1, 1, 128),
    "many_rows": (26, 70, 110, 10, 1, 128),              # 128 rows (float32: 32)
}
CASES = [(name, *plan[:5], dim) for name, plan in PLANS.items() for dim in (64, 128)]
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

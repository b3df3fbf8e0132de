"""The operators of the 8-bit decoder step, as cases to be measured: RMSNorm with the residual's addition and 8-bit rows out,
8-bit rows of an activation or of a SwiGLU product, the int8 product with scales per token and channel, the int8 key / value
cache as it is written and read back, and the attention that reads it.

Codes are int8 in [-127, 127] with one float32 scale per row: scale = max |x| / 127, code = round-half-even(x / scale).  Rows are
laid out as the library's own producers lay them out: a row's codes start at a multiple of 16 bytes.
Sizes: Qwen3-ASR-1.7B (hidden 2048, 16 query heads on 8 key/value heads of 128, ffn 6144) and Whisper large-v3 (1280, 20 heads
of 64, 1500 encoder positions), and odd sizes around them.
"""
import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # one clip's next token: the first norm of a layer, 2048 columns, the attention's output joining the residual stream
        {"name": "norm_token", "op": "norm", "rows": 1, "cols": 2048, "dtype": "float32", "delta": "float16"},
        # the prompts of 32 half-minute clips in one pass
        {"name": "norm_prompt", "op": "norm", "rows": 16384, "cols": 2048, "dtype": "float32", "delta": "float16"},
        # SwiGLU of a decode batch of 24 clips: gate / up columns interleaved in blocks of 16, as the packed weights leave them
        {"name": "swiglu_step", "op": "quantize", "rows": 24, "cols": 6144, "dtype": "float16", "block": 16},
        # attention outputs of a prompt pass, one row short of a whole block and columns that are no multiple of 16
        {"name": "quantize_prompt", "op": "quantize", "rows": 16383, "cols": 2040, "dtype": "bfloat16", "block": 0},
        # one token through the fused q/k/v projection
        {"name": "gemm_token", "op": "gemm", "m": 1, "n": 4096, "k": 2048, "dtype": "float16", "bias": False},
        # a decode batch of 240 clips through the gate-up projection
        {"name": "gemm_batch", "op": "gemm", "m": 240, "n": 12288, "k": 2048, "dtype": "float16", "bias": False},
        # a prompt pass through the same projection
        {"name": "gemm_prompt", "op": "gemm", "m": 16384, "n": 12288, "k": 2048, "dtype": "bfloat16", "bias": False},
        # the caches of a decode batch of 48 clips take one position each
        {"name": "cache_step", "op": "cache", "seqs": 48, "len": 700, "new": 1, "kind": "step", "heads": 16, "kv": 8, "dim": 128, "ctx": 1024,
         "dtype": "float16"},
        # the caches of 32 clips take their prompts
        {"name": "cache_prompt", "op": "cache", "seqs": 32, "len": 1000, "new": 1000, "kind": "prompt", "heads": 16, "kv": 8, "dim": 128, "ctx": 1024,
         "dtype": "float16"},
        # one clip's next token
        {"name": "attend_token", "op": "attend", "seqs": 1, "len": 448, "new": 1, "kind": "step", "heads": 16, "kv": 8, "dim": 128, "ctx": 512,
         "dtype": "float16"},
        # the next tokens of a large decode batch, clips of unequal age
        {"name": "attend_batch", "op": "attend", "seqs": 512, "len": 1000, "new": 1, "kind": "step", "heads": 16, "kv": 8, "dim": 128, "ctx": 1024,
         "dtype": "float16"},
        # the prompts of 32 clips
        {"name": "attend_prompt", "op": "attend", "seqs": 32, "len": 1000, "new": 1000, "kind": "prompt", "heads": 16, "kv": 8, "dim": 128, "ctx": 1024,
         "dtype": "bfloat16"},
    ]


def _log(rng, low, high):
    """A whole number, spread over its logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["norm", "quantize", "gemm", "gemm", "cache", "attend", "attend"])
    dtype = rng.choice(["float16", "bfloat16", "float32"])
    if op == "norm":
        rows = _log(rng, 1, 16384)
        cols = _log(rng, 33, max(34, min(8192, 16384 * 2048 // rows)))
        return {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "delta": rng.choice(["", "float16", "bfloat16", "float32"])}
    if op == "quantize":
        rows = _log(rng, 1, 16384)
        cols = _log(rng, 33, max(34, min(8192, 16384 * 2040 // rows)))
        block = rng.choice([0, 16, cols])
        if block == 16:
            cols = max(16, cols // 16 * 16)
        if block:
            rows = max(1, rows // 2)
        if dtype == "float32":
            rows = max(1, rows // 2)
        return {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "block": block}
    if op == "gemm":
        m, n, k = _log(rng, 1, 16384), _log(rng, 33, 12288), _log(rng, 33, 6144)
        if dtype == "float32" and m * n > 16384 * 6144:
            m = 16384 * 6144 // n
        while m * n * k > 16384 * 12288 * 2048:
            k //= 2
        return {"op": op, "m": m, "n": n, "k": k, "dtype": dtype, "bias": rng.random() < 0.5}
    dim = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8, 20])
    group = rng.choice([1, 2, 4])
    kind = rng.choice(["step", "verify", "prompt", "cross"])
    seqs = _log(rng, 1, 512 if kind in ("step", "verify") else 32)
    length = _log(rng, 1, 1500 if kind != "prompt" else 1000)
    new = {"step": 1, "verify": min(length, rng.randint(2, 16)), "prompt": length, "cross": rng.randint(1, 6)}[kind]
    if op == "cache" and kind == "cross":
        new = length            # an encoder's states, all written at once
    most = 512 * 8 * 1000 * 128 if op == "attend" else 32 * 8 * 1000 * 128      # the largest listed case's codes
    while seqs > 1 and seqs * kv * (length if op == "attend" else new) * dim > most // 2:
        seqs //= 2
    if kind == "prompt" and op == "attend":
        while seqs > 1 and seqs * kv * group * length * length * dim > 32 * 16 * 1000 * 1000 * 128 // 2:
            seqs //= 2
        while length > 1 and seqs * kv * group * length * length * dim > 32 * 16 * 1000 * 1000 * 128 // 2:
            length //= 2
            new = length
    return {"op": op, "seqs": seqs, "len": length, "new": new, "kind": kind, "heads": kv * group, "kv": kv, "dim": dim,
            "ctx": length + rng.choice([0, 1, 37]), "dtype": dtype}


# ---- inputs -------------------------------------------------------------------------------------------------------------------

def _spans(case):
    """(positions after the call, new rows) of every sequence: clips of unequal length, the first the longest."""
    lens, news = [], []
    for b in range(case["seqs"]):
        part = (b * 0.6180339887498949) % 1.0
        n = case["len"] if case["kind"] == "cross" else max(1, int(case["len"] * (1.0 - 0.75 * part)))
        lens.append(n)
        if case["kind"] in ("prompt",) or (case["kind"] == "cross" and case["op"] == "cache"):
            news.append(n)
        elif case["kind"] == "verify":
            news.append(min(n, 1 + (case["new"] - 1 + b) % case["new"]))
        else:
            news.append(case["new"])
    return lens, news


def _codes(gen, rows, cols, amax=127):
    """int8 rows in storage whose rows start at multiples of 16 bytes, bell-shaped as quantised activations and weights are, each with
    one value at the end of the range."""
    pad = (cols + 15) // 16 * 16
    x = (torch.randn((rows, pad), generator=gen, device="cuda") * 32).round_().clamp_(-amax, amax).to(torch.int8)[:, :cols]
    top = torch.randint(0, cols, (rows, 1), generator=gen, device="cuda")
    x.scatter_(1, top, torch.full((rows, 1), amax, dtype=torch.int8, device="cuda"))
    return x


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    op, dtype = case["op"], DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    state = {"case": case, "dtype": dtype}
    if op == "norm":
        outlier = 1 + 9 * (torch.rand((case["cols"],), generator=gen, device="cuda") < 0.01)      # the few large coordinates of a residual stream
        state["x"] = (randn(case["rows"], case["cols"]) * outlier).to(dtype)
        state["delta"] = (randn(case["rows"], case["cols"]) * 0.5).to(DTYPES[case["delta"]]) if case["delta"] else None
        state["weight"] = 1 + 0.1 * randn(case["cols"])
        state["eps"] = 1e-6
    elif op == "quantize":
        state["x"] = randn(case["rows"], case["cols"] * (2 if case["block"] else 1)).to(dtype)
    elif op == "gemm":
        state["a"], state["w"] = _codes(gen, case["m"], case["k"]), _codes(gen, case["n"], case["k"])
        state["a_scale"] = (0.5 + torch.rand((case["m"],), generator=gen, device="cuda")) * (3 / 127)
        state["w_scale"] = (0.5 + torch.rand((case["n"],), generator=gen, device="cuda")) * (3 / 127 / case["k"] ** 0.5)
        state["bias"] = randn(case["n"]) if case["bias"] else None
    else:
        lens, news = _spans(case)
        slots = case["seqs"] + 1                                  # a slot that no sequence of the call owns
        kv, dim, ctx, rows = case["kv"], case["dim"], case["ctx"], sum(news)
        starts = [0]
        for n in news:
            starts.append(starts[-1] + n)

        def ints(v):
            return torch.tensor(v, dtype=torch.int32, device="cuda")

        state["batch"] = (torch.randperm(slots, generator=gen, device="cuda")[: case["seqs"]].to(torch.int32), ints(starts), ints(lens))
        state["max_new"], state["max_len"], state["rows"] = max(news), max(lens), rows
        state["causal"] = case["kind"] != "cross"
        if op == "cache":
            state["k"], state["v"] = randn(rows, kv, dim).to(dtype), randn(rows, kv, dim).to(dtype)
            state["cache"] = (torch.zeros((slots, kv, ctx, dim), dtype=torch.int8, device="cuda"), torch.zeros((slots, kv, ctx), device="cuda"),
                              torch.zeros((slots, kv, ctx, dim), dtype=torch.int8, device="cuda"), torch.zeros((slots, kv, ctx), device="cuda"))
        else:
            def half():
                codes = torch.randint(-127, 128, (slots, kv, ctx, dim), generator=gen, device="cuda", dtype=torch.int8)
                return codes, (0.5 + torch.rand((slots, kv, ctx), generator=gen, device="cuda")) * (2 / 127)
            state["cache"] = half() + half()
            state["q"] = (randn(rows, case["heads"], dim) * 1.5).to(dtype)
    return state


# ---- the plain forms ------------------------------------------------------------------------------------------------------------

def _quantize(y):
    scale = y.abs().amax(-1) / 127
    return torch.round(y / scale.clamp_min(1e-38)[..., None]).clamp(-127, 127), scale


def _swiglu(x, block):
    """Gate and up columns in alternating blocks of `block` columns."""
    parts = x.reshape(x.shape[0], -1, 2, block)
    gate, up = parts[:, :, 0], parts[:, :, 1]
    return (gate / (1 + torch.exp(-gate)) * up).reshape(x.shape[0], -1)


def _rows_of(state):
    """(sequence, place in it, position in its cache) of every row."""
    slots, starts, lens = state["batch"]
    row = torch.arange(state["rows"], device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1
    place = row - starts[seq]
    return seq, place, lens[seq] - (starts[seq + 1] - starts[seq]) + place


def _plain_attention(state, q, k, v):
    """q [rows][heads][dim], k and v [sequence][kv head][position][dim] as values, in q's type."""
    case = state["case"]
    slots, starts, lens = state["batch"]
    group = case["heads"] // case["kv"]
    place = torch.arange(state["max_new"], device="cuda")
    new = starts[1:] - starts[:-1]
    rows = (starts[:-1, None] + place).clamp_max(state["rows"] - 1)                       # [sequence][place]
    qs = q[rows].reshape(len(slots), -1, case["kv"], group, case["dim"]).permute(0, 2, 1, 3, 4)
    qs = qs.reshape(len(slots), case["kv"], -1, case["dim"])                              # [sequence][kv head][place x group][dim]
    s = torch.matmul(qs, k.transpose(2, 3).contiguous()) * case["dim"] ** -0.5
    key = torch.arange(k.shape[2], device="cuda")
    if state["causal"]:
        sees = key <= (lens - new)[:, None, None] + place[None, :, None]
    else:
        sees = (key < lens[:, None, None]).expand(-1, state["max_new"], -1)
    s = s.masked_fill_(~sees.repeat_interleave(group, 1)[:, None], float("-inf"))
    s = s.sub_(s.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(s, v) / s.sum(-1, keepdim=True)
    o = o.reshape(len(slots), case["kv"], state["max_new"], group, case["dim"]).permute(0, 2, 1, 3, 4)
    seq, at, _ = _rows_of(state)
    return o.reshape(len(slots), state["max_new"], case["heads"], case["dim"])[seq, at]


def _plain(state):
    case, op, dtype = state["case"], state["case"]["op"], state["dtype"]
    if op == "norm":
        r = state["x"].float()
        if state["delta"] is not None:
            r = r + state["delta"].float()
        y = r * torch.rsqrt(r.square().mean(-1, keepdim=True) + state["eps"]) * state["weight"]
        codes, scale = _quantize(y)
        return {"residual": r.to(dtype), "values": (codes * scale[:, None]).half(), "scale": scale}
    if op == "quantize":
        x = state["x"].float()
        codes, scale = _quantize(_swiglu(x, case["block"]) if case["block"] else x)
        return {"values": (codes * scale[:, None]).half(), "scale": scale}
    if op == "gemm":
        c = torch.matmul(state["a"].float(), state["w"].float().t()) * state["a_scale"][:, None] * state["w_scale"]
        return (c if state["bias"] is None else c + state["bias"]).to(dtype)
    slots = state["batch"][0].long()
    if op == "cache":
        seq, _, pos = _rows_of(state)
        kc, ks, vc, vs = state["cache"]
        at = (slots[seq], slice(None), pos.long())
        for codes, scales, x in ((kc, ks, state["k"]), (vc, vs, state["v"])):
            c, s = _quantize(x.float())
            codes[at], scales[at] = c.to(torch.int8), s
        return {"k": (kc[at] * ks[at][..., None]).half(), "v": (vc[at] * vs[at][..., None]).half()}
    kc, ks, vc, vs = (t[slots, :, : state["max_len"]] for t in state["cache"])
    return _plain_attention(state, state["q"].float(), kc.float() * ks[..., None], vc.float() * vs[..., None]).to(dtype)


def _own(state):
    from whisperjav_amd import q8
    op, dtype = state["case"]["op"], state["dtype"]
    if op == "norm":
        r = torch.empty_like(state["x"])
        codes, scale = q8.rmsnorm(state["x"], state["weight"], state["eps"], delta=state["delta"], residual=r)
        return {"residual": r, "values": q8.dequantize(codes, scale), "scale": scale}
    if op == "quantize":
        codes, scale = q8.quantize(state["x"], swiglu_block=state["case"]["block"])
        return {"values": q8.dequantize(codes, scale), "scale": scale}
    if op == "gemm":
        return q8.gemm(state["a"], state["a_scale"], state["w"], state["w_scale"], bias=state["bias"], dtype=dtype)
    cache = q8.KV8Cache(*state["cache"])
    batch = q8.Batch(*state["batch"], max_new=state["max_new"], max_len=state["max_len"])
    if op == "cache":
        q8.kv_write(cache, state["k"], state["v"], batch)
        k, v = q8.kv_read(cache, batch, state["rows"])
        return {"k": k, "v": v}
    return q8.kv_attention(state["q"], cache, batch, causal=state["causal"])


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ---- what a pass cannot do without, and the definition in 64 bits ------------------------------------------------------------------

def work(case):
    size = {"float32": 4, "float16": 2, "bfloat16": 2, "": 0}
    op = case["op"]
    if op == "norm":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (2 * size[case["dtype"]] + size[case["delta"]] + 2) + 4 * (case["cols"] + case["rows"]), "flops": 8 * n}
    if op == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (size[case["dtype"]] * (2 if case["block"] else 1) + 2) + 4 * case["rows"], "flops": (8 if case["block"] else 4) * n}
    if op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + m * n * size[case["dtype"]] + 4 * (m + n * (2 if case["bias"] else 1)), "flops": 2 * m * n * k}
    lens, news = _spans(case)
    if op == "cache":
        n = sum(news) * case["kv"]
        return {"bytes": 2 * n * (case["dim"] * (size[case["dtype"]] + 1 + 2) + 4), "flops": 8 * n * case["dim"]}
    seen = sum(n * w - (w * (w - 1) // 2 if case["kind"] != "cross" else 0) for n, w in zip(lens, news))
    return {"bytes": 2 * sum(lens) * case["kv"] * (case["dim"] + 4) + 2 * sum(news) * case["heads"] * case["dim"] * size[case["dtype"]],
            "flops": 4 * seen * case["heads"] * case["dim"]}


def _exact_codes(y):
    top = y.abs().max(-1, keepdim=True).values
    step = top / 127
    return torch.where(top > 0, torch.round(y / torch.where(top > 0, step, torch.ones_like(step))) * step, torch.zeros_like(y)), step[..., 0]


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        r = state["x"].double() + (0 if state["delta"] is None else state["delta"].double())
        y = r / torch.sqrt(torch.sum(r * r, -1, keepdim=True) / case["cols"] + state["eps"]) * state["weight"].double()
        values, step = _exact_codes(y)
        return {"residual": r, "values": values, "scale": step}
    if op == "quantize":
        x = state["x"].double()
        if case["block"]:
            col = torch.arange(case["cols"], device="cuda")
            gate = col // case["block"] * 2 * case["block"] + col % case["block"]
            x = x[:, gate] * torch.sigmoid(x[:, gate]) * x[:, gate + case["block"]]
        values, step = _exact_codes(x)
        return {"values": values, "scale": step}
    if op == "gemm":
        c = torch.matmul(state["a"].double() * state["a_scale"].double()[:, None], (state["w"].double() * state["w_scale"].double()[:, None]).t().contiguous())
        return c if state["bias"] is None else c + state["bias"].double()
    if op == "cache":
        return {"k": _exact_codes(state["k"].double())[0], "v": _exact_codes(state["v"].double())[0]}
    lens, news = _spans(case)
    slots = state["batch"][0].tolist()
    kc, ks, vc, vs = state["cache"]
    out, first = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda"), 0
    for slot, n, w in zip(slots, lens, news):
        q = state["q"][first: first + w].double().transpose(0, 1)                           # [head][row][dim]
        per = case["heads"] // case["kv"]
        k = (kc[slot, :, :n].double() * ks[slot, :, :n, None].double()).repeat_interleave(per, 0)
        v = (vc[slot, :, :n].double() * vs[slot, :, :n, None].double()).repeat_interleave(per, 0)
        s = torch.matmul(q, k.transpose(1, 2).contiguous()) / case["dim"] ** 0.5
        if case["kind"] != "cross":
            hidden = torch.ones((w, n), dtype=torch.bool, device="cuda").triu(n - w + 1)
            s = s.masked_fill(hidden, float("-inf"))
        out[first: first + w] = torch.matmul(torch.softmax(s, -1), v).transpose(0, 1)
        first += w
    return out

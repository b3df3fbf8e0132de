"""8-bit operators of a decoder step on torch tensors (``wj_q8_*`` / ``wj_kv8_*``, ``include/wjhip.h``).

A row of values is held as int8 codes in [-127, 127], 127 x / max |x| to the nearest, and one float32 scale, max |x| / 127: ``rmsnorm`` and ``quantize``
produce such rows, ``gemm`` multiplies them with weights held the same way (a scale per token and per channel), ``KV8Cache`` holds keys and values
like that, ``kv_write`` / ``kv_read`` / ``kv_attention`` fill, read back and attend to it.

Every function launches on torch's current stream of the tensors' device and returns at once; outputs come from torch's allocator.  The
calls may be captured into a ``torch.cuda.graph``.  They serve inference and refuse tensors that want a gradient or carry a tangent.  What they
write in place (``x`` or ``residual``, ``out``, the cache) is marked as modified, so that a ``backward`` which saved it raises.  Arguments are checked
on the host (``ValueError``); the library's own refusals raise ``hipbind.WjError``.  There is no CPU path.

A decoder layer::

    codes, scale = q8.rmsnorm(x, ln1, eps, delta=mlp_out)                       # x += mlp_out, in place
    qkv = q8.gemm(codes, scale, w_qkv, w_qkv_scale, dtype=torch.float16)
    ...                                                                         # head norms, rotary embedding
    q8.kv_write(cache, k, v, batch)
    o = q8.kv_attention(q, cache, batch)
    attn_out = q8.gemm(*q8.quantize(o.flatten(1)), w_o, w_o_scale)
    codes, scale = q8.rmsnorm(x, ln2, eps, delta=attn_out)
    gate_up = q8.gemm(codes, scale, w_gate_up, w_gate_up_scale)
    mlp_out = q8.gemm(*q8.quantize(gate_up, swiglu_block=16), w_down, w_down_scale)
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad as _forward
from torch.autograd.graph import increment_version as _modified

from . import hipbind
from .hipbind import WJ_BF16, WJ_F16, WJ_F32

_TYPE = {torch.float32: WJ_F32, torch.float16: WJ_F16, torch.bfloat16: WJ_BF16}
_INT = 2 ** 31 - 1                       # sizes that the library takes as 32-bit integers
_STREAM_DEFAULT = C.c_void_p(-1)        # include/wjhip.h: WJ_STREAM_DEFAULT


class Kv8C(C.Structure):
    _fields_ = [("k", C.c_void_p), ("k_scale", C.c_void_p), ("v", C.c_void_p), ("v_scale", C.c_void_p),
                ("slots", C.c_int32), ("heads", C.c_int32), ("ctx", C.c_int32), ("dim", C.c_int32)]


class Kv8BatchC(C.Structure):
    _fields_ = [("slots", C.c_void_p), ("starts", C.c_void_p), ("lens", C.c_void_p),
                ("seqs", C.c_int32), ("rows", C.c_int32), ("max_new", C.c_int32), ("max_len", C.c_int32)]


def _launch(index: int):
    """(library, context handle, stream) for tensors on GPU ``index``.  The calls of a decode step are bound by the host: the raw stream
    handle costs 0.1 us where a ``torch.cuda.Stream`` object costs 2."""
    stream = torch._C._cuda_getCurrentRawStream(index)
    ctx = hipbind._contexts.get(index)
    if ctx is None:
        with torch.cuda.device(index):          # wj_init makes its GPU the thread's current one: put it back
            ctx = hipbind.context(index)
    return hipbind.lib(), ctx.handle, stream or _STREAM_DEFAULT


def _fail(name: str, rc: int) -> None:
    hipbind.check(rc, name)


def _no_gradient(t: torch.Tensor, what: str) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: requires a gradient; these operators have none (torch.no_grad() to go on)")
    if _forward._current_level >= 0 and _forward.unpack_dual(t).tangent is not None:
        raise ValueError(f"{what}: carries a tangent; these operators have none")


def _float_rows(t: torch.Tensor, what: str, index: Optional[int] = None, rows: int = -1, cols: int = -1) -> int:
    """Check a ``[rows, cols]`` float tensor whose rows are contiguous (on GPU ``index``); its type code."""
    code = _TYPE.get(t.dtype)
    if code is None:
        raise ValueError(f"{what}: float32, float16 or bfloat16 expected, got {t.dtype}")
    shape = t.shape
    if len(shape) != 2 or (index is not None and (shape[0] != rows or shape[1] != cols)):
        raise ValueError(f"{what}: {'[rows, cols]' if index is None else [rows, cols]} expected, got {list(shape)}")
    if shape[1] > _INT:
        raise ValueError(f"{what}: {shape[1]} columns (at most 2^31 - 1)")
    if not t.is_cuda or (index is not None and t.get_device() != index):
        raise ValueError(f"{what}: on {t.device}, expected {'a GPU' if index is None else f'cuda:{index}'}")
    if t.stride(1) != 1 and shape[1] > 1:
        raise ValueError(f"{what}: the elements of a row must be contiguous (stride {t.stride(1)})")
    _no_gradient(t, what)
    return code


def _codes(t: torch.Tensor, scale: torch.Tensor, what: str, index: Optional[int] = None) -> int:
    """Check int8 rows and their scales; the GPU's index."""
    if t.dtype != torch.int8 or t.dim() != 2:
        raise ValueError(f"{what}: int8 [rows, cols] expected, got {t.dtype} {list(t.shape)}")
    if t.shape[1] > _INT:
        raise ValueError(f"{what}: {t.shape[1]} columns (at most 2^31 - 1)")
    if not t.is_cuda or (index is not None and t.get_device() != index):
        raise ValueError(f"{what}: on {t.device}, expected {'a GPU' if index is None else f'cuda:{index}'}")
    if t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError(f"{what}: the elements of a row must be contiguous (stride {t.stride(1)})")
    index = t.get_device()
    _vector(scale, what + " scale", t.shape[0], index)
    return index


def _vector(t: torch.Tensor, what: str, n: int, index: int) -> None:
    if t.dtype != torch.float32 or t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1) or t.get_device() != index:
        raise ValueError(f"{what}: contiguous float32 [{n}] on cuda:{index} expected, got {t.dtype} {list(t.shape)} on {t.device}")
    _no_gradient(t, what)


def _output(t: torch.Tensor, what: str) -> None:
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"{what}: rows overlap")


def _new_codes(rows: int, cols: int, device: torch.device) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows that start at multiples of 16 bytes, as the product's fast kernels want them."""
    pad = (cols + 15) & ~15
    codes = torch.empty(rows, pad, dtype=torch.int8, device=device)
    return codes if pad == cols else codes[:, :cols], torch.empty(rows, dtype=torch.float32, device=device)


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *, delta: Optional[torch.Tensor] = None,
            residual: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(codes, scale)`` of the rows of ``(x + delta) / rms(x + delta) * weight``.

    ``residual`` receives ``x + delta`` in x's type; left out, the sum is written back into ``x`` (when there is a ``delta``).  The squares
    are summed in float32, as in the plain form: their sum must stay below 3e38."""
    xt = _float_rows(x, "x")
    rows, cols = x.shape
    index = x.get_device()
    _vector(weight, "weight", cols, index)
    if delta is None:
        dt, dp, ld = 0, None, 0
    else:
        dt, dp, ld = _float_rows(delta, "delta", index, rows, cols), delta.data_ptr(), delta.stride(0)
        if residual is None:
            residual = x
    if residual is None:
        rp, lr = None, 0
    else:
        if _float_rows(residual, "residual", index, rows, cols) != xt:
            raise ValueError(f"residual: {x.dtype} expected, got {residual.dtype}")
        _output(residual, "residual")
        rp, lr = residual.data_ptr(), residual.stride(0)
    codes, scale = _new_codes(rows, cols, x.device)
    lib, ctx, stream = _launch(index)
    rc = lib.wj_q8_rmsnorm(ctx, xt, x.data_ptr(), x.stride(0), dt, dp, ld, weight.data_ptr(), eps, rp, lr, codes.data_ptr(), codes.stride(0),
                           scale.data_ptr(), rows, cols, stream)
    if rc:
        _fail("wj_q8_rmsnorm", rc)
    if residual is not None:
        _modified(residual)
    return codes, scale


def quantize(x: torch.Tensor, *, swiglu_block: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(codes, scale)`` of the rows of ``x``, or of ``silu(gate) * up`` where ``x`` holds gate and up columns in alternating blocks of
    ``swiglu_block`` (half of x's columns: ``[gate | up]``; 16: the engine's packed gate-up rows)."""
    xt = _float_rows(x, "x")
    rows, cols = x.shape
    if swiglu_block:
        if swiglu_block < 0 or cols % (2 * swiglu_block):
            raise ValueError(f"x: {cols} columns are no whole number of gate / up blocks of {swiglu_block}")
        cols //= 2
    codes, scale = _new_codes(rows, cols, x.device)
    lib, ctx, stream = _launch(x.get_device())
    rc = lib.wj_q8_quantize(ctx, xt, x.data_ptr(), x.stride(0), swiglu_block, codes.data_ptr(), codes.stride(0), scale.data_ptr(), rows, cols, stream)
    if rc:
        _fail("wj_q8_quantize", rc)
    return codes, scale


def dequantize(codes: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """``codes * scale`` in ``dtype``."""
    index = _codes(codes, scale, "codes")
    if dtype not in _TYPE:
        raise ValueError(f"dtype: float32, float16 or bfloat16 expected, got {dtype}")
    rows, cols = codes.shape
    out = torch.empty(rows, cols, dtype=dtype, device=codes.device)
    lib, ctx, stream = _launch(index)
    rc = lib.wj_q8_dequantize(ctx, codes.data_ptr(), codes.stride(0), scale.data_ptr(), _TYPE[dtype], out.data_ptr(), cols, rows, cols, stream)
    if rc:
        _fail("wj_q8_dequantize", rc)
    return out


def gemm(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, *, bias: Optional[torch.Tensor] = None,
         dtype: torch.dtype = torch.float16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[i, j] = a_scale[i] * w_scale[j] * sum_k a[i, k] w[j, k] + bias[j]``, the sum exact, in ``dtype`` (or ``out``'s type).

    ``a`` int8 ``[m, k]``, ``w`` int8 ``[n, k]``; rows that start at multiples of 16 bytes (what ``rmsnorm`` / ``quantize`` return) take the
    fast kernels."""
    index = _codes(a, a_scale, "a")
    _codes(w, w_scale, "w", index)
    (m, k), n = a.shape, w.shape[0]
    if w.shape[1] != k:
        raise ValueError(f"a has {k} columns, w has {w.shape[1]}")
    if n > _INT:
        raise ValueError(f"w: {n} rows (at most 2^31 - 1)")
    if bias is not None:
        _vector(bias, "bias", n, index)
    given = out
    if out is None:
        dt = _TYPE.get(dtype)
        if dt is None:
            raise ValueError(f"dtype: float32, float16 or bfloat16 expected, got {dtype}")
        out = torch.empty(m, n, dtype=dtype, device=a.device)
    else:
        dt = _float_rows(out, "out", index, m, n)
        _output(out, "out")
    lib, ctx, stream = _launch(index)
    need = lib.wj_q8_gemm_workspace(ctx, m, n, k)
    work = torch.empty(need, dtype=torch.uint8, device=a.device) if need else None      # freed in stream order by torch's allocator
    rc = lib.wj_q8_gemm(ctx, a.data_ptr(), a.stride(0), a_scale.data_ptr(), w.data_ptr(), w.stride(0), w_scale.data_ptr(),
                        bias.data_ptr() if bias is not None else None, dt, out.data_ptr(), out.stride(0), m, n, k,
                        work.data_ptr() if need else None, need, stream)
    if rc:
        _fail("wj_q8_gemm", rc)
    if given is not None:
        _modified(given)
    return out


class _CacheTensors(NamedTuple):
    k: torch.Tensor
    k_scale: torch.Tensor
    v: torch.Tensor
    v_scale: torch.Tensor


class KV8Cache(_CacheTensors):
    """One layer's keys and values in 8 bits: codes int8 ``[slots, heads, ctx, dim]`` and scales float32 ``[slots, heads, ctx]``.
    A program keeps it like a handle: the tensors are checked at its first use, and again when one of them has other memory."""

    @classmethod
    def empty(cls, slots: int, heads: int, ctx: int, dim: int, device: torch.device = torch.device("cuda", 0)) -> "KV8Cache":
        def codes():
            return torch.zeros((slots, heads, ctx, dim), dtype=torch.int8, device=device)

        def scale():
            return torch.zeros((slots, heads, ctx), dtype=torch.float32, device=device)
        return cls(codes(), scale(), codes(), scale())

    def __reduce__(self):                        # a copy describes its own tensors
        return type(self), tuple(self)


class _BatchArrays(NamedTuple):
    slots: torch.Tensor
    starts: torch.Tensor
    lens: torch.Tensor
    max_new: int
    max_len: int


class Batch(_BatchArrays):
    """The sequences of a call, int32 on the device: sequence b owns rows ``starts[b] .. starts[b + 1] - 1`` of the row tensors and has
    ``lens[b]`` positions in slot ``slots[b]`` of the cache once they are written, the rows being the last ones.  A slot of -1 is padding.
    ``max_new`` / ``max_len``: the most new rows / positions of any sequence; they size the launch.  A call is right whatever they say, but they choose
    the kernel and with it the order of the sums: attention under other hints may differ in its last bits.  The
    arrays may change between replays of a captured graph.  Slots are distinct where the batch is written."""

    def __reduce__(self):
        return type(self), tuple(self)


def _storages(tensors) -> list:
    """Kept beside addresses: while memory is held, no other tensor can come to lie at its address."""
    return [t.untyped_storage() for t in tensors]


def _cache(cache: KV8Cache) -> Kv8C:
    k, ks, v, vs = cache
    _no_gradient(ks, "cache scale")
    _no_gradient(vs, "cache scale")
    at = (k.data_ptr(), ks.data_ptr(), v.data_ptr(), vs.data_ptr())
    known = cache.__dict__.get("_c")             # checked and laid out at the object's first use; see _storages
    if known is not None and known[0] == at:
        return known[1]
    shape = k.shape
    if len(shape) != 4 or v.shape != shape or ks.shape != shape[:3] or vs.shape != shape[:3]:
        raise ValueError(f"cache: codes [slots, heads, ctx, dim] and scales [slots, heads, ctx] expected, got {list(k.shape)}, {list(ks.shape)}, "
                         f"{list(v.shape)}, {list(vs.shape)}")
    if k.dtype != torch.int8 or v.dtype != torch.int8 or ks.dtype != torch.float32 or vs.dtype != torch.float32:
        raise ValueError("cache: int8 codes and float32 scales expected")
    if not (k.is_cuda and k.device == v.device == ks.device == vs.device):
        raise ValueError("cache: the four tensors must be on one GPU")
    if max(shape) > _INT:
        raise ValueError(f"cache: {list(shape)} (sizes of at most 2^31 - 1)")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError("cache: contiguous tensors expected")
    c = Kv8C(*at, *shape)
    cache.__dict__["_c"] = (at, c, _storages(cache))
    return c


def _batch(batch: Batch, rows: int, index: int) -> Kv8BatchC:
    slots, starts, lens, max_new, max_len = batch
    at = (slots.data_ptr(), starts.data_ptr(), lens.data_ptr(), rows, index)
    known = batch.__dict__.get("_c")
    if known is not None and known[0] == at:
        return known[1]
    if rows > _INT:
        raise ValueError(f"{rows} rows (at most 2^31 - 1)")
    n = slots.shape[0] if slots.dim() == 1 else -1
    for t, what, want in ((slots, "slots", n), (starts, "starts", n + 1), (lens, "lens", n)):
        if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != want or t.get_device() != index or not t.is_contiguous():
            raise ValueError(f"batch.{what}: contiguous int32 [{want if want >= 0 else 'seqs'}] on cuda:{index} expected, got {t.dtype} {list(t.shape)} on {t.device}")
    b = Kv8BatchC(*at[:3], n, rows, min(max_new, _INT), min(max_len, _INT))
    batch.__dict__["_c"] = (at, b, _storages(batch[:3]))
    return b


def _head_rows(t: torch.Tensor, what: str, cache: Kv8C, index: int, heads: Optional[int] = None) -> int:
    """Check ``[rows, heads, dim]`` whose rows may be strided and whose heads lie one after the other; its type code."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != cache.dim or (heads is not None and shape[1] != heads):
        raise ValueError(f"{what}: [rows, {heads if heads is not None else 'heads'}, {cache.dim}] expected, got {list(shape)}")
    code = _TYPE.get(t.dtype)
    if code is None:
        raise ValueError(f"{what}: float32, float16 or bfloat16 expected, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{what}: on {t.device}, expected cuda:{index}")
    _no_gradient(t, what)
    stride = t.stride()
    if stride[2] != 1 or (shape[1] > 1 and stride[1] != cache.dim):
        raise ValueError(f"{what}: the heads of a row must lie one after the other, their elements too (strides {stride})")
    return code


def kv_write(cache: KV8Cache, k: torch.Tensor, v: torch.Tensor, batch: Batch) -> None:
    """Quantise the rows ``k`` and ``v`` ``[rows, heads, dim]`` (they may be views of one projection's output) into the cache."""
    c, index = _cache(cache), cache.k.get_device()
    dt = _head_rows(k, "k", c, index, c.heads)
    if _head_rows(v, "v", c, index, c.heads) != dt or v.shape[0] != k.shape[0]:
        raise ValueError(f"v: {list(k.shape)} in {k.dtype} expected, got {list(v.shape)} in {v.dtype}")
    b = _batch(batch, k.shape[0], index)
    lib, ctx, stream = _launch(index)
    rc = lib.wj_kv8_write(ctx, C.byref(c), C.byref(b), dt, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), stream)
    if rc:
        _fail("wj_kv8_write", rc)
    _modified(cache)


def kv_read(cache: KV8Cache, batch: Batch, rows: int, dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values ``[rows, heads, dim]`` of the batch's rows as the cache holds them (rows behind ``starts[-1]`` are not written)."""
    c, index = _cache(cache), cache.k.get_device()
    if dtype not in _TYPE:
        raise ValueError(f"dtype: float32, float16 or bfloat16 expected, got {dtype}")
    if rows < 0:
        raise ValueError(f"rows: {rows}")
    b = _batch(batch, rows, index)
    heads, dim, device = c.heads, c.dim, cache.k.device
    k = torch.empty(rows, heads, dim, dtype=dtype, device=device)
    v = torch.empty(rows, heads, dim, dtype=dtype, device=device)
    lib, ctx, stream = _launch(index)
    rc = lib.wj_kv8_read(ctx, C.byref(c), C.byref(b), _TYPE[dtype], k.data_ptr(), heads * dim, v.data_ptr(), heads * dim, stream)
    if rc:
        _fail("wj_kv8_read", rc)
    return k, v


def kv_attention(q: torch.Tensor, cache: KV8Cache, batch: Batch, *, causal: bool = True, scale: Optional[float] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the rows ``q`` ``[rows, n_heads, dim]`` over the cached positions of their sequences: up to the row's own position
    (``causal``), or all ``lens[b]`` of them.  ``scale`` defaults to ``dim ** -0.5``.  A row that sees nothing is zeros; rows behind
    ``starts[-1]`` are not written."""
    c, index = _cache(cache), cache.k.get_device()
    dt = _head_rows(q, "q", c, index)
    rows, heads, dim = q.shape
    given = out
    if out is None:
        out = torch.empty(rows, heads, dim, dtype=q.dtype, device=q.device)
    elif _head_rows(out, "out", c, index, heads) != dt or out.shape[0] != rows or (rows > 1 and out.stride(0) < heads * dim):
        raise ValueError(f"out: {list(q.shape)} in {q.dtype} expected, rows apart, got {list(out.shape)} in {out.dtype}")
    b = _batch(batch, rows, index)
    lib, ctx, stream = _launch(index)
    cp, bp = C.byref(c), C.byref(b)
    need = lib.wj_kv8_attention_workspace(ctx, cp, bp, heads)
    work = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None      # freed in stream order by torch's allocator
    rc = lib.wj_kv8_attention(ctx, cp, bp, dt, q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), heads, dim ** -0.5 if scale is None else scale,
                              1 if causal else 0, work.data_ptr() if need else None, need, stream)
    if rc:
        _fail("wj_kv8_attention", rc)
    if given is not None:
        _modified(given)
    return out

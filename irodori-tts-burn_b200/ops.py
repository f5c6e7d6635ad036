"""Attention over context states as operators on torch CUDA tensors: cross
attention to an encoder's states, and the context cache held in 4 bits.

The engine's joint attention (src/model/attention.rs:403-418, :619-664) reads
its latent frames and its text / speaker rows in one pass.  These calls are for
programs that keep queries and context rows themselves: ``kv4_attention`` reads
both as the engine does, from a 4-bit context; ``cross_attention`` reads a
native context alone.

    table = attention_table(q_lens, k_lens, device=0)           # once per batch
    out = cross_attention(q, k, v, table, max(q_lens), max(k_lens))

    cache = Kv4Cache(rows, kv_heads=16, head_dim=128, device=0)  # 4.5 bits a value
    kv4_append(cache, k, v)
    out = kv4_attention(q, cache, table, max(q_lens), max(k_lens), k_self=ks, v_self=vs)

Unlike ``InferenceEngine.sample`` the calls queue their work and return: with
``stream=None`` on torch's current stream of the tensors' GPU (whichever GPU is
current), so they order like torch's own operators and can be captured into a
CUDA graph.  On an explicit ``stream`` the caller orders the work before and
after; the tensors' memory is kept until that stream is done with it.  They are
forward only: a tensor that requires a gradient is refused while gradients are
recorded, one with a forward-mode tangent too, and so is torch.jit.trace, which
would record a call's allocations and not its kernel.
"""

from __future__ import annotations

import ctypes
import struct

from . import IrodoriError, PREC, _check, lib


# The header's structures, as their bytes: irt_rows; irt_attn_args (device, dtype, heads, kv_heads, head_dim, num_seqs,
# max_q_len, max_k_len, scale, q_rows, seqs, q, gate, out, key_mask, lse); irt_kv4_cache.
_ROWS = struct.Struct("@Pqq")
_ATTN = struct.Struct("@8ifqPPqqPqqPqqPP")
_CACHE = struct.Struct("@qiiPPPP")

_P, _I, _L = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
SIGNATURES = {
    "irt_cross_attention": (_I, [_P, _P, _P, _L, _P]),
    "irt_kv4_append": (_I, [_I, _I, _P, _L, _L, _P, _P, _L, _P, _P]),
    "irt_kv4_read": (_I, [_I, _I, _P, _L, _L, _P, _P, _P]),
    "irt_kv4_attention": (_I, [_P, _P, _P, _P, _P]),
    "irt_attention_check": (_I, [_I]),
}

GROUP = 32  # values that share a scale in the 4-bit cache

_torch = None
_forward_ad = None
_dtype_code = None  # torch dtype -> irt_precision
_INT32 = _MASKS = None


def _t():
    """torch, imported at the first call (the package itself does not need it)."""
    global _torch, _forward_ad, _dtype_code, _INT32, _MASKS
    if _torch is None:
        import torch
        import torch.autograd.forward_ad
        _torch, _forward_ad = torch, torch.autograd.forward_ad
        _INT32, _MASKS = (torch.int32,), (torch.uint8, torch.bool)
        _dtype_code = {torch.bfloat16: PREC["bf16"], torch.float32: PREC["f32"]}
    return _torch


def _no_gradient(name, t):
    if t.requires_grad and _torch.is_grad_enabled():
        raise IrodoriError(4, f"Unsupported mode: {name} requires a gradient; the operators are forward only "
                              "(call them under torch.no_grad())")
    if _forward_ad._current_level >= 0 and _forward_ad.unpack_dual(t).tangent is not None:
        raise IrodoriError(4, f"Unsupported mode: {name} has a forward-mode tangent, which the operators would lose "
                              "(pass its primal)")


def _no_tracing():
    if _torch._C._is_tracing():
        raise IrodoriError(4, "Unsupported mode: torch.jit.trace records torch's own operators only")


def _heads(name, t, device, dtype, shape):
    """(address, row stride, head stride) of a [rows, heads, head_dim] tensor (any strides, the last one 1)."""
    if not isinstance(t, _torch.Tensor):
        raise IrodoriError(22, f"{name} must be a torch CUDA tensor")
    if t.dtype is dtype and t.get_device() == device and t.shape == shape and not t.requires_grad and \
            _forward_ad._current_level < 0:
        row, head, one = t.stride()
        if one == 1:
            return t.data_ptr(), row, head
    if t.dtype is not dtype:
        raise IrodoriError(9, f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise IrodoriError(2, f"Shape mismatch: {name} must be {list(shape)}, got {list(t.shape)}")
    if t.get_device() != device:
        raise IrodoriError(22, f"{name} must be on cuda:{device}, got {t.device}")
    _no_gradient(name, t)
    if t.stride(2) != 1 and t.numel():
        raise IrodoriError(22, f"{name}: the values of a head must be contiguous")
    return t.data_ptr(), t.stride(0), t.stride(1)


def _first(name, t):
    torch = _t()
    _no_tracing()
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise IrodoriError(22, f"{name} must be a torch CUDA tensor")
    if t.dim() != 3:
        raise IrodoriError(2, f"Shape mismatch: {name} must be [rows, heads, head_dim], got {list(t.shape)}")
    if t.dtype not in _dtype_code:
        raise IrodoriError(9, f"{name} must be bfloat16 or float32, got {t.dtype}")
    return torch


def _plain(name, t, device, dtypes, shape):
    """Address of a contiguous helper tensor (table, mask, index, cache buffer)."""
    if isinstance(t, _torch.Tensor) and t.dtype in dtypes and t.get_device() == device and t.shape == shape and \
            t.is_contiguous() and not t.requires_grad and _forward_ad._current_level < 0:
        return t.data_ptr()
    if not isinstance(t, _torch.Tensor) or t.get_device() != device:
        raise IrodoriError(22, f"{name} must be a tensor on cuda:{device}")
    if t.dtype not in dtypes:
        raise IrodoriError(9, f"{name} must be {dtypes[0]}, got {t.dtype}")
    if t.shape != shape:
        raise IrodoriError(2, f"Shape mismatch: {name} must be {list(shape)}, got {list(t.shape)}")
    if not t.is_contiguous():
        raise IrodoriError(22, f"{name} must be contiguous")
    _no_gradient(name, t)
    return t.data_ptr()


def _stream(stream, device):
    """(handle, torch stream or None) of one call.  Without an explicit stream: torch's current one on the tensors' GPU."""
    if stream is None:
        return _torch._C._cuda_getCurrentRawStream(device), None
    if isinstance(stream, int):
        stream = _torch.cuda.ExternalStream(stream, device=device)
    return stream.cuda_stream, stream


def _empty(side, shape, dtype, device):
    """Memory for a result, of the stream that writes it."""
    if side is None:
        return _torch.empty(shape, dtype=dtype, device=device)
    with _torch.cuda.stream(side):
        return _torch.empty(shape, dtype=dtype, device=device)


def _empty_like(side, t):
    if side is None:
        return _torch.empty_like(t)
    with _torch.cuda.stream(side):
        return _torch.empty_like(t)


def _keep(side, *tensors):
    """Keeps the allocator from handing out these tensors' memory before an explicit stream is done with them."""
    for t in tensors:
        if t is not None:
            t.record_stream(side)


def attention_table(q_lens, k_lens, k_starts=None, device=0):
    """The sequence table of ``cross_attention`` / ``kv4_attention``: int32
    [n, 4] rows (q_start, q_len, k_start, k_len) on the GPU.  Queries are
    packed in order; context rows too, unless ``k_starts`` places them (ranges
    may overlap)."""
    torch = _t()
    q_lens, k_lens = [int(x) for x in q_lens], [int(x) for x in k_lens]
    if len(q_lens) != len(k_lens) or (k_starts is not None and len(k_starts) != len(k_lens)):
        raise IrodoriError(2, "Shape mismatch: q_lens, k_lens and k_starts must have one entry per sequence")
    if any(x < 0 for x in q_lens + k_lens):
        raise IrodoriError(2, "Shape mismatch: lengths must not be negative")
    if sum(q_lens) >= 1 << 30 or max(k_lens, default=0) >= 1 << 30 or \
            (sum(k_lens) if k_starts is None else max(map(int, k_starts), default=0)) >= 1 << 30:
        raise IrodoriError(2, "Shape mismatch: the query rows and the context rows must stay below 2^30")
    if k_starts is not None and min(map(int, k_starts), default=0) < 0:
        raise IrodoriError(2, "Shape mismatch: k_starts must not be negative")
    rows, q, k = [], 0, 0
    for i, (a, b) in enumerate(zip(q_lens, k_lens)):
        rows.append([q, a, k if k_starts is None else int(k_starts[i]), b])
        q, k = q + a, k + b
    if not rows:
        return torch.zeros((0, 4), dtype=torch.int32, device=torch.device("cuda", device))
    return torch.tensor(rows, dtype=torch.int32, device=torch.device("cuda", device))


def _row_range(cache, row_start, n):
    if not isinstance(cache, Kv4Cache):
        raise IrodoriError(22, "cache must be a Kv4Cache")
    if not 0 <= row_start <= cache.rows or not 0 <= n <= cache.rows - row_start:
        raise IrodoriError(2, f"Shape mismatch: rows [{row_start}, {row_start} + {n}) are outside the cache's {cache.rows}")


class Kv4Cache:
    """Context cache in 4 bits (``irt_kv4_cache``): K and V rows as codes of 4
    bits with one bf16 scale per 32 values of a head's row.  Holds values of a
    relative error of about 0.1 (normal data) in 0.28 of a bf16 cache's bytes;
    every value it holds is a bf16 number.  Rows start as zeros."""

    def __init__(self, rows: int, kv_heads: int, head_dim: int, device=0):
        torch = _t()
        dev = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        if rows < 0 or kv_heads <= 0 or head_dim < 8 or head_dim > 256 or head_dim % 8:
            raise IrodoriError(2, "Shape mismatch: a 4-bit cache has rows >= 0, kv_heads > 0 and a head_dim that is a "
                                  f"multiple of 8 in 8..256, got {rows}, {kv_heads}, {head_dim}")
        g = -(-head_dim // GROUP)
        self._set(torch.zeros((kv_heads, rows, head_dim // 2), dtype=torch.uint8, device=dev),
                  torch.zeros((kv_heads, rows, g), dtype=torch.bfloat16, device=dev),
                  torch.zeros((kv_heads, rows, head_dim // 2), dtype=torch.uint8, device=dev),
                  torch.zeros((kv_heads, rows, g), dtype=torch.bfloat16, device=dev))

    @classmethod
    def from_buffers(cls, k_codes, k_scales, v_codes, v_scales) -> "Kv4Cache":
        """A cache over tensors of the caller: codes uint8 [kv_heads, rows,
        head_dim / 2] (c + 8, the even index in the low half), scales bfloat16
        [kv_heads, rows, ceil(head_dim / 32)].  ``kv4_append`` writes scales of
        5 significant bits, whose values c s are bf16 numbers.  Scales of your
        own may be any bf16 number: float32 calls read c s exactly, bfloat16
        calls may round it to bfloat16."""
        self = cls.__new__(cls)
        self._set(k_codes, k_scales, v_codes, v_scales)
        return self

    def _set(self, k_codes, k_scales, v_codes, v_scales):
        torch = _t()
        if not isinstance(k_codes, torch.Tensor) or not k_codes.is_cuda or k_codes.dim() != 3:
            raise IrodoriError(22, "k_codes must be a CUDA tensor [kv_heads, rows, head_dim / 2]")
        h, n, half = shape = k_codes.shape
        scale_shape, dev = (h, n, -(-2 * half // GROUP)), k_codes.get_device()
        u8, b16 = (torch.uint8,), (torch.bfloat16,)
        self.buffers = (k_codes, k_scales, v_codes, v_scales)
        self.rows, self.kv_heads, self.head_dim, self.device = n, h, 2 * half, dev
        self._c = _CACHE.pack(n, h, 2 * half, _plain("k_codes", k_codes, dev, u8, shape),
                              _plain("k_scales", k_scales, dev, b16, scale_shape),
                              _plain("v_codes", v_codes, dev, u8, shape),
                              _plain("v_scales", v_scales, dev, b16, scale_shape))


def kv4_append(cache: Kv4Cache, k, v, row_start: int = 0, src_rows=None, stream=None) -> None:
    """Writes rows of ``k``, ``v`` [rows, kv_heads, head_dim] into ``cache``
    from ``row_start`` on (``irt_kv4_append``): all of them, or rows
    ``src_rows`` (int32 tensor; an index outside the source leaves its cache
    row as it was)."""
    torch = _first("k", k)
    if not isinstance(cache, Kv4Cache):
        raise IrodoriError(22, "cache must be a Kv4Cache")
    n_src = k.shape[0]
    shape = (n_src, cache.kv_heads, cache.head_dim)
    kr = _ROWS.pack(*_heads("k", k, cache.device, k.dtype, shape))
    vr = _ROWS.pack(*_heads("v", v, cache.device, k.dtype, shape))
    n, idx = n_src, None
    if src_rows is not None:
        n = src_rows.shape[0] if isinstance(src_rows, torch.Tensor) and src_rows.dim() == 1 else -1
        idx = _plain("src_rows", src_rows, cache.device, _INT32, (n,))
    _row_range(cache, row_start, n)
    handle, side = _stream(stream, cache.device)
    status = lib().irt_kv4_append(cache.device, _dtype_code[k.dtype], cache._c, row_start, n, kr, vr, n_src, idx, handle)
    if status:
        _check(status)
    if side is not None:
        _keep(side, k, v, src_rows, *cache.buffers)


def kv4_read(cache: Kv4Cache, row_start: int = 0, rows=None, dtype=None, stream=None):
    """The values that cache rows [row_start, row_start + rows) hold, as
    (k, v) [rows, kv_heads, head_dim] of ``dtype`` (bfloat16, the default, or
    float32; exact in both for scales of 5 significant bits, in float32 for
    any)."""
    torch = _t()
    _no_tracing()
    dtype = torch.bfloat16 if dtype is None else dtype
    if dtype not in _dtype_code:
        raise IrodoriError(9, f"dtype must be bfloat16 or float32, got {dtype}")
    n = cache.rows - row_start if rows is None else rows
    _row_range(cache, row_start, n)
    handle, side = _stream(stream, cache.device)
    shape = (n, cache.kv_heads, cache.head_dim)
    k = _empty(side, shape, dtype, cache.device)
    v = _empty_like(side, k)
    row, head, _ = k.stride()
    status = lib().irt_kv4_read(cache.device, _dtype_code[dtype], cache._c, row_start, n,
                                _ROWS.pack(k.data_ptr(), row, head), _ROWS.pack(v.data_ptr(), row, head), handle)
    if status:
        _check(status)
    if side is not None:
        _keep(side, *cache.buffers)
    return k, v


def _attention(call, q, kv_heads, k_rows, seqs, max_q_len, max_k_len, key_mask, gate, scale, out, return_lse, stream,
               context, keep):
    torch = _torch
    n, h, d = shape = q.shape
    dev, dtype = q.get_device(), q.dtype
    handle, side = _stream(stream, dev)
    given = out is not None
    if not given:
        out = _empty_like(side, q)
        out_row, out_head, _ = out.stride()
        out_p = out.data_ptr()
    else:
        out_p, out_row, out_head = _heads("out", out, dev, dtype, shape)
    lse = _empty(side, (n, h), torch.float32, dev) if return_lse else None
    if seqs is None:
        nseq, tab = (n // max_q_len if max_q_len > 0 else 0), 0
        if nseq * max_q_len != n or nseq * max_k_len != k_rows:
            raise IrodoriError(2, f"Shape mismatch: without a table {n} query rows and {k_rows} context rows must be "
                                  f"the same number of sequences of {max_q_len} and {max_k_len}")
    else:
        nseq = seqs.shape[0] if isinstance(seqs, torch.Tensor) and seqs.dim() == 2 else -1
        tab = _plain("seqs", seqs, dev, _INT32, (nseq, 4))
    mask = 0
    if key_mask is not None:
        mask = _plain("key_mask", key_mask, dev, _MASKS, (k_rows,))
    g = (0, 0, 0) if gate is None else _heads("gate", gate, dev, dtype, shape)
    try:
        a = _ATTN.pack(dev, _dtype_code[dtype], h, kv_heads, d, nseq, max_q_len, max_k_len,
                       d ** -0.5 if scale is None else scale, n, tab, *_heads("q", q, dev, dtype, shape), *g, out_p,
                       out_row, out_head, mask, 0 if lse is None else lse.data_ptr())
    except (struct.error, OverflowError) as e:
        raise IrodoriError(22, f"max_q_len, max_k_len or scale is out of range: {e}") from None
    status = call(a, *context, handle)
    if status:
        _check(status)
    if given:
        torch.autograd.graph.increment_version(out)  # autograd's record of in-place writes
    if side is not None:
        _keep(side, q, seqs, key_mask, gate, out, *keep)
    return (out, lse) if return_lse else out


def cross_attention(q, k, v, seqs, max_q_len: int, max_k_len: int, key_mask=None, gate=None, scale=None, out=None,
                    return_lse: bool = False, stream=None):
    """Attention of packed queries ``q`` [q_rows, heads, head_dim] to an
    encoder's states ``k``, ``v`` [k_rows, kv_heads, head_dim]
    (``irt_cross_attention``); bfloat16 or float32, any row and head strides.

    ``seqs`` is an ``attention_table`` (or None: equal sequences of
    ``max_q_len`` query and ``max_k_len`` context rows, in order); ``max_q_len``
    and ``max_k_len`` bound its lengths.  A table of your own may place
    sequences anywhere and let them share context rows, but not query rows
    (which of those are written is not defined).  Query head h reads KV head
    h // (heads // kv_heads).  ``key_mask`` uint8 / bool [k_rows]: non-zero =
    attend.  ``gate``, shaped like ``q``, is multiplied into the output.
    ``scale`` defaults to 1 / sqrt(head_dim).

    Returns [q_rows, heads, head_dim], with ``return_lse`` also the float32
    [q_rows, heads] log of the softmax's sum.  A query without any key gives 0
    and -inf; rows that no sequence covers (and sequences that reach outside
    the tensors or the bounds) are left as they were: pass ``out`` where that
    matters."""
    _first("q", q)
    _first("k", k)
    n, kv_heads, _ = k.shape
    shape = (n, kv_heads, q.shape[2])
    dev = q.get_device()
    context = (_ROWS.pack(*_heads("k", k, dev, q.dtype, shape)), _ROWS.pack(*_heads("v", v, dev, q.dtype, shape)), n)
    return _attention(lib().irt_cross_attention, q, kv_heads, n, seqs, max_q_len, max_k_len, key_mask, gate, scale,
                      out, return_lse, stream, context, (k, v))


def kv4_attention(q, cache: Kv4Cache, seqs, max_q_len: int, max_k_len: int, k_self=None, v_self=None, key_mask=None,
                  gate=None, scale=None, out=None, return_lse: bool = False, stream=None):
    """Attention of packed queries over a 4-bit context cache
    (``irt_kv4_attention``).  With ``k_self``, ``v_self`` [q_rows, kv_heads,
    head_dim] a sequence's queries attend to the rows of their own range too,
    as in the model's joint attention.  The other arguments and the result are
    those of ``cross_attention``, the cache's rows in the place of ``k``, ``v``."""
    _first("q", q)
    dev = q.get_device()
    if not isinstance(cache, Kv4Cache):
        raise IrodoriError(22, "cache must be a Kv4Cache")
    if cache.device != dev:
        raise IrodoriError(22, f"the cache must be on cuda:{dev}, got cuda:{cache.device}")
    shape = (q.shape[0], cache.kv_heads, q.shape[2])
    kr = None if k_self is None else _ROWS.pack(*_heads("k_self", k_self, dev, q.dtype, shape))
    vr = None if v_self is None else _ROWS.pack(*_heads("v_self", v_self, dev, q.dtype, shape))
    return _attention(lib().irt_kv4_attention, q, cache.kv_heads, cache.rows, seqs, max_q_len, max_k_len, key_mask,
                      gate, scale, out, return_lse, stream, (cache._c, kr, vr),
                      (k_self, v_self, *cache.buffers))


def attention_check(device: int = 0) -> None:
    """Waits for the GPU and raises if a bounded wait inside an attention
    operator's kernel has expired since the last check; until then the attention
    calls on that GPU raise too."""
    _check(lib().irt_attention_check(device))

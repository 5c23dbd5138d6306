"""Serving ops: a paged key-value cache, attention of single tokens over it and
the log probabilities of the answer, on gfx950.

They continue where the prefill ends.  The reference has no counterpart (its
path stops at the prefill's output); the conventions are those of ``ops``: the
hand-written kernels behind ``include/kfmi.h``, no fallback, forward only, BF16 activations,
ValueError before anything is launched, torch's current stream, no
synchronisation, so every call can be captured in a HIP graph.

A cache is plain tensors (``make_cache``): ``k_cache`` and ``v_cache``
``[pages, Hkv, page_size, D]`` in BF16, or in ``float8_e4m3fn`` with one
power-of-two scale per row, ``k_scale`` and ``v_scale`` ``[pages, Hkv,
page_size]`` in ``float8_e8m0fnu``.  Other memory orders are views of that
shape (``cache.transpose(1, 2)`` of ``[pages, page_size, Hkv, D]`` tensors, a layer's slice of a larger
tensor).  ``page_size`` is a power of two, at least 16; slot ``z`` is row ``z % page_size``
of page ``z // page_size``.

Indices (positions, slots, pages, lengths, ids) are int32 or int64 tensors on
the device.  Their values are not checked on the host, which would have to wait
for the GPU; the kernels never leave the tensors whatever the values are, and
answer a wrong one with NaN, as each function says.  Other work may not write them
while a call that reads them runs.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import NORM_STYLES
from .ops import EPS, device_arch

_I32, _I64, _F32 = torch.int32, torch.int64, torch.float32
_BF16, _E4M3, _E8M0 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu


def make_cache(pages: int, hkv: int, page_size: int, d: int, dtype=torch.bfloat16, device="cuda"):
    """An empty cache: ``(k_cache, v_cache, k_scale, v_scale)``, the scales None
    for BF16.  ``dtype``: ``torch.bfloat16`` or ``torch.float8_e4m3fn``."""
    if dtype not in (_BF16, _E4M3):
        raise ValueError("a cache holds bfloat16 or float8_e4m3fn")
    if page_size < 16 or page_size & (page_size - 1):
        raise ValueError("page_size must be a power of two, at least 16")
    if pages < 1 or hkv < 1 or d not in (128, 256):
        raise ValueError("Expected pages and hkv >= 1 and D in (128, 256)")
    kv = [torch.zeros(pages, hkv, page_size, d, dtype=dtype, device=device) for _ in range(2)]
    if dtype is _BF16:
        return kv[0], kv[1], None, None
    sc = [torch.zeros(pages, hkv, page_size, dtype=torch.uint8, device=device).view(_E8M0) for _ in range(2)]
    return kv[0], kv[1], sc[0], sc[1]


# ---------------------------------------------------------------------------
# Checks
# ---------------------------------------------------------------------------

# The checks read each property once and without helper objects: an eager call
# of one token is bound by them, not by its kernel (a property costs 70 to 160 ns).

_checked_devices: set[int] = set()


def _check_gpu(index, *tensors):
    """All tensors on the gfx950 device of this index (-1: the CPU)."""
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError("Inputs must be on one GPU device")
    if index not in _checked_devices:
        if index < 0:
            raise ValueError("Inputs must be on one GPU device")
        arch = device_arch(torch.device("cuda", index))
        if not arch.startswith("gfx950"):
            raise ValueError(f"This implementation targets gfx950 (MI355X); device is {arch}")
        _checked_devices.add(index)


def _call(index, entry, packed, work=None):
    """One entry point on the current stream of the device.  ``work``: a function of the stream that
    gives (address, bytes, tensor) of the workspace, whose place in ``packed`` it fills."""
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            return _call(index, entry, packed, work)
    stream = _raw_stream(index)
    if work is not None:
        wp, wb, buf = work(stream)
        packed = packed(wp, wb)
    _lib.call(entry, packed, stream)


def _raw_stream(index):
    raw = _lib._raw_stream
    return torch.cuda.current_stream(index).cuda_stream if raw is None else raw(index)


def _check_grad(name, *tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} is forward-only")


def _check_cache(k_cache, v_cache, k_scale, v_scale):
    """The cache's (pages, Hkv, page_size, D), strides, scale strides and type."""
    shape, strides, dtype = k_cache.shape, k_cache.stride(), k_cache.dtype
    if len(shape) != 4 or v_cache.shape != shape or v_cache.stride() != strides or v_cache.dtype is not dtype:
        raise ValueError("Expected k_cache and v_cache [pages,Hkv,page_size,D], alike in shape, strides and type")
    pages, hkv, page, d = shape
    if d not in (128, 256) or page < 16 or page & (page - 1) or pages < 1 or hkv < 1:
        raise ValueError("Expected D in (128, 256) and a page_size that is a power of two, at least 16")
    if dtype is _BF16:
        if k_scale is not None or v_scale is not None:
            raise ValueError("a bfloat16 cache has no scales")
        kind, unit, es = _lib.CACHE_BF16, 8, (0, 0)
    elif dtype is _E4M3:
        if k_scale is None or v_scale is None:
            raise ValueError("a float8_e4m3fn cache needs k_scale and v_scale")
        es = k_scale.stride()
        if (k_scale.shape != shape[:3] or v_scale.shape != shape[:3] or k_scale.dtype is not _E8M0
                or v_scale.dtype is not _E8M0 or v_scale.stride() != es):
            raise ValueError("Expected k_scale and v_scale [pages,Hkv,page_size] in float8_e8m0fnu, alike in strides")
        if es[2] != 1 or es[0] % 4 or es[1] % 4:
            raise ValueError("k_scale and v_scale need contiguous rows and strides that are multiples of 4")
        kind, unit, es = _lib.CACHE_E4M3, 16, es[:2]
    else:
        raise ValueError("a cache holds bfloat16 or float8_e4m3fn")
    if strides[3] != 1 or strides[0] % unit or strides[1] % unit or strides[2] % unit:
        raise ValueError("k_cache and v_cache need contiguous rows and strides that are multiples of 16 bytes")
    return shape, strides, es, kind


def _wide(t, flag, name):
    """The index flag of an int64 tensor, 0 for int32."""
    if t.dtype is _I64:
        return flag
    if t.dtype is _I32:
        return 0
    raise ValueError(f"{name} must be int32 or int64")


def _row_strides(t, name):
    """Strides of B, H and S of a [B,H,S,D] tensor with contiguous, aligned rows."""
    st = t.stride()
    if st[3] != 1 or st[0] % 8 or st[1] % 8 or st[2] % 8:
        raise ValueError(f"{name} needs contiguous rows and strides that are multiples of 8 elements")
    return st[:3]


# ---------------------------------------------------------------------------
# Workspaces: one per (device, stream) for eager calls, kept zeroed where the
# kernels count arrivals, as in ops; one of the graph's own under capture.
# ---------------------------------------------------------------------------

COUNTER_BYTES = 8192  # KFMI_DECODE_COUNTER_BYTES, KFMI_LOGPROBS_COUNTER_BYTES

_work_cache: dict[tuple[int, int], tuple[int, int, torch.Tensor]] = {}
_work_retired: list[torch.Tensor] = []
_size_cache: dict[tuple, int] = {}


def _ask_workspace(entry, packed):
    """Bytes that a workspace query answers for these arguments."""
    got = ctypes.c_int64()
    lib = _lib.load()
    if getattr(lib, entry)(packed, ctypes.byref(got)) != _lib.KFMI_OK:
        raise ValueError(f"{entry}: {lib.kfmi_last_error().decode(errors='replace')}")
    return got.value


def _workspace(index, stream, nbytes):
    """(address, bytes, tensor) of a workspace with zeroed counters for a launch
    on ``stream`` of the current device ``index``."""
    if nbytes <= 0:
        return 0, 0, None
    if torch.cuda.is_current_stream_capturing():
        buf = torch.empty(nbytes, dtype=torch.uint8, device=index)
        buf[:COUNTER_BYTES].zero_()  # a fill kernel inside the graph, not a memset node
        return buf.data_ptr(), nbytes, buf
    key = (index, stream)
    buf = _work_cache.get(key)
    if buf is None or buf[1] < nbytes:
        if buf is not None:
            _work_retired.append(buf[2])  # launches that hold its address may still run
        t = torch.zeros(max(nbytes, 0 if buf is None else 2 * buf[1]), dtype=torch.uint8, device=index)
        buf = _work_cache[key] = (t.data_ptr(), t.numel(), t)
    return buf


def _given_work(work, index):
    if work.get_device() != index or not work.is_contiguous():
        raise ValueError("work must be a contiguous tensor on the inputs' device")
    return work.data_ptr(), work.numel() * work.element_size(), work


# ---------------------------------------------------------------------------
# The cache
# ---------------------------------------------------------------------------

def norm_rope_to_cache(q, k, v, gq, gk, cos, sin, positions, slots, k_cache, v_cache, k_scale=None, v_scale=None, *,
                       norm_style="hf", eps=EPS, qn=None, kn=None):
    """Q/K RMSNorm*gamma (+ rotate-half RoPE) of new tokens, K and V written into
    the cache, in one launch.  Returns ``qn`` (None when ``q`` is).

    ``q`` ``[B,Hq,S,D]`` (or None: K and V only), ``k``, ``v`` ``[B,Hkv,S,D]``: BF16 rows of any strides, so the
    transposed views of projections ``[B,S,H,D]`` need no copy.  ``cos``/``sin``: BF16 tables ``[P,D]``, both
    None without RoPE; ``positions`` ``[B,S]``: each token's row of them (None without tables).  ``slots``
    ``[B,S]``: where each token goes; a negative slot is a padding token, which
    is not written.  The other slots of a call must differ.  Strides of both are free (``expand``).

    ``norm_style``: ``'hf'``, ``'legacy'`` or ``'fp32'`` as in ``optimized_attention``; Q and K rows are
    ``norm_rope``'s bit for bit.  A ``float8_e4m3fn`` cache takes the BF16 rows divided by
    the row's power-of-two scale (the smallest with ``max|row| / scale <= 448``), rounded to nearest even.  ``qn``
    and ``kn``: contiguous buffers for the prepared Q rows and (only where given) for
    the BF16 K rows, which a prefill over the same tokens reads; ``qn`` may be a contiguous ``q``.

    A position outside the tables makes its token's rows of ``qn``, ``kn`` and
    the cached K NaN; a slot behind the cache makes its rows of ``qn`` and ``kn`` NaN and is not written.
    """
    style = NORM_STYLES.get(norm_style)
    if style is None:
        raise ValueError("norm_style must be 'hf', 'legacy' or 'fp32'")
    if (cos is None) != (sin is None):
        raise ValueError("Pass both rotary tables (cos and sin) or neither")
    if k is None or v is None or gk is None or (q is not None and gq is None):
        raise ValueError("Expected k, v and gk (and gq with q)")
    _check_grad("norm_rope_to_cache", q, k, v, gq, gk, cos, sin, k_cache, v_cache)
    shape, d1 = k.shape, (k.shape[-1],)
    if len(shape) != 4 or v.shape != shape:
        raise ValueError("Expected q [B,Hq,S,D] and k, v [B,Hkv,S,D]")
    b, hk, s, d = shape
    if d not in (128, 256) or b < 1 or hk < 1 or s < 1:
        raise ValueError("Expected D in (128, 256), B, S >= 1 and Hq a multiple of Hkv")
    if k.dtype is not _BF16 or v.dtype is not _BF16 or gk.dtype is not _BF16:
        raise ValueError("Inputs must be BF16 tensors")
    if gk.shape != d1:
        raise ValueError("Expected gamma vectors [D]")
    ks, vs = _row_strides(k, "k"), _row_strides(v, "v")
    index = k.get_device()
    hq, qs, q_ptr, gq_ptr = 0, (0, 0, 0), 0, 0
    if q is not None:
        qshape = q.shape
        if len(qshape) != 4 or qshape[0] != b or qshape[2] != s or qshape[3] != d:
            raise ValueError("Expected q [B,Hq,S,D] and k, v [B,Hkv,S,D]")
        hq = qshape[1]
        if hq < 1 or hq % hk:
            raise ValueError("Expected D in (128, 256), B, S >= 1 and Hq a multiple of Hkv")
        if q.dtype is not _BF16 or gq.dtype is not _BF16:
            raise ValueError("Inputs must be BF16 tensors")
        if gq.shape != d1:
            raise ValueError("Expected gamma vectors [D]")
        if not gq.is_contiguous():
            raise ValueError("gamma vectors and rotary tables must be contiguous")
        qs, q_ptr, gq_ptr = _row_strides(q, "q"), q.data_ptr(), gq.data_ptr()
    flags = _wide(slots, _lib.I64_SLOTS, "slots")
    if slots.shape != (b, s):
        raise ValueError("Expected slots [B,S]")
    table_rows, cos_ptr, sin_ptr, pos_ptr, pos_strides = 0, 0, 0, 0, (0, 0)
    if cos is not None:
        if positions is None or positions.shape != (b, s):
            raise ValueError("Expected positions [B,S] with rotary tables")
        tshape = cos.shape
        if len(tshape) != 2 or tshape[1] != d or sin.shape != tshape or tshape[0] < 1:
            raise ValueError("Expected rotary tables [P,D]")
        if cos.dtype is not _BF16 or sin.dtype is not _BF16:
            raise ValueError("Inputs must be BF16 tensors")
        if not cos.is_contiguous() or not sin.is_contiguous():
            raise ValueError("gamma vectors and rotary tables must be contiguous")
        flags |= _wide(positions, _lib.I64_POSITIONS, "positions")
        table_rows, cos_ptr, sin_ptr = tshape[0], cos.data_ptr(), sin.data_ptr()
        pos_ptr, pos_strides = positions.data_ptr(), positions.stride()
    if not gk.is_contiguous():
        raise ValueError("gamma vectors and rotary tables must be contiguous")
    cshape, cs, es, kind = _check_cache(k_cache, v_cache, k_scale, v_scale)
    if cshape[1] != hk or cshape[3] != d:
        raise ValueError("The cache's Hkv and D must be those of k and v")
    if b * s * max(hq, hk) * d >= 2 ** 31:
        raise ValueError("Tensors must have fewer than 2**31 elements")
    if qn is not None:
        _check_out("qn", qn, None if q is None else qshape)
    if kn is not None:
        _check_out("kn", kn, shape)
    _check_gpu(index, q, v, gq if q is not None else None, gk, cos, sin, positions if cos is not None else None, slots,
               k_cache, v_cache, k_scale, v_scale, qn, kn)
    if not eps >= 0.0:
        raise ValueError("eps must be >= 0")
    if q is not None and qn is None:
        qn = torch.empty(qshape, dtype=_BF16, device=index)
    _call(index, "kfmi_norm_rope_to_cache_bf16", _lib.CACHE_WRITE_ARGS.pack(
        q_ptr, k.data_ptr(), v.data_ptr(), gq_ptr, gk.data_ptr(), cos_ptr, sin_ptr, pos_ptr, slots.data_ptr(),
        0 if q is None else qn.data_ptr(), 0 if kn is None else kn.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
        0 if k_scale is None else k_scale.data_ptr(), 0 if k_scale is None else v_scale.data_ptr(), *qs, *ks, *vs,
        *pos_strides, *slots.stride(), cs[0], cs[1], cs[2], *es, b, hq, hk, s, d, table_rows, cshape[0], cshape[2],
        eps, style, kind, flags, 0))
    return qn


def _check_out(name, out, shape):
    if shape is None or out.shape != shape or out.dtype is not _BF16 or not out.is_contiguous():
        raise ValueError(f"{name} must be a contiguous BF16 tensor shaped like its input on the same device")


def _pages_and_lengths(pages, lengths, b):
    """Their index flags, the pages per sequence and the stride between them."""
    shape, stride = pages.shape, pages.stride()
    if len(shape) != 2 or shape[0] != b or shape[1] < 1 or stride[1] != 1:
        raise ValueError("Expected pages [B,max_pages] with contiguous rows")
    if lengths.shape != (b,):
        raise ValueError("Expected lengths [B]")
    return (_wide(pages, _lib.I64_PAGES, "pages") | _wide(lengths, _lib.I64_LENGTHS, "lengths"), shape[1], stride[0])


def cache_to_dense(k_cache, v_cache, pages, lengths, max_length, k_scale=None, v_scale=None, *, k=None, v=None):
    """The first ``max_length`` cached rows of each sequence as contiguous BF16
    ``(k, v)`` ``[B,Hkv,max_length,D]`` (allocated unless given): an e4m3 row is
    its payload times its scale, exactly.  ``pages`` ``[B,max_pages]``: each
    sequence's pages in order; ``lengths`` ``[B]``.  Rows behind a sequence's
    length are zeros.  Rows of a page outside the cache, and all rows of a sequence whose length is
    negative or more than its pages hold, are NaN."""
    _check_grad("cache_to_dense", k_cache, v_cache)
    shape, cs, es, kind = _check_cache(k_cache, v_cache, k_scale, v_scale)
    num_pages, hk, page, d = shape
    b, l = lengths.shape[0] if lengths.ndim == 1 else 0, int(max_length)
    flags, _, _ = _pages_and_lengths(pages, lengths, b)
    if b < 1 or l < 1:
        raise ValueError("Expected B and max_length >= 1")
    if b * hk * l * d >= 2 ** 31:
        raise ValueError("Tensors must have fewer than 2**31 elements")
    for name, out in (("k", k), ("v", v)):
        if out is not None and (out.shape != (b, hk, l, d) or out.dtype is not _BF16 or not out.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous BF16 tensor [B,Hkv,max_length,D]")
    index = k_cache.get_device()
    _check_gpu(index, v_cache, pages, lengths, k, v, k_scale, v_scale)
    if k is None:
        k = torch.empty((b, hk, l, d), dtype=_BF16, device=index)
    if v is None:
        v = torch.empty((b, hk, l, d), dtype=_BF16, device=index)
    _call(index, "kfmi_cache_to_dense_bf16", _lib.CACHE_READ_ARGS.pack(
        k_cache.data_ptr(), v_cache.data_ptr(), 0 if k_scale is None else k_scale.data_ptr(),
        0 if v_scale is None else v_scale.data_ptr(), pages.data_ptr(), lengths.data_ptr(), k.data_ptr(),
        v.data_ptr(), cs[0], cs[1], cs[2], *es, pages.stride(0), lengths.stride(0), b, hk, l, d, num_pages, page,
        pages.shape[1], kind, flags))
    return k, v


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------

def attention_decode(q, k_cache, v_cache, pages, lengths, k_scale=None, v_scale=None, *, scale=None, window=None,
                     softcap=None, out=None, work=None):
    """Attention of each sequence's last S tokens over its paged cache; returns
    ``out`` ``[B,Hq,S,D]`` BF16 (which may be a contiguous ``q``).

    ``q`` ``[B,Hq,S,D]``: prepared queries (``norm_rope_to_cache``'s ``qn``) of
    any strides, 1 <= S <= 16: one token per sequence, or a few drafted ones.  ``pages`` ``[B,max_pages]``: each
    sequence's pages in order; ``lengths`` ``[B]``: its keys, the S new ones among them.  Query i has
    position ``lengths[b] - S + i`` and sees the keys up to its own; with ``window``
    only the last ``window`` of them.  ``scale`` defaults to D^-1/2; with ``softcap``
    the scores are ``softcap * tanh(score / softcap)``.  A query that sees
    no key (a padding sequence of length 0) gives zeros.

    Entries of ``pages`` behind a sequence's last key or before its window are
    not read, and what lies in rows that a query does not see, NaN or not, does not
    reach its result.  A length that is negative or more than the pages hold, or a page outside the cache, makes
    the sequence's rows of ``out`` NaN.

    ``work``: the workspace that joins the parts of split sequences (a
    zero-filled tensor of ``attention_decode_workspace_bytes``, left ready for the next call; calls that
    overlap in time need one each); None uses one that the package keeps per stream, or, while a
    graph is captured, one of the graph's own, zeroed on each replay.  The
    result's bits depend on the lengths in the batch, not on timing.
    """
    _check_grad("attention_decode", q, k_cache, v_cache)
    qshape = q.shape
    if len(qshape) != 4 or q.dtype is not _BF16:
        raise ValueError("Expected q [B,Hq,S,D] in BF16")
    b, hq, s, d = qshape
    shape, cs, es, kind = _check_cache(k_cache, v_cache, k_scale, v_scale)
    num_pages, hk, page, cd = shape
    if d != cd or b < 1 or hq < 1 or s < 1 or hq % hk:
        raise ValueError("Expected the cache's D and Hq a multiple of its Hkv")
    if s > 16:
        raise ValueError("attention_decode takes at most 16 tokens per sequence")
    flags, max_pages, pages_stride = _pages_and_lengths(pages, lengths, b)
    if window is None:
        window = 0
    elif int(window) < 1:
        raise ValueError("window must be >= 1")
    else:
        window = min(int(window), 1 << 40)
    if softcap is None:
        softcap = 0.0
    elif not 1e-30 <= softcap <= 1e30:
        raise ValueError("softcap must be from 1e-30 to 1e30")
    if scale is None:
        scale = d ** -0.5
    elif not 1e-30 <= scale <= 1e30:
        raise ValueError("scale must be from 1e-30 to 1e30")
    if b * hq * s * d >= 2 ** 31:
        raise ValueError("Tensors must have fewer than 2**31 elements")
    if out is not None and (out.shape != qshape or out.dtype is not _BF16 or not out.is_contiguous()):
        raise ValueError("out must be a contiguous BF16 tensor shaped like q")
    qs = _row_strides(q, "q")
    index = q.get_device()
    _check_gpu(index, k_cache, v_cache, pages, lengths, k_scale, v_scale, out)
    if out is None:
        out = torch.empty(qshape, dtype=_BF16, device=index)

    def space(stream):
        if work is not None:
            return _given_work(work, index)
        return _workspace(index, stream, attention_decode_workspace_bytes(b, hq, hk, s, d, max_pages * page))

    def packed(wp, wb):
        return _lib.DECODE_ARGS.pack(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), 0 if k_scale is None else k_scale.data_ptr(),
            0 if k_scale is None else v_scale.data_ptr(), pages.data_ptr(), lengths.data_ptr(), out.data_ptr(), wp,
            wb, *qs, cs[0], cs[1], cs[2], *es, pages_stride, lengths.stride(0), b, hq, hk, s, d, num_pages, page,
            max_pages, window, scale, softcap, kind, flags)

    _call(index, "kfmi_attention_decode_bf16", packed, space)
    return out


def attention_decode_workspace_bytes(b: int, hq: int, hkv: int, s: int, d: int, max_keys: int) -> int:
    """Bytes of ``attention_decode``'s workspace for sequences of up to ``max_keys``."""
    key = (b, hq, hkv, s, d, max_keys)
    n = _size_cache.get(key)
    if n is None:
        pages = -(-max_keys // 16)
        n = _size_cache[key] = _ask_workspace("kfmi_attention_decode_workspace", _lib.DECODE_ARGS.pack(
            *[0] * 9, 0, *[0] * 8, 0, 0, b, hq, hkv, s, d, 1, 16, pages, 0, 1.0, 0.0, 0, 0))
    return n


# ---------------------------------------------------------------------------
# Log probabilities
# ---------------------------------------------------------------------------

class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor  # [...] float32
    entropy: torch.Tensor  # [...] float32
    top_logprobs: Optional[torch.Tensor]  # [..., top] float32, largest first (None when top is 0)
    top_ids: Optional[torch.Tensor]  # [..., top] int64


def token_logprobs(logits, ids, top=0, *, work=None) -> TokenLogprobs:
    """Log probabilities of the tokens ``ids`` under ``logits``, the entropy of each
    distribution (nats) and its ``top`` (0 to 32) likeliest tokens, largest first,
    equal logits by the lower index; one pass over the logits.

    ``logits`` ``[..., V]`` in float32, BF16 or float16 with at most two leading
    dimensions of any strides (``logits[:, :-1]`` needs no copy) and contiguous rows; ``ids`` ``[...]`` int32 or
    int64.  Sums are 32-bit.  An id outside the vocabulary has log probability NaN.  A row that holds NaN or +infinity, or
    nothing but -infinity, is no distribution: NaN everywhere and top_ids -1.

    ``work``: as for ``attention_decode`` (``token_logprobs_workspace_bytes``)."""
    _check_grad("token_logprobs", logits)
    kind = _lib.LOGITS_TYPES.get(logits.dtype)
    if kind is None:
        raise ValueError("logits must be float32, bfloat16 or float16")
    shape, ls, is_ = logits.shape, logits.stride(), ids.stride()
    lead = shape[:-1]
    if not 1 <= len(shape) <= 3 or ids.shape != lead:
        raise ValueError("Expected logits [...,V] with up to two leading dimensions and ids [...]")
    flags = _wide(ids, _lib.I64_IDS, "ids")
    v, top = shape[-1], int(top)
    if v < 1 or v >= 2 ** 30 or (v > 1 and ls[-1] != 1):
        raise ValueError("logits need contiguous rows of 1 to 2**30 - 1 values")
    if not 0 <= top <= min(_lib.LOGPROBS_TOP_MAX, v):
        raise ValueError(f"top must be from 0 to {_lib.LOGPROBS_TOP_MAX} and at most V")
    n0, n1 = (1, 1, *lead)[-2:]
    if n0 * n1 >= 2 ** 25:
        raise ValueError("Expected fewer than 2**25 rows")
    index = logits.get_device()
    _check_gpu(index, ids)
    out, entropy = torch.empty((2, *lead), dtype=_F32, device=index).unbind(0)
    tops = (None, None)
    if top:
        tops = (torch.empty((*lead, top), dtype=_F32, device=index), torch.empty((*lead, top), dtype=_I64, device=index))
    if n0 * n1 == 0:
        return TokenLogprobs(out, entropy, *tops)

    def space(stream):
        if work is not None:
            return _given_work(work, index)
        return _workspace(index, stream, token_logprobs_workspace_bytes(n0 * n1, v, top, logits.dtype))

    def packed(wp, wb):
        return _lib.LOGPROBS_ARGS.pack(
            logits.data_ptr(), ids.data_ptr(), out.data_ptr(), entropy.data_ptr(), tops[0].data_ptr() if top else 0,
            tops[1].data_ptr() if top else 0, wp, wb, *(0, 0, *ls[:-1])[-2:], *(0, 0, *is_)[-2:], n0, n1, v, top, kind,
            flags, 0)

    _call(index, "kfmi_token_logprobs", packed, space)
    return TokenLogprobs(out, entropy, *tops)


def token_logprobs_workspace_bytes(n: int, v: int, top: int, dtype=torch.float32) -> int:
    """Bytes of ``token_logprobs``'s workspace for ``n`` rows of ``v`` logits."""
    key = (n, v, top, dtype)
    size = _size_cache.get(key)
    if size is None:
        size = _size_cache[key] = _ask_workspace("kfmi_token_logprobs_workspace", _lib.LOGPROBS_ARGS.pack(
            *[0] * 7, 0, 0, 0, 0, 0, 1, n, v, top, _lib.LOGITS_TYPES[dtype], 0, 0))
    return size

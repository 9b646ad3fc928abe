"""A quantised, paged K/V cache and the operators around it, for programs that generate tokens.

    rotary = SageRotary(128, base=10000.0)
    cache = SageCache.empty(num_pages, page_size, num_kv_heads, head_dim, dtype=torch.bfloat16)
    q, k = sage_rotary(q, k, positions, rotary)                 # q (tokens, Hq, D), k (tokens, Hkv, D)
    sage_cache_write(cache, k, v, slots)                        # quantised as it is written
    out = sageattn_cached(q, cache, page_table, seqlens_k)      # one new token per sequence
    out = sageattn_cached(q, cache, page_table, seqlens_k, cu_seqlens_q, max_seqlen_q, tree_mask=mask)
    out = sageattn_cached(q, cache, page_table, seqlens_k, cu_seqlens_q, max_seqlen_q)      # the next chunk of a prompt: a chain
    k16, v16 = sage_cache_read(cache, page_table, cu_seqlens_k, total)      # e.g. for sageattn_varlen without a causal mask

The reference keeps no cache: its callers hand over the whole K and V with every call, which are then
quantised again (sageattention/core.py:1037-1252).  Codes and scales here are those of its quantiser
(kernels/hip/h34_prologue.hip:116-211): one fp32 scale per token and head, int8 or e4m3 K, e4m3 V.
Index tensors (slots, page tables, lengths) stay on the GPU and are never read on the host: no call
synchronises, and every call can be captured into a CUDA graph.
"""
from __future__ import annotations

import math
import operator
import struct
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _native
from . import b200_backend as _be
from .b200_backend import HEAD_DIM, _WS_GRANULE, _counters, _dtype_code, _report_to, _state, packed_view_reason, strided_view_reason

_E4M3 = torch.float8_e4m3fn


def _refuse(what: str, kind=ValueError):
    _counters["refusals"] += 1
    raise kind("%s (B200 path)" % what)


def _check_head_dim(d: int):
    if d < 8 or d > HEAD_DIM or d % 8:
        _refuse("head_dim must be a multiple of 8 in 8..128, got %d" % d, NotImplementedError)


# The C calls take their arguments as 64-bit words: those that change from call to call, then those of the plan, kept as bytes
# (27 arguments that are converted one by one take 6 us, the words one).
_WRITE, _READ, _ATTEND, _ROTATE = range(4)           # SAGE_WORDS_* in sage_b200.h
_COUNT = (21, 24, 34, 32)
_FIRST = tuple(struct.Struct("%dQ" % n).pack for n in (4, 5, 11, 7))


def _kept(*words) -> bytes:
    return struct.pack("".join("d" if isinstance(x, float) else "q" for x in words), *words)


def _call(what, dev, words):
    """The C call, on `dev` as the current device."""
    prev = torch.cuda.current_device()
    if prev == dev.index:
        return _native.load().sage_call_words(what, words, _COUNT[what])
    torch.cuda.set_device(dev)
    try:
        return _native.load().sage_call_words(what, words, _COUNT[what])
    finally:
        torch.cuda.set_device(prev)


_PACKED = torch.contiguous_format


def _fresh(t):
    """Packed memory for an output like t."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty_like(t, memory_format=_PACKED)


def _like(shape, dtype, dev):
    """A tensor of one element in that shape, for `empty_like`, which is twice as fast as `empty`."""
    return torch.empty((1,) * len(shape), dtype=dtype, device=dev).expand(shape)


# A step of generation is a handful of calls whose GPU work takes a few microseconds each, so that the host path must
# not take longer.  A call signature (shapes, strides, dtypes, devices, alignment) that has passed the checks once is
# remembered with what the C call is given for it, as for `sageattn`.
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)
_PLANS = 256


def _sig(t: torch.Tensor):
    return t.shape, t.stride(), t.dtype, t.device, t.data_ptr() & 15


def _fixed(self, name, value):
    """`__setattr__` of objects whose buffers' addresses are worked out once."""
    if hasattr(self, "_plans"):
        raise AttributeError("%s.%s is fixed when the object is made" % (type(self).__name__, name))
    object.__setattr__(self, name, value)


def _written(tensors):
    """Tell autograd that these were written over, as it is told of torch's own writes."""
    for t in tensors:
        if t.requires_grad and torch.is_grad_enabled():
            _refuse("an output must not require gradients")
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _remember(plans: dict, key, plan):
    if len(plans) >= _PLANS:
        plans.clear()
    plans[key] = plan
    return plan


class SageCache:
    """The buffers of a paged cache, which the caller may own.

    k_codes : ``(pages, Hkv, page_size, width)`` int8 or float8_e4m3fn; v_codes the same shape,
        float8_e4m3fn; ``width`` is 64 for ``head_dim`` up to 64 and 128 above
    k_scale, v_scale : ``(pages, Hkv, page_size)`` float32
    k_shift : optional ``(Hkv, head_dim)`` float32 that is subtracted from K before it is quantised (the mean
        that `smooth_k` takes off, taken once over a prompt and kept).  Attention does not change by it: all
        keys of a head move alike.  The cache keeps a copy of it, which is what the attribute of that name shows.
    The buffers stay the cache's for good (what they hold may change).
    page_size is a power of two, 16 .. 256.  The code buffers must start as zeros (`empty` does that): codes that
    no write has set may be read behind a mask, and must not be the e4m3 NaN.
    """

    __slots__ = ("k_codes", "k_scale", "v_codes", "v_scale", "k_shift", "head_dim", "num_pages", "page_size",
                 "num_kv_heads", "device", "_mode", "_args", "_sizes", "_tracked", "_plans")
    __setattr__ = _fixed

    def __init__(self, k_codes: torch.Tensor, k_scale: torch.Tensor, v_codes: torch.Tensor, v_scale: torch.Tensor,
                 head_dim: int, k_shift: Optional[torch.Tensor] = None):
        if k_codes.dim() != 4 or k_codes.dtype not in (torch.int8, _E4M3):
            _refuse("k_codes must be a (pages, heads, page_size, width) tensor of int8 or float8_e4m3fn")
        pages, heads, page, width = (int(x) for x in k_codes.shape)
        head_dim = int(head_dim)
        _check_head_dim(head_dim)
        if width != (64 if head_dim <= 64 else 128):
            _refuse("rows of a cache are 64 bytes wide for head_dim up to 64, else 128; got %d" % width)
        if page < 16 or page > 256 or page & (page - 1):
            _refuse("page_size must be a power of two in 16..256, got %d" % page, NotImplementedError)
        if pages < 1 or heads < 1:
            _refuse("a cache needs at least one page and one head")
        if v_codes.dtype != _E4M3 or tuple(v_codes.shape) != tuple(k_codes.shape):
            _refuse("v_codes must be float8_e4m3fn of k_codes' shape")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t.dtype != torch.float32 or tuple(t.shape) != (pages, heads, page):
                _refuse("%s must be float32 (pages, heads, page_size)" % name)
        for t in (k_codes, k_scale, v_codes, v_scale):
            if not t.is_cuda or t.device != k_codes.device:
                _refuse("a cache lives on one CUDA device; there is no CPU path")
            if not t.is_contiguous() or t.data_ptr() % 16:
                _refuse("the buffers of a cache must be contiguous and 16-byte aligned")
        if k_shift is not None:
            if tuple(k_shift.shape) != (heads, head_dim) or k_shift.device != k_codes.device:
                _refuse("k_shift must be (heads, head_dim) on the cache's device")
            padded = torch.zeros((heads, width), dtype=torch.float32, device=k_codes.device)
            padded[:, :head_dim] = k_shift.detach()
            k_shift = padded[:, :head_dim]
        self.k_codes, self.k_scale, self.v_codes, self.v_scale, self.k_shift = k_codes, k_scale, v_codes, v_scale, k_shift
        self.head_dim, self.num_pages, self.page_size, self.num_kv_heads = head_dim, pages, page, heads
        self.device = k_codes.device
        self._mode = _native.SAGE_QK_INT8 if k_codes.dtype == torch.int8 else _native.SAGE_QK_E4M3
        self._args = (k_codes.data_ptr(), k_scale.data_ptr(), v_codes.data_ptr(), v_scale.data_ptr(),
                      0 if k_shift is None else k_shift.data_ptr())
        self._sizes = (pages, page)
        self._tracked = [t for t in (k_codes, k_scale, v_codes, v_scale) if not t.is_inference()]
        self._plans = {}                             # call signature -> what the C call is given for it

    def __reduce__(self):                            # a copy has buffers, and addresses, of its own
        return type(self), (self.k_codes, self.k_scale, self.v_codes, self.v_scale, self.head_dim, self.k_shift)

    @classmethod
    def empty(cls, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, dtype: torch.dtype = torch.float16,
              int8: Optional[bool] = None, device="cuda", k_shift: Optional[torch.Tensor] = None) -> "SageCache":
        """A cache of zeros for keys and values of `dtype`.  ``int8=None`` follows the rule of `sageattn`: int8 K
        codes for float16, e4m3 for bfloat16."""
        _dtype_code(dtype)
        _check_head_dim(int(head_dim))
        if int8 is None:
            int8 = dtype == torch.float16
        shape = (int(num_pages), int(num_kv_heads), int(page_size))
        width = 64 if head_dim <= 64 else 128
        codes = [torch.zeros(shape + (width,), dtype=torch.uint8, device=device) for _ in range(2)]
        scales = [torch.zeros(shape, dtype=torch.float32, device=device) for _ in range(2)]
        return cls(codes[0].view(torch.int8 if int8 else _E4M3), scales[0], codes[1].view(_E4M3), scales[1], head_dim, k_shift)


def _check_rows(name: str, t: torch.Tensor, heads: int, d: int, dev, output: bool = False):
    """A packed (tokens, heads, head_dim) tensor next to a cache; in an output every row has memory of its own."""
    if t.device != dev:
        _refuse("%s must be on the cache's device" % name)
    if t.dtype not in (torch.float16, torch.bfloat16):
        _refuse("%s must be float16 or bfloat16" % name)
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != d:
        _refuse("%s must be (tokens, %d, %d), got %s" % (name, heads, d, tuple(t.shape)))
    if t.numel():
        reason = packed_view_reason(t)
        if reason is not None:
            _refuse("cannot serve %s: %s" % (name, reason))
    reach = d
    for stride, n in sorted(zip(t.stride()[:2], t.shape[:2])) if output else ():
        if n > 1:
            if stride < reach:
                _refuse("the rows of %s must not overlap" % name)
            reach += stride * (n - 1)


def _check_index(name: str, t: torch.Tensor, dev, dims: int, dtypes=(torch.int32,)):
    if t.device != dev:
        _refuse("%s must be on the cache's device" % name)
    if t.dtype not in dtypes or t.dim() != dims:
        _refuse("%s must be a %d-D tensor of %s" % (name, dims, " or ".join(str(x) for x in dtypes)))
    if t.numel() and t.stride(-1) != 1:
        _refuse("%s must be contiguous along its last axis" % name)


def sage_cache_write(cache: SageCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantise `k` and `v`, ``(tokens, Hkv, head_dim)`` float16 or bfloat16, into the cache.

    slots : ``(tokens,)`` int32 or int64 on the GPU, ``page * page_size + offset``.  A token whose slot lies below
    0 or past the last page is left out (the padding of a batch).  Slots of one call are distinct: of two tokens
    with one slot, each part of the row may come from either.  A row that holds a NaN or an infinity reads back as
    NaN throughout.
    """
    _counters["calls"] += 1
    key = ("write", _sig(k), _sig(v), _sig(slots))
    plan = cache._plans.get(key)
    if plan is None:
        plan = _remember(cache._plans, key, _plan_write(cache, k, v, slots))
    if plan:
        torch.autograd.graph.increment_version(cache._tracked)       # as for torch's own writes
        dev = cache.device
        rc = _call(_WRITE, dev, _FIRST[_WRITE](k.data_ptr(), v.data_ptr(), slots.data_ptr(), _raw_stream(dev.index)) + plan)
        if rc:
            _native.check(rc, "sage_cache_write")


def _plan_write(cache, k, v, slots):
    dev, heads, d = cache.device, cache.num_kv_heads, cache.head_dim
    _check_rows("k", k, heads, d, dev)
    _check_rows("v", v, heads, d, dev)
    if k.dtype != v.dtype or k.shape[0] != v.shape[0]:
        _refuse("k and v must have the same dtype and tokens")
    _check_index("slots", slots, dev, 1, (torch.int32, torch.int64))
    if slots.shape[0] != k.shape[0]:
        _refuse("slots must hold one entry per token")
    if k.shape[0] == 0:
        return b""
    return _kept(slots.dtype == torch.int64, *cache._args, k.shape[0], heads, d, *cache._sizes, k.stride(0), k.stride(1), v.stride(0),
                 v.stride(1), _dtype_code(k.dtype), cache._mode)


def sage_cache_read(cache: SageCache, page_table: torch.Tensor, cu_seqlens: torch.Tensor, total: int,
                    dtype: torch.dtype = torch.float16, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
                    ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Sequences of the cache as packed 16-bit keys and values, each ``(total, Hkv, head_dim)``.

    page_table : ``(batch, width)`` int32 page ids on the GPU; cu_seqlens : ``(batch + 1,)`` int32 prefix sums of the
    token counts on the GPU, ``cu_seqlens[-1]`` at most `total`.  Rows from ``cu_seqlens[-1]`` on are left as they are
    (in fresh outputs: undefined); tokens on a page that does not exist read as zeros.
    """
    _counters["calls"] += 1
    dev = cache.device
    if total.__class__ is not int:
        _refuse("total must be an int, not negative")
    key = ("read", _sig(page_table), _sig(cu_seqlens), total, dtype, None if out is None else tuple(_sig(t) for t in out))
    plan = cache._plans.get(key)
    if plan is None:
        plan = _remember(cache._plans, key, _plan_read(cache, page_table, cu_seqlens, total, dtype, out))
    words, like = plan
    if out is None:
        k, v = torch.empty_like(like, memory_format=_PACKED), torch.empty_like(like, memory_format=_PACKED)
    else:
        k, v = out
        if words and _overlap(k, v):
            _refuse("the two outputs must not overlap")
        _written(out)
    if words:
        rc = _call(_READ, dev, _FIRST[_READ](page_table.data_ptr(), cu_seqlens.data_ptr(), k.data_ptr(), v.data_ptr(), _raw_stream(dev.index)) + words)
        if rc:
            _native.check(rc, "sage_cache_read")
    return k, v


def _plan_read(cache, page_table, cu_seqlens, total, dtype, out):
    dev, heads, d = cache.device, cache.num_kv_heads, cache.head_dim
    code = _dtype_code(dtype)
    _check_index("page_table", page_table, dev, 2)
    _check_index("cu_seqlens", cu_seqlens, dev, 1)
    if page_table.shape[0] < 1 or page_table.shape[1] < 1 or cu_seqlens.shape[0] != page_table.shape[0] + 1:
        _refuse("page_table and cu_seqlens must describe the same sequences, at least one")
    if total < 0:
        _refuse("total must be an int, not negative")
    strides = (heads * d, d) * 2
    if out is not None:
        if len(out) != 2:
            _refuse("out must be a pair")
        for name, t in (("out[0]", out[0]), ("out[1]", out[1])):
            _check_rows(name, t, heads, d, dev, output=True)
            if t.shape[0] != total or t.dtype != dtype:
                _refuse("%s must hold total rows of dtype" % name)
        strides = [n for t in out for n in t.stride()[:2]]
    like = _like((total, heads, d), dtype, dev)
    if total == 0:
        return b"", like
    return _kept(*cache._args, page_table.stride(0), page_table.shape[1], page_table.shape[0], total, heads, d, *cache._sizes, *strides, code,
                 cache._mode), like


def sageattn_cached(q: torch.Tensor, cache: SageCache, page_table: torch.Tensor, seqlens_k: torch.Tensor,
                    cu_seqlens_q: Optional[torch.Tensor] = None, max_seqlen_q: Optional[int] = None,
                    tree_mask: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None,
                    return_lse: bool = False, out: Optional[torch.Tensor] = None):
    """Attention of new tokens over the cached keys of their sequences.

    q : ``(tokens, Hq, head_dim)`` packed, float16 or bfloat16, ``Hq`` a multiple of the cache's heads.
    page_table : ``(batch, width)`` int32; seqlens_k : ``(batch,)`` int32: cached keys of each sequence, those of its
        new tokens among them (the last ones, written before this call).
    cu_seqlens_q : ``(batch + 1,)`` int32 prefix sums of the new tokens per sequence, with `max_seqlen_q` the largest
        count (a longer sequence is cut off there, as in `sageattn_varlen`).  None: ``tokens / batch`` for each.
    tree_mask : None, and a new token sees every key up to its own (one token: all of them; several: a chain);
        or ``(tokens, >= max_seqlen_q)`` bool (or uint8): token t sees the new token j of its sequence where
        ``tree_mask[t, j]``, and all keys before the new tokens.  A tree of drafted tokens sets a token's
        ancestors and itself.
    sm_scale : default ``head_dim ** -0.5``.
    return_lse : also return the fp32 log-sum-exp ``(tokens, Hq)`` of ``sm_scale * q.k``.
    out : optional output of q's shape and dtype, which shares no memory with q.
    A token that sees no key gets zeros and an LSE of -infinity; one that sees a key whose row of K or V held a NaN or an
    infinity gets NaN (its LSE: NaN, or for V alone that of the keys' scores), and so does one that sees a key and whose query
    holds one (its LSE too).  A key on a page that does not exist is not seen.  Rows of no sequence, and those past
    `max_seqlen_q` of theirs, are left as they are (in fresh outputs: undefined).  The lengths stay on the GPU; the last bits
    of a result depend on the lengths of the other sequences of the call (fp32 sums in another order).  Forward only: the
    result carries no gradient, as that of `sageattn`.
    """
    dev = cache.device
    if torch.cuda.current_device() != dev.index:     # (its current stream, and whether that is being captured)
        with torch.cuda.device(dev):
            return sageattn_cached(q, cache, page_table, seqlens_k, cu_seqlens_q, max_seqlen_q, tree_mask, sm_scale, return_lse, out)
    _counters["calls"] += 1
    if max_seqlen_q is not None:
        max_seqlen_q = operator.index(max_seqlen_q)
    if sm_scale is not None:
        sm_scale = float(sm_scale)
    key = ("attend", _sig(q), _sig(page_table), _sig(seqlens_k), None if cu_seqlens_q is None else _sig(cu_seqlens_q), max_seqlen_q,
           None if tree_mask is None else _sig(tree_mask), sm_scale, None if out is None else _sig(out))
    plan = cache._plans.get(key)
    if plan is None:
        plan = _remember(cache._plans, key, _plan_attend(cache, q, page_table, seqlens_k, cu_seqlens_q, max_seqlen_q, tree_mask, sm_scale, out))
    words, ws_bytes, like_lse = plan
    if out is None:
        out = _fresh(q)
    else:
        if words and _overlap(q, out):
            _refuse("out must not overlap q")
        _written((out,))
    lse = torch.empty_like(like_lse, memory_format=_PACKED) if return_lse else None
    if words:
        stream = _raw_stream(dev.index)
        capturing = torch.cuda.is_current_stream_capturing()
        st = _state(dev, stream)                     # host word of the stream, as for `sageattn`
        if st.host_word is not None and st.host_word.value:
            st.raise_if_failed("the next call on the stream")
        with st.cache_lock:                          # the call's two kernels share a workspace: another thread's do not come between them
            if capturing:                            # a captured call has memory of its graph's own: two graphs may run at once
                ws = torch.empty((ws_bytes,), dtype=torch.uint8, device=dev)
            else:
                ws = st.cache_ws
                if ws is None or ws.numel() < ws_bytes:
                    st.cache_ws = None               # release first: the two need not be resident together
                    ws = st.cache_ws = torch.empty(((ws_bytes + _WS_GRANULE - 1) // _WS_GRANULE * _WS_GRANULE,), dtype=torch.uint8, device=dev)
            rc = _native.load().sage_call_words(_ATTEND, _FIRST[_ATTEND](
                q.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(), page_table.data_ptr(), seqlens_k.data_ptr(),
                0 if cu_seqlens_q is None else cu_seqlens_q.data_ptr(), 0 if tree_mask is None else tree_mask.data_ptr(), ws.data_ptr(), ws_bytes,
                _report_to(st, capturing), stream) + words, _COUNT[_ATTEND])
        if rc:
            _native.check(rc, "sage_cache_attention")
        if _be._STRICT and not capturing:
            torch.cuda.current_stream(dev).synchronize()
            st.raise_if_failed("this call (strict mode)")
    return (out, lse) if return_lse else out


def _plan_attend(cache, q, page_table, seqlens_k, cu_seqlens_q, max_seqlen_q, tree_mask, sm_scale, out):
    dev, hkv, d = cache.device, cache.num_kv_heads, cache.head_dim
    if q.dim() != 3 or q.shape[1] < 1 or q.shape[1] % hkv:
        _refuse("q must be (tokens, heads, head_dim) with a multiple of the cache's %d heads" % hkv)
    tokens, hq = int(q.shape[0]), int(q.shape[1])
    _check_rows("q", q, hq, d, dev)
    _check_index("page_table", page_table, dev, 2)
    _check_index("seqlens_k", seqlens_k, dev, 1)
    batch, width = int(page_table.shape[0]), int(page_table.shape[1])
    if batch < 1 or width < 1 or seqlens_k.shape[0] != batch:
        _refuse("page_table and seqlens_k must describe the same sequences, at least one")
    if cu_seqlens_q is None:
        if tokens % batch or (max_seqlen_q is not None and max_seqlen_q * batch != tokens):
            _refuse("without cu_seqlens_q every sequence needs the same number of new tokens")
        max_q = tokens // batch
    else:
        _check_index("cu_seqlens_q", cu_seqlens_q, dev, 1)
        if cu_seqlens_q.shape[0] != batch + 1:
            _refuse("cu_seqlens_q must have batch + 1 entries")
        if max_seqlen_q is None or max_seqlen_q < 1:
            _refuse("cu_seqlens_q needs max_seqlen_q, at least 1")
        max_q = min(max_seqlen_q, tokens)
    if tree_mask is not None:
        _check_index("tree_mask", tree_mask, dev, 2, (torch.bool, torch.uint8))
        if tree_mask.shape[0] != tokens or tree_mask.shape[1] < max_q:
            _refuse("tree_mask must be (tokens, >= max_seqlen_q)")
    scale = d ** -0.5 if sm_scale is None else sm_scale
    if not (0.0 < scale < float("inf")):
        _refuse("sm_scale must be finite and positive, got %r" % (sm_scale,))
    if out is not None:
        _check_rows("out", out, hq, d, dev, output=True)
        if out.shape != q.shape or out.dtype != q.dtype:
            _refuse("out must have q's shape and dtype")
    like_lse = _like((tokens, hq), torch.float32, dev)
    if tokens == 0:
        return b"", 0, like_lse
    words = _kept(*cache._args, page_table.stride(0), width, 0 if tree_mask is None else tree_mask.stride(0), batch, hq, hkv, tokens, max_q, d,
                  *cache._sizes, q.stride(0), q.stride(1), *((hq * d, d) if out is None else out.stride()[:2]), _dtype_code(q.dtype), cache._mode, scale)
    return words, int(_native.load().sage_cache_attention_workspace_bytes(batch, hq, hkv, max_q)), like_lse


# ---- rotary positions --------------------------------------------------------------------------------------------

class SageRotary:
    """The frequencies of a rotary position encoding, in 64 bits on the GPU.

    rotary_dim : columns of a head that turn (default all of them), a multiple of 8
    interleaved : pairs (2i, 2i + 1) instead of (i, i + rotary_dim / 2)
    scaling : ``"none"``; ``"linear"``, all frequencies divided by `factor`; ``"ntk"``, the base raised to
        ``base * factor ** (rotary_dim / (rotary_dim - 2))``; ``"parts"``: frequencies that turn more than `fast` times
        within `original_length` positions stay, those that turn less than `slow` times are divided by `factor`, a
        linear ramp between, and the result is scaled by ``0.1 ln(factor) + 1``.
    """

    __slots__ = ("head_dim", "rotary_dim", "interleaved", "inv_freq", "magnitude", "device", "_plans")
    __setattr__ = _fixed

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, base: float = 10000.0, interleaved: bool = False,
                 scaling: str = "none", factor: float = 1.0, original_length: int = 4096, fast: float = 32.0, slow: float = 1.0,
                 device="cuda"):
        head_dim = int(head_dim)
        _check_head_dim(head_dim)
        rot = head_dim if rotary_dim is None else int(rotary_dim)
        if rot < 8 or rot > head_dim or rot % 8:
            _refuse("rotary_dim must be a multiple of 8 in 8..head_dim, got %d" % rot, NotImplementedError)
        if scaling not in ("none", "linear", "ntk", "parts"):
            _refuse("scaling must be 'none', 'linear', 'ntk' or 'parts'")
        if not (base > 1.0 and math.isfinite(base)) or not (factor >= 1.0 and math.isfinite(factor)):
            _refuse("base must be above 1 and factor at least 1")
        if scaling == "parts" and not (original_length > 0 and fast > slow > 0):
            _refuse("'parts' needs original_length > 0 and fast > slow > 0")
        if scaling == "ntk":
            base = base * factor ** (rot / (rot - 2))
        freq = [base ** (-i / rot) for i in range(0, rot, 2)]
        magnitude = 1.0
        if scaling == "linear":
            freq = [f / factor for f in freq]
        elif scaling == "parts":
            keep = [min(1.0, max(0.0, (original_length * f / (2 * math.pi) - slow) / (fast - slow))) for f in freq]
            freq = [f * (k + (1 - k) / factor) for f, k in zip(freq, keep)]
            magnitude = 0.1 * math.log(factor) + 1.0
        self._set(head_dim, rot, bool(interleaved), torch.tensor(freq, dtype=torch.float64).to(device), magnitude)

    def _set(self, head_dim, rotary_dim, interleaved, inv_freq, magnitude):
        self.head_dim, self.rotary_dim, self.interleaved, self.inv_freq, self.magnitude = head_dim, rotary_dim, interleaved, inv_freq, magnitude
        self.device = inv_freq.device
        self._plans = {}

    def __reduce__(self):                            # a copy has frequencies, and their address, of its own
        return _rotary_of, (self.head_dim, self.rotary_dim, self.interleaved, self.inv_freq, self.magnitude)


def _rotary_of(*parts):
    rotary = object.__new__(SageRotary)
    rotary._set(*parts)
    return rotary


def _rotary_views(x, layout):
    """A logical (B, H, N, D) view of a packed or batched tensor."""
    if x.dim() == 3:
        return x.unsqueeze(0).transpose(1, 2)
    if x.dim() == 4:
        return x if layout == "HND" else x.transpose(1, 2)
    _refuse("rotary takes (tokens, heads, head_dim) or 4-D tensors")


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two views share an element.  Views of one buffer with the same strides (the parts of a fused projection)
    are told apart exactly where each stride steps over all that the smaller ones reach, as those of servable views do;
    others that reach into one another count as sharing."""
    def span(t):
        return t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))
    (a0, a1), (b0, b1) = span(a), span(b)
    if not (a0 < b1 and b0 < a1):
        return False
    if a.stride() != b.stride():
        return True
    # (an axis of one element has no say, whatever its stride)
    axes = sorted(((s, na, nb) for s, na, nb in zip(a.stride(), a.shape, b.shape) if na > 1 or nb > 1), reverse=True)
    reach = 0
    for stride, na, nb in reversed(axes):
        if stride <= reach:
            return True
        reach += stride * (max(na, nb) - 1)

    def reachable(rest, k):
        # is rest = sum over the axes of (index in b - index in a) * stride?
        if k == len(axes):
            return rest == 0
        stride, na, nb = axes[k]
        near = rest // stride
        return any(-(na - 1) <= i <= nb - 1 and reachable(rest - i * stride, k + 1) for i in (near, near + 1))

    return reachable((a0 - b0) // a.element_size(), 0)


def _rotate(q, k, positions, rotary, layout, backward, out):
    # (an output that is its input needs no more of a plan than that the two inputs share nothing: their distance; a plan
    # holds the outputs' strides, so that fresh outputs, marked by None, have plans of their own)
    in_place = out is not None and (out is q if k is None else len(out) == 2 and out[0] is q and out[1] is k)
    kept = out is None or in_place
    distance = None if not in_place else 0 if k is None else k.data_ptr() - q.data_ptr()
    key = (_sig(q), None if k is None else _sig(k), _sig(positions), layout, distance)
    plan = rotary._plans.get(key) if kept else None
    if plan is None:
        plan = _plan_rotary(q, k, positions, rotary, layout, out)
        if kept:
            _remember(rotary._plans, key, plan)
    dev = rotary.device
    if out is None:
        outs = (_fresh(q),) if k is None else (_fresh(q), _fresh(k))
    else:
        outs = (out,) if isinstance(out, torch.Tensor) else tuple(out)
        _written(outs)
    if plan:
        rc = _call(_ROTATE, dev, _FIRST[_ROTATE](
            q.data_ptr(), outs[0].data_ptr(), 0 if k is None else k.data_ptr(), 0 if k is None else outs[1].data_ptr(), positions.data_ptr(),
            backward, _raw_stream(dev.index)) + plan)
        if rc:
            _native.check(rc, "sage_rotary")
    return outs


def _plan_rotary(q, k, positions, rotary, layout, out):
    ins = [x for x in (q, k) if x is not None]
    if ins[-1].dim() != q.dim():
        _refuse("q and k must both be packed or both be 4-D")
    views = [_rotary_views(x, layout) for x in ins]
    dev = q.device
    o_views = []
    if out is not None:
        outs = [out] if isinstance(out, torch.Tensor) else list(out)
        if len(outs) != len(ins):
            _refuse("out must hold one tensor per input")
        for i, (x, o) in enumerate(zip(ins, outs)):
            if o.shape != x.shape or o.dtype != x.dtype or o.device != x.device:
                _refuse("out must have the inputs' shapes, dtypes and device")
            for j, y in enumerate(ins + outs[:i]):
                own = j == i and o.data_ptr() == y.data_ptr() and o.stride() == y.stride()
                if x.numel() and y.numel() and not own and _overlap(o, y):
                    _refuse("out may be its own input, and overlaps nothing else")
        o_views = [_rotary_views(x, layout) for x in outs]
    b, _, n, d = views[0].shape
    for v in views + o_views:
        if v.device != dev or not v.is_cuda:
            _refuse("rotary needs CUDA tensors on one device; there is no CPU path")
        if v.dtype not in (torch.float16, torch.bfloat16) or v.dtype != q.dtype:
            _refuse("q and k must share one dtype, float16 or bfloat16")
        if v.shape[0] != b or v.shape[2] != n or v.shape[3] != d or v.shape[1] < 1:
            _refuse("q and k must agree in all but their heads")
        reason = strided_view_reason(v) if v.numel() else None
        if reason is not None:
            _refuse("cannot serve this call: %s" % reason)
    if d != rotary.head_dim or rotary.device != dev:
        _refuse("the rotary was made for head_dim %d on %s" % (rotary.head_dim, rotary.device))
    if positions.device != dev or positions.dtype not in (torch.int32, torch.int64):
        _refuse("positions must be int32 or int64 on the tensors' device")
    if positions.dim() == 1 and positions.shape[0] == n:
        p2 = (0, positions.stride(0))
    elif positions.dim() == 2 and q.dim() == 4 and tuple(positions.shape) == (b, n):
        p2 = positions.stride()
    else:
        _refuse("positions must be (N,) or (B, N)")
    if not b * n:
        return b""

    def triple(v):
        return v.stride()[:3]

    def packed(v):                                   # strides of a contiguous tensor in the inputs' layout
        h = v.shape[1]
        return (n * h * d, d, h * d) if q.dim() == 3 or layout == "NHD" else (h * n * d, n * d, d)
    s3 = []
    for i in (0, len(ins) - 1):
        s3 += [*triple(views[i]), *(triple(o_views[i]) if o_views else packed(views[i]))]
    return _kept(rotary.inv_freq.data_ptr(), positions.dtype == torch.int64, rotary.magnitude, b, views[0].shape[1],
                 views[1].shape[1] if k is not None else 0, n, d, rotary.rotary_dim, rotary.interleaved, *s3, *p2, _dtype_code(q.dtype))


def _tangent(t: torch.Tensor) -> bool:
    """Whether t carries a forward-mode derivative.  (Outside of every dual level, which is where calls are made that take
    a few microseconds, none does: asking the tensor takes 0.4.)"""
    return getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(t).tangent is not None


def _servable(grad: torch.Tensor) -> torch.Tensor:
    """A gradient as the kernel takes it: autograd hands over whatever the next operation left, broadcast or cut out of
    something larger at any offset."""
    grad = grad.contiguous()
    if grad.data_ptr() & 15 or any(s <= 0 or s % 8 for s in grad.stride()[:-1]):     # (the stride of an axis of one may be anything)
        grad = grad.clone(memory_format=_PACKED)
    return grad


class _Rotary(torch.autograd.Function):
    """The map is linear: its gradient is the transposed map of the outputs' gradients."""

    @staticmethod
    def forward(ctx, q, k, positions, rotary, layout, backward):
        ctx.save_for_backward(positions)
        ctx.rest = (rotary, layout, backward)
        res = _rotate(q, k, positions, rotary, layout, backward, None)
        return res if k is not None else res[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        rotary, layout, backward = ctx.rest
        res = _rotate(_servable(grads[0]), _servable(grads[1]) if len(grads) > 1 else None, ctx.saved_tensors[0], rotary, layout,
                      not backward, None)
        return res[0], res[1] if len(grads) > 1 else None, None, None, None, None


def sage_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rotary: SageRotary,
                tensor_layout: str = "HND", backward: bool = False, out=None):
    """Turn queries and keys to their positions; returns ``(q, k)``, or q alone where `k` is None.

    q, k : packed ``(tokens, heads, head_dim)``, or 4-D in `tensor_layout`; float16 or bfloat16; strided views as in
        `sageattn`.  They differ in their heads at most.
    positions : int32 or int64 on the GPU, ``(tokens,)``, for 4-D tensors also ``(B, N)``; any value (angles are
        worked out in 64 bits).
    backward : the transposed map, which takes the gradient of the outputs to that of the inputs (for a magnitude
        of 1, the inverse).  Inputs that require gradients get them by it; a backward pass that is captured
        into a graph is warmed up on the capture stream, with no eager graph of the same leaves left alive.  Forward-mode
        derivatives are refused.
    out : optional output (for two inputs a pair), each its input itself or memory of its own; not differentiable.
    """
    _counters["calls"] += 1
    if tensor_layout not in ("HND", "NHD"):
        _refuse("tensor_layout must be 'HND' or 'NHD'")
    if _tangent(q) or (k is not None and _tangent(k)):
        _refuse("forward-mode derivatives are not carried", NotImplementedError)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        if out is not None:
            _refuse("out cannot be given for inputs that require gradients")
        return _Rotary.apply(q, k, positions, rotary, tensor_layout, bool(backward))
    res = _rotate(q, k, positions, rotary, tensor_layout, bool(backward), out)
    return res if k is not None else res[0]

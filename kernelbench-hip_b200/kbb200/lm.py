"""Language-model operators over the C ABI (include/kbb200.h): what decoding
needs beside the norms, products and softmax of `kbb200.ops`.

  qk_norm_rope, qk_norm_rope_backward   norms of queries and keys for each
                                        head with the position rotation
  cache_reserve, cache_append, cache_fork, cache_free, cache_compact,
  cache_copy                            a paged key/value cache
  shared_prefix_attention               attention over it, the pages that all
                                        sequences share read once
  penalize_logits                       repetition, presence and frequency
                                        penalties, biases, grammar masks

Tensors are fp32, fp16 or bf16 on one CUDA device.  Every function checks its
tensors, allocates outputs and scratch through torch's caching allocator and
launches on torch's current stream; it never waits for the GPU.  A C-ABI error
raises KbError.
"""
from __future__ import annotations

from functools import lru_cache

import torch

from ._lib import LIB, KbError
from .ops import _get_raw_stream, _ptr
from .ops import _stream as _stream_of

__all__ = ["qk_norm_rope", "qk_norm_rope_backward", "rope_tables", "shared_prefix_attention", "cache_reserve",
           "cache_append", "cache_fork", "cache_free", "cache_compact", "cache_copy", "penalize_logits"]

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_INTS = {torch.int32: 0, torch.int64: 1}
_POOLS = (torch.float32, torch.float16, torch.bfloat16, torch.uint8, torch.int8)

# Decoding makes these calls once per layer and token, so a call's time on the
# host counts: each function first asks one compact question that all right
# arguments answer with yes, and only on a no goes through the checks one by
# one, to say what is wrong.
_empty, _empty_like = torch.empty, torch.empty_like
_F32, _I32 = torch.float32, torch.int32


def _stream(dev: int, t: torch.Tensor) -> int:
    return _get_raw_stream(dev) if _get_raw_stream is not None else _stream_of(t)


def _like(x: torch.Tensor) -> torch.Tensor:
    """A new contiguous tensor of x's shape and type (empty_like costs half of empty; it keeps another order of
    memory than the contiguous one where x has one)."""
    y = _empty_like(x)
    return y if y.is_contiguous() else _empty(x.shape, device=x.device, dtype=x.dtype)


def _scratch(nbytes: int, like: torch.Tensor) -> torch.Tensor:
    """Workspace of nbytes, made of `like`'s 32-bit elements."""
    return like.new_empty((nbytes + 3) // 4 if nbytes > 16 else 4)


def check(fn: str, status: int) -> None:
    if status != 0:
        raise KbError(fn, status, LIB.kb_last_error().decode(errors="replace"))


def _is(t, dtype, dev, dims) -> bool:
    return isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == dev and t.dim() == dims


def _is_row(t, dtype, dev, n) -> bool:
    """A contiguous tensor [n]."""
    return (isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == dev and t.dim() == 1
            and t.shape[0] == n and t.is_contiguous())


@lru_cache(maxsize=4096)
def _attention_bytes(*sizes) -> int:
    return LIB.kb_shared_prefix_attention_workspace_size(*sizes)


@lru_cache(maxsize=4096)
def _rope_backward_bytes(*sizes) -> int:
    return LIB.kb_qk_norm_rope_backward_workspace_size(*sizes)


@lru_cache(maxsize=4096)
def _reserve_bytes(*sizes) -> int:
    return LIB.kb_cache_reserve_workspace_size(*sizes)


@lru_cache(maxsize=4096)
def _fork_bytes(*sizes) -> int:
    return LIB.kb_cache_fork_workspace_size(*sizes)


def _tensor(name: str, what: str, t, dev: torch.device | None, dtypes, dims: int | None = None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: {what} must be a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise RuntimeError(f"{name}: {what} must be on a CUDA device (got {t.device})")
    if dev is not None and t.device != dev:
        raise RuntimeError(f"{name}: tensors on different devices ({dev} vs {t.device})")
    if t.dtype not in dtypes:
        raise RuntimeError(f"{name}: {what} is {t.dtype}, expected one of {[str(d) for d in dtypes]}")
    if dims is not None and t.dim() != dims:
        raise RuntimeError(f"{name}: {what} must have {dims} dimensions, got {tuple(t.shape)}")
    return t


def _contiguous(name: str, what: str, t: torch.Tensor, shape=None) -> torch.Tensor:
    if not t.is_contiguous():
        raise RuntimeError(f"{name}: {what} must be contiguous")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise RuntimeError(f"{name}: {what} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t


def _vectors(name: str, what: str, t: torch.Tensor) -> torch.Tensor:
    """Head vectors are contiguous; the other strides are free."""
    if t.shape[-1] > 1 and t.stride(-1) != 1 and t.numel():
        raise RuntimeError(f"{name}: the last dimension of {what} must be contiguous")
    return t


def _out(name: str, t: torch.Tensor | None, like: torch.Tensor, shape, dtype=None) -> torch.Tensor:
    dtype = like.dtype if dtype is None else dtype
    if t is None:
        return _empty(shape, device=like.device, dtype=dtype)
    _tensor(name, "out", t, like.device, (dtype,))
    return _contiguous(name, "out", t, shape)


# ------------------------------------------------------------------ norms of queries and keys, rotation
def rope_tables(length: int, rotary: int, base: float = 10000.0, device="cuda"):
    """The cos and sin tables [length, rotary / 2] of angles p * base^(-2 i / rotary), computed in fp64 and
    rounded to fp32 once; a program makes them once and keeps them."""
    f = base ** (-torch.arange(0, rotary, 2, device=device, dtype=torch.float64) / max(rotary, 1))
    a = torch.arange(length, device=device, dtype=torch.float64)[:, None] * f
    return a.cos().float().contiguous(), a.sin().float().contiguous()


def _rope_args(name, q, k, q_weight, k_weight, cos, sin, positions):
    if isinstance(q, torch.Tensor) and q.dim() == 3 and q.is_cuda:
        T, hq, d = q.shape
        dt, dev = q.dtype, q.get_device()
        qs, ps = q.stride(), None
        if (_is(k, dt, dev, 3) and dt in _DTYPES and isinstance(positions, torch.Tensor)
                and (q_weight is None) == (k_weight is None) and T and hq and d > 1 and qs[2] == 1):
            ks, wt, ps = k.stride(), _F32 if q_weight is None else q_weight.dtype, positions.dtype
            n = k.shape
            if (n[0] == T and n[2] == d and n[1] and ks[2] == 1 and (wt is dt or wt is _F32)
                    and (q_weight is None or (_is_row(q_weight, wt, dev, d) and _is_row(k_weight, wt, dev, d)))
                    and _is(cos, _F32, dev, 2) and _is(sin, _F32, dev, 2) and cos.shape == sin.shape
                    and cos.is_contiguous() and sin.is_contiguous() and ps in _INTS and _is_row(positions, ps, dev, T)):
                rows, half = cos.shape
                return ((T, hq, n[1], d, 2 * half, rows, qs[0], qs[1], ks[0], ks[1]),
                        (_DTYPES[dt], _DTYPES[wt], _INTS[ps]), dev)
    _tensor(name, "q", q, None, _DTYPES, 3)
    dev, dt = q.device, q.dtype
    _tensor(name, "k", k, dev, (dt,), 3)
    T, hq, d = q.shape
    hkv = k.shape[1]
    if k.shape[0] != T or k.shape[2] != d:
        raise RuntimeError(f"{name}: q {tuple(q.shape)} and k {tuple(k.shape)} must be [tokens, heads, dim]")
    _vectors(name, "q", q)
    _vectors(name, "k", k)
    wt = None
    for what, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            continue
        _tensor(name, what, w, dev, (dt, torch.float32), 1)
        _contiguous(name, what, w, (d,))
        if wt is not None and w.dtype != wt:
            raise RuntimeError(f"{name}: weights of different types ({wt} and {w.dtype})")
        wt = w.dtype
    _tensor(name, "cos", cos, dev, (torch.float32,), 2)
    _tensor(name, "sin", sin, dev, (torch.float32,), 2)
    _contiguous(name, "cos", cos)
    _contiguous(name, "sin", sin, cos.shape)
    _tensor(name, "positions", positions, dev, _INTS, 1)
    _contiguous(name, "positions", positions, (T,))
    shape = (T, hq, hkv, d, 2 * cos.shape[1], cos.shape[0], q.stride(0), q.stride(1), k.stride(0), k.stride(1))
    kinds = (_DTYPES[dt], _DTYPES[wt if wt is not None else torch.float32], _INTS[positions.dtype])
    return shape, kinds, q.get_device()


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps: float = 1e-6, interleaved: bool = False,
                 q_out=None, k_out=None):
    """RMS norm of every head vector of q [tokens, heads_q, dim] and k [tokens, heads_kv, dim], times the
    weights [dim] (None: ones), then the rotation of the first 2 * cos.shape[1] elements by row positions[t] of
    cos and sin (`rope_tables`): pairs (i, i + rotary / 2), or (2 i, 2 i + 1) with `interleaved`.

    q and k may be views of one packed projection.  Weights are fp32 or of q's type, positions int64 or int32; a
    position outside the tables gives NaN in the rotated elements.  Returns new (or the given, contiguous) q
    and k."""
    fn = "kb_qk_norm_rope"
    shape, kinds, dev = _rope_args(fn, q, k, q_weight, k_weight, cos, sin, positions)
    qo = _like(q) if q_out is None else _out(fn, q_out, q, q.shape)
    ko = _like(k) if k_out is None else _out(fn, k_out, k, k.shape)
    check(fn, LIB.kb_qk_norm_rope(q.data_ptr(), k.data_ptr(), _ptr(q_weight), _ptr(k_weight), cos.data_ptr(),
                                  sin.data_ptr(), positions.data_ptr(), qo.data_ptr(), ko.data_ptr(), *shape,
                                  *kinds, 1 if interleaved else 0, eps, _stream(dev, q)))
    return qo, ko


def qk_norm_rope_backward(dq_out, dk_out, q, k, q_weight, k_weight, cos, sin, positions, eps: float = 1e-6,
                          interleaved: bool = False):
    """The gradients (dq, dk, dq_weight, dk_weight) of qk_norm_rope at its inputs, from those of its outputs
    (contiguous).  A weight that is None has None.  Weight gradients have the weights' type; they are summed in
    fp64 in a fixed order."""
    fn = "kb_qk_norm_rope_backward"
    shape, kinds, dev = _rope_args(fn, q, k, q_weight, k_weight, cos, sin, positions)
    dt = q.dtype
    for what, g, x in (("dq_out", dq_out, q), ("dk_out", dk_out, k)):
        if not (_is(g, dt, dev, 3) and g.shape == x.shape and g.is_contiguous()):
            _tensor(fn, what, g, q.device, (dt,))
            _contiguous(fn, what, g, x.shape)
    dq, dk = torch.empty_like(dq_out), torch.empty_like(dk_out)
    dqw = None if q_weight is None else torch.empty_like(q_weight)
    dkw = None if k_weight is None else torch.empty_like(k_weight)
    need = _rope_backward_bytes(shape[0], shape[1], shape[2], shape[3])
    ws = _scratch(need, cos)
    check(fn, LIB.kb_qk_norm_rope_backward(dq_out.data_ptr(), dk_out.data_ptr(), q.data_ptr(), k.data_ptr(),
                                           _ptr(q_weight), _ptr(k_weight), cos.data_ptr(), sin.data_ptr(),
                                           positions.data_ptr(), dq.data_ptr(), dk.data_ptr(), _ptr(dqw), _ptr(dkw),
                                           *shape, *kinds, 1 if interleaved else 0, eps, ws.data_ptr(),
                                           need, _stream(dev, q)))
    return dq, dk, dqw, dkw


# ------------------------------------------------------------------ attention over the cache
def shared_prefix_attention(q, k_pages, v_pages, prefix, table, lens, scale: float | None = None, out=None):
    """Attention of the newest tokens of a batch, q [batch, queries, heads_q, dim], over the paged cache
    k_pages, v_pages [pages, page_size, heads_kv, dim], whose pages prefix [n] int32 (the full pages of the
    prompt that all sequences share) hold the first keys of every sequence.

    table [batch, width] int32 holds each sequence's pages from its first key on, as cache_fork leaves it; its
    first n columns are not read.  lens [batch] int32 counts a sequence's keys, those of the queries included:
    query t sees the keys below lens - queries + t + 1.  scale: dim ** -0.5 unless given.

    Returns (out, lse): out like q, contiguous, and lse [batch, queries, heads_q] fp32, the logarithm of the sum
    of the exponentials; a query without keys (a slot whose lens is 0) gets zeros and -inf."""
    fn = "kb_shared_prefix_attention"
    sizes = _attention_sizes(q, k_pages, v_pages, prefix, table, lens)
    if sizes is None:
        sizes = _attention_checks(fn, q, k_pages, v_pages, prefix, table, lens)
    B, Q, hq, hkv, d, n_pre, width, pages, page_size, qs, ks, vs = sizes
    code = _DTYPES[q.dtype]
    o = _like(q) if out is None else _out(fn, out, q, q.shape)
    lse = q.new_empty((B, Q, hq), dtype=_F32)
    need = _attention_bytes(B, Q, hq, hkv, d, n_pre, width, page_size, code)
    ws = _scratch(need, lens) if need else None
    check(fn, LIB.kb_shared_prefix_attention(
        q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), prefix.data_ptr(), table.data_ptr(), lens.data_ptr(),
        o.data_ptr(), lse.data_ptr(), B, Q, hq, hkv, d, n_pre, width, pages, page_size, qs[0], qs[1], qs[2],
        ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], d ** -0.5 if scale is None else scale, code,
        _ptr(ws), need, _stream(q.get_device(), q)))
    return o, lse


def _attention_sizes(q, k_pages, v_pages, prefix, table, lens):
    """The sizes of right arguments, else None."""
    if not (isinstance(q, torch.Tensor) and q.dim() == 4 and q.is_cuda):
        return None
    dt, dev = q.dtype, q.get_device()
    if not (dt in _DTYPES and _is(k_pages, dt, dev, 4) and _is(v_pages, dt, dev, 4) and _is(table, _I32, dev, 2)
            and _is(prefix, _I32, dev, 1)):
        return None
    B, Q, hq, d = q.shape
    n = k_pages.shape
    pages, page_size, hkv, dk = n
    qs, ks, vs = q.stride(), k_pages.stride(), v_pages.stride()
    rows, width = table.shape
    if (dk != d or d < 2 or n != v_pages.shape or qs[3] != 1 or ks[3] != 1 or vs[3] != 1 or rows != B
            or not prefix.is_contiguous() or not table.is_contiguous() or not _is_row(lens, _I32, dev, B)):
        return None
    return B, Q, hq, hkv, d, prefix.shape[0], width, pages, page_size, qs, ks, vs


def _attention_checks(fn, q, k_pages, v_pages, prefix, table, lens):
    _tensor(fn, "q", q, None, _DTYPES, 4)
    dev, dt = q.device, q.dtype
    _tensor(fn, "k_pages", k_pages, dev, (dt,), 4)
    _tensor(fn, "v_pages", v_pages, dev, (dt,), 4)
    B, Q, hq, d = q.shape
    pages, page_size, hkv, dk = k_pages.shape
    if v_pages.shape != k_pages.shape or dk != d:
        raise RuntimeError(f"{fn}: k_pages {tuple(k_pages.shape)} and v_pages {tuple(v_pages.shape)} must both be "
                           f"[pages, page_size, heads, {d}]")
    for what, t in (("q", q), ("k_pages", k_pages), ("v_pages", v_pages)):
        _vectors(fn, what, t)
    _tensor(fn, "prefix", prefix, dev, (torch.int32,), 1)
    _contiguous(fn, "prefix", prefix)
    _tensor(fn, "table", table, dev, (torch.int32,), 2)
    _contiguous(fn, "table", table)
    _tensor(fn, "lens", lens, dev, (torch.int32,), 1)
    _contiguous(fn, "lens", lens, (B,))
    if table.shape[0] != B:
        raise RuntimeError(f"{fn}: table has {table.shape[0]} rows for {B} sequences")
    return (B, Q, hq, hkv, d, prefix.shape[0], table.shape[1], pages, page_size, q.stride(), k_pages.stride(),
            v_pages.stride())


# ------------------------------------------------------------------ the paged cache
def _state(fn, table, lens, refs):
    if isinstance(table, torch.Tensor) and table.is_cuda and table.dtype is _I32 and table.dim() == 2 and table.is_contiguous():
        dev = table.get_device()
        if ((lens is None or _is_row(lens, _I32, dev, table.shape[0]))
                and (refs is None or (_is(refs, _I32, dev, 1) and refs.is_contiguous()))):
            return table.device
    _tensor(fn, "table", table, None, (torch.int32,), 2)
    dev = table.device
    _contiguous(fn, "table", table)
    if lens is not None:
        _tensor(fn, "lens", lens, dev, (torch.int32,), 1)
        _contiguous(fn, "lens", lens, (table.shape[0],))
    if refs is not None:
        _tensor(fn, "refs", refs, dev, (torch.int32,), 1)
        _contiguous(fn, "refs", refs)
    return dev


def _slots(fn, what, t, dev, n=None):
    if (isinstance(t, torch.Tensor) and t.dtype is _I32 and t.device == dev and t.dim() == 1 and t.is_contiguous()
            and (n is None or t.shape[0] == n)):
        return t
    _tensor(fn, what, t, dev, (torch.int32,), 1)
    return _contiguous(fn, what, t, None if n is None else (n,))


def _pool(fn, what, pool, dev, pages=None):
    if not (isinstance(pool, torch.Tensor) and pool.dtype in _POOLS and pool.device == dev and pool.is_contiguous()):
        _tensor(fn, what, pool, dev, _POOLS)
        _contiguous(fn, what, pool)
    if pool.dim() < 3:
        raise RuntimeError(f"{fn}: {what} must be [planes, pages, page_size, ...], got {tuple(pool.shape)}")
    if pages is not None and pool.shape[1] != pages:
        raise RuntimeError(f"{fn}: {what} has {pool.shape[1]} pages, refs {pages}")
    return pool.stride(1) * pool.element_size() if pool.numel() else 0


def cache_reserve(table, lens, refs, seqs, tokens: int, page_size: int):
    """Grows the slots seqs [n] int32 by `tokens` keys each: lens += tokens, with the free pages that takes
    (lowest first, in the order of seqs).  table [slots, width], lens [slots] and refs [pages] are int32 and
    changed in place.  Returns granted [n] int32: 0 for a request that got nothing (the row or the pool is
    full, or the slot is out of range or listed again)."""
    fn = "kb_cache_reserve"
    dev = _state(fn, table, lens, refs)
    n = _slots(fn, "seqs", seqs, dev).shape[0]
    granted = _empty_like(seqs)
    sizes = (table.shape[0], table.shape[1], refs.shape[0], int(page_size))
    need = _reserve_bytes(n, int(tokens), *sizes)
    ws = _scratch(need, refs)
    check(fn, LIB.kb_cache_reserve(table.data_ptr(), lens.data_ptr(), refs.data_ptr(), seqs.data_ptr(),
                                   granted.data_ptr(), n, int(tokens), *sizes, ws.data_ptr(), need,
                                   _stream(table.get_device(), table)))
    return granted


def cache_append(k, v, k_pages, v_pages, table, lens, seqs) -> None:
    """Writes k, v [n, tokens, heads, dim] into the last `tokens` places of the slots seqs [n] int32 (which
    cache_reserve has made), in one layer's planes k_pages, v_pages [pages, page_size, heads, dim]."""
    fn = "kb_cache_append"
    dev = _state(fn, table, lens, None)
    n = _slots(fn, "seqs", seqs, dev).shape[0]
    ks = _append_strides(k, v, k_pages, v_pages, dev, n)
    if ks is None:
        _append_checks(fn, k, v, k_pages, v_pages, dev, n)
        ks = k.stride(), v.stride()
    (ksn, kst, *_), (vsn, vst, *_) = ks
    pages, page_size, h, d = k_pages.shape
    e = k_pages.element_size()
    check(fn, LIB.kb_cache_append(k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                                  table.data_ptr(), lens.data_ptr(), seqs.data_ptr(), n, k.shape[1], table.shape[0],
                                  table.shape[1], pages, page_size, page_size * h * d * e, h * d * e,
                                  ksn * e, kst * e, vsn * e, vst * e,
                                  _stream(table.get_device(), table)))


def _append_strides(k, v, k_pages, v_pages, dev, n):
    """The strides of right arguments, else None."""
    if not (isinstance(k_pages, torch.Tensor) and k_pages.dim() == 4 and k_pages.device == dev):
        return None
    dt, i = k_pages.dtype, k_pages.get_device()
    if not (dt in _DTYPES and _is(v_pages, dt, i, 4) and _is(k, dt, i, 4) and _is(v, dt, i, 4)
            and k_pages.is_contiguous() and v_pages.is_contiguous()):
        return None
    size, kv, ks, vs = k_pages.shape, k.shape, k.stride(), v.stride()
    d = size[3]
    if (v_pages.shape != size or v.shape != kv or kv[0] != n or kv[2] != size[2] or kv[3] != d
            or ks[2:] != (d, 1) or vs[2:] != (d, 1)):
        return None
    return ks, vs


def _append_checks(fn, k, v, k_pages, v_pages, dev, n):
    _tensor(fn, "k_pages", k_pages, dev, _DTYPES, 4)
    dt = (k_pages.dtype,)
    _tensor(fn, "v_pages", v_pages, dev, dt, 4)
    _contiguous(fn, "k_pages", k_pages)
    _contiguous(fn, "v_pages", v_pages, k_pages.shape)
    pages, page_size, h, d = k_pages.shape
    for what, t in (("k", k), ("v", v)):
        _tensor(fn, what, t, dev, dt, 4)
        if t.shape[0] != n or t.shape[2:] != k_pages.shape[2:] or t.shape[1] != k.shape[1]:
            raise RuntimeError(f"{fn}: {what} has shape {tuple(t.shape)}, expected ({n}, {k.shape[1]}, {h}, {d})")
        if t.numel() and ((d > 1 and t.stride(3) != 1) or (h > 1 and t.stride(2) != d)):
            raise RuntimeError(f"{fn}: the heads of a token of {what} must be contiguous")


def cache_fork(pool, table, lens, refs, parents, children):
    """Makes the slots children [n] int32 copies of the slots parents [n] int32, whatever they held: full pages
    are shared (refs + 1), a last page that is not full is copied to a free one in every plane of pool
    [planes, pages, page_size, ...].  All parents are read before any child is replaced (a beam may be
    permuted), and pages are taken before those of replaced children are given back.  Returns granted [n] int32
    as cache_reserve does."""
    fn = "kb_cache_fork"
    dev = _state(fn, table, lens, refs)
    page_bytes = _pool(fn, "pool", pool, dev, refs.shape[0])
    n = _slots(fn, "parents", parents, dev).shape[0]
    _slots(fn, "children", children, dev, n)
    granted = _empty_like(parents)
    slots, width = table.shape
    need = _fork_bytes(n, slots, width)
    ws = _scratch(need, refs)
    check(fn, LIB.kb_cache_fork(pool.data_ptr(), table.data_ptr(), lens.data_ptr(), refs.data_ptr(),
                                parents.data_ptr(), children.data_ptr(), granted.data_ptr(), n, slots, width,
                                *pool.shape[:3], page_bytes, ws.data_ptr(), need,
                                _stream(table.get_device(), table)))
    return granted


def cache_free(table, lens, refs, seqs) -> None:
    """Empties the slots seqs [n] int32: their pages are given back, lens = 0, rows = -1."""
    fn = "kb_cache_free"
    dev = _state(fn, table, lens, refs)
    n = _slots(fn, "seqs", seqs, dev).shape[0]
    check(fn, LIB.kb_cache_free(table.data_ptr(), lens.data_ptr(), refs.data_ptr(), seqs.data_ptr(), n,
                                table.shape[0], table.shape[1], refs.shape[0], _stream(table.get_device(), table)))


def cache_compact(pool, table, refs):
    """Moves the live pages to the low end of pool [planes, pages, ...]: with n live pages, the i-th live page at
    or above n goes to the i-th free one below; table and refs follow.  Returns n as an int32 tensor [1]."""
    fn = "kb_cache_compact"
    dev = _state(fn, table, None, refs)
    page_bytes = _pool(fn, "pool", pool, dev, refs.shape[0])
    live = refs.new_empty(1)
    need = LIB.kb_cache_compact_workspace_size(refs.shape[0])
    ws = _scratch(need, refs)
    check(fn, LIB.kb_cache_compact(pool.data_ptr(), table.data_ptr(), refs.data_ptr(), live.data_ptr(),
                                   table.shape[0], table.shape[1], pool.shape[0], pool.shape[1], page_bytes,
                                   ws.data_ptr(), need, _stream(table.get_device(), table)))
    return live


def cache_copy(src_pool, src, dst_pool, dst) -> None:
    """Copies pages src [n] int32 of src_pool to pages dst [n] int32 of dst_pool, in every plane: into another
    pool, or within one.  The dst are distinct and, in one pool, none is also a src.  Ids out of range are passed
    over."""
    fn = "kb_cache_copy"
    _tensor(fn, "src_pool", src_pool, None, _POOLS)
    dev = src_pool.device
    page_bytes = _pool(fn, "src_pool", src_pool, dev)
    if _pool(fn, "dst_pool", dst_pool, dev) != page_bytes or dst_pool.shape[0] != src_pool.shape[0]:
        raise RuntimeError(f"{fn}: pools {tuple(src_pool.shape)} and {tuple(dst_pool.shape)} differ in planes or pages")
    n = _slots(fn, "src", src, dev).shape[0]
    _slots(fn, "dst", dst, dev, n)
    check(fn, LIB.kb_cache_copy(src_pool.data_ptr(), src.data_ptr(), dst_pool.data_ptr(), dst.data_ptr(), n,
                                src_pool.shape[0], page_bytes, src_pool.shape[1], dst_pool.shape[1],
                                _stream(src_pool.get_device(), src_pool)))


# ------------------------------------------------------------------ logits
def penalize_logits(logits, prompt=None, output=None, repetition=None, presence=None, frequency=None, bias_ids=None,
                    bias_values=None, mask=None, out=None):
    """Penalties for repeated tokens, biases and a grammar's mask on logits [rows, vocab], in this order:

      seen in `prompt` or `output`:  l / repetition if l > 0 else l * repetition
      c times in `output`:           l - frequency * c - presence
      listed in bias_ids:            l + bias_values (an id listed twice: the last)
      mask bit clear:                -inf

    prompt, output, bias_ids: [rows, n] int64 or int32 (one type), ids outside the vocabulary (padding) ignored;
    repetition, presence, frequency: [rows] fp32; bias_values [rows, n] fp32; mask: int32 words
    [rows or 1, ceil(vocab / 32)], token v at bit v % 32 of word v // 32.  All may be None.  `out` may be logits
    itself (contiguous)."""
    fn = "kb_penalize_logits"
    if not (isinstance(logits, torch.Tensor) and logits.is_cuda and logits.dtype in _DTYPES and logits.dim() == 2
            and logits.stride(1) == 1):
        _tensor(fn, "logits", logits, None, _DTYPES, 2)
        _vectors(fn, "logits", logits)
    dev, index = logits.device, logits.get_device()
    B, V = logits.shape
    ids = None
    lengths = []
    for what, t in (("prompt", prompt), ("output", output), ("bias_ids", bias_ids)):
        if t is None:
            lengths.append(0)
            continue
        if not (_is(t, ids if ids is not None else torch.int64, index, 2) and t.is_contiguous() and t.shape[0] == B):
            _tensor(fn, what, t, dev, _INTS if ids is None else (ids,), 2)
            _contiguous(fn, what, t, (B, t.shape[1]))
        ids = t.dtype
        lengths.append(t.shape[1])
    for what, t in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
        if t is not None and not _is_row(t, _F32, index, B):
            _tensor(fn, what, t, dev, (torch.float32,), 1)
            _contiguous(fn, what, t, (B,))
    if (bias_ids is None) != (bias_values is None):
        raise RuntimeError(f"{fn}: bias_ids and bias_values go together")
    if bias_values is not None and not (_is(bias_values, _F32, index, 2) and bias_values.is_contiguous()
                                        and bias_values.shape == bias_ids.shape):
        _tensor(fn, "bias_values", bias_values, dev, (torch.float32,), 2)
        _contiguous(fn, "bias_values", bias_values, bias_ids.shape)
    mask_stride = 0
    if mask is not None:
        _tensor(fn, "mask", mask, dev, (torch.int32,), 2)
        words = -(-V // 32)
        if tuple(mask.shape) not in ((B, words), (1, words)):
            raise RuntimeError(f"{fn}: mask has shape {tuple(mask.shape)}, expected ({B} or 1, {words})")
        _contiguous(fn, "mask", mask)
        mask_stride = words if mask.shape[0] == B else 0
    y = _like(logits) if out is None else _out(fn, out, logits, logits.shape)
    check(fn, LIB.kb_penalize_logits(logits.data_ptr(), y.data_ptr(), _ptr(prompt), _ptr(output), _ptr(repetition),
                                     _ptr(presence), _ptr(frequency), _ptr(bias_ids), _ptr(bias_values), _ptr(mask),
                                     B, V, logits.stride(0), *lengths, mask_stride, _DTYPES[logits.dtype],
                                     1 if ids is torch.int64 else 0, _stream(index, logits)))
    return y

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
raises KbError.  Outputs take no part in autograd, whatever the inputs require.

Decoding makes these calls once per layer and token, so the way of right
arguments is native (csrc/lm_host.cpp): it checks them, allocates and calls the
C ABI (whose errors it raises), and answers None where anything is not plainly
right.  Then the checks here run one by one and say what is wrong, or the call
is made from here.
"""
from __future__ import annotations

import ctypes

import torch

from ._lib import LIB, SIGNATURES, check
from .ops import _ptr, _stream, _workspace

try:
    from . import _lm_host as _host
except ImportError as e:
    raise ImportError("kbb200/_lm_host.so is missing or was built for another torch: build it with "
                      "`python kernelbench-hip_b200/build.py`") from e

_ENTRIES = {name: ctypes.cast(getattr(LIB, name), ctypes.c_void_p).value for name in SIGNATURES}
_host.init({**_ENTRIES, "check": check})

__all__ = ["qk_norm_rope", "qk_norm_rope_backward", "rope_tables", "shared_prefix_attention", "cache_reserve",
           "cache_append", "cache_fork", "cache_free", "cache_compact", "cache_copy", "penalize_logits"]

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_INTS = {torch.int32: 0, torch.int64: 1}
_POOLS = (torch.float32, torch.float16, torch.bfloat16, torch.uint8, torch.int8)

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
        return torch.empty(shape, device=like.device, dtype=dtype)
    _tensor(name, "out", t, like.device, (dtype,))
    return _contiguous(name, "out", t, shape)


# ------------------------------------------------------------------ norms of queries and keys, rotation
def rope_tables(length: int, rotary: int, base: float = 10000.0, device="cuda"):
    """The cos and sin tables [length, rotary / 2] of angles p * base^(-2 i / rotary), computed in fp64 and
    rounded to fp32 once; a program makes them once and keeps them."""
    if rotary < 0 or rotary % 2:
        raise RuntimeError(f"rope_tables: rotary must be even (whole pairs), got {rotary}")
    f = base ** (-torch.arange(0, rotary, 2, device=device, dtype=torch.float64) / max(rotary, 1))
    a = torch.arange(length, device=device, dtype=torch.float64)[:, None] * f
    return a.cos().float().contiguous(), a.sin().float().contiguous()


def _rope_args(name, q, k, q_weight, k_weight, cos, sin, positions):
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
    return shape, kinds


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps: float = 1e-6, interleaved: bool = False,
                 q_out=None, k_out=None):
    """RMS norm of every head vector of q [tokens, heads_q, dim] and k [tokens, heads_kv, dim], times the
    weights [dim] (None: ones), then the rotation of the first 2 * cos.shape[1] elements by row positions[t] of
    cos and sin (`rope_tables`): pairs (i, i + rotary / 2), or (2 i, 2 i + 1) with `interleaved`.

    q and k may be views of one packed projection.  Weights are fp32 or of q's type, positions int64 or int32; a
    position outside the tables gives NaN in the rotated elements.  Returns new (or the given, contiguous) q
    and k."""
    fn = "kb_qk_norm_rope"
    if q_out is None and k_out is None:
        out = _host.rope(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
        if out is not None:
            return out
    shape, kinds = _rope_args(fn, q, k, q_weight, k_weight, cos, sin, positions)
    qo, ko = _out(fn, q_out, q, q.shape), _out(fn, k_out, k, k.shape)
    check(fn, LIB.kb_qk_norm_rope(q.data_ptr(), k.data_ptr(), _ptr(q_weight), _ptr(k_weight), cos.data_ptr(),
                                  sin.data_ptr(), positions.data_ptr(), qo.data_ptr(), ko.data_ptr(), *shape,
                                  *kinds, 1 if interleaved else 0, float(eps), _stream(q)))
    return qo, ko


def qk_norm_rope_backward(dq_out, dk_out, q, k, q_weight, k_weight, cos, sin, positions, eps: float = 1e-6,
                          interleaved: bool = False):
    """The gradients (dq, dk, dq_weight, dk_weight) of qk_norm_rope at its inputs, from those of its outputs
    (contiguous).  A weight that is None has None.  Weight gradients have the weights' type; they are summed in
    fp64 in a fixed order."""
    fn = "kb_qk_norm_rope_backward"
    out = _host.rope_backward(dq_out, dk_out, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
    if out is not None:
        return out
    shape, kinds = _rope_args(fn, q, k, q_weight, k_weight, cos, sin, positions)
    for what, g, x in (("dq_out", dq_out, q), ("dk_out", dk_out, k)):
        _tensor(fn, what, g, q.device, (q.dtype,))
        _contiguous(fn, what, g, x.shape)
    dq, dk = torch.empty_like(dq_out), torch.empty_like(dk_out)
    dqw = None if q_weight is None else torch.empty_like(q_weight)
    dkw = None if k_weight is None else torch.empty_like(k_weight)
    ws = _workspace(q, LIB.kb_qk_norm_rope_backward_workspace_size(*shape[:4]))
    check(fn, LIB.kb_qk_norm_rope_backward(dq_out.data_ptr(), dk_out.data_ptr(), q.data_ptr(), k.data_ptr(),
                                           _ptr(q_weight), _ptr(k_weight), cos.data_ptr(), sin.data_ptr(),
                                           positions.data_ptr(), dq.data_ptr(), dk.data_ptr(), _ptr(dqw), _ptr(dkw),
                                           *shape, *kinds, 1 if interleaved else 0, float(eps), ws.data_ptr(),
                                           ws.numel(), _stream(q)))
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
    of the exponentials; a query without keys (a slot whose lens is 0) gets zeros and -inf.  What stands in slots that
    no query sees does not matter, and infinite or NaN keys and values reach the queries that see them only."""
    fn = "kb_shared_prefix_attention"
    if out is None:
        made = _host.attention(q, k_pages, v_pages, prefix, table, lens, scale)
        if made is not None:
            return made
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
    n_pre, width, code = prefix.shape[0], table.shape[1], _DTYPES[dt]
    o = _out(fn, out, q, q.shape)
    lse = torch.empty((B, Q, hq), device=dev, dtype=torch.float32)
    ws = _workspace(q, LIB.kb_shared_prefix_attention_workspace_size(B, Q, hq, hkv, d, n_pre, width, page_size, code))
    check(fn, LIB.kb_shared_prefix_attention(
        q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), prefix.data_ptr(), table.data_ptr(), lens.data_ptr(),
        o.data_ptr(), lse.data_ptr(), B, Q, hq, hkv, d, n_pre, width, pages, page_size, *q.stride()[:3],
        *k_pages.stride()[:3], *v_pages.stride()[:3], float(d ** -0.5 if scale is None else scale), code,
        ws.data_ptr(), ws.numel(), _stream(q)))
    return o, lse


# ------------------------------------------------------------------ the paged cache
def _state(fn, table, lens, refs):
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
    _tensor(fn, what, t, dev, (torch.int32,), 1)
    return _contiguous(fn, what, t, None if n is None else (n,))


def _pool(fn, what, pool, dev, pages=None):
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
    full, or the slot is out of range or listed again).

    To drop a slot's newest keys (drafts that were rejected), lower its lens, though not into pages that other slots
    share: the pages past it stay in its row, where its next reserve uses them first."""
    fn = "kb_cache_reserve"
    granted = _host.reserve(table, lens, refs, seqs, tokens, page_size)
    if granted is not None:
        return granted
    dev = _state(fn, table, lens, refs)
    n = _slots(fn, "seqs", seqs, dev).shape[0]
    granted = torch.empty_like(seqs)
    sizes = (table.shape[0], table.shape[1], refs.shape[0], int(page_size))
    ws = _workspace(table, LIB.kb_cache_reserve_workspace_size(n, int(tokens), *sizes))
    check(fn, LIB.kb_cache_reserve(table.data_ptr(), lens.data_ptr(), refs.data_ptr(), seqs.data_ptr(),
                                   granted.data_ptr(), n, int(tokens), *sizes, ws.data_ptr(), ws.numel(),
                                   _stream(table)))
    return granted


def cache_append(k, v, k_pages, v_pages, table, lens, seqs, granted=None) -> None:
    """Writes k, v [n, tokens, heads, dim] into the last `tokens` places of the slots seqs [n] int32 (which
    cache_reserve has made), in one layer's planes k_pages, v_pages [pages, page_size, heads, dim].

    granted [n] int32 is what that cache_reserve returned.  A slot that it refused has not grown: its last places
    hold older keys, which other slots may share, and it is passed over.  Without granted all of seqs are written."""
    fn = "kb_cache_append"
    if _host.append(k, v, k_pages, v_pages, table, lens, seqs, granted):
        return
    dev = _state(fn, table, lens, None)
    n = _slots(fn, "seqs", seqs, dev).shape[0]
    if granted is not None:
        _slots(fn, "granted", granted, dev, n)
    _tensor(fn, "k_pages", k_pages, dev, _DTYPES, 4)
    dt = (k_pages.dtype,)
    _tensor(fn, "v_pages", v_pages, dev, dt, 4)
    _contiguous(fn, "k_pages", k_pages)
    _contiguous(fn, "v_pages", v_pages, k_pages.shape)
    pages, page_size, h, d = k_pages.shape
    e = k_pages.element_size()
    for what, t in (("k", k), ("v", v)):
        _tensor(fn, what, t, dev, dt, 4)
        if t.shape[0] != n or t.shape[2:] != k_pages.shape[2:] or t.shape[1] != k.shape[1]:
            raise RuntimeError(f"{fn}: {what} has shape {tuple(t.shape)}, expected ({n}, {k.shape[1]}, {h}, {d})")
        if t.numel() and ((d > 1 and t.stride(3) != 1) or (h > 1 and t.stride(2) != d)):
            raise RuntimeError(f"{fn}: the heads of a token of {what} must be contiguous")
    check(fn, LIB.kb_cache_append_granted(k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                                          table.data_ptr(), lens.data_ptr(), seqs.data_ptr(), _ptr(granted), n,
                                          k.shape[1], table.shape[0], table.shape[1], pages, page_size,
                                          page_size * h * d * e, h * d * e, k.stride(0) * e, k.stride(1) * e,
                                          v.stride(0) * e, v.stride(1) * e, _stream(table)))


def cache_fork(pool, table, lens, refs, parents, children):
    """Makes the slots children [n] int32 copies of the slots parents [n] int32, whatever they held: full pages
    are shared (refs + 1), a last page that is not full is copied to a free one in every plane of pool
    [planes, pages, page_size, ...].  All parents are read before any child is replaced (a beam may be
    permuted), and pages are taken before those of replaced children are given back.  Returns granted [n] int32
    as cache_reserve does."""
    fn = "kb_cache_fork"
    granted = _host.fork(pool, table, lens, refs, parents, children)
    if granted is not None:
        return granted
    dev = _state(fn, table, lens, refs)
    page_bytes = _pool(fn, "pool", pool, dev, refs.shape[0])
    n = _slots(fn, "parents", parents, dev).shape[0]
    _slots(fn, "children", children, dev, n)
    granted = torch.empty_like(parents)
    slots, width = table.shape
    ws = _workspace(table, LIB.kb_cache_fork_workspace_size(n, slots, width))
    check(fn, LIB.kb_cache_fork(pool.data_ptr(), table.data_ptr(), lens.data_ptr(), refs.data_ptr(),
                                parents.data_ptr(), children.data_ptr(), granted.data_ptr(), n, slots, width,
                                *pool.shape[:3], page_bytes, ws.data_ptr(), ws.numel(),
                                _stream(table)))
    return granted


def cache_free(table, lens, refs, seqs) -> None:
    """Empties the slots seqs [n] int32: their pages are given back, lens = 0, rows = -1."""
    fn = "kb_cache_free"
    if _host.release(table, lens, refs, seqs):
        return
    dev = _state(fn, table, lens, refs)
    n = _slots(fn, "seqs", seqs, dev).shape[0]
    check(fn, LIB.kb_cache_free(table.data_ptr(), lens.data_ptr(), refs.data_ptr(), seqs.data_ptr(), n,
                                table.shape[0], table.shape[1], refs.shape[0], _stream(table)))


def cache_compact(pool, table, refs):
    """Moves the live pages to the low end of pool [planes, pages, ...]: with n live pages, the i-th live page at
    or above n goes to the i-th free one below; table and refs follow.  Returns n as an int32 tensor [1]."""
    fn = "kb_cache_compact"
    live = _host.compact(pool, table, refs)
    if live is not None:
        return live
    dev = _state(fn, table, None, refs)
    page_bytes = _pool(fn, "pool", pool, dev, refs.shape[0])
    live = torch.empty(1, device=dev, dtype=torch.int32)
    ws = _workspace(table, LIB.kb_cache_compact_workspace_size(refs.shape[0]))
    check(fn, LIB.kb_cache_compact(pool.data_ptr(), table.data_ptr(), refs.data_ptr(), live.data_ptr(),
                                   table.shape[0], table.shape[1], pool.shape[0], pool.shape[1], page_bytes,
                                   ws.data_ptr(), ws.numel(), _stream(table)))
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
                                _stream(src_pool)))


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
    if out is None:
        made = _host.logits(logits, prompt, output, repetition, presence, frequency, bias_ids, bias_values, mask)
        if made is not None:
            return made
    _tensor(fn, "logits", logits, None, _DTYPES, 2)
    _vectors(fn, "logits", logits)
    dev = logits.device
    B, V = logits.shape
    ids = None
    lengths = []
    for what, t in (("prompt", prompt), ("output", output), ("bias_ids", bias_ids)):
        if t is None:
            lengths.append(0)
            continue
        _tensor(fn, what, t, dev, _INTS if ids is None else (ids,), 2)
        ids = t.dtype
        _contiguous(fn, what, t, (B, t.shape[1]))
        lengths.append(t.shape[1])
    for what, t in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
        if t is not None:
            _tensor(fn, what, t, dev, (torch.float32,), 1)
            _contiguous(fn, what, t, (B,))
    if (bias_ids is None) != (bias_values is None):
        raise RuntimeError(f"{fn}: bias_ids and bias_values go together")
    if bias_values is not None:
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
    y = _out(fn, out, logits, logits.shape)
    check(fn, LIB.kb_penalize_logits(logits.data_ptr(), y.data_ptr(), _ptr(prompt), _ptr(output), _ptr(repetition),
                                     _ptr(presence), _ptr(frequency), _ptr(bias_ids), _ptr(bias_values), _ptr(mask),
                                     B, V, logits.stride(0), *lengths, mask_stride, _DTYPES[logits.dtype],
                                     1 if ids is torch.int64 else 0, _stream(logits)))
    return y

"""GPU: the language-model operators (kbb200.lm) against the 64-bit oracle.

Tolerances, from the formats alone: u is the unit roundoff of the output's
type (2^-24 fp32, 2^-11 fp16, 2^-8 bf16: 24, 11 and 8 bits) and U = 2^-24 that of the
fp32 arithmetic.
  norms and rotation   a sum of at most 512 squares over 32 lanes, rsqrt and
                       five products: 32 U of the pair's magnitude, + u
  weight gradients     each term 16 U of its magnitude (summed in fp64), + u
  attention            scores are off by at most e = (dim + 16) U scale sum
                       |q k|, so weights by 2 e + 2^-21 (ex2, joins); 16-bit
                       values meet weights rounded to u: all of softmax @ |v|
  logits               six operations: 8 U of the magnitudes met, + u
Page operations move bits and whole numbers: equal.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import lm as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}  # below normal numbers
TYPES = list(UNIT)


def f64(t):
    return t.detach().double().cpu().numpy()


def within(got, want, tol, what=""):
    got = f64(got) if isinstance(got, torch.Tensor) else got
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN in other places"
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), f"{what}: infinities differ"
    err, tol = np.abs(got - np.where(fine, want, 0))[fine], np.broadcast_to(tol, want.shape)[fine]
    assert (err <= tol).all(), f"{what}: {err.max():.3e} off, {(err / np.maximum(tol, 1e-300)).max():.2f} of the tolerance"


# ------------------------------------------------------------ norms of queries and keys, rotation
ROPE = [  # tokens, heads_q, heads_kv, dim, rotary
    (1, 1, 1, 64, 64), (7, 4, 2, 128, 128), (33, 32, 8, 128, 128), (5, 3, 1, 96, 32), (9, 7, 1, 80, 40),
    (3, 2, 2, 256, 256), (4, 2, 1, 72, 0), (6, 2, 1, 50, 26), (2, 1, 1, 1, 0), (3, 5, 2, 512, 512), (11, 0, 2, 64, 64),
    (301, 14, 2, 64, 64),
]


def rope_inputs(shape, dt, dev, weights, seed):
    T, hq, hkv, d, r = shape
    g = torch.Generator(device=dev).manual_seed(seed)
    packed = torch.randn(T, (hq + 2 * hkv) * d, device=dev, generator=g).to(dt)
    q = packed[:, : hq * d].view(T, hq, d)
    k = packed[:, hq * d: (hq + hkv) * d].view(T, hkv, d)
    wt = {"same": dt, "f32": torch.float32, "none": None}[weights]
    w = [None if wt is None else (1 + 0.3 * torch.randn(d, device=dev, generator=g)).to(wt) for _ in range(2)]
    from kbb200 import lm
    cos, sin = lm.rope_tables(200, r, device=dev)
    pos = torch.randint(0, 200, (T,), device=dev, generator=g)
    return q, k, w, cos, sin, pos


def weight64(w, d):
    return np.ones(d) if w is None else f64(w)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", ROPE)
def test_qk_norm_rope(shape, dt, interleaved, cuda_device):
    from kbb200 import lm

    T, hq, hkv, d, r = shape
    q, k, w, cos, sin, pos = rope_inputs(shape, dt, cuda_device, "same" if d % 3 else "f32", sum(shape))
    if T % 2:
        pos = pos.int()
    outs = lm.qk_norm_rope(q, k, w[0], w[1], cos, sin, pos, eps=1e-5, interleaved=interleaved)
    c, s = f64(cos)[pos.cpu().numpy()], f64(sin)[pos.cpu().numpy()]
    for x, wt, z in zip((q, k), w, outs):
        assert z.shape == x.shape and z.dtype == dt and z.is_contiguous()
        want = O.norm_rope(f64(x), weight64(wt, d), c, s, r, interleaved, 1e-5)
        mag = O.norm_rope(np.abs(f64(x)), np.abs(weight64(wt, d)), np.abs(c), -np.abs(s), r, interleaved, 1e-5)
        mag = np.maximum(mag, O.norm_rope(np.abs(f64(x)), np.abs(weight64(wt, d)), np.abs(c), np.abs(s), r, interleaved, 1e-5))
        within(z, want, UNIT[dt] * np.abs(want) + 32 * U * mag + TINY[dt], f"{shape} {dt}")


@pytest.mark.parametrize("weights", ["same", "f32", "none"])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", ROPE)
def test_qk_norm_rope_backward(shape, dt, weights, cuda_device):
    from kbb200 import lm

    T, hq, hkv, d, r = shape
    interleaved = bool(T % 2)
    q, k, w, cos, sin, pos = rope_inputs(shape, dt, cuda_device, weights, 7 + sum(shape))
    g = torch.Generator(device=cuda_device).manual_seed(5)
    dq = torch.randn(T, hq, d, device=cuda_device, generator=g).to(dt)
    dk = torch.randn(T, hkv, d, device=cuda_device, generator=g).to(dt)
    got = lm.qk_norm_rope_backward(dq, dk, q, k, w[0], w[1], cos, sin, pos, eps=1e-5, interleaved=interleaved)
    again = lm.qk_norm_rope_backward(dq, dk, q, k, w[0], w[1], cos, sin, pos, eps=1e-5, interleaved=interleaved)
    c, s = f64(cos)[pos.cpu().numpy()], f64(sin)[pos.cpu().numpy()]
    for i, (x, wt, dz) in enumerate(((q, w[0], dq), (k, w[1], dk))):
        x64, w64, dz64 = f64(x), weight64(wt, d), f64(dz)
        want, dw = O.norm_rope_backward(dz64, x64, w64, c, s, r, interleaved, 1e-5)
        rstd = 1 / np.sqrt((x64 * x64).mean(-1, keepdims=True) + 1e-5)
        dy = np.maximum(O.rotate(np.abs(dz64), np.abs(c), np.abs(s), r, interleaved),
                        O.rotate(np.abs(dz64), np.abs(c), np.abs(s), r, interleaved, back=True))
        xh = np.abs(x64) * rstd
        mag = rstd * (dy * np.abs(w64) + xh * (dy * np.abs(w64) * xh).mean(-1, keepdims=True))
        within(got[i], want, UNIT[dt] * np.abs(want) + 48 * U * mag + TINY[dt], f"dx {shape} {dt}")
        if weights == "none":
            assert got[2 + i] is None
        else:
            assert got[2 + i].dtype == wt.dtype
            within(got[2 + i], dw, UNIT[wt.dtype] * np.abs(dw) + 32 * U * (dy * xh).sum((0, 1)) + TINY[wt.dtype],
                   f"dw {shape} {dt}")
            assert torch.equal(got[2 + i], again[2 + i])


def test_rope_positions_outside_the_table(cuda_device):
    from kbb200 import lm

    q, k, w, cos, sin, _ = rope_inputs((4, 2, 1, 64, 32), torch.float32, cuda_device, "same", 3)
    pos = torch.tensor([0, 200, -1, 199], device=cuda_device)
    z, _ = lm.qk_norm_rope(q, k, w[0], w[1], cos, sin, pos)
    bad = torch.isnan(z)
    assert bad[1:3, :, :32].all() and not bad[[0, 3]].any() and not bad[:, :, 32:].any()


def test_rope_no_tokens(cuda_device):
    from kbb200 import lm

    q, k, w, cos, sin, pos = rope_inputs((0, 2, 1, 64, 32), torch.bfloat16, cuda_device, "f32", 3)
    assert lm.qk_norm_rope(q, k, w[0], w[1], cos, sin, pos)[0].shape == (0, 2, 64)
    e = torch.empty_like(q), torch.empty_like(k)
    _, _, dw, _ = lm.qk_norm_rope_backward(e[0].contiguous(), e[1].contiguous(), q, k, w[0], w[1], cos, sin, pos)
    assert (dw == 0).all()


def test_rope_any_strides(cuda_device):
    """Heads in another order of memory, and a base that is not 16-byte aligned."""
    from kbb200 import lm

    T, h, d = 5, 3, 64
    base = torch.randn(h, T, d + 3, device=cuda_device).bfloat16()
    q = base.transpose(0, 1)[..., 1: d + 1]
    w = torch.ones(d, device=cuda_device)
    cos, sin = lm.rope_tables(50, d, device=cuda_device)
    pos = torch.arange(T, device=cuda_device)
    a = lm.qk_norm_rope(q, q, w, w, cos, sin, pos)
    b = lm.qk_norm_rope(q.contiguous(), q.contiguous(), w, w, cos, sin, pos)
    within(a[0], f64(b[0]), 2 * UNIT[torch.bfloat16] * np.abs(f64(b[0])))
    assert torch.equal(a[0], a[1])


# ------------------------------------------------------------ attention over the cache
def attention_inputs(dev, dt, B, Q, hq, hkv, d, page, n_pre, suffix, lens=None, seed=0, spread=2.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    n_own = -(-suffix // page)
    pages = n_pre + B * n_own + 2
    k, v = (torch.randn(pages, page, hkv, d, device=dev, generator=g).to(dt) for _ in range(2))
    q = (spread * torch.randn(B, Q, hq, d, device=dev, generator=g)).to(dt)
    order = torch.randperm(pages, device=dev, generator=g).int()
    prefix = order[:n_pre].contiguous()
    table = torch.cat((prefix[None].expand(B, -1), order[n_pre: n_pre + B * n_own].view(B, n_own)), 1).contiguous()
    if lens is None:
        lens = n_pre * page + torch.randint(0, suffix + 1, (B,), device=dev, generator=g)
        lens[0] = n_pre * page + suffix
    return q, k, v, prefix, table, torch.as_tensor(lens, device=dev, dtype=torch.int32)


def check_attention(args, dt, scale=None):
    from kbb200 import lm

    q, k, v, prefix, table, lens = args
    d = q.shape[-1]
    out, lse = lm.shared_prefix_attention(*args, scale=scale)
    sc = d ** -0.5 if scale is None else scale
    q64, k64, v64 = f64(q), f64(k), f64(v)
    tab, n = table.cpu().numpy(), lens.cpu().numpy()
    want, want_lse, mag = O.shared_prefix_attention(q64, k64, v64, prefix.cpu().numpy(), tab, n, sc)
    e = (d + 16) * U * abs(sc) * np.abs(q64).sum(-1).max() * np.abs(k64).max()
    top = np.abs(want_lse[np.isfinite(want_lse)]).max() if np.isfinite(want_lse).any() else 0.0
    e = min(e, (d + 16) * U * abs(sc) * np.sqrt((q64 ** 2).sum(-1).max() * (k64 ** 2).sum(-1).max()) * 2)
    rounded = 0.0 if dt == torch.float32 else UNIT[dt]
    within(out, want, UNIT[dt] * np.abs(want) + (rounded + 2 * e + 2.0 ** -20) * mag + TINY[dt], "out")
    within(lse, want_lse, e + 2.0 ** -20 + 4 * U * top, "lse")
    return out, lse


ATTN = [  # B, Q, hq, hkv, d, page, prefix pages, suffix
    (1, 1, 1, 1, 64, 16, 0, 1), (1, 1, 4, 1, 64, 16, 1, 0), (2, 1, 8, 2, 128, 16, 3, 20), (3, 2, 6, 2, 64, 8, 5, 33),
    (9, 1, 8, 1, 128, 16, 17, 65), (5, 3, 4, 4, 80, 32, 2, 70), (2, 8, 16, 2, 96, 16, 4, 40), (17, 1, 10, 2, 128, 64, 9, 130),
    (4, 1, 2, 1, 256, 16, 6, 50), (3, 1, 5, 5, 16, 1, 7, 9), (2, 1, 40, 2, 128, 128, 2, 200), (33, 1, 16, 2, 64, 32, 30, 12),
    (2, 5, 20, 1, 128, 24, 11, 77), (70, 2, 4, 1, 128, 16, 40, 17),
]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", ATTN)
def test_shared_prefix_attention(shape, dt, cuda_device):
    check_attention(attention_inputs(cuda_device, dt, *shape, seed=sum(shape)), dt)


LARGE = [  # past 1.2e9 operations over the prefix: fp32 in halves on the tensor cores
    (40, 1, 16, 4, 64, 16, 460, 30), (33, 2, 8, 2, 80, 24, 300, 50), (18, 1, 32, 4, 128, 32, 140, 0),
]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", LARGE)
def test_attention_long_prefix(shape, dt, cuda_device):
    check_attention(attention_inputs(cuda_device, dt, *shape, seed=sum(shape)), dt)


def test_attention_long_prefix_in_fp32_of_uneven_magnitudes(cuda_device):
    """Keys and values over six orders of magnitude, short and ended sequences, NaN where nobody looks, a negative
    scale."""
    shape = (40, 1, 16, 4, 64, 16, 460, 30)
    q, k, v, prefix, table, lens = attention_inputs(cuda_device, torch.float32, *shape, seed=3)
    g = torch.Generator(device=cuda_device).manual_seed(3)
    q, k, v = (x * 10 ** (3 * torch.rand(x.shape[:-1] + (1,), device=cuda_device, generator=g) - 2.5) for x in (q, k, v * 1e5))
    lens = 7000 + torch.arange(40, device=cuda_device, dtype=torch.int32)
    lens[5], lens[6], lens[7] = 0, 1, 130
    args = (q, k, v, prefix, table, lens)
    out, lse = check_attention(args, torch.float32)
    assert (out[5] == 0).all()
    check_attention(args, torch.float32, scale=-0.05)
    last = prefix[7039 // 16:].long()
    for t in (k, v):
        t[last[1:]] = float("nan")
        t[last[0], 7039 % 16:] = float("inf")
    from kbb200 import lm
    again = lm.shared_prefix_attention(*args)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("dt", TYPES)
def test_attention_empty_and_short_rows(dt, cuda_device):
    """Ended slots, sequences with fewer keys than queries, and shorter than the prefix."""
    lens = [0, 64, 0, 1, 2, 3, 70, 40, 33, 200, -5]
    args = attention_inputs(cuda_device, dt, len(lens), 3, 8, 2, 64, 16, 4, 136, lens=lens, seed=1)
    out, lse = check_attention(args, dt)
    assert (out[0] == 0).all() and torch.isinf(lse[0]).all() and (out[3, :2] == 0).all() and (out[10] == 0).all()


@pytest.mark.parametrize("dt", TYPES)
def test_attention_no_keys_at_all(dt, cuda_device):
    args = attention_inputs(cuda_device, dt, 3, 1, 4, 2, 64, 16, 0, 0, lens=[0, 0, 0])
    out, lse = check_attention(args, dt)
    assert (out == 0).all()


@pytest.mark.parametrize("dt", TYPES)
def test_attention_unused_slots_hold_anything(dt, cuda_device):
    """NaN and infinities past a sequence's end, in pages that no sequence holds, and ids past a row's end."""
    shape = (6, 1, 8, 2, 128, 16, 9, 100)
    q, k, v, prefix, table, lens = args = attention_inputs(cuda_device, dt, *shape, seed=4)
    want, want_lse = check_attention(args, dt)
    used = torch.zeros(k.shape[:2], dtype=torch.bool, device=cuda_device)
    used[prefix.long()] = True
    for b, n in enumerate(lens.tolist()):
        for j in range(n):
            used[table[b, j // 16].long(), j % 16] = True
        table[b, -(-n // 16):] = -1 if b % 2 else 2 ** 31 - 1
    table[:, :9] = -7  # not read: the prefix stands in for them
    for t in (k, v):
        t[~used] = float("nan")
        t[~used & (torch.rand(used.shape, device=cuda_device) < 0.5)] = float("inf")
    from kbb200 import lm
    out, lse = lm.shared_prefix_attention(q, k, v, prefix, table, lens)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_attention_nan_of_one_sequence_stays_there(cuda_device):
    dt = torch.bfloat16
    q, k, v, prefix, table, lens = args = attention_inputs(cuda_device, dt, 4, 1, 8, 2, 128, 16, 5, 60, seed=9)
    from kbb200 import lm
    want, _ = lm.shared_prefix_attention(*args)
    k[table[0, 5].long(), 3] = float("nan")
    out, lse = lm.shared_prefix_attention(*args)
    assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all() and torch.equal(out[1:], want[1:])


@pytest.mark.parametrize("dt", TYPES)
def test_attention_strides_and_scale(dt, cuda_device):
    """q as a view of a packed projection, keys and values interleaved in one pool, another stream."""
    shape = (5, 2, 8, 2, 64, 16, 6, 40)
    q, k, v, prefix, table, lens = attention_inputs(cuda_device, dt, *shape, seed=2)
    pool = torch.stack((k, v), 2)  # [pages, page, 2, heads, dim]
    packed = torch.cat((q.flatten(2), q.flatten(2)), -1)
    args = (packed[..., : 8 * 64].view(5, 2, 8, 64), pool[:, :, 0], pool[:, :, 1], prefix, table, lens)
    assert not args[0].is_contiguous() and not args[1].is_contiguous()
    check_attention(args, dt, scale=0.05)
    check_attention(args, dt, scale=-0.2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        check_attention(args, dt)
    torch.cuda.current_stream().wait_stream(s)


@pytest.mark.parametrize("dt", TYPES)
def test_attention_large_scores(dt, cuda_device):
    """Scores of hundreds: the running maximum moves and one key takes nearly all the weight."""
    args = attention_inputs(cuda_device, dt, 9, 1, 8, 2, 128, 16, 40, 150, seed=11, spread=60.0)
    check_attention(args, dt)


def test_attention_offsets_past_32_bits(cuda_device):
    """A pool of over 2^31 elements, with the pages used at its end."""
    dt, page, h, d = torch.bfloat16, 16, 8, 128
    pages = 2 ** 31 // (page * h * d) + 40
    k = torch.empty(pages, page, h, d, device=cuda_device, dtype=dt)
    k[-40:] = torch.randn(40, page, h, d, device=cuda_device).to(dt)
    q = torch.randn(16, 1, 32, d, device=cuda_device).to(dt)
    prefix = torch.arange(pages - 20, pages, device=cuda_device).int()
    table = torch.full((16, 21), pages - 30, device=cuda_device).int()
    table[:, 20] = torch.arange(pages - 40, pages - 24, device=cuda_device).int()
    lens = torch.full((16,), 20 * page + 5, device=cuda_device).int()
    from kbb200 import lm
    out, lse = lm.shared_prefix_attention(q, k, k, prefix, table, lens)
    low = k[-40:].clone()
    want, want_lse = lm.shared_prefix_attention(q, low, low, prefix - (pages - 40), table - (pages - 40), lens)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_attention_refusals(cuda_device):
    from kbb200 import KbError, lm

    q, k, v, prefix, table, lens = attention_inputs(cuda_device, torch.bfloat16, 2, 1, 4, 2, 64, 16, 2, 20)
    with pytest.raises(KbError, match="16-byte"):
        lm.shared_prefix_attention(q[..., :60].contiguous(), k[..., :60].contiguous(), v[..., :60].contiguous(), prefix,
                                   table, lens)
    with pytest.raises(KbError, match="key heads"):
        lm.shared_prefix_attention(q[:, :, :3].contiguous(), k, v, prefix, table, lens)
    with pytest.raises(RuntimeError, match="float32"):
        lm.shared_prefix_attention(q.float(), k, v, prefix, table, lens)
    with pytest.raises(RuntimeError, match="int64"):
        lm.shared_prefix_attention(q, k, v, prefix.long(), table, lens)
    with pytest.raises(RuntimeError, match="last dimension"):
        lm.shared_prefix_attention(q.transpose(2, 3).contiguous().transpose(2, 3), k, v, prefix, table, lens)
    with pytest.raises(RuntimeError, match="CUDA"):
        lm.shared_prefix_attention(q.cpu(), k, v, prefix, table, lens)
    with pytest.raises(RuntimeError, match="rows"):
        lm.shared_prefix_attention(q, k, v, prefix, table[:1].contiguous(), lens)
    with pytest.raises(KbError, match="head dim"):
        big = torch.zeros(2, 1, 4, 264, device=cuda_device, dtype=torch.bfloat16)
        pages = torch.zeros(4, 16, 2, 264, device=cuda_device, dtype=torch.bfloat16)
        lm.shared_prefix_attention(big, pages, pages, prefix, table, lens)


# ------------------------------------------------------------ the paged cache
def cache_state(dev, dt, planes, pages, page, h, d, lens, width, seed=0):
    """Slots of the given lengths on scattered pages."""
    g = torch.Generator(device=dev).manual_seed(seed)
    pool = torch.randn(planes, pages, page, h, d, device=dev, generator=g).to(dt)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    for s, n in enumerate(lens):
        for j in range(-(-n // page)):
            table[s, j] = order.pop()
            refs[table[s, j]] = 1
    state = pool, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), refs.to(dev)
    return state, O.Cache(f64(pool), table.numpy(), np.array(lens), refs.numpy())


def same_cache(state, want):
    pool, table, lens, refs = state
    assert np.array_equal(table.cpu().numpy(), want.table)
    assert np.array_equal(lens.cpu().numpy(), want.lens)
    assert np.array_equal(refs.cpu().numpy(), want.refs)
    assert np.array_equal(f64(pool), want.pool)


def ints(dev, v):
    return torch.tensor(v, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("page,h,d", [(16, 2, 64), (8, 1, 80), (5, 1, 3), (1, 2, 8)])
def test_cache_rounds(page, h, d, dt, cuda_device):
    """Random rounds of every operation, compared after each."""
    from kbb200 import lm

    rng = np.random.default_rng(page)
    slots, width, planes = 12, 9, 6
    lens = [int(n) for n in rng.integers(0, width * page // 2 + 1, slots)]
    state, want = cache_state(cuda_device, dt, planes, 70, page, h, d, lens, width, seed=page)
    pool, table, lens, refs = state
    for step in range(12):
        some = rng.permutation(slots)
        parents, children = some[: slots // 2], some[slots // 2:]
        if step % 3 == 2:  # a beam: parents replaced by each other's children
            parents, children = rng.integers(0, slots, slots), rng.permutation(slots)
        got = lm.cache_fork(pool, table, lens, refs, ints(cuda_device, parents.tolist()), ints(cuda_device, children.tolist()))
        assert got.tolist() == want.fork(parents.tolist(), children.tolist())
        same_cache(state, want)
        seqs, tokens = rng.permutation(slots)[:7].tolist(), int(rng.integers(0, 2 * page + 2))
        got = lm.cache_reserve(table, lens, refs, ints(cuda_device, seqs), tokens, page)
        granted = want.reserve(seqs, tokens)
        assert got.tolist() == granted
        same_cache(state, want)
        seqs = [s for s, ok in zip(seqs, granted) if ok]
        k, v = (torch.randn(len(seqs), tokens, h, d, device=cuda_device).to(dt) for _ in range(2))
        lm.cache_append(k, v, pool[0], pool[1], table, lens, ints(cuda_device, seqs))
        want.append(f64(k), f64(v), seqs)
        same_cache(state, want)
        gone = rng.integers(0, slots, 4).tolist()  # with repeats
        lm.cache_free(table, lens, refs, ints(cuda_device, gone))
        want.free(gone)
        same_cache(state, want)
        if step % 2:
            assert lm.cache_compact(pool, table, refs).tolist() == [want.compact()]
            same_cache(state, want)


def test_cache_requests_that_are_refused(cuda_device):
    from kbb200 import lm

    state, want = cache_state(cuda_device, torch.float32, 2, 9, 4, 1, 4, [6, 3, 8, 0, 0, 0], 4)
    pool, table, lens, refs = state  # 5 pages held, 4 free
    parents, children = [0, 0, 1, 9, 0, 2, -1, 1], [3, 3, 4, 5, -2, 5, 0, 1]
    got = lm.cache_fork(pool, table, lens, refs, ints(cuda_device, parents), ints(cuda_device, children))
    assert got.tolist() == want.fork(parents, children) == [1, 0, 1, 0, 0, 0, 0, 1]
    same_cache(state, want)
    for seqs, tokens in (([0, 1, 2], 9), ([0, 0, 7, 1], 1), ([2, 1], 5), ([2, 1, 0], 4), ([0], 100)):
        assert lm.cache_reserve(table, lens, refs, ints(cuda_device, seqs), tokens, 4).tolist() == want.reserve(seqs, tokens)
        same_cache(state, want)
    lm.cache_free(table, lens, refs, ints(cuda_device, [-1, 6, 2, 2]))
    want.free([-1, 6, 2, 2])
    same_cache(state, want)


def test_cache_many_pages_and_requests(cuda_device):
    """More pages, slots and requests than one block has threads."""
    from kbb200 import lm

    rng = np.random.default_rng(0)
    lens = [int(n) for n in rng.integers(0, 40, 1500)] + [0] * 1600
    state, want = cache_state(cuda_device, torch.float16, 2, 9000, 8, 1, 8, lens, 6, seed=3)
    pool, table, lens, refs = state
    parents, children = list(range(1500)), list(range(1500, 3000))
    got = lm.cache_fork(pool, table, lens, refs, ints(cuda_device, parents), ints(cuda_device, children))
    assert got.tolist() == want.fork(parents, children)
    seqs = rng.permutation(3100).tolist()
    got = lm.cache_reserve(table, lens, refs, ints(cuda_device, seqs), 9, 8)
    assert got.tolist() == want.reserve(seqs, 9)
    gone = list(range(0, 3100, 3))
    lm.cache_free(table, lens, refs, ints(cuda_device, gone))
    want.free(gone)
    assert lm.cache_compact(pool, table, refs).tolist() == [want.compact()]
    same_cache(state, want)


@pytest.mark.parametrize("d", [8, 3])
def test_cache_copy_between_pools(d, cuda_device):
    from kbb200 import lm

    a = torch.randn(4, 30, 2, 1, d, device=cuda_device)
    b = torch.zeros(4, 11, 2, 1, d, device=cuda_device)
    src, dst = [3, 29, 0, 30, -1, 7, 5], [10, 0, 4, 1, 2, 11, 5]
    lm.cache_copy(a, ints(cuda_device, src), b, ints(cuda_device, dst))
    want = torch.zeros_like(b)
    for s, t in zip(src, dst):
        if 0 <= s < 30 and 0 <= t < 11:
            want[:, t] = a[:, s]
    assert torch.equal(b, want)
    lm.cache_copy(a, ints(cuda_device, []), b, ints(cuda_device, []))
    assert torch.equal(b, want)


def test_cache_refusals(cuda_device):
    from kbb200 import KbError, lm

    (pool, table, lens, refs), _ = cache_state(cuda_device, torch.float16, 2, 9, 4, 1, 8, [6, 3], 4)
    one = ints(cuda_device, [0])
    with pytest.raises(RuntimeError, match="contiguous"):
        lm.cache_fork(pool.transpose(2, 4), table, lens, refs, one, one)
    with pytest.raises(RuntimeError, match="pages"):
        lm.cache_fork(pool, table, lens, refs[:8].contiguous(), one, one)
    with pytest.raises(RuntimeError, match="int64"):
        lm.cache_free(table.long(), lens, refs, one)
    with pytest.raises(KbError, match="token count"):
        lm.cache_reserve(table, lens, refs, one, -1, 4)
    with pytest.raises(KbError, match="token count"):
        lm.cache_reserve(table, lens, refs, one, 1, 0)
    k = torch.zeros(1, 1, 1, 8, device=cuda_device, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="float32"):
        lm.cache_append(k.float(), k, pool[0], pool[1], table, lens, one)
    with pytest.raises(RuntimeError, match="shape"):
        lm.cache_append(k, k[:0], pool[0], pool[1], table, lens, one)
    with pytest.raises(RuntimeError, match="planes"):
        lm.cache_copy(pool, one, pool[:1].contiguous(), one)


# ------------------------------------------------------------ logits
def mask_words(allowed):
    """bool [rows, vocab] -> int32 words."""
    rows, vocab = allowed.shape
    pad = np.zeros((rows, -(-vocab // 32) * 32), dtype=np.uint8)
    pad[:, :vocab] = allowed
    return torch.from_numpy(np.packbits(pad, axis=1, bitorder="little").view(np.int32).copy())


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("ids", [torch.int64, torch.int32])
@pytest.mark.parametrize("rows,vocab,n_prompt,n_output,n_bias,masked", [
    (1, 1, 1, 1, 1, True), (3, 100, 7, 200, 5, True), (2, 8192, 0, 50, 0, False), (5, 8193, 30, 0, 300, True),
    (4, 50257, 500, 700, 40, False), (2, 131072, 64, 64, 2000, True), (7, 33, 3, 3, 0, True), (1, 200001, 3, 2000, 1, True),
])
def test_penalize_logits(rows, vocab, n_prompt, n_output, n_bias, masked, ids, dt, cuda_device):
    from kbb200 import lm

    rng = np.random.default_rng(vocab)
    x = torch.from_numpy(4 * rng.standard_normal((rows, vocab))).to(cuda_device).to(dt)
    x[0, 0] = float("-inf")
    x[-1, vocab // 2] = float("inf")

    def hist(n):
        if not n:
            return None
        h = (vocab * rng.random((rows, n)) ** 3).astype(np.int64)
        h[rng.random((rows, n)) < 0.2] = -1
        h[rng.random((rows, n)) < 0.05] = vocab
        return h

    prompt, output, bias = hist(n_prompt), hist(n_output), hist(n_bias)
    values = rng.standard_normal((rows, n_bias)).astype(np.float32) if n_bias else None
    rep = (1 + rng.random(rows)).astype(np.float32)
    pres, freq = (rng.standard_normal(rows).astype(np.float32) for _ in range(2))
    allowed = None
    if masked:
        allowed = rng.random((rows, vocab)) < 0.6
        allowed[rows // 2] = False

    def dev(v, t=None):
        return None if v is None else torch.as_tensor(v, dtype=t).to(cuda_device)

    args = (dev(prompt, ids), dev(output, ids), dev(rep), dev(pres), dev(freq), dev(bias, ids), dev(values),
            None if allowed is None else mask_words(allowed).to(cuda_device))
    got = lm.penalize_logits(x, *args)
    want = O.penalize_logits(f64(x), prompt, output, rep.astype(np.float64), pres.astype(np.float64), freq.astype(np.float64),
                             bias, values, allowed)
    mag = 2 * np.abs(f64(x)) + n_output * np.abs(freq)[:, None] + np.abs(pres)[:, None] + 6
    tol = UNIT[dt] * np.abs(want) + 8 * U * mag + TINY[dt]
    within(got, want, np.where(np.isfinite(tol), tol, 0), "logits")
    same = x.clone()
    lm.penalize_logits(same, *args, out=same)
    assert torch.equal(same, got)


@pytest.mark.parametrize("dt", TYPES)
def test_penalize_leaves_other_logits_alone(dt, cuda_device):
    from kbb200 import lm

    x = torch.randn(3, 1001, device=cuda_device).to(dt)
    assert torch.equal(lm.penalize_logits(x), x)
    out = torch.tensor([[5], [6], [-1]], device=cuda_device)
    got = lm.penalize_logits(x, output=out, presence=torch.ones(3, device=cuda_device))
    changed = (got != x).nonzero().tolist()
    assert changed == [[0, 5], [1, 6]]


def test_penalize_strided_rows_and_one_mask(cuda_device):
    from kbb200 import lm

    wide = torch.randn(4, 300, device=cuda_device)
    x = wide[:, 7:257]
    allowed = np.random.default_rng(0).random((1, 250)) < 0.5
    got = lm.penalize_logits(x, mask=mask_words(allowed).to(cuda_device))
    keep = torch.from_numpy(allowed).to(cuda_device)
    assert torch.equal(got, torch.where(keep, x, torch.full_like(x, float("-inf"))))
    assert lm.penalize_logits(x[:0]).shape == (0, 250) and lm.penalize_logits(x[:, :0]).shape == (4, 0)


def test_penalize_refusals(cuda_device):
    from kbb200 import KbError, lm

    x = torch.zeros(2, 64, device=cuda_device)
    ids = torch.zeros(2, 3, device=cuda_device, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="go together"):
        lm.penalize_logits(x, bias_ids=ids)
    with pytest.raises(RuntimeError, match="mask"):
        lm.penalize_logits(x, mask=torch.zeros(2, 3, device=cuda_device, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="int32"):
        lm.penalize_logits(x, prompt=ids, output=ids.int())
    with pytest.raises(RuntimeError, match="float64"):
        lm.penalize_logits(x.double())
    with pytest.raises(RuntimeError, match="shape"):
        lm.penalize_logits(x, repetition=torch.ones(3, device=cuda_device))
    with pytest.raises(KbError, match="biases"):
        many = torch.zeros(2, 2048, device=cuda_device, dtype=torch.int64)
        lm.penalize_logits(x, bias_ids=many, bias_values=many.float())

"""GPU: sizes from which the language-model operators take other ways than the small ones of test_gpu_lm: logits of 8 MB
and more with histories (copy, then a hash table of the changed tokens), histories past that table, and enough tokens
that the warps of the norms' backward pass walk on and move their sums to fp64.  Tolerances as in test_gpu_lm."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import lm as O
from tests.test_gpu_lm import TINY, U, UNIT, f64, mask_words, within

pytestmark = pytest.mark.gpu

TYPES = list(UNIT)


# ------------------------------------------------------------ logits
def histories(rng, rows, vocab, n, step=1):
    """Ids that repeat within a row and meet those of the other lists; some are padding or past the vocabulary."""
    if not n:
        return None
    h = ((vocab // step) * rng.random((rows, n)) ** 3).astype(np.int64) * step
    h[rng.random((rows, n)) < 0.1] = -1
    h[rng.random((rows, n)) < 0.02] = vocab
    return h


LOGITS = [  # vocab, prompt, output, biases, mask (None, rows of their own, one for all), ids are multiples of
    (131072, 1000, 900, 300, "rows", 1), (100003, 40, 0, 7, "one", 1), (131072, 5000, 2000, 1192, "rows", 1),
    (131072, 5000, 2000, 1193, "rows", 1), (50257, 20000, 5000, 20, None, 1), (131072, 0, 16, 0, None, 4096),
    (131072, 0, 700, 0, "one", 128), (200001, 1, 1, 1, "rows", 1),
]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("vocab,n_prompt,n_output,n_bias,masked,step", LOGITS)
def test_penalize_large_batches(vocab, n_prompt, n_output, n_bias, masked, step, dt, cuda_device):
    from kbb200 import lm

    rng = np.random.default_rng(vocab + n_output)
    size = torch.empty((), dtype=dt).element_size()
    rows = -(-(8 << 20) // (vocab * size)) + 1  # past 8 MB
    x = torch.from_numpy(4 * rng.standard_normal((rows, vocab))).to(cuda_device).to(dt)
    x[0, 0], x[-1, vocab // 2] = float("-inf"), float("inf")
    prompt, output, bias = (histories(rng, rows, vocab, n, step) for n in (n_prompt, n_output, n_bias))
    values = rng.standard_normal((rows, n_bias)).astype(np.float32) if n_bias else None
    rep = (1 + rng.random(rows)).astype(np.float32)
    pres, freq = (rng.standard_normal(rows).astype(np.float32) for _ in range(2))
    allowed = None
    if masked:
        allowed = rng.random((rows if masked == "rows" else 1, vocab)) < 0.6
        allowed[allowed.shape[0] // 2, ::3] = False

    def dev(v, t=None):
        return None if v is None else torch.as_tensor(v, dtype=t).to(cuda_device)

    ids = torch.int32 if rows % 2 else torch.int64
    args = (dev(prompt, ids), dev(output, ids), dev(rep), dev(pres), dev(freq), dev(bias, ids), dev(values),
            None if allowed is None else mask_words(allowed).to(cuda_device))
    got = lm.penalize_logits(x, *args)
    want = O.penalize_logits(f64(x), prompt, output, rep.astype(np.float64), pres.astype(np.float64), freq.astype(np.float64),
                             bias, values, None if allowed is None else np.broadcast_to(allowed, x.shape))
    mag = 2 * np.abs(f64(x)) + n_output * np.abs(freq)[:, None] + np.abs(pres)[:, None] + 6
    tol = UNIT[dt] * np.abs(want) + 8 * U * mag + TINY[dt]
    within(got, want, np.where(np.isfinite(tol), tol, 0), "logits")
    same = x.clone()
    lm.penalize_logits(same, *args, out=same)
    assert torch.equal(same, got)
    wide = torch.full((rows, vocab + 3), 7.0, device=cuda_device, dtype=dt)  # rows of another alignment
    wide[:, 1: vocab + 1] = x
    assert torch.equal(lm.penalize_logits(wide[:, 1: vocab + 1], *args), got)


@pytest.mark.parametrize("in_graph", [False, True])
@pytest.mark.parametrize("dt", TYPES)
def test_penalize_large_batches_without_pauses(dt, in_graph, cuda_device):
    """Behind a slow producer of logits and histories, in place and not, with the next call right after."""
    from kbb200 import lm

    g = torch.Generator(device=cuda_device).manual_seed(1)
    rows, vocab = 40, 131072
    source = torch.randn(rows, vocab, device=cuda_device, generator=g)
    ids = torch.randint(0, vocab, (rows, 3000), device=cuda_device, generator=g)
    x, history = torch.zeros(rows, vocab, device=cuda_device, dtype=dt), torch.zeros_like(ids)
    ones = torch.full((rows,), 1.5, device=cuda_device)
    slow = torch.randn(1 << 25, device=cuda_device, generator=g)

    def run(between=lambda: None):
        x.zero_(), history.zero_()
        between()
        for _ in range(3):
            slow.mul_(-1.0)
        x.copy_(source), history.copy_(ids)
        between()
        y = lm.penalize_logits(x, prompt=history, output=history[:, :900].contiguous(), repetition=ones, frequency=ones)
        between()
        lm.penalize_logits(x, prompt=history, repetition=ones, out=x)
        between()
        z = lm.penalize_logits(x, output=history, presence=ones)
        between()
        return y, x.clone(), z

    run(torch.cuda.synchronize)
    if in_graph:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run()
    for i in range(3):
        source.normal_(generator=torch.Generator(device=cuda_device).manual_seed(i))
        want = run(torch.cuda.synchronize)
        if in_graph:
            graph.replay()
        else:
            got = run()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


# ------------------------------------------------------------ norms of queries and keys, rotation
ROPE = [  # tokens, heads_q, heads_kv, dim, rotary, interleaved; a warp of the backward pass sums 128 terms and more
    (20500, 32, 8, 128, 128, False), (20500, 32, 8, 128, 64, True), (41000, 30, 6, 64, 64, False), (21000, 32, 4, 72, 36, False),
    (10400, 30, 8, 256, 256, False), (5000, 8, 3, 320, 64, True),
]


def rotated(y, c, s, rotary, interleaved, back=False):
    s = -s if back else s
    a, b = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, rotary // 2), slice(rotary // 2, rotary))
    z = y.clone()
    z[..., a] = y[..., a] * c - y[..., b] * s
    z[..., b] = y[..., b] * c + y[..., a] * s
    return z


def close(got, want, tol, what):
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"{what}: {float(err.max()):.3e} off, {float((err / tol).max()):.2f} of the tolerance"


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", ROPE)
def test_qk_norm_rope_of_many_tokens(shape, dt, cuda_device):
    """Values and gradients against the formula in 64 bits, on the device: there is too much for the host."""
    from kbb200 import lm

    T, hq, hkv, d, r, interleaved = shape
    g = torch.Generator(device=cuda_device).manual_seed(T)
    packed = torch.randn(T, (hq + 2 * hkv) * d, device=cuda_device, generator=g).to(dt)
    q, k = packed[:, : hq * d].view(T, hq, d), packed[:, hq * d: (hq + hkv) * d].view(T, hkv, d)
    w = [(1 + 0.3 * torch.randn(d, device=cuda_device, generator=g)).to(dt if d % 3 else torch.float32) for _ in range(2)]
    cos, sin = lm.rope_tables(4000, r, device=cuda_device)
    pos = torch.randint(0, 4000, (T,), device=cuda_device, generator=g)
    dz = [torch.randn(T, h, d, device=cuda_device, generator=g).to(dt) for h in (hq, hkv)]
    z = lm.qk_norm_rope(q, k, *w, cos, sin, pos, eps=1e-5, interleaved=interleaved)
    got = lm.qk_norm_rope_backward(*dz, q, k, *w, cos, sin, pos, eps=1e-5, interleaved=interleaved)
    again = lm.qk_norm_rope_backward(*dz, q, k, *w, cos, sin, pos, eps=1e-5, interleaved=interleaved)
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    for i, x in enumerate((q, k)):
        x, w64, g64 = x.double(), w[i].double(), dz[i].double()
        rstd = (x.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
        xh = x * rstd
        mag = rotated((xh * w64).abs(), c.abs(), -s.abs(), r, interleaved).maximum(
            rotated((xh * w64).abs(), c.abs(), s.abs(), r, interleaved))
        want = rotated(xh * w64, c, s, r, interleaved)
        close(z[i], want, UNIT[dt] * want.abs() + 32 * U * mag + TINY[dt], f"z {shape} {dt}")
        dy = rotated(g64, c, s, r, interleaved, back=True)
        big = rotated(g64.abs(), c.abs(), s.abs(), r, interleaved).maximum(
            rotated(g64.abs(), c.abs(), s.abs(), r, interleaved, back=True))
        h = dy * w64
        want = rstd * (h - xh * (h * xh).mean(-1, keepdim=True))
        mag = rstd * ((big * w64).abs() + xh.abs() * ((big * w64) * xh).abs().mean(-1, keepdim=True))
        close(got[i], want, UNIT[dt] * want.abs() + 48 * U * mag + TINY[dt], f"dx {shape} {dt}")
        dw = (dy * xh).sum((0, 1))
        wt = w[i].dtype
        close(got[2 + i], dw, UNIT[wt] * dw.abs() + 32 * U * (big * xh.abs()).sum((0, 1)) + TINY[wt], f"dw {shape} {dt}")
        assert torch.equal(got[i], again[i]) and torch.equal(got[2 + i], again[2 + i])

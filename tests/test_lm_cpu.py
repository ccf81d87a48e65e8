"""CPU: the language-model entries refuse bad arguments on the host, before any launch, and the 64-bit oracle's
gradients agree with differences."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import lm as O

INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3


def _rope(LIB, tokens=4, hq=2, hkv=1, dim=64, rotary=64, dtype=2, weight=0, q=16, pos=16):
    return LIB.kb_qk_norm_rope(q, 16, 16, 16, 16, 16, pos, 16, 16, tokens, hq, hkv, dim, rotary, 100, dim * hq, dim, dim * hkv,
                               dim, dtype, weight, 1, 0, 1e-6, None)


@pytest.mark.parametrize("bad,status", [
    (dict(tokens=-1), INVALID), (dict(dim=0), UNSUPPORTED), (dict(dim=513, rotary=2), UNSUPPORTED),
    (dict(rotary=65), INVALID), (dict(rotary=66), INVALID), (dict(dtype=3), INVALID), (dict(weight=1), INVALID),
    (dict(q=None), INVALID), (dict(pos=None), INVALID), (dict(hq=70000), UNSUPPORTED)])
def test_qk_norm_rope_refusals(bad, status):
    from kbb200 import LIB

    assert _rope(LIB, **bad) == status
    assert b"kb_qk_norm_rope" in LIB.kb_last_error()


def test_qk_norm_rope_nothing_to_do():
    from kbb200 import LIB

    assert _rope(LIB, tokens=0, q=None) == 0
    assert LIB.kb_qk_norm_rope_backward_workspace_size(0, 2, 1, 64) == 0
    assert LIB.kb_qk_norm_rope_backward_workspace_size(10, 2, 1, 64) >= 2 * 64 * 8


def test_qk_norm_rope_backward_wants_its_workspace():
    from kbb200 import LIB

    args = [16] * 13 + [4, 2, 1, 64, 64, 100, 128, 64, 64, 64, 2, 0, 1, 0, 1e-6]
    assert LIB.kb_qk_norm_rope_backward(*args, None, 0, None) == WORKSPACE
    assert LIB.kb_qk_norm_rope_backward(*args, 16, 8, None) == WORKSPACE
    assert LIB.kb_qk_norm_rope_backward(*args, 24, 1 << 30, None) == INVALID  # not 16-byte aligned


def _attention(LIB, B=2, Q=1, hq=4, hkv=2, d=64, pre=2, width=4, pages=9, page=16, dtype=2, q=16, stride=None, k=16, table=16,
               ws=16, ws_bytes=1 << 40):
    s = hq * d if stride is None else stride
    return LIB.kb_shared_prefix_attention(q, k, 16, 16, table, 16, 16, 16, B, Q, hq, hkv, d, pre, width, pages, page, s, s, d,
                                          page * hkv * d, hkv * d, d, page * hkv * d, hkv * d, d, 0.1, dtype, ws, ws_bytes, None)


@pytest.mark.parametrize("bad,status", [
    (dict(B=-1), INVALID), (dict(page=0), INVALID), (dict(hkv=0), INVALID), (dict(hkv=3), INVALID), (dict(dtype=7), INVALID),
    (dict(q=None), INVALID), (dict(k=None), INVALID), (dict(table=None), INVALID), (dict(pages=0), INVALID),
    (dict(d=264), UNSUPPORTED), (dict(d=60), UNSUPPORTED), (dict(q=24), UNSUPPORTED), (dict(stride=257), UNSUPPORTED),
    (dict(width=1 << 40), UNSUPPORTED), (dict(ws=None), WORKSPACE), (dict(ws_bytes=64), WORKSPACE), (dict(ws=20), INVALID)])
def test_attention_refusals(bad, status):
    from kbb200 import LIB

    assert _attention(LIB, **bad) == status
    assert b"kb_shared_prefix_attention" in LIB.kb_last_error()


def test_attention_nothing_to_do():
    from kbb200 import LIB

    assert _attention(LIB, B=0) == 0 and _attention(LIB, Q=0) == 0
    assert LIB.kb_shared_prefix_attention_workspace_size(0, 1, 4, 2, 64, 2, 4, 16, 2) == 0


def test_cache_refusals():
    from kbb200 import LIB

    assert LIB.kb_cache_reserve(16, 16, 16, 16, 16, 2, -1, 4, 8, 9, 16, 16, 1 << 30, None) == INVALID
    assert LIB.kb_cache_reserve(16, 16, 16, 16, 16, 2, 1, 4, 8, 9, 0, 16, 1 << 30, None) == INVALID
    assert LIB.kb_cache_reserve(16, 16, 16, 16, 16, 2, 1, 4, 8, (1 << 20) + 1, 16, 16, 1 << 30, None) == UNSUPPORTED
    assert LIB.kb_cache_reserve(16, 16, 16, None, 16, 2, 1, 4, 8, 9, 16, 16, 1 << 30, None) == INVALID
    assert LIB.kb_cache_reserve(16, 16, 16, 16, 16, 2, 1, 4, 8, 9, 16, None, 0, None) == WORKSPACE
    assert LIB.kb_cache_reserve(None, None, None, None, None, 0, 1, 4, 8, 9, 16, None, 0, None) == 0
    assert LIB.kb_cache_fork(16, 16, 16, 16, 16, 16, 16, 2, 4, 8, 2, 9, 16, 64, None, 0, None) == WORKSPACE
    assert LIB.kb_cache_fork(None, 16, 16, 16, 16, 16, 16, 2, 4, 8, 2, 9, 16, 64, 16, 1 << 30, None) == INVALID
    assert LIB.kb_cache_fork(16, 16, 16, 16, 16, 16, 16, -2, 4, 8, 2, 9, 16, 64, 16, 1 << 30, None) == INVALID
    assert LIB.kb_cache_fork(16, 16, 16, 16, 16, 16, 16, 2, 4, 8, 2, 9, 0, 64, 16, 1 << 30, None) == INVALID
    assert LIB.kb_cache_append(16, 16, 16, 16, 16, 16, 16, 2, 1, 4, 8, 9, 16, 15, 1, 1, 1, 1, 1, None) == INVALID
    assert LIB.kb_cache_append(16, 16, 16, 16, 16, 16, 16, 2, 0, 4, 8, 9, 16, 16, 1, 1, 1, 1, 1, None) == 0
    assert LIB.kb_cache_free(16, None, 16, 16, 2, 4, 8, 9, None) == INVALID
    assert LIB.kb_cache_free(None, None, None, None, 0, 4, 8, 9, None) == 0
    assert LIB.kb_cache_compact(16, 16, 16, None, 4, 8, 2, 9, 64, 16, 1 << 30, None) == INVALID
    assert LIB.kb_cache_compact(16, 16, 16, 16, 4, 8, 2, 9, 64, 16, 8, None) == WORKSPACE
    assert LIB.kb_cache_copy(16, None, 16, 16, 3, 2, 64, 9, 9, None) == INVALID
    assert LIB.kb_cache_copy(None, None, None, None, 0, 2, 64, 9, 9, None) == 0


@pytest.mark.parametrize("bad,status", [
    (dict(rows=-1), INVALID), (dict(dtype=5), INVALID), (dict(logits=None), INVALID), (dict(stride=10), INVALID),
    (dict(prompt=None), INVALID), (dict(n_output=1 << 20), UNSUPPORTED), (dict(n_bias=2048), UNSUPPORTED),
    (dict(rows=70000), UNSUPPORTED), (dict(rows=0), 0), (dict(vocab=0), 0)])
def test_penalize_refusals(bad, status):
    from kbb200 import LIB

    c = dict(rows=2, vocab=100, stride=100, n_prompt=3, n_output=3, n_bias=3, dtype=0, logits=16, prompt=16) | bad
    assert LIB.kb_penalize_logits(c["logits"], 16, c["prompt"], 16, None, None, None, 16, 16, None, c["rows"], c["vocab"],
                                  c["stride"], c["n_prompt"], c["n_output"], c["n_bias"], 0, c["dtype"], 1, None) == status


def test_tensors_are_checked_before_the_library():
    import torch

    from kbb200 import lm

    x = torch.zeros(2, 1, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        lm.qk_norm_rope(x, x, None, None, x[0], x[0], torch.zeros(2, dtype=torch.int64))
    with pytest.raises(TypeError, match="tensor"):
        lm.penalize_logits([1.0])
    with pytest.raises(RuntimeError, match="CUDA"):
        lm.cache_free(x.int()[0], None, None, None)


# ------------------------------------------------------------ the oracle itself
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rotary", [0, 6, 10])
def test_oracle_gradients_agree_with_differences(rotary, interleaved):
    rng = np.random.default_rng(rotary)
    x, w, dz = rng.standard_normal((3, 2, 10)), rng.standard_normal(10), rng.standard_normal((3, 2, 10))
    a = rng.standard_normal((3, rotary // 2))
    args = (np.cos(a), np.sin(a), rotary, interleaved, 1e-5)
    dx, dw = O.norm_rope_backward(dz, x, w, *args)
    h = 1e-6

    def value(x, w):
        return (dz * O.norm_rope(x, w, *args)).sum()

    for at in np.ndindex(x.shape):
        e = np.zeros(x.shape)
        e[at] = h
        assert abs((value(x + e, w) - value(x - e, w)) / (2 * h) - dx[at]) < 1e-7
    for at in range(10):
        e = np.zeros(10)
        e[at] = h
        assert abs((value(x, w + e) - value(x, w - e)) / (2 * h) - dw[at]) < 1e-7


def test_oracle_attention_of_one_sequence_is_softmax():
    rng = np.random.default_rng(0)
    k, v = rng.standard_normal((2, 5, 4, 1, 6))
    q = rng.standard_normal((1, 1, 2, 6))
    out, lse, _ = O.shared_prefix_attention(q, k, v, [3, 0], np.array([[9, 9, 4]]), [10], 0.5)
    keys = np.concatenate((k[3], k[0], k[4]))[:10, 0]
    values = np.concatenate((v[3], v[0], v[4]))[:10, 0]
    s = 0.5 * q[0, 0] @ keys.T
    p = np.exp(s)
    np.testing.assert_allclose(out[0, 0], p @ values / p.sum(-1, keepdims=True), rtol=1e-12)
    np.testing.assert_allclose(lse[0, 0], np.log(p.sum(-1)), rtol=1e-12)

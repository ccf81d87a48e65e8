"""GPU: the decoding example against the same model computed plainly, in 64 bits and without a cache."""
from __future__ import annotations

import importlib.util
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import lm as O

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parent.parent / "kernelbench-hip_b200" / "examples" / "best_of_n.py"


def load_example():
    spec = importlib.util.spec_from_file_location("best_of_n", EXAMPLE)
    mod = importlib.util.module_from_spec(spec)
    sys.modules["best_of_n"] = mod
    spec.loader.exec_module(mod)
    return mod


def plain_logits(model, tokens):
    """Logits [length, vocab] of one sequence, in 64 bits."""
    s = model.s

    def d(t):
        return t.double().cpu().numpy()

    def norm(x, w):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5) * d(w)

    n = len(tokens)
    x = d(model.embedding)[tokens]
    cos, sin = d(model.cos)[:n], d(model.sin)[:n]
    for w in model.layers:
        qkv = norm(x, w["norm"]) @ d(w["qkv"])
        hq, hkv, dim = s.heads_q, s.heads_kv, s.dim
        q = O.norm_rope(qkv[:, : hq * dim].reshape(n, hq, dim), d(w["q_norm"]), cos, sin, dim, False, 1e-6)
        k = O.norm_rope(qkv[:, hq * dim: (hq + hkv) * dim].reshape(n, hkv, dim), d(w["k_norm"]), cos, sin, dim, False, 1e-6)
        v = qkv[:, (hq + hkv) * dim:].reshape(n, hkv, dim)
        o, _, _ = O.shared_prefix_attention(q[None], k[None], v[None], [], np.zeros((1, 1), dtype=int), [n], dim ** -0.5)
        x = x + o[0].reshape(n, -1) @ d(w["out"])
        h = norm(x, w["norm2"]) @ d(w["up"])
        x = x + (0.5 * h * (1 + np.tanh(np.sqrt(2 / np.pi) * (h + 0.044715 * h ** 3)))) @ d(w["down"])
    return norm(x, model.norm) @ d(model.head)


@pytest.mark.parametrize("length,samples,steps", [(37, 5, 12), (32, 3, 20), (1, 2, 3)])
def test_generate_matches_the_model_without_a_cache(length, samples, steps, cuda_device):
    ex = load_example()
    model = ex.Decoder(ex.Sizes(vocab=120, heads_q=4, heads_kv=2, dim=32, hidden=64, page=8, longest=128))
    prompt = torch.randint(0, 120, (length,), device=cuda_device)
    made, logits = ex.generate(model, prompt, samples, steps, seed=1)
    assert ((made >= 0) & (made < 120)).all()
    for i in range(samples):
        want = plain_logits(model, prompt.tolist() + made[i, :-1].tolist())[length - 1:]
        # two layers of fp32 products of depth 128: the library's tolerance for contractions
        np.testing.assert_allclose(logits[i].double().cpu().numpy(), want, rtol=1e-3, atol=1e-3)


def test_generate_with_an_end_token(cuda_device):
    ex = load_example()
    model = ex.Decoder(ex.Sizes(vocab=8, heads_q=4, heads_kv=2, dim=32, hidden=64, page=8, longest=128))
    prompt = torch.randint(0, 8, (11,), device=cuda_device)
    made, _ = ex.generate(model, prompt, 16, 24, seed=2, end_token=3)
    rows = made.tolist()
    assert any(3 in r for r in rows)
    for r in rows:
        if 3 in r[:-1]:
            at = r.index(3)
            assert all(t == -1 for t in r[at + 1:])
        assert all(t != -1 for t in (r[: r.index(3) + 1] if 3 in r else r))


def test_the_command_runs():
    r = subprocess.run([sys.executable, str(EXAMPLE), "--samples", "3", "--steps", "4"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    assert len(r.stdout.splitlines()) == 3

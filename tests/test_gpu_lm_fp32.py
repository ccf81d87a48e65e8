"""GPU: long fp32 prefixes, whose kernel holds every operand as two fp16 halves: the magnitudes of other heads, of
other sequences' queries and of ended slots cost a result none of its bits.

Tolerances, per result: a score is off by at most e = (dim + 16) U scale max_j sum |q k_j| (as in test_gpu_lm), and by
what elements far below a head's largest lose, 2^-38 of that largest against each of q's elements; values likewise
2^-38 of their head's largest, and out by 2 e + 2^-20 of softmax @ |v|."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import lm as O
from tests.test_gpu_lm import U, attention_inputs, f64, within

pytestmark = pytest.mark.gpu

SHAPES = [(40, 1, 16, 4, 64, 16, 460, 30), (33, 2, 8, 2, 80, 24, 300, 50)]  # past 1.2e9 operations


def check_rows(args, scale=None):
    from kbb200 import lm

    q, k, v, prefix, table, lens = args
    out, lse = lm.shared_prefix_attention(*args, scale=scale)
    B, Q, hq, d = q.shape
    sc = d ** -0.5 if scale is None else scale
    q64, k64, v64, n = f64(q), f64(k), f64(v), lens.cpu().numpy()
    group = hq // k.shape[2]
    want, want_lse, mag = O.shared_prefix_attention(q64, k64, v64, prefix.cpu().numpy(), table.cpu().numpy(), n, sc)
    e, tiny = np.zeros((B, Q, hq)), np.zeros(hq)
    for h in range(hq):
        used = [np.unique(prefix.cpu().numpy())] + [np.unique(table.cpu().numpy()[:, prefix.numel():])]
        kh = np.concatenate([np.abs(k64[u, :, h // group]).reshape(-1, d) for u in used])
        vh = np.concatenate([np.abs(v64[u, :, h // group]).reshape(-1, d) for u in used])
        for b in range(B):
            a = np.abs(q64[b, :, h])
            e[b, :, h] = (d + 16) * U * abs(sc) * (a @ kh.T).max(-1) + 2.0 ** -38 * abs(sc) * a.sum(-1) * kh.max()
        tiny[h] = 2.0 ** -37 * vh.max()
    top = np.where(np.isfinite(want_lse), np.abs(want_lse), 0)
    within(out, want, U * np.abs(want) + (2 * e + 2.0 ** -20)[..., None] * mag + tiny[:, None], "out")
    within(lse, want_lse, e + 2.0 ** -20 + 4 * U * top, "lse")
    return out


@pytest.mark.parametrize("shape", SHAPES)
def test_heads_of_different_magnitudes(shape, cuda_device):
    """Keys and values of one head 2^30 below the others', its queries as far above them: ordinary scores."""
    q, k, v, prefix, table, lens = attention_inputs(cuda_device, torch.float32, *shape, seed=21)
    group = shape[2] // shape[3]
    k[:, :, 1] *= 2.0 ** -30
    v[:, :, 1] *= 2.0 ** -30
    q[:, :, group: 2 * group] *= 2.0 ** 30
    check_rows((q, k, v, prefix, table, lens))


@pytest.mark.parametrize("shape", SHAPES)
def test_queries_of_different_magnitudes(shape, cuda_device):
    """One sequence's queries 2^30 times the others', whose scores are ordinary."""
    q, k, v, prefix, table, lens = attention_inputs(cuda_device, torch.float32, *shape, seed=22)
    q[3] *= 2.0 ** 30
    q[4] *= 2.0 ** -20
    check_rows((q, k, v, prefix, table, lens))


@pytest.mark.parametrize("garbage", [1e30, float("inf"), float("nan")])
@pytest.mark.parametrize("shape", SHAPES)
def test_ended_slots_hold_anything(shape, garbage, cuda_device):
    """The queries of a slot without keys are whatever stood in the buffer."""
    from kbb200 import lm

    q, k, v, prefix, table, lens = args = attention_inputs(cuda_device, torch.float32, *shape, seed=23)
    lens[5] = 0
    want = check_rows(args)
    q[5] = garbage
    out, lse = lm.shared_prefix_attention(*args)
    assert torch.equal(out, want) and (out[5] == 0).all() and torch.isinf(lse[5]).all()


@pytest.mark.parametrize("of_q,of_k", [(1e-25, 1e-25), (1e-30, 1e20), (1e25, 1e-25), (1e-38, 1.0)])
def test_magnitudes_near_the_ends_of_fp32(of_q, of_k, cuda_device):
    q, k, v, prefix, table, lens = attention_inputs(cuda_device, torch.float32, *SHAPES[0], seed=24)
    check_rows((q * of_q, k * of_k, v, prefix, table, lens))

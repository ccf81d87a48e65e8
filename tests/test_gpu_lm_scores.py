"""GPU: attention with scores so large that only the largest key counts, down to ties: the kernels that hold a row's
reference in units of log2 must not lose it to the last place of a large number.

Queries and keys are small whole numbers and the scale a power of two, so that raw scores are exact and lie at least
2^10 apart: all weight is on the largest.  How keys that tie share it is not the formula's to say here, for a score of
2^24 has no place for the rounding of one unit in a part's lse.  So an output lies between the least and the largest of
their values, give or take the type's rounding of weights (u) and output (u) and 2^-20, and in fp32 2^-37 of the
largest value, as in test_gpu_lm_fp32; lse by eight roundings of its magnitude and the logarithm of the number of
ties."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.test_gpu_lm import U, UNIT, attention_inputs, f64, within

pytestmark = pytest.mark.gpu

SHAPES = [  # the kernels for few rows, for more of them, and on tensor cores (fp32: in halves)
    (3, 1, 8, 2, 64, 16, 5, 40), (30, 2, 8, 1, 256, 16, 40, 20), (150, 3, 6, 2, 64, 8, 60, 33), (40, 1, 16, 4, 64, 16, 460, 30)]


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("power", [10, 18, 22, 25, 27, 31, 36])
@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_only_the_largest_key_counts(shape, dt, power, sign, cuda_device):
    from kbb200 import lm

    q, k, v, prefix, table, lens = attention_inputs(cuda_device, dt, *shape, seed=power)
    q, k = (x.sign() * (x.abs() > 0.7) for x in (q, k))  # -1, 0, 1
    scale = sign * 2.0 ** power
    out, lse = lm.shared_prefix_attention(q, k, v, prefix, table, lens, scale=scale)
    B, Q, hq, d = q.shape
    page, group, q64, k64, v64 = k.shape[1], hq // k.shape[2], f64(q), f64(k), f64(v)
    rows = torch.cat([prefix[None].expand(B, -1), table[:, prefix.numel():]], 1).cpu().numpy()
    low, high, mag, want_lse = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape), np.full((B, Q, hq), -np.inf)
    for b in range(B):
        n = int(lens[b])
        ks, vs = (x[rows[b]].reshape(-1, *x.shape[2:]) for x in (k64, v64))
        for t in range(Q):
            m = n - Q + 1 + t
            if m <= 0:
                continue
            for h in range(hq):
                s = scale * (ks[:m, h // group] @ q64[b, t, h])
                top = s == s.max()
                values = vs[:m, h // group][top]
                low[b, t, h], high[b, t, h], mag[b, t, h] = values.min(0), values.max(0), np.abs(values).max(0)
                want_lse[b, t, h] = s.max() + np.log(top.sum())
    rounded = 0.0 if dt == torch.float32 else UNIT[dt]
    got, tiny = f64(out), 2.0 ** -37 * np.abs(v64).max() if dt == torch.float32 else 0.0
    within(got, np.clip(got, low, high), (UNIT[dt] + rounded + 2.0 ** -20) * mag + tiny, "out")
    lse_tol = 8 * U * np.where(np.isfinite(want_lse), np.abs(want_lse), 0) + 2.0 ** -20
    within(lse, want_lse, lse_tol, "lse")

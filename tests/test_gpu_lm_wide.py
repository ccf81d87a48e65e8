"""GPU: attention over a shared prefix with enough query rows for the wide kernels (tensor cores for fp16 and bf16,
16 rows a warp for fp32) at short and ragged prefixes, with the tolerances of test_gpu_lm."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_lm import attention_inputs, check_attention

pytestmark = pytest.mark.gpu

HALF = [torch.float16, torch.bfloat16]
WIDE = [  # B, Q, hq, hkv, d, page, prefix pages, suffix; rows x dim x keys past 3e7
    (430, 1, 4, 1, 128, 16, 9, 20), (150, 3, 6, 2, 64, 8, 60, 33), (260, 2, 4, 2, 96, 32, 11, 5),
    (81, 1, 8, 1, 128, 128, 3, 60), (51, 1, 16, 2, 80, 256, 4, 9), (9, 1, 8, 1, 128, 16, 300, 0),
    (500, 1, 5, 1, 16, 64, 44, 3), (129, 1, 1, 1, 64, 24, 160, 1), (33, 4, 7, 1, 72, 16, 33, 2),
]


@pytest.mark.parametrize("dt", HALF + [torch.float32])
@pytest.mark.parametrize("shape", WIDE)
def test_wide(shape, dt, cuda_device):
    check_attention(attention_inputs(cuda_device, dt, *shape, seed=sum(shape)), dt)


@pytest.mark.parametrize("dt", HALF + [torch.float32])
@pytest.mark.parametrize("scale", [None, -0.07, 0.0])
def test_wide_scales_and_strides(dt, scale, cuda_device):
    q, k, v, prefix, table, lens = attention_inputs(cuda_device, dt, 200, 1, 8, 2, 64, 16, 50, 40, seed=5)
    pool = torch.stack((k, v), 2)  # [pages, page, 2, heads, dim]
    packed = torch.cat((q.flatten(2), q.flatten(2)), -1)
    args = (packed[..., : 8 * 64].view(200, 1, 8, 64), pool[:, :, 0], pool[:, :, 1], prefix, table, lens)
    check_attention(args, dt, scale=scale)


def test_long_fp32_prefix_without_a_scale(cuda_device):
    """All keys alike, by scale or by one that vanishes next to the keys' magnitude."""
    q, k, v, prefix, table, lens = attention_inputs(cuda_device, torch.float32, 40, 1, 16, 4, 64, 16, 460, 30, seed=12)
    lens[3:6] = torch.tensor([0, 1, 100], device=cuda_device)
    for scale in (0.0, 1e-37):
        check_attention((q, k, v, prefix, table, lens), torch.float32, scale=scale)


@pytest.mark.parametrize("dt", HALF + [torch.float32])
def test_wide_empty_and_short_rows(dt, cuda_device):
    """Ended slots, sequences shorter than the prefix and than their queries, whole tiles of rows without keys."""
    B = 300
    lens = torch.arange(B) % 290
    lens[:70] = 0
    lens[100:103] = torch.tensor([1, 2, -4])
    lens[299] = 330
    args = attention_inputs(cuda_device, dt, B, 2, 4, 1, 128, 16, 18, 50, lens=lens, seed=6)
    out, lse = check_attention(args, dt)
    assert (out[:70] == 0).all() and torch.isinf(lse[:70]).all()


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("longest", [1, 100, 129, 250, 287])
def test_wide_end_inside_a_tile(dt, longest, cuda_device):
    """No sequence reaches the end of the prefix; what lies past the longest is NaN and infinity."""
    q, k, v, prefix, table, lens = attention_inputs(cuda_device, dt, 300, 1, 4, 1, 128, 16, 18, 10, seed=longest)
    lens = torch.randint(0, longest + 1, (300,), device=cuda_device, dtype=torch.int32)
    lens[7] = longest
    args = (q, k, v, prefix, table, lens)
    out, lse = check_attention(args, dt)
    for t in (k, v):
        t[prefix[longest // 16].long(), longest % 16:] = float("nan")
        t[prefix[longest // 16 + 1:].long()] = float("inf")
        t[table[:, 18:].long()] = float("nan")
    from kbb200 import lm
    again = lm.shared_prefix_attention(*args)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("dt", HALF)
def test_wide_large_scores(dt, cuda_device):
    """The running maximum moves by hundreds, and grows from tile to tile."""
    q, k, v, prefix, table, lens = attention_inputs(cuda_device, dt, 200, 1, 4, 1, 128, 16, 96, 20, seed=8, spread=20.0)
    k[prefix.long()] *= torch.linspace(0.1, 2.0, 96, device=cuda_device).to(dt)[:, None, None, None]
    check_attention((q, k, v, prefix, table, lens), dt)

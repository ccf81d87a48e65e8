"""GPU: attention with heads above 128 columns and more rows than the 16-row kernel takes, with the tolerances of
test_gpu_lm."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_lm import attention_inputs, check_attention

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
# B, Q, hq, hkv, d, page, prefix pages, suffix; rows x dim x keys past 3e7 over the prefix
PREFIX = [(100, 1, 1, 1, 256, 16, 76, 20), (42, 2, 4, 2, 192, 32, 31, 40), (80, 1, 1, 1, 136, 24, 120, 3)]
# the same over the sequences' own keys: prompts, with and without a prefix before them
PROMPT = [(1, 301, 4, 1, 256, 16, 0, 301), (2, 200, 2, 1, 192, 16, 3, 600), (1, 260, 3, 1, 144, 8, 0, 260)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", PREFIX + PROMPT)
def test_large_heads(shape, dt, cuda_device):
    check_attention(attention_inputs(cuda_device, dt, *shape, seed=sum(shape)), dt)


def test_large_heads_in_fp32_of_any_whole_vectors(cuda_device):
    """132 columns: whole 16-byte vectors of fp32 that are not whole tiles of eight."""
    check_attention(attention_inputs(cuda_device, torch.float32, 90, 1, 1, 1, 132, 16, 180, 30, seed=1), torch.float32)

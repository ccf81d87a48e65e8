"""GPU: calls at the limits that the entries state."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_lm import ints

pytestmark = pytest.mark.gpu


def test_fork_into_the_most_slots(cuda_device):
    """2^20 requests: every slot a copy of slot 0, which stays what it is."""
    from kbb200 import lm

    n, page = 1 << 20, 2
    pool = torch.randn(2, 3, page, 1, 4, device=cuda_device)
    table = torch.full((n, 1), -1, device=cuda_device, dtype=torch.int32)
    lens, refs = torch.zeros(n, device=cuda_device, dtype=torch.int32), ints(cuda_device, [0, 1, 0])
    table[0], lens[0], before = 1, page, pool.clone()
    granted = lm.cache_fork(pool, table, lens, refs, torch.zeros_like(lens), torch.arange(n, device=cuda_device).int())
    assert (granted == 1).all() and (table == 1).all() and (lens == page).all()
    assert refs.tolist() == [0, n, 0] and torch.equal(pool, before)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,n_pre", [(3, 5), (200, 70)])
def test_attention_of_the_least_length(batch, n_pre, dt, cuda_device):
    """A length of -2^31, as a sentinel or left over, is a slot without keys."""
    from kbb200 import lm
    from tests.test_gpu_lm import attention_inputs

    args = q, k, v, prefix, table, lens = attention_inputs(cuda_device, dt, batch, 4, 4, 1, 128, 16, n_pre, 40, seed=2)
    lens[1] = 0
    want, want_lse = lm.shared_prefix_attention(*args)
    lens[1] = -2 ** 31
    out, lse = lm.shared_prefix_attention(*args)
    assert (out[1] == 0).all() and (lse[1] == -float("inf")).all()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_append_to_the_least_length(cuda_device):
    from kbb200 import lm

    width, page = 1 << 20, 1 << 12  # a row of 2^32 places
    pool = torch.zeros(2, 2, page, 1, 4, device=cuda_device)
    table = torch.zeros(1, width, device=cuda_device, dtype=torch.int32)
    k = torch.ones(1, 3, 1, 4, device=cuda_device)
    lm.cache_append(k, k, pool[0], pool[1], table, ints(cuda_device, [-2 ** 31]), ints(cuda_device, [0]))
    assert (pool == 0).all()

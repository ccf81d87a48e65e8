"""GPU: a request that the cache refuses leaves everyone's keys as they were, through the append that follows it."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.test_gpu_lm import ints
from tests.test_gpu_lm_example import load_example, plain_logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens", [1, 3, 6])
@pytest.mark.parametrize("free", [0, 1, 2])
def test_append_passes_refused_slots_over(free, tokens, dt, cuda_device):
    """A slot of two full pages and two forks of it, which share them; a pool with too few pages for all."""
    from kbb200 import lm

    page, h, d, held = 4, 2, 8, 2
    pages = held + free
    g = torch.Generator(device=cuda_device).manual_seed(free)
    pool = torch.randn(2, pages, page, h, d, device=cuda_device, generator=g).to(dt)
    table = torch.full((3, 5), -1, dtype=torch.int32, device=cuda_device)
    table[0, :held] = torch.arange(held, device=cuda_device, dtype=torch.int32)
    lens, refs = ints(cuda_device, [held * page, 0, 0]), torch.zeros(pages, dtype=torch.int32, device=cuda_device)
    refs[:held] = 1
    lm.cache_fork(pool, table, lens, refs, ints(cuda_device, [0, 0]), ints(cuda_device, [1, 2]))
    want = pool.clone()
    seqs = ints(cuda_device, [2, 0, 1])
    granted = lm.cache_reserve(table, lens, refs, seqs, tokens, page)
    each = -(-tokens // page)
    assert granted.tolist() == [int((i + 1) * each <= free) for i in range(3)]
    k, v = (torch.randn(3, tokens, h, d, device=cuda_device, generator=g).to(dt) for _ in range(2))
    lm.cache_append(k, v, pool[0], pool[1], table, lens, seqs, granted)
    for i, (slot, ok) in enumerate(zip(seqs.tolist(), granted.tolist())):
        for t in range(tokens if ok else 0):
            at = int(table[slot, held + t // page])
            want[0, at, t % page], want[1, at, t % page] = k[i, t], v[i, t]
    assert torch.equal(pool, want)


def test_append_checks_granted(cuda_device):
    from kbb200 import lm

    pool = torch.zeros(2, 3, 4, 1, 8, device=cuda_device)
    table, lens = ints(cuda_device, [[0, 1]]), ints(cuda_device, [5])
    k, one = torch.ones(1, 1, 1, 8, device=cuda_device), ints(cuda_device, [0])
    with pytest.raises(RuntimeError, match="granted"):
        lm.cache_append(k, k, pool[0], pool[1], table, lens, one, ints(cuda_device, [1, 1]))
    with pytest.raises(RuntimeError, match="granted"):
        lm.cache_append(k, k, pool[0], pool[1], table, lens, one, one.long())
    with pytest.raises(TypeError, match="granted"):
        lm.cache_append(k, k, pool[0], pool[1], table, lens, one, [1])
    assert (pool == 0).all()


@pytest.mark.parametrize("spare", [0, 1, 2])
def test_samples_end_where_the_cache_is_full(spare, cuda_device):
    """The prompt fills whole pages, which all samples share; only `spare` of five samples get a page of their own."""
    ex = load_example()
    model = ex.Decoder(ex.Sizes(vocab=120, heads_q=4, heads_kv=2, dim=32, hidden=64, page=8, longest=128))
    prompt = torch.randint(0, 120, (16,), device=cuda_device, generator=torch.Generator(cuda_device).manual_seed(spare))
    made, logits = ex.generate(model, prompt, 5, 8, seed=1, pages=2 + spare)
    for i in range(5):
        n = 8 if i < spare else 1  # the prompt's own logits give every sample its first token
        assert (made[i, :n] >= 0).all() and (made[i, n:] == -1).all()
        want = plain_logits(model, prompt.tolist() + made[i, : n - 1].tolist())[15:]
        np.testing.assert_allclose(logits[i, :n].double().cpu().numpy(), want, rtol=1e-3, atol=1e-3)


def test_a_prompt_that_does_not_fit(cuda_device):
    ex = load_example()
    model = ex.Decoder(ex.Sizes(vocab=120, heads_q=4, heads_kv=2, dim=32, hidden=64, page=8, longest=128))
    with pytest.raises(RuntimeError, match="fit"):
        ex.generate(model, torch.zeros(17, device=cuda_device, dtype=torch.int64), 2, 4, pages=3)

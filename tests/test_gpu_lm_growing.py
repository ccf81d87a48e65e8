"""GPU: sequences that grow: reserve, append and attention read one another's table and lengths in place, step after
step without a pause, and give the bits of the same steps with a synchronisation after every call."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

# dtype, sequences, prefix pages of 16 keys, dim: no prefix; one launch for the prefix and the own keys; a launch each
# (16-row tiles beside wider ones, tensor cores, tensor cores in halves)
GROWING = [(torch.bfloat16, 9, 0, 128), (torch.float16, 4, 3, 64), (torch.bfloat16, 60, 60, 192), (torch.bfloat16, 48, 120, 128),
           (torch.float16, 40, 300, 64), (torch.float32, 48, 480, 128)]


@pytest.mark.parametrize("in_graph", [False, True])
@pytest.mark.parametrize("dt,batch,n_pre,dim", GROWING)
def test_growing_sequences_without_pauses(dt, batch, n_pre, dim, in_graph, cuda_device):
    from kbb200 import lm

    page, hkv, group, own, steps = 16, 2, 4, 4, 25
    pages = n_pre + batch * own
    g = torch.Generator(device=cuda_device).manual_seed(batch)
    pool0 = torch.randn(2, pages, page, hkv, dim, device=cuda_device, generator=g).to(dt)
    prefix = torch.arange(n_pre, device=cuda_device, dtype=torch.int32)
    table0 = torch.full((batch, n_pre + own), -1, device=cuda_device, dtype=torch.int32)
    table0[:, :n_pre] = prefix
    refs0 = torch.zeros(pages, device=cuda_device, dtype=torch.int32)
    refs0[:n_pre] = batch
    seqs = torch.arange(batch, device=cuda_device, dtype=torch.int32)
    q = torch.randn(steps, batch, 1, hkv * group, dim, device=cuda_device, generator=g).to(dt)
    kv = torch.randn(steps, 2, batch, 2, hkv, dim, device=cuda_device, generator=g).to(dt)
    pool, table, refs, lens = pool0.clone(), table0.clone(), refs0.clone(), torch.empty_like(seqs)

    def run(between=lambda: None):
        pool.copy_(pool0), table.copy_(table0), refs.copy_(refs0), lens.fill_(n_pre * page)
        between()
        made = []
        for i in range(steps):
            granted = lm.cache_reserve(table, lens, refs, seqs, 2, page)
            between()
            lm.cache_append(kv[i, 0], kv[i, 1], pool[0], pool[1], table, lens, seqs, granted)
            between()
            made += lm.shared_prefix_attention(q[i], pool[0], pool[1], prefix, table, lens)
            between()
        return made

    want = [t.clone() for t in run(torch.cuda.synchronize)]
    if in_graph:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run()
    for _ in range(4):
        if in_graph:
            graph.replay()
        else:
            got = run()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)

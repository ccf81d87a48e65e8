"""GPU: calls that follow one another without a pause.  The launches of the language-model operators begin while
the launch before them ends, so a chain of calls behind a slow producer has to give the bits of the same chain
with a synchronisation after every call; in a captured graph, too."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

# dtype, sequences, prefix pages of 16 keys: each of the kernels that can take the prefix (16-row tiles, wider
# ones, tensor cores, tensor cores in halves), and no prefix
STEPS = [(torch.bfloat16, 2, 3, 128), (torch.bfloat16, 24, 40, 128), (torch.float16, 40, 20, 192),
         (torch.float32, 6, 5, 64), (torch.float32, 48, 480, 128), (torch.bfloat16, 5, 0, 128)]


class Step:
    """One decoding step of `batch` sequences: rotation, append, attention, penalties."""

    def __init__(self, dev, dt, batch, n_pre, dim):
        from kbb200 import lm

        g = torch.Generator(device=dev).manual_seed(batch)
        self.page, self.hkv, self.group, own = 16, 2, 4, 4
        pages = n_pre + batch * own
        self.source = torch.randn(batch, (2 + self.group) * self.hkv * dim, device=dev, generator=g)
        self.packed = torch.zeros(batch, (2 + self.group) * self.hkv * dim, device=dev, dtype=dt)
        self.pool0 = torch.randn(2, pages, self.page, self.hkv, dim, device=dev, generator=g).to(dt)
        self.pool = self.pool0.clone()
        self.prefix = torch.arange(n_pre, device=dev, dtype=torch.int32)
        own_pages = n_pre + torch.randperm(batch * own, device=dev, generator=g, dtype=torch.int32).view(batch, own)
        self.table = torch.cat([self.prefix.expand(batch, n_pre), own_pages], 1).contiguous()
        self.lens = n_pre * self.page + torch.randint(1, own * self.page + 1, (batch,), device=dev, generator=g,
                                                      dtype=torch.int32)
        self.seqs = torch.arange(batch, device=dev, dtype=torch.int32)
        self.cos, self.sin = lm.rope_tables(8192, dim, device=dev)
        self.ones = torch.ones(dim, device=dev)
        self.logits = torch.randn(batch, 5000, device=dev, generator=g).to(dt)
        self.history = torch.randint(0, 5000, (batch, 40), device=dev, generator=g)
        self.recent = self.history[:, :7].contiguous()
        self.repetition = torch.full((batch,), 1.25, device=dev)
        self.slow = torch.randn(1 << 25, device=dev, generator=g)
        self.dim, self.dt, self.batch = dim, dt, batch

    def run(self, between=lambda: None):
        from kbb200 import lm

        self.pool.copy_(self.pool0)
        self.packed.zero_()
        between()
        for _ in range(3):
            self.slow.mul_(-1.0)
        self.packed.copy_(self.source)  # by a kernel (it converts) or a copy
        between()
        x = self.packed.view(self.batch, -1, self.dim)
        hq = self.group * self.hkv
        q, k = lm.qk_norm_rope(x[:, :hq], x[:, hq:hq + self.hkv], self.ones, None, self.cos, self.sin, self.lens - 1)
        between()
        lm.cache_append(k[:, None], x[:, None, hq + self.hkv:], self.pool[0], self.pool[1], self.table, self.lens,
                        self.seqs)
        between()
        out, lse = lm.shared_prefix_attention(q[:, None], self.pool[0], self.pool[1], self.prefix, self.table, self.lens)
        between()
        y = lm.penalize_logits(self.logits + lse[:, 0, :1].to(self.dt), prompt=self.history, output=self.recent,
                               repetition=self.repetition, presence=self.repetition)
        between()
        kept = [t.clone() for t in (q, k, out, lse, y, self.pool)]
        dx = lm.qk_norm_rope_backward(q, k, x[:, :hq], x[:, hq:hq + self.hkv], self.ones, None, self.cos, self.sin,
                                      self.lens - 1)
        between()
        return kept + [t for t in dx if t is not None]


@pytest.mark.parametrize("dt,batch,n_pre,dim", STEPS)
def test_step_without_pauses(dt, batch, n_pre, dim, cuda_device):
    s = Step(cuda_device, dt, batch, n_pre, dim)
    for i in range(4):
        s.source.normal_(generator=torch.Generator(device=cuda_device).manual_seed(i))
        want = s.run(torch.cuda.synchronize)
        got = s.run()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dt,batch,n_pre,dim", STEPS)
def test_step_in_a_graph(dt, batch, n_pre, dim, cuda_device):
    s = Step(cuda_device, dt, batch, n_pre, dim)
    s.run(torch.cuda.synchronize)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = s.run()
    for i in range(4):
        s.source.normal_(generator=torch.Generator(device=cuda_device).manual_seed(i))
        want = s.run(torch.cuda.synchronize)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


# children and table width: the fork whose plan writes the rows, and the one of three launches
@pytest.mark.parametrize("children,width", [(5, 8), (40, 60)])
def test_cache_calls_without_pauses(children, width, cuda_device):
    from kbb200 import lm

    def ints(*v):
        return torch.tensor(v, device=cuda_device, dtype=torch.int32)

    page, held = 8, width - 2
    pages = held + 4 * children + 9
    pool0 = torch.randn(4, pages, page, 2, 64, device=cuda_device)
    slow = torch.randn(1 << 25, device=cuda_device)

    def run(between=lambda: None):
        table = torch.full((children + 2, width), -1, device=cuda_device, dtype=torch.int32)
        lens = torch.zeros(children + 2, device=cuda_device, dtype=torch.int32)
        refs = torch.zeros(pages, device=cuda_device, dtype=torch.int32)
        pool = pool0.clone()
        between()
        for _ in range(3):
            slow.mul_(-1.0)
        refs[:3] = 1  # pages of someone else, so that the compaction has what to move
        between()
        made = [lm.cache_reserve(table, lens, refs, ints(1), held * page - 3, page)]
        between()
        refs[:3] = 0
        kids = torch.arange(2, children + 2, device=cuda_device, dtype=torch.int32)
        made.append(lm.cache_fork(pool, table, lens, refs, torch.ones_like(kids), kids))
        between()
        made.append(lm.cache_reserve(table, lens, refs, kids, 7, page))
        between()
        kv = torch.randn(children, 7, 2, 64, device=cuda_device, generator=torch.Generator(device=cuda_device).manual_seed(3))
        lm.cache_append(kv, -kv, pool[0], pool[1], table, lens, kids)
        between()
        lm.cache_free(table, lens, refs, kids[::2].contiguous())
        between()
        made.append(lm.cache_compact(pool, table, refs))
        between()
        # swapped: each is the other's parent
        made.append(lm.cache_fork(pool, table, lens, refs, ints(3, 1), ints(1, 3)))
        between()
        lm.cache_copy(pool, ints(0, 1), pool, ints(pages - 1, pages - 2))
        between()
        return made + [table, lens, refs, pool]

    for _ in range(4):
        want = run(torch.cuda.synchronize)
        got = run()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)

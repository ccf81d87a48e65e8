"""GPU: drafts that are rejected.  Their program lowers a slot's lens; no page is lost by that."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_lm import ints

pytestmark = pytest.mark.gpu


def holders(table, pages):
    flat = table[table >= 0].long()
    return torch.bincount(flat, minlength=pages).int()


@pytest.mark.parametrize("page", [1, 3, 4, 16])
@pytest.mark.parametrize("drafts", [1, 5, 13])
def test_no_page_is_lost(page, drafts, cuda_device):
    """Rounds of drafts with any number accepted, in a pool that is just large enough; then everything is freed."""
    from kbb200 import lm

    slots, rounds = 7, 20
    g = torch.Generator().manual_seed(page + drafts)
    width = -(-(rounds * drafts + 1) // page) + 1
    pages = slots * width
    table = torch.full((slots, width), -1, device=cuda_device, dtype=torch.int32)
    lens, refs = torch.zeros(slots, device=cuda_device, dtype=torch.int32), torch.zeros(pages, device=cuda_device, dtype=torch.int32)
    pool = torch.zeros(2, pages, page, 1, 4, device=cuda_device)
    seqs = torch.arange(slots, device=cuda_device, dtype=torch.int32)
    want = [[] for _ in range(slots)]  # every slot's keys
    for i in range(rounds):
        assert (lm.cache_reserve(table, lens, refs, seqs, drafts, page) == 1).all()
        k = torch.randn(slots, drafts, 1, 4, generator=g).to(cuda_device)
        lm.cache_append(k, -k, pool[0], pool[1], table, lens, seqs)
        accepted = torch.randint(0, drafts + 1, (slots,), generator=g)
        lens -= (drafts - accepted).int().to(cuda_device)
        for s in range(slots):
            want[s] += [k[s, t] for t in range(accepted[s])]
        assert torch.equal(refs, holders(table, pages))
        if i % 7 == 6:
            lm.cache_compact(pool, table, refs)
            assert torch.equal(refs, holders(table, pages))
    for s in range(slots):
        assert int(lens[s]) == len(want[s])
        for j, x in enumerate(want[s]):
            assert torch.equal(pool[0, table[s, j // page], j % page], x)
    lens[2] = 0  # all dropped: what is left in the row is given back, too
    lm.cache_free(table, lens, refs, ints(cuda_device, [0, 1, 2, 3, 4, 5, 6, 2]))
    assert (refs == 0).all() and (table == -1).all() and (lens == 0).all()


def test_a_shortened_slot_as_parent_and_child(cuda_device):
    from kbb200 import lm

    page, pages = 4, 12
    table = torch.full((3, 5), -1, device=cuda_device, dtype=torch.int32)
    lens, refs = torch.zeros(3, device=cuda_device, dtype=torch.int32), torch.zeros(pages, device=cuda_device, dtype=torch.int32)
    pool = torch.randn(2, pages, page, 1, 4, device=cuda_device)
    lm.cache_reserve(table, lens, refs, ints(cuda_device, [0, 1]), 14, page)
    lens[0] -= 8  # two pages, the second half full, and two that stay in the row
    lm.cache_fork(pool, table, lens, refs, ints(cuda_device, [0, 0]), ints(cuda_device, [2, 1]))
    assert lens.tolist() == [6, 6, 6] and torch.equal(refs, holders(table, pages))
    assert table[1, 0] == table[0, 0] and table[1, 1] != table[0, 1] and (table[1:, 2:] == -1).all()
    before = table[0].clone()
    # the kept pages serve a request that the free ones alone would not
    assert lm.cache_reserve(table, lens, refs, ints(cuda_device, [0, 1]), 14, page).tolist() == [1, 1]
    assert torch.equal(table[0, :4], before[:4]) and torch.equal(refs, holders(table, pages)) and lens.tolist() == [20, 20, 6]


def test_a_refused_reserve_keeps_the_pages(cuda_device):
    from kbb200 import lm

    table = torch.full((2, 6), -1, device=cuda_device, dtype=torch.int32)
    lens, refs = torch.zeros(2, device=cuda_device, dtype=torch.int32), torch.zeros(5, device=cuda_device, dtype=torch.int32)
    assert lm.cache_reserve(table, lens, refs, ints(cuda_device, [0, 1]), 8, 4).tolist() == [1, 1]
    lens[0] = 2
    row = table[0].tolist()
    assert lm.cache_reserve(table, lens, refs, ints(cuda_device, [0]), 15, 4).tolist() == [0]  # 17 keys: three pages more
    assert table[0].tolist() == row and lens.tolist() == [2, 8] and refs.tolist() == [1, 1, 1, 1, 0]
    assert lm.cache_reserve(table, lens, refs, ints(cuda_device, [0]), 10, 4).tolist() == [1]
    assert table[0].tolist() == row[:2] + [4, -1, -1, -1] and refs.tolist() == [1] * 5

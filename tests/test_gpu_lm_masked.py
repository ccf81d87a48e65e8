"""GPU: infinite and NaN keys and values reach the queries that see them, and no others: later drafts of a sequence,
later tokens of a prompt, and prefixes that are longer than some sequences."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_lm import attention_inputs

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")
TYPES = [torch.float32, torch.float16, torch.bfloat16]
# B, Q, hq, hkv, d, page, prefix pages, suffix; the kernel for few rows, and the one for more
OWN = [(3, 3, 8, 2, 64, 16, 2, 60), (2, 8, 16, 2, 96, 16, 4, 40), (2, 5, 4, 1, 128, 24, 0, 33), (2, 4, 4, 2, 192, 16, 1, 50),
       (1, 150, 4, 2, 128, 16, 3, 200), (2, 130, 3, 1, 64, 8, 0, 140), (1, 400, 2, 1, 256, 16, 0, 400)]
# rows x dim x keys past 3e7 over the prefix: tensor cores for the 16-bit types
PREFIX = [(260, 1, 4, 1, 128, 16, 24, 5), (200, 1, 6, 2, 64, 64, 16, 20), (150, 2, 4, 1, 96, 128, 4, 9),
          (81, 1, 8, 1, 72, 256, 3, 30), (300, 1, 1, 1, 128, 24, 40, 3), (90, 1, 2, 1, 192, 16, 70, 10)]
LONG = [(40, 1, 16, 4, 64, 16, 460, 30), (33, 2, 8, 2, 80, 24, 300, 50)]  # fp32 in halves


def visible(lens, Q):
    """[batch, queries]: how many keys each query sees."""
    return lens.long()[:, None] - Q + 1 + torch.arange(Q, device=lens.device)


def check(args, places, what):
    """places: (page, slot, key, sequence or None for all): `what` in some columns of the values there."""
    from kbb200 import lm

    q, k, v, prefix, table, lens = args
    Q, d, hkv, group = q.shape[1], q.shape[3], k.shape[2], q.shape[2] // k.shape[2]
    want, want_lse = lm.shared_prefix_attention(*args)
    bad = v.clone()
    touched = torch.zeros(q.shape, dtype=torch.bool, device=q.device)
    for i, (page, slot, key, batch) in enumerate(places):
        h, cols = i % hkv, slice(i % 3, d, 7 + i % 5)
        bad[page, slot, h, cols] = what
        sees = visible(lens, Q) > key
        if batch is not None:
            sees &= (torch.arange(q.shape[0], device=q.device) == batch)[:, None]
        touched[:, :, h * group: (h + 1) * group, cols] |= sees[:, :, None, None]
    out, lse = lm.shared_prefix_attention(q, k, bad, prefix, table, lens)
    assert touched.any() and not touched.all()
    assert not torch.isfinite(out[touched]).any()
    assert torch.equal(out[~touched], want[~touched]) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("what", [NAN, INF, -INF])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", OWN)
def test_values_of_later_tokens(shape, dt, what, cuda_device):
    args = q, k, v, prefix, table, lens = attention_inputs(cuda_device, dt, *shape, seed=sum(shape))
    B, Q, page = shape[0], shape[1], shape[5]
    lens.clamp_(min=prefix.numel() * page + Q)
    places = []
    for b in range(B):
        for back in {0, 1, Q // 2, Q - 2}:
            key = int(lens[b]) - 1 - back
            places.append((int(table[b, key // page]), key % page, key, b))
    check(args, places, what)


@pytest.mark.parametrize("what", [NAN, INF, -INF])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", PREFIX + LONG)
def test_values_past_short_sequences(shape, dt, what, cuda_device):
    args = q, k, v, prefix, table, lens = attention_inputs(cuda_device, dt, *shape, seed=sum(shape))
    B, page, keys = shape[0], shape[5], prefix.numel() * shape[5]
    lens[1: B // 2] = torch.randint(1, keys, (B // 2 - 1,), device=cuda_device, dtype=torch.int32)
    lens[B // 2] = 0
    places = [(int(prefix[key // page]), key % page, key, None) for key in (int(lens[1]) - 1, int(lens[2]), keys - 1, keys // 2)]
    check(args, places, what)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", [OWN[0], OWN[4], PREFIX[0], PREFIX[1], LONG[0]])
def test_keys_that_some_do_not_see(shape, dt, cuda_device):
    from kbb200 import lm

    args = q, k, v, prefix, table, lens = attention_inputs(cuda_device, dt, *shape, seed=sum(shape))
    B, Q, page, keys = shape[0], shape[1], shape[5], prefix.numel() * shape[5]
    lens.clamp_(min=keys + Q)
    if Q == 1:
        lens[1: B // 2] = torch.randint(1, keys, (B // 2 - 1,), device=cuda_device, dtype=torch.int32)
        at, page_id, batch = int(lens[1]), int(prefix[int(lens[1]) // page]), torch.ones(B, dtype=torch.bool, device=cuda_device)
    else:
        at = int(lens[0]) - 2
        page_id, batch = int(table[0, at // page]), torch.arange(B, device=cuda_device) == 0
    want, want_lse = lm.shared_prefix_attention(*args)
    for what in (NAN, INF, -INF):
        bad = k.clone()
        bad[page_id, at % page] = what
        out, lse = lm.shared_prefix_attention(q, bad, v, prefix, table, lens)
        same = ~((visible(lens, Q) > at) & batch[:, None])
        assert same.any() and not same.all()
        assert torch.equal(out[same], want[same]) and torch.equal(lse[same], want_lse[same])


@pytest.mark.parametrize("what", [NAN, INF])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("length", [1, 130, 1000, 2048])
@pytest.mark.parametrize("shape", [(140, 1, 4, 1, 128, 16, 200, 5), (160, 1, 8, 2, 64, 32, 100, 20), (70, 1, 16, 4, 64, 16, 460, 3)])
def test_values_that_only_other_row_tiles_see(shape, length, dt, what, cuda_device):
    """The second half of the batch has one length, inside a tile of keys or at its end."""
    args = q, k, v, prefix, table, lens = attention_inputs(cuda_device, dt, *shape, seed=sum(shape))
    page = shape[5]
    lens[shape[0] // 2:] = length
    check(args, [(int(prefix[key // page]), key % page, key, None) for key in (length, length + 1, length + 40)], what)


@pytest.mark.parametrize("what", [NAN, INF])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("length", [5, 130, 1001, 2047])
@pytest.mark.parametrize("shape", [(140, 1, 4, 1, 128, 16, 200, 5), (160, 1, 8, 2, 64, 32, 100, 20), (70, 1, 16, 4, 64, 16, 460, 3)])
def test_values_beside_those_that_nobody_sees(shape, length, dt, what, cuda_device):
    """All sequences have one length, inside a page: what lies before it is everyone's, what lies after it nobody's."""
    args = q, k, v, prefix, table, lens = attention_inputs(cuda_device, dt, *shape, seed=sum(shape))
    page = shape[5]
    lens[:] = length
    check(args, [(int(prefix[key // page]), key % page, key, None) for key in (length - 1, length, length + 1, length // 2)], what)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", [(2, 3, 2, 1, 64, 16, 0, 40), (1, 90, 2, 1, 128, 16, 0, 100), (200, 1, 2, 1, 128, 16, 30, 0)])
def test_a_query_of_nan_stays_so(shape, dt, cuda_device):
    """The newest query of a sequence is NaN, and it alone sees values that are infinite."""
    from kbb200 import lm

    q, k, v, prefix, table, lens = args = attention_inputs(cuda_device, dt, *shape, seed=sum(shape))
    page = shape[5]
    if shape[1] > 1:
        lens.clamp_(min=shape[1])
        last = int(lens[0]) - 1
        page_id = int(table[0, last // page])
    else:  # one query a sequence: all others end a key earlier
        last = prefix.numel() * page - 1
        lens[:], page_id = last, int(prefix[-1])
        lens[0] = last + 1
    want, want_lse = lm.shared_prefix_attention(*args)
    q[0, -1] = NAN
    v[page_id, last % page] = INF
    out, lse = lm.shared_prefix_attention(*args)
    assert torch.isnan(out[0, -1]).all() and torch.isnan(lse[0, -1]).all()
    others = torch.ones(out.shape[:2], dtype=torch.bool, device=cuda_device)
    others[0, -1] = False
    assert torch.equal(out[others], want[others]) and torch.equal(lse[others], want_lse[others])

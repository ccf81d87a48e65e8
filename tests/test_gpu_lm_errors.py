"""GPU: an error of the C ABI reaches the caller of kbb200.lm from the one call that was made."""
from __future__ import annotations

import ctypes

import pytest
import torch

from tests.test_gpu_lm import ints

pytestmark = pytest.mark.gpu

KB_ERR_CUDA = 4
CHANGE_STATE = ["kb_cache_reserve", "kb_cache_append_granted", "kb_cache_fork", "kb_cache_free", "kb_cache_compact"]


class NotAgain:
    """Stands for the library in the Python half of the calls: sizes may be asked for, nothing may be launched."""

    def __getattr__(self, name):
        from kbb200 import LIB

        if not name.endswith("_size"):
            raise AssertionError(f"{name} was called again")
        return getattr(LIB, name)


@pytest.mark.parametrize("entry", CHANGE_STATE)
def test_a_failed_call_is_not_made_again(entry, cuda_device, monkeypatch):
    from kbb200 import KbError, lm
    from kbb200._lib import SIGNATURES, check

    pool = torch.zeros(2, 6, 4, 1, 8, device=cuda_device)
    table, lens = ints(cuda_device, [[0, 1], [-1, -1]]), ints(cuda_device, [5, 0])
    refs = ints(cuda_device, [1, 1, 0, 0, 0, 0])
    k, one, two = torch.ones(1, 1, 1, 8, device=cuda_device), ints(cuda_device, [0]), ints(cuda_device, [1])
    calls = {"kb_cache_reserve": lambda: lm.cache_reserve(table, lens, refs, one, 1, 4),
             "kb_cache_append_granted": lambda: lm.cache_append(k, k, pool[0], pool[1], table, lens, one),
             "kb_cache_fork": lambda: lm.cache_fork(pool, table, lens, refs, one, two),
             "kb_cache_free": lambda: lm.cache_free(table, lens, refs, one),
             "kb_cache_compact": lambda: lm.cache_compact(pool, table, refs)}
    made = []
    result, args = SIGNATURES[entry]

    def fails(*_):
        made.append(entry)
        return KB_ERR_CUDA

    fake = ctypes.CFUNCTYPE(result, *args)(fails)
    state = [t.clone() for t in (pool, table, lens, refs)]
    monkeypatch.setattr(lm, "LIB", NotAgain())
    lm._host.init({**lm._ENTRIES, entry: ctypes.cast(fake, ctypes.c_void_p).value, "check": check})
    try:
        with pytest.raises(KbError) as e:
            calls[entry]()
    finally:
        lm._host.init({**lm._ENTRIES, "check": check})
    assert made == [entry] and e.value.status == KB_ERR_CUDA and e.value.fn == entry.replace("_granted", "")
    assert all(torch.equal(a, b) for a, b in zip(state, (pool, table, lens, refs)))
    calls[entry]()  # the library's own entry again

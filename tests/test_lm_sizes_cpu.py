"""CPU: sizes whose sums or products pass 64 bits are refused, rather than wrapping around to one that looks right."""
from __future__ import annotations

import pytest

UNSUPPORTED, INVALID = 2, 1
HUGE = 1 << 62


def _rope(LIB, tokens=4, hq=2, hkv=1, dim=64):
    return LIB.kb_qk_norm_rope(16, 16, 16, 16, 16, 16, 16, 16, 16, tokens, hq, hkv, dim, dim, 100, dim, dim, dim, dim, 2, 0, 1, 0,
                               1e-6, None)


def _rope_backward(LIB, tokens=4, hq=2, hkv=1, dim=64):
    return LIB.kb_qk_norm_rope_backward(*[16] * 13, tokens, hq, hkv, dim, dim, 100, dim, dim, dim, dim, 2, 0, 1, 0, 1e-6, 16,
                                        1 << 40, None)


@pytest.mark.parametrize("call", [_rope, _rope_backward])
@pytest.mark.parametrize("bad", [dict(tokens=HUGE), dict(tokens=HUGE + 1), dict(tokens=(1 << 31) + 1), dict(tokens=HUGE, dim=512),
                                 dict(hq=HUGE, hkv=HUGE), dict(hq=(1 << 63) - 1, hkv=(1 << 63) - 1)])
def test_norms_and_rotation(call, bad):
    from kbb200 import LIB

    assert call(LIB, **bad) == UNSUPPORTED


@pytest.mark.parametrize("bad", [dict(batch=HUGE, queries=4), dict(batch=1 << 32, queries=1 << 32), dict(queries=1 << 62, hq=4),
                                 dict(batch=1 << 31, queries=1 << 31, hq=4), dict(page=HUGE, width=4), dict(page=HUGE, pre=4),
                                 dict(pre=HUGE, width=HUGE, page=4), dict(width=(1 << 63) - 1)])
def test_attention(bad):
    from kbb200 import LIB

    c = dict(batch=2, queries=1, hq=4, pre=2, width=4, page=16) | bad
    assert LIB.kb_shared_prefix_attention(16, 16, 16, 16, 16, 16, 16, 16, c["batch"], c["queries"], c["hq"], 2, 64, c["pre"],
                                          c["width"], 9, c["page"], 64, 64, 64, 64, 64, 64, 64, 64, 64, 0.1, 2, 16, 1 << 40,
                                          None) == UNSUPPORTED
    for dtype in (0, 1, 2):
        assert LIB.kb_shared_prefix_attention_workspace_size(c["batch"], c["queries"], c["hq"], 2, 64, c["pre"], c["width"],
                                                             c["page"], dtype) == 0


def test_cache():
    from kbb200 import LIB

    big = 1 << 40  # of a workspace
    for page in (HUGE, 1 << 61, (1 << 61) + 1, 1 << 32):  # times a width of 4 or 8
        assert LIB.kb_cache_reserve(16, 16, 16, 16, 16, 2, 1, 4, 8, 9, page, 16, big, None) == UNSUPPORTED
        assert LIB.kb_cache_fork(16, 16, 16, 16, 16, 16, 16, 2, 4, 8, 2, 9, page, 64, 16, big, None) == UNSUPPORTED
    # a row that holds 2^30 keys or more cannot take one page more in 32 bits
    assert LIB.kb_cache_fork(16, 16, 16, 16, 16, 16, 16, 2, 4, 1, 2, 9, 0x7fffffff, 64, 16, big, None) == UNSUPPORTED
    assert LIB.kb_cache_fork(16, 16, 16, 16, 16, 16, 16, 2, 4, 8, HUGE, 9, 16, 64, 16, big, None) == UNSUPPORTED
    assert LIB.kb_cache_compact(16, 16, 16, 16, 4, 8, HUGE, 9, 64, 16, big, None) == UNSUPPORTED
    assert LIB.kb_cache_copy(16, 16, 16, 16, 4, HUGE, 64, 9, 9, None) == UNSUPPORTED
    for entry, extra in ((LIB.kb_cache_append, []), (LIB.kb_cache_append_granted, [None])):
        sizes = [4, 8, 9]
        assert entry(16, 16, 16, 16, 16, 16, 16, *extra, 4, HUGE, *sizes, 16, 16, 1, 1, 1, 1, 1, None) == UNSUPPORTED
        assert entry(16, 16, 16, 16, 16, 16, 16, *extra, 8, (1 << 61) + 1, *sizes, 16, 16, 1, 1, 1, 1, 1, None) == UNSUPPORTED
        # pages of 2^32 keys of 2^32 bytes: more than page_bytes
        assert entry(16, 16, 16, 16, 16, 16, 16, *extra, 2, 1, *sizes, 1 << 32, 64, 1 << 32, 1, 1, 1, 1, None) == INVALID


def test_logits():
    from kbb200 import LIB

    for n in ((1 << 63) - 1, HUGE):
        assert LIB.kb_penalize_logits(16, 16, 16, 16, None, None, None, 16, 16, None, 2, 100, 100, n, 3, 3, 0, 0, 1,
                                      None) == UNSUPPORTED

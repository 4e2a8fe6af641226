"""What the C entry of eviction refuses about arrays that share memory, on the host before
anything touches a GPU."""

from __future__ import annotations

import ctypes

import pytest

from sglang_restomod_b200 import _lib
from tests.test_attention_capi import desc, err
from tests.test_serving_capi import EVICT, call


def at(n):
    return ctypes.c_void_p(n)


# 3 sequences, 2 heads, a budget of 20: kept takes 480 bytes, lens and kv_lens 12, a table 24
APART = dict(EVICT, table=at(1 << 16), kv_lens=at(2 << 16), out_table=at(3 << 16), kept=at(4 << 16),
             lens=at(5 << 16))


def evict(cache=None, **kw):
    return call("b200_kv_cache_evict", APART, kw, cache or desc())


@pytest.mark.parametrize("kw", [
    dict(lens=2 << 16),  # the lengths updated in place
    dict(lens=(2 << 16) + 8), dict(lens=(2 << 16) - 8),
    dict(lens=(1 << 16) + 20), dict(lens=(3 << 16) + 20), dict(lens=(4 << 16) + 476),
    dict(lens=(4 << 16) - 8),
    dict(kept=2 << 16), dict(kept=(2 << 16) - 476), dict(kept=(2 << 16) + 8),
    dict(kept=1 << 16), dict(kept=(1 << 16) - 476), dict(kept=(3 << 16) - 476),
    dict(kv_lens=4 << 16), dict(table=(5 << 16) - 20), dict(out_table=(4 << 16) + 400),
    dict(lens=2 << 16, out_table=None),
])
def test_results_with_memory_of_an_input(kw):
    kw = {name: v and at(v) for name, v in kw.items()}
    assert "memory of their own" in err(evict(**kw), _lib.ERR_INVALID)


def test_the_same_table_with_another_stride():
    """In place or not: rows after the first would be other pages."""
    assert "page_table's stride" in err(evict(out_table=at(1 << 16), out_stride=3, out_width=3),
                                        _lib.ERR_INVALID)


def test_keys_that_are_the_values():
    """Each moves without waiting for the other."""
    for out_table in (None, at(3 << 16)):
        assert "same memory" in err(evict(desc(v=4096), out_table=out_table), _lib.ERR_INVALID)

"""Values, log-sums and page numbers out of the ordinary, at more rows a sequence than the
streaming kernel of the scores takes, for each cache type, with tensor copies (pages of 16
tokens) and without (pages of one)."""

from __future__ import annotations

import math

import pytest
import torch

from sglang_restomod_b200 import ops
from tests.test_gpu_attention import TYPES
from tests.test_gpu_scores_hidden import slots, tiled

pytestmark = pytest.mark.gpu

PAGES = [1, 16]


def same(a, b):
    return torch.equal(torch.nan_to_num(a, 3.0), torch.nan_to_num(b, 3.0))


@pytest.mark.parametrize("q_dtype,store", TYPES)
@pytest.mark.parametrize("page", PAGES)
def test_infinite_log_sums(cuda_device, q_dtype, store, page):
    """Rows of -inf and of +inf add nothing."""
    c = tiled(1, [40, 50], [300, 50], 128, page, 4, q_dtype, store)
    c.lse[3:9] = -math.inf
    c.lse[30, 5:] = math.inf
    c.lse[60:70, 2] = -math.inf
    c.all()
    c.lse.fill_(-math.inf)
    c.all()


@pytest.mark.parametrize("q_dtype,store", TYPES)
@pytest.mark.parametrize("page", PAGES)
def test_a_keys_nan_stays_with_its_token(cuda_device, q_dtype, store, page):
    c = tiled(2, [40, 33], [300, 170], 64, page, 4, q_dtype, store)
    want = c.run().cpu()
    keys = c.cache.k if store.itemsize > 1 else c.cache.k.view(torch.uint8)
    for s, token in ((0, 5), (0, 280), (1, 128)):
        p, o = (int(t[token]) for t in slots(c, s))
        keys[p, o, 1, 17] = math.nan if store.itemsize > 1 else 0x7f
        want[p, o, 1] = math.nan
    got = c.run().cpu()
    assert same(got, want)
    for s in range(2):
        assert int(got[slots(c, s)].isnan().sum()) == 2 - s
    assert ops.attention_status() == 0


@pytest.mark.parametrize("q_dtype,store", TYPES)
@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("bad", [-1, -9, 1 << 30, "pages"])
def test_bad_pages(cuda_device, q_dtype, store, page, bad):
    """Tokens on pages outside the cache are left out and reported; the others have their bits."""
    c = tiled(3, [40, 33], [300, 170], 128, page, 4, q_dtype, store)
    want = c.run().cpu()
    bad = c.cache.num_pages if bad == "pages" else bad
    table, untouched = c.dev[2].clone(), c.scores().cpu()
    for s, entry in ((0, 3), (0, 299 // page), (1, 9)):
        table[s, entry] = bad
        want[int(c.table[s, entry])] = untouched[int(c.table[s, entry])]
    c.dev = (*c.dev[:2], table, *c.dev[3:])
    assert ops.attention_status() == 0
    got = c.run().cpu()
    assert ops.attention_status() == 16
    assert same(got, want)
    assert ops.attention_status() == 0


@pytest.mark.parametrize("q_dtype,store", TYPES)
@pytest.mark.parametrize("page", PAGES)
def test_sequences_within_a_tile(cuda_device, q_dtype, store, page):
    """Rows of one tile belong to several sequences in memory: another's NaN stays there."""
    c = tiled(4, [9, 9, 9, 9, 9], [90, 9, 190, 300, 20], 128, page, 8, q_dtype, store)
    want = c.run().cpu()
    c.dev[0][9:18] = math.nan
    c.dev[0][27:36] = math.nan
    got = c.run().cpu()
    for s in range(5):
        x, y = got[slots(c, s)], want[slots(c, s)]
        assert x.isnan().all() if s in (1, 3) else torch.equal(x, y)

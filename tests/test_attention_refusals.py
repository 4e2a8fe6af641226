"""Refusals of the attention half's C entry points that need no GPU."""

from __future__ import annotations

import ctypes

import pytest

from sglang_restomod_b200 import _lib
from tests.test_attention_capi import attention, desc, err


def test_device_status_wants_a_place_for_its_bits():
    assert "null pointer" in err(_lib.load().b200_device_status(None, 1, None), _lib.ERR_INVALID)


@pytest.mark.parametrize("scale", [3e38, -3e38, float("inf")])
def test_scales_that_are_not_finite_in_log2(scale):
    d = desc()
    assert "finite" in err(attention(ctypes.addressof(d), scale=scale), _lib.ERR_INVALID)

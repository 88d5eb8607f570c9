"""Refusals of the attention entry points that need no GPU."""
from __future__ import annotations

import ctypes

import pytest

from test_attention_validation import ENTRY, GOOD, PTR, SHAPE, _structs, lib  # noqa: F401  (lib: a fixture)


@pytest.mark.parametrize("max_tree", [65, 1 << 20])
def test_a_masked_tree_has_at_most_64_tokens(lib, max_tree):
    mirror, _ = _structs()["tree"]
    args = mirror(**{**GOOD["tree"], "mask": PTR, "max_tree": max_tree})
    assert getattr(lib, ENTRY["tree"])(ctypes.addressof(args), None) == SHAPE

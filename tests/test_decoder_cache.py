"""The list of free pages behind my_int4.decoder.KV8Cache (host side)."""
from __future__ import annotations

import pytest
import torch

from my_int4.decoder import KV8Cache


def cache(pages=8):
    return KV8Cache(pages, 1, 64, page_size=16, device="cpu"), torch.full((2, 6), -1, dtype=torch.int32)


def owned(table):
    return [p for p in table.flatten().tolist() if p >= 0]


def test_growing_without_held_keeps_the_rows_pages():
    c, t = cache()
    assert c.grow(t, 0, 20) == 2
    first = t[0].tolist()
    assert c.grow(t, 0, 20) == 2 and t[0].tolist() == first and len(c.free) == 6
    assert c.grow(t, 0, 40) == 3 and t[0, :2].tolist() == first[:2] and len(c.free) == 5
    assert c.grow(t, 0, 50, 1) == 4 and t[0, :2].tolist() == first[:2] and len(c.free) == 4
    assert c.grow(t, 1, 64) == 4 and not c.free
    assert sorted(owned(t)) == list(range(8))
    with pytest.raises(MemoryError):
        c.grow(t, 0, 65)
    c.release(t, 0, 6)                                # entries without a page give none back
    c.release(t, 1, 4)
    assert sorted(c.free) == list(range(8)) and not owned(t)


def test_pages_taken_back_from_the_front():
    # a window that has passed a sequence's first page: its entry is -1, and is filled only on demand
    c, t = cache()
    c.grow(t, 0, 48)
    c.release(t, 0, 1)
    assert t[0, 0] == -1 and len(c.free) == 6
    assert c.grow(t, 0, 64, 1) == 4 and t[0, 0] == -1 and len(c.free) == 5
    assert len(set(owned(t))) == 3


def test_a_table_of_zeros_is_refused():
    # 0 is a page: without this, rows would share it
    c, _ = cache()
    with pytest.raises(ValueError, match="-1"):
        c.grow(torch.zeros(2, 6, dtype=torch.int32), 0, 20)
    assert len(c.free) == 8

"""Calls over a paged cache at the ends of what they allow, on the CPU: which are
refused, and with what; none of them reaches a kernel."""
from __future__ import annotations

import pytest
import torch

from proteus_attention import _hip, evict_kv_tokens, new_kv_pages

ONE = torch.ones(1, dtype=torch.int32)


def test_two_tables_without_pages_are_two_tables():
    """Neither has an address: they pass as any two do, and then miss their device."""
    pages, w = new_kv_pages(4, 2, 16, 32, device="cpu"), torch.zeros(1, 2, 32)
    none, table = torch.zeros(1, 0, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32)
    for a, b in ((none, none), (none, none.clone()), (table, none), (none, table), (table[:, :0], table[:, 1:1])):
        with pytest.raises(_hip.HipLibraryError):
            evict_kv_tokens(pages, w, a, ONE, 3, b)
    for a, b in ((table, table), (table, table[:, :1])):
        with pytest.raises(ValueError):
            evict_kv_tokens(pages, w, a, ONE, 3, b)

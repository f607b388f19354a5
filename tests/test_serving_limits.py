"""The limits of the serving entry points without a GPU: sizes whose positions or launches
would leave 32 bits are refused on the host, before anything runs."""

from __future__ import annotations

import ctypes

import pytest
import torch

from switchyard import _lib
from switchyard.cache_op import paged_append, paged_attention

FAKE = 0x1000  # never dereferenced
OK, SHAPE = 0, -2


def _paged(**kw):
    base = dict(k=FAKE, v=FAKE, table=FAKE, lengths=FAKE, starts=None, page_stride=8 << 20, head_stride=8 << 20,
                row_stride=8, table_stride=4, n_seq=1, n_tok=1, n_pages=2, table_cols=4, page=1 << 20, heads=1,
                kv_heads=1, hd=8, dtype=_lib.SY_BF16)
    return _lib.Paged(**{**base, **kw})


@pytest.mark.parametrize("prefix_len", [(1 << 30) + 1, 2**31 - 64, 2**31 - 1])
def test_a_prefix_past_the_positions_is_refused(prefix_len):
    """The last tile's look-ahead would pass 2^31 and index before the list of pages."""
    lib, c = _lib.lib(), ctypes.byref(_paged())
    assert lib.sy_paged_attention_workspace_bytes(c, 1 << 30) >= 0
    assert lib.sy_paged_attention_workspace_bytes(c, prefix_len) == SHAPE
    assert lib.sy_paged_attention(c, FAKE, 8, 8, FAKE, FAKE, prefix_len, 1.0, 0, FAKE, 1 << 40, None) == SHAPE
    assert lib.sy_paged_append(c, FAKE, 24, 8, FAKE, FAKE, 8, prefix_len, FAKE, 0, None) == SHAPE


def test_a_table_past_the_positions_is_refused():
    lib = _lib.lib()
    for cols in (1025, 2047):
        c = ctypes.byref(_paged(table_cols=cols, table_stride=cols))
        assert lib.sy_paged_attention_workspace_bytes(c, 0) == SHAPE
        assert lib.sy_paged_append(c, FAKE, 24, 8, FAKE, FAKE, 8, 0, FAKE, 0, None) == SHAPE
    assert lib.sy_paged_attention_workspace_bytes(ctypes.byref(_paged(table_cols=1024, table_stride=1024)), 0) >= 0


@pytest.mark.parametrize("fn", [paged_append, paged_attention])
def test_the_functions_refuse_them_too(fn):
    page = 1 << 20
    k = torch.zeros(1, 1, page, 8)
    lengths, cos = torch.zeros(1, dtype=torch.int32), torch.zeros(4, 4)
    rows = torch.zeros(1, 3 if fn is paged_append else 1, 8)
    head = (rows, cos, cos) if fn is paged_append else (rows,)
    with pytest.raises(ValueError, match="prefix_len"):
        fn(*head, k, k, torch.zeros(1, 4, dtype=torch.int32), lengths, prefix_len=(1 << 30) + 1)
    with pytest.raises(ValueError, match="page_table"):
        fn(*head, k, k, torch.zeros(1, 1025, dtype=torch.int32), lengths)


def test_launches_of_2_to_32_threads_are_refused():
    """A workgroup of 256 threads for every token of 2^24 sequences, or for its merge."""
    lib = _lib.lib()
    more = dict(page=1, page_stride=8, head_stride=8, table_cols=1, table_stride=1)
    for n, prefix, rc in ((1 << 24, 0, SHAPE), ((1 << 24) - 1, 0, OK), (1 << 24, 100, SHAPE), (1 << 23, 100, OK)):
        need = lib.sy_paged_attention_workspace_bytes(ctypes.byref(_paged(n_seq=n, n_tok=n, **more)), prefix)
        assert need == rc if rc else need >= 0, (n, prefix, need)
    wide = ctypes.byref(_paged(n_seq=1 << 21, n_tok=1 << 21, heads=8, kv_heads=8, **more))
    assert lib.sy_paged_attention_workspace_bytes(wide, 0) == SHAPE

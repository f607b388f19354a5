"""The serving entry points without a GPU: what they refuse, and with which error."""

from __future__ import annotations

import ctypes

import pytest
import torch

from switchyard import _lib
from switchyard.cache_op import paged_append, paged_attention
from switchyard.sample_op import sample_tokens

OK, NULL, SHAPE, DTYPE, WORKSPACE, STRIDE = 0, -1, -2, -3, -4, -5
FAKE = 0x1000  # never dereferenced: every call below fails validation first


def _paged(**kw):
    base = dict(k=FAKE, v=FAKE, table=FAKE, lengths=FAKE, starts=None, page_stride=2 * 16 * 64, head_stride=16 * 64,
                row_stride=64, table_stride=4, n_seq=3, n_tok=3, n_pages=10, table_cols=4, page=16, heads=4, kv_heads=2,
                hd=64, dtype=_lib.SY_BF16)
    base.update(kw)
    return _lib.Paged(**base)


BAD = [
    (dict(dtype=7), DTYPE), (dict(n_seq=-1), SHAPE), (dict(n_tok=-1), SHAPE), (dict(n_tok=4), SHAPE),
    (dict(n_seq=0), SHAPE), (dict(n_pages=0), SHAPE), (dict(table_cols=-1), SHAPE), (dict(table_cols=0), SHAPE), (dict(page=0), SHAPE),
    (dict(page=24), SHAPE), (dict(page=1 << 21), SHAPE), (dict(table_cols=1 << 28), SHAPE), (dict(heads=3), SHAPE),
    (dict(kv_heads=0), SHAPE), (dict(heads=0), SHAPE), (dict(heads=1 << 16), SHAPE), (dict(hd=0), SHAPE),
    (dict(hd=60), SHAPE), (dict(hd=264), SHAPE), (dict(n_tok=1 << 31, starts=FAKE), SHAPE), (dict(k=None), NULL),
    (dict(v=None), NULL), (dict(table=None), NULL), (dict(lengths=None), NULL), (dict(k=FAKE + 8), SHAPE),
    (dict(page_stride=-16), STRIDE), (dict(row_stride=65), STRIDE), (dict(head_stride=12), STRIDE), (dict(page_stride=1 << 31), STRIDE), (dict(row_stride=1 << 27), STRIDE),
]


@pytest.mark.parametrize("change,code", BAD, ids=[str(i) for i in range(len(BAD))])
def test_a_bad_cache_is_refused(change, code):
    lib, c = _lib.lib(), _paged(**change)
    r = ctypes.byref(c)
    assert lib.sy_paged_append(r, FAKE, 512, 64, FAKE, FAKE, 8, 0, FAKE, 0, None) == code
    assert lib.sy_paged_attention(r, FAKE, 256, 64, FAKE, None, 0, 1.0, 0, FAKE, 1 << 40, None) == code
    assert lib.sy_paged_attention_workspace_bytes(r, 0) == code


def test_other_bad_arguments_are_refused():
    lib, c = _lib.lib(), _paged()
    r = ctypes.byref(c)
    assert lib.sy_paged_append(None, FAKE, 512, 64, FAKE, FAKE, 8, 0, FAKE, 0, None) == NULL
    assert lib.sy_paged_append(r, None, 512, 64, FAKE, FAKE, 8, 0, FAKE, 0, None) == NULL
    assert lib.sy_paged_append(r, FAKE, 512, 64, None, FAKE, 8, 0, FAKE, 0, None) == NULL
    assert lib.sy_paged_append(r, FAKE, 512, 64, FAKE, FAKE, 8, 0, None, 0, None) == NULL
    assert lib.sy_paged_append(r, FAKE, -1, 64, FAKE, FAKE, 8, 0, FAKE, 0, None) == STRIDE
    assert lib.sy_paged_append(r, FAKE, 512, 64, FAKE, FAKE, -1, 0, FAKE, 0, None) == SHAPE
    assert lib.sy_paged_append(r, FAKE, 512, 64, FAKE, FAKE, 8, -1, FAKE, 0, None) == SHAPE
    assert lib.sy_paged_append(r, FAKE, 512, 64, FAKE, FAKE, 8, 0, FAKE, 2, None) == SHAPE
    assert lib.sy_paged_append(r, FAKE, 512, 64, FAKE, FAKE, 8, 0, FAKE + 2, 0, None) == SHAPE
    attend = lib.sy_paged_attention
    assert attend(None, FAKE, 256, 64, FAKE, None, 0, 1.0, 0, FAKE, 1 << 40, None) == NULL
    assert attend(r, None, 256, 64, FAKE, None, 0, 1.0, 0, FAKE, 1 << 40, None) == NULL
    assert attend(r, FAKE, 256, 64, None, None, 0, 1.0, 0, FAKE, 1 << 40, None) == NULL
    assert attend(r, FAKE, 256, 64, FAKE, None, 5, 1.0, 0, FAKE, 1 << 40, None) == NULL
    assert attend(r, FAKE, 250, 64, FAKE, None, 0, 1.0, 0, FAKE, 1 << 40, None) == STRIDE
    assert attend(r, FAKE + 2, 256, 64, FAKE, None, 0, 1.0, 0, FAKE, 1 << 40, None) == SHAPE
    assert attend(r, FAKE, 256, 64, FAKE, FAKE, -1, 1.0, 0, FAKE, 1 << 40, None) == SHAPE
    need = lib.sy_paged_attention_workspace_bytes(r, 100)
    assert need > 0
    assert attend(r, FAKE, 256, 64, FAKE, FAKE, 100, 1.0, 0, FAKE, need - 1, None) == WORKSPACE
    assert attend(r, FAKE, 256, 64, FAKE, FAKE, 100, 1.0, 0, None, need, None) == WORKSPACE
    # tiles past 32 bits
    big = _paged(n_tok=1 << 29, n_seq=1 << 29, table_cols=1 << 20)
    assert lib.sy_paged_attention_workspace_bytes(ctypes.byref(big), 0) == SHAPE
    # no rows: nothing is launched, and no pointer is needed
    none = ctypes.byref(_paged(n_tok=0, k=None, v=None, table=None, lengths=None))
    assert lib.sy_paged_append(none, None, 0, 0, None, None, 0, 0, None, 0, None) == OK
    assert attend(none, None, 0, 0, None, None, 0, 1.0, 0, None, 0, None) == OK


def test_sampling_arguments_are_refused():
    lib, how = _lib.lib(), ctypes.byref(_lib.Sampling(1.0, 1.0, 0.0, 0))
    assert lib.sy_sample(FAKE, FAKE, FAKE, None, 2, 10, 10, _lib.SY_F32, None) == NULL
    assert lib.sy_sample(None, FAKE, FAKE, how, 2, 10, 10, _lib.SY_F32, None) == NULL
    assert lib.sy_sample(FAKE, None, FAKE, how, 2, 10, 10, _lib.SY_F32, None) == NULL
    assert lib.sy_sample(FAKE, FAKE, None, how, 2, 10, 10, _lib.SY_F32, None) == NULL
    assert lib.sy_sample(FAKE, FAKE, FAKE, how, 2, 10, 10, 9, None) == DTYPE
    assert lib.sy_sample(FAKE, FAKE, FAKE, how, -1, 10, 10, _lib.SY_F32, None) == SHAPE
    assert lib.sy_sample(FAKE, FAKE, FAKE, how, 2, 0, 10, _lib.SY_F32, None) == SHAPE
    assert lib.sy_sample(FAKE, FAKE, FAKE, how, 2, (1 << 18) + 1, 10, _lib.SY_F32, None) == SHAPE
    assert lib.sy_sample(FAKE, FAKE, FAKE, how, 2, 10, -1, _lib.SY_F32, None) == STRIDE
    assert lib.sy_sample(None, None, None, how, 0, 10, 10, _lib.SY_F32, None) == OK


def _call(fn, **change):
    i = torch.int32
    a = dict(rows=torch.zeros(3, 8 if fn is paged_append else 4, 64), k=torch.zeros(10, 2, 16, 64),
             table=torch.zeros(3, 4, dtype=i), lengths=torch.zeros(3, dtype=i), starts=None, cos=torch.zeros(99, 32))
    a["v"] = torch.zeros_like(change.get("k", a["k"]))
    more = {k: change.pop(k) for k in list(change) if k in ("prefix_len", "prefix_pages", "out")}
    a.update(change)
    if fn is paged_append:
        return fn(a["rows"], a["cos"], a["cos"], a["k"], a["v"], a["table"], a["lengths"], a["starts"], **more)
    return fn(a["rows"], a["k"], a["v"], a["table"], a["lengths"], a["starts"], **more)


REFUSED = [
    (dict(), "CUDA"),
    (dict(k=torch.zeros(10, 2, 24, 64)), "power of two"),
    (dict(k=torch.zeros(10, 2, 16, 60)), "multiple of 8"),
    (dict(k=torch.zeros(10, 2, 16, 264)), "at most 256"),
    (dict(k=torch.zeros(0, 2, 16, 64)), "page"),
    (dict(v=torch.zeros(10, 2, 16, 32)), "same shape"),
    (dict(k=torch.zeros(10, 2, 16, 64, dtype=torch.float64), v=torch.zeros(10, 2, 16, 64, dtype=torch.float64)), "dtype"),
    (dict(k=torch.zeros(10, 2, 16, 64, dtype=torch.bfloat16), v=torch.zeros(10, 2, 16, 64, dtype=torch.bfloat16)), "dtype"),
    (dict(k=torch.zeros(10, 2, 64, 16).transpose(2, 3), v=torch.zeros(10, 2, 64, 16).transpose(2, 3)), "dense"),
    (dict(table=torch.zeros(3, 4)), "int32"),
    (dict(table=torch.zeros(4, dtype=torch.int32)), "page_table"),
    (dict(table=torch.zeros(0, 4, dtype=torch.int32)), "page_table"),
    (dict(lengths=torch.zeros(4, dtype=torch.int32)), "lengths"),
    (dict(lengths=torch.zeros(3, dtype=torch.int64)), "int32"),
    (dict(lengths=torch.zeros(6, dtype=torch.int32)[::2]), "dense"),
    (dict(starts=torch.zeros(3, dtype=torch.int32)), "starts"),
    (dict(rows=torch.zeros(4, 8, 64)), "divide"),
    (dict(rows=torch.zeros(3, 8)), "must be"),
    (dict(rows=torch.zeros(3, 7, 64)), "kv heads"),
    (dict(prefix_len=-1), "prefix_len"),
]


@pytest.mark.parametrize("fn", [paged_append, paged_attention])
@pytest.mark.parametrize("change,match", REFUSED, ids=[str(i) for i in range(len(REFUSED))])
def test_the_functions_say_what_is_wrong(change, match, fn):
    with pytest.raises(ValueError, match=match):
        _call(fn, **dict(change))


def test_settings_are_checked():
    x, u = torch.zeros(2, 5), torch.zeros(2)
    for kw, match in ((dict(temperature=-1.0), "temperature"), (dict(min_p=float("nan")), "min_p"),
                      (dict(top_k=1.5), "top_k"), (dict(top_p="x"), "top_p"), (dict(min_p=-0.1), "min_p"),
                      (dict(), "CUDA")):
        with pytest.raises(ValueError, match=match):
            sample_tokens(x, u, **kw)
    with pytest.raises(ValueError, match="columns"):
        sample_tokens(torch.zeros(2, 0), u)
    with pytest.raises(ValueError, match=r"\[B, V\]"):
        sample_tokens(torch.zeros(5), u)

"""Edges of the paged cache's operators on the GPU, against float64 with the bounds of
``test_cache_op``."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a HIP device", allow_module_level=True)

from switchyard.cache_op import paged_append  # noqa: E402

DEV = "cuda"
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def test_a_length_past_the_longest_row():
    """A row of 2^30 tokens and a length five past it: the first new tokens have the row's last
    places, the others none."""
    page, n = 1 << 20, 10
    k = torch.zeros(1, 1, page, 8, dtype=BF, device=DEV)
    v = torch.zeros_like(k)
    turn = torch.empty(1 << 30, 4, device=DEV)  # (only the last rows are read)
    turn[-16:] = 0.5
    qkv = torch.randn(n, 3, 8, generator=torch.Generator().manual_seed(1)).to(BF).to(DEV)
    table = torch.zeros(1, 1024, dtype=torch.int32, device=DEV)
    lengths = torch.full((1,), (1 << 30) + 5, dtype=torch.int32, device=DEV)
    q = paged_append(qkv, turn, turn, k, v, table, lengths)
    assert torch.equal(torch.isnan(q).all(-1)[:, 0], torch.arange(n, device=DEV) >= 5)
    assert torch.equal(v[0, 0, -5:], qkv[:5, 2]) and (v[0, 0, :-5] == 0).all() and (k[0, 0, :-5] == 0).all()

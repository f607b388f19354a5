"""Sampling more rows than one launch has threads for."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a HIP device", allow_module_level=True)

from switchyard.sample_op import sample_tokens  # noqa: E402


def test_more_rows_than_a_launch():
    """2^22 + 3 rows of three logits with settings of their own: every launch's rows are those of
    a call of their own."""
    n = (1 << 22) + 3
    g = torch.Generator(device="cuda").manual_seed(1)
    x = 2 * torch.randn(n, 3, device="cuda", generator=g)
    u = torch.rand(n, device="cuda", generator=g)
    t = 0.5 + torch.rand(n, device="cuda", generator=g)
    k = torch.randint(0, 3, (n,), device="cuda", generator=g, dtype=torch.int32)
    p, m = 0.5 + torch.rand(n, device="cuda", generator=g), 0.2 * torch.rand(n, device="cuda", generator=g)
    got = sample_tokens(x, u, temperature=t, top_k=k, top_p=p, min_p=m)
    for lo, hi in ((0, 1000), ((1 << 21) - 500, (1 << 21) + 500), (n - 1000, n)):
        rows = slice(lo, hi)
        want = sample_tokens(x[rows], u[rows], temperature=t[rows], top_k=k[rows], top_p=p[rows], min_p=m[rows])
        assert torch.equal(got[rows], want)
    assert ((got >= 0) & (got < 3)).all()

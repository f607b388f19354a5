"""Sampling more rows than one launch has threads for, and rows whose range is far wider than
their candidates'; the definition is ``test_sample_op``'s."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a HIP device", allow_module_level=True)

from test_sample_op import BF, F, HF, check, rows  # noqa: E402

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
        at = slice(lo, hi)
        want = sample_tokens(x[at], u[at], temperature=t[at], top_k=k[at], top_p=p[at], min_p=m[at])
        assert torch.equal(got[at], want)
    assert ((got >= 0) & (got < 3)).all()


@pytest.mark.parametrize("v", [5000, 50257])
@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_tokens_ruled_out_by_the_lowest_number(dtype, v):
    """Some or most of a row at the type's lowest number, with more other tokens than are ranked;
    cuts within the candidates, behind the last one with a weight (low temperatures, large k)
    and among those that are ruled out."""
    x, u = rows(12, v, dtype, seed=21)
    g = torch.Generator().manual_seed(22)
    lowest = torch.finfo(dtype).min
    x[:4, 7] = lowest
    x[4:8][(torch.rand(4, v, generator=g) < 0.5).to(x.device)] = lowest
    x[8:] = lowest
    for r in range(8, 12):
        x[r, torch.randperm(v, generator=g)[:1500].to(x.device)] = torch.randn(1500, generator=g).to(x)
    for t in (1e-3, 0.05, 0.8, 30.0):
        for k in (1, 40, 1400, 1499, 1501, v - 1):
            check(x, u, t, k)
            check(x, u, t, k, 0.8, 0.01)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("top", [0.0, 1e5, -1e5, 3e-30])
def test_ties_of_the_largest_at_any_place(top, dtype):
    """Equal largest logits are cut by their index, whatever the temperature and their size."""
    x, u = rows(6, 5000, dtype, seed=23)
    x = torch.where(x > 0, torch.full_like(x, top), torch.full_like(x, torch.finfo(dtype).min))
    x[:, 3::7] = top - 1.0 if abs(top) < 1e4 else top - 2048.0
    for t in (1e-38, 1e-4, 0.02, 1.0, 1e3):
        for k in (1, 5, 900, 1300, 3500, 4990):
            check(x, u, t, k)
            check(x, u, t, k, 0.6)

"""Sampling on the GPU against the definition in whole numbers (numpy, row by row).

The weights come from an exponential whose last bits may differ between the two sides, so
a weight may differ by one unit of 2^-44 and a token whose border the random number hits
to about 2^-40 may differ: none of the few thousand draws here should (probability below
1e-7), so tokens are compared exactly."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a HIP device", allow_module_level=True)

from switchyard.sample_op import sample_tokens  # noqa: E402

DEV = "cuda"
BF, HF, F = torch.bfloat16, torch.float16, torch.float32
ONE = 1 << 44


def reference(logits, u, t, k, p, m):
    """One row: ``logits`` float64, NaN already as -inf."""
    if not (logits > -math.inf).any():
        return -1
    top = logits.max()
    if not t > 0:
        return int(np.flatnonzero(logits == top)[0])
    with np.errstate(invalid="ignore"):
        e = np.where(logits == top, 1.0, np.exp((logits - top) / t))
    e = np.where(np.isnan(e) | (logits == -math.inf), 0.0, e)
    w = np.rint(e * ONE).astype(np.int64)
    order = np.argsort(-logits, kind="stable")
    if 1 <= k < len(logits):
        order = order[:k]
    if p < 1:
        before = np.concatenate(([0], np.cumsum(w[order])[:-1]))
        keep = before < p * float(w[order].sum())
        keep[0] = True
        order = order[keep]
    chosen = np.sort(order[e[order] >= min(m, 1.0)])
    cum = np.cumsum(w[chosen])
    goal = min(int(u * float(cum[-1])), int(cum[-1]) - 1)
    return int(chosen[np.searchsorted(cum, goal, side="right")])


def expected(logits, u, t, k, p, m):
    x = logits.double().cpu().numpy()
    x = np.where(np.isnan(x), -math.inf, x)
    cols = [y.double().cpu().numpy() if torch.is_tensor(y) else np.full(len(x), float(y)) for y in (t, k, p, m)]
    return torch.tensor([reference(r, float(v), a, int(b), c, d)
                         for r, v, a, b, c, d in zip(x, u.double().cpu().numpy(), *cols)])


def check(logits, u, t=1.0, k=0, p=1.0, m=0.0):
    got = sample_tokens(logits, u, temperature=t, top_k=k, top_p=p, min_p=m)
    assert got.dtype == torch.int64 and got.shape == u.shape
    want = expected(logits, u, t, k, p, m)
    assert torch.equal(got.cpu(), want), (got.cpu() != want).nonzero().flatten().tolist()
    return got


def rows(b, v, dtype, seed, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    x = scale * torch.randn(b, v, generator=g)
    return x.to(dtype).to(DEV), torch.rand(b, generator=g).to(DEV)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.8, 50, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (1.5, 0, 1.0, 0.1), (0.7, 1, 1.0, 0.0),
            (1.0, 3, 0.5, 0.3), (0.0, 5, 0.5, 0.1), (3.0, 400, 0.99, 0.001), (1.0, 10**9, 0.0, 0.0), (1e-4, 0, 0.9, 0.0),
            (1e4, 0, 0.7, 0.0), (1.0, 0, 0.3, 1.0), (math.inf, 7, 0.6, 0.0)]


@pytest.mark.parametrize("settings", SETTINGS, ids=[str(i) for i in range(len(SETTINGS))])
@pytest.mark.parametrize("v", [1, 2, 63, 1000, 8193, 32000])
@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_sampling(v, dtype, settings):
    check(*rows(9, v, dtype, seed=v), *settings)


@pytest.mark.parametrize("v", [50257, 65537, 131072, 262144])
@pytest.mark.parametrize("dtype", [BF, F])
def test_wide_rows(v, dtype):
    for settings in SETTINGS[:4]:
        check(*rows(3, v, dtype, seed=1), *settings)


@pytest.mark.parametrize("dtype", [BF, F])
def test_every_border_of_the_draw(dtype):
    """A row sampled with many numbers, 0 and the largest below 1 among them."""
    x, _ = rows(1, 300, dtype, seed=2)
    u = torch.linspace(0, 1, 1001)
    u[-1] = 1 - 2.0**-24
    for settings in ((1.0, 0, 1.0, 0.0), (0.5, 20, 0.8, 0.0)):
        check(x.expand(1001, -1), u.to(DEV), *settings)  # rows of stride 0
    assert (sample_tokens(x.expand(2, -1), torch.tensor([1.0, math.nan], device=DEV)) >= 0).all()


@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_ties_go_to_the_lowest_index(dtype):
    g = torch.Generator().manual_seed(3)
    few = torch.randint(-3, 4, (16, 5000), generator=g).to(dtype).to(DEV)  # seven values in all
    u = torch.rand(16, generator=g).to(DEV)
    for k in (1, 2, 700, 1500, 4999, 5000):
        check(few, u, 1.0, k)
        check(few, u, 2.0, k, 0.6)
    same = torch.zeros(16, 20000, dtype=dtype, device=DEV)
    same[:, ::2] = -0.0  # equal to 0
    for settings in ((1.0, 0, 1.0), (1.0, 0, 0.37), (1.0, 777, 1.0), (1.0, 1025, 0.5), (0.0, 0, 1.0)):
        check(same, u, *settings)


@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_infinities_and_nan(dtype):
    x, u = rows(8, 3000, dtype, seed=4)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, 1:] = -math.inf
    x[3, ::2] = math.nan
    x[4, ::3] = -math.inf
    x[5, 7::500] = math.inf
    x[6, :] = torch.finfo(dtype).min
    x[7, 5] = torch.finfo(dtype).max
    for settings in SETTINGS[:6]:
        got = check(x, u, *settings)
        assert (got[:2] == -1).all() and got[2] == 0 and got[5] % 500 == 7


def test_spread_past_the_largest_number():
    """fp32 logits whose range overflows, alone and with equals."""
    x, u = rows(4, 3000, F, seed=5)
    x[:, 10] = torch.finfo(F).min
    x[:, 20] = torch.finfo(F).max
    x[2:, 30] = torch.finfo(F).max
    for settings in SETTINGS[:4]:
        check(x, u, *settings)


@pytest.mark.parametrize("v", [1200, 40001])
def test_settings_of_each_row(v):
    g = torch.Generator().manual_seed(6)
    b = 40
    x, u = rows(b, v, BF, seed=7)
    t = (2 * torch.rand(b, generator=g)).to(DEV)
    t[3], t[4], t[5] = 0.0, -1.0, math.nan  # the first largest
    k = torch.randint(-5, 100, (b,), generator=g, dtype=torch.int32).to(DEV)
    p = (0.3 + torch.rand(b, generator=g)).to(DEV)
    m = (0.3 * torch.rand(b, generator=g)).to(DEV)
    check(x, u, t, k, p, m)
    check(x, u, 0.9, k, 0.8, m)


def test_strides_and_streams():
    wide, u = rows(6, 4 * 1001, F, seed=8)
    x = wide.view(6, 4, 1001)[:, -1]  # the last position's logits; rows of odd starts
    assert x.stride(0) == 4004
    want = check(x, u, 0.8, 50, 0.9)
    columns = x.t().contiguous().t()
    assert torch.equal(sample_tokens(columns, u, temperature=0.8, top_k=50, top_p=0.9), want)
    half = x.to(BF)
    odd = torch.zeros(6 * 1001 + 1, dtype=BF, device=DEV)[1:].view(6, 1001)
    odd.copy_(half)
    assert torch.equal(sample_tokens(odd, u, top_p=0.9), sample_tokens(half, u, top_p=0.9))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = [sample_tokens(x, u, temperature=0.8, top_k=50, top_p=0.9) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_a_captured_draw_follows_its_inputs():
    x, u = rows(5, 32000, BF, seed=9)
    t = torch.full((5,), 0.8, device=DEV)
    sample_tokens(x, u, temperature=t, top_p=0.9)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = sample_tokens(x, u, temperature=t, top_p=0.9)
    for turn in range(4):
        y, r = rows(5, 32000, BF, seed=10 + turn)
        x.copy_(y), u.copy_(r), t.fill_(0.5 + 0.4 * turn)
        want = sample_tokens(x, u, temperature=t, top_p=0.9)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_no_rows():
    assert sample_tokens(torch.zeros(0, 10, device=DEV), torch.zeros(0, device=DEV)).shape == (0,)

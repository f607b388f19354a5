"""Edges of the paged cache's operators on the GPU, against float64 with the bounds of
``test_cache_op``."""

from __future__ import annotations

import contextlib

import pytest
import torch
from torch.autograd import forward_ad
from torch.overrides import TorchFunctionMode

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a HIP device", allow_module_level=True)

from test_cache_op import Case  # noqa: E402

from switchyard.cache_op import paged_append, paged_attention  # noqa: E402

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


def scaled(c, scale, **more):
    """``paged_attention`` with a scale, checked; a negative one is a positive one of turned queries."""
    got = c.call(scale=scale, **more).cpu().double()
    q = c.q
    c.q = q if scale >= 0 else -q
    want, tol = c.expected(abs(scale))
    c.q = q
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol.clamp_min(1e-30)).max().item()


SCALES = [
    # new, past, kv, group, hd, page, prefix
    ([1, 1, 3], [5, 70, 300], 2, 2, 64, 16, 0),  # few rows
    ([65, 129], [0, 77], 1, 1, 128, 64, 0),  # many
    ([17, 1, 40], [15, 0, 130], 2, 2, 80, 16, 0),  # both, of a padded width
    ([1] * 20, list(range(20)), 1, 3, 64, 32, 200),  # a prefix's pass of many rows
    ([1, 1], [9, 40], 2, 2, 128, 16, 333),  # and of few
    ([90, 41], [0, 7], 1, 2, 64, 16, 100),  # a prefix before many rows of each
]


@pytest.mark.parametrize("scale", [0.0, 1e-42, -0.2, 0.5, -0.0])
@pytest.mark.parametrize("shape", SCALES, ids=[str(i) for i in range(len(SCALES))])
@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_scales(dtype, shape, scale):
    """Any scale: none gives the mean of what a row sees."""
    new, past, kv, group, hd, page, prefix = shape
    scaled(Case(new, past, kv=kv, group=group, hd=hd, page=page, dtype=dtype, prefix=prefix, seed=31), scale)


def test_a_query_of_nan_without_a_scale():
    """Only its own row is NaN."""
    c = Case([65, 40], [0, 30], kv=1, group=2, hd=64, page=16, dtype=BF, seed=32)
    c.q[50, 1, 3] = float("nan")
    bad = torch.zeros(105, 2, dtype=torch.bool)
    bad[50, 1] = True
    assert torch.equal(torch.isnan(c.call(scale=0.0).cpu()).all(-1), bad)
    assert torch.equal(torch.isnan(c.call(scale=0.0).cpu()).any(-1), bad)


def _serving(seed):
    """A case's tensors for both functions: (append's arguments, attention's), by name."""
    c = Case([1, 2], [5, 20], kv=1, group=2, hd=64, page=16, dtype=F, seed=seed)
    d = dict(qkv=torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(seed)).to(DEV),
             cos=torch.ones(64, 32, device=DEV), sin=torch.zeros(64, 32, device=DEV), q=c.q.to(DEV), k=c.k.to(DEV),
             v=c.v.to(DEV))
    rest = (c.table.to(DEV), c.lengths.to(DEV), c.starts.to(DEV))
    return d, rest


def _both(d, rest, out=None):
    q = paged_append(d["qkv"], d["cos"], d["sin"], d["k"], d["v"], *rest, out=out)
    return q, paged_attention(d["q"], d["k"], d["v"], *rest, out=out)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", ["qkv", "cos", "sin", "q", "k", "v"])
def test_tangents_are_refused(name, grad):
    """A tangent must not get lost: no_grad does not switch forward mode off."""
    d, rest = _serving(41)
    _both(d, rest)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual = {**d, name: forward_ad.make_dual(d[name], torch.ones_like(d[name]))}
        with pytest.raises(RuntimeError, match="no derivative"):
            _both(dual, rest)
    def one(x):  # the function that takes it, inside a transform
        e = {**d, name: x}
        if name in ("qkv", "cos", "sin"):
            return paged_append(e["qkv"], e["cos"], e["sin"], e["k"], e["v"], *rest)
        return paged_attention(e["q"], e["k"], e["v"], *rest)

    with pytest.raises(RuntimeError, match="no derivative"):
        torch.func.jvp(one, (d[name],), (torch.ones_like(d[name]),))
    _both(d, rest)


class _Mode(TorchFunctionMode):
    def __torch_function__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("mode", [contextlib.nullcontext, _Mode], ids=["native", "python"])
def test_autograd_notices_what_is_written(mode):
    """A tensor that a backward saved and a call then overwrote."""
    d, rest = _serving(42)
    w = torch.randn((), device=DEV, requires_grad=True)
    out = torch.zeros(3, 2, 64, device=DEV)
    for name, t in (("k", d["k"]), ("v", d["v"]), ("out", out)):
        loss = (w * t).sum()
        with torch.no_grad(), mode():
            before = t._version
            _both(d, rest, out=out if name == "out" else None)
            assert t._version == before + (2 if name == "out" else 1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode(), mode():  # such tensors have no version
        e, rest = _serving(42)
        _both(e, rest, out=torch.zeros(3, 2, 64, device=DEV))

"""Edges of the paged cache's operators on the GPU, against float64 with the bounds of
``test_cache_op``.

fp16 ends where bf16 goes on: its steps are 2^-24 below 2^-14. A weight (relative to the
largest) is therefore off by at most half of such a step over what the kernels lift weights
by, 2^-25 2^-15 where a sequence has up to 16 rows and 2^-25 2^-7 where it has more, if that is
more than its own rounding. Over n keys that is n step / l (max|v| + |o|) of the result, with
l the sum of the weights."""

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
from switchyard.sample_op import sample_tokens  # noqa: E402

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


FAINT = [
    # new, past, kv, group, prefix, what a weight may be off by
    ([1, 1], [3000, 40], 2, 2, 0, 2.0**-40),  # whole sequences in one workgroup
    ([1, 3], [20000, 64], 1, 1, 0, 2.0**-40),  # one shared out
    ([65, 30], [3000, 100], 1, 2, 0, 2.0**-32),
    ([1] * 20, list(range(20)), 1, 2, 3000, 2.0**-32),  # a prefix's pass
    ([1, 1], [9, 40], 2, 2, 3000, 2.0**-40),
    ([40, 20], [0, 7], 1, 2, 3000, 2.0**-32),
]


@pytest.mark.parametrize("below", [14.0, 20.0, 24.5])
@pytest.mark.parametrize("shape", FAINT, ids=[str(i) for i in range(len(FAINT))])
@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_many_faint_tokens(dtype, shape, below):
    """Every 32nd token is strong and has no value; all the others are 2^-below and fainter,
    and are the result."""
    new, past, kv, group, prefix, step = shape
    c = Case(new, past, kv=kv, group=group, hd=64, page=32, dtype=dtype, prefix=prefix, seed=51)
    g = torch.Generator().manual_seed(52)
    c.q.zero_()
    c.q[..., 0] = 8.0  # (the scale is 1/8)
    c.k.zero_()
    c.k[..., 0] = -(below + 3 * torch.rand(c.k.shape[:3], generator=g)) * 0.6931
    c.v.copy_(512 * (1 + 0.25 * torch.randn(c.v.shape, generator=g)))
    c.k[:, :, 0], c.v[:, :, 0] = 0.0, 0.0
    want, tol = c.expected()
    got = c.call().cpu().double()
    assert (want > 0).any()
    if dtype == HF:
        tol = tol + 2.0**-25 + 32 * step * (c.v.double().abs().max() + want)  # (l is at least n / 32)
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol.clamp_min(1e-30)).max().item()


@pytest.mark.parametrize("q", [300.0, 3000.0, 60000.0, -300.0, -3000.0, -60000.0])
@pytest.mark.parametrize("shape", FAINT, ids=[str(i) for i in range(len(FAINT))])
@pytest.mark.parametrize("dtype,times", [(HF, 1.0), (BF, 1.0), (BF, 1e12), (F, 1.0)])
@pytest.mark.parametrize("hd", [64, 80])
def test_scores_past_every_step(hd, dtype, times, shape, q):
    """Scores of 2^21 to 2^29 (bf16 to 2^109) of either sign: the nearest other is thousands
    below the largest, so that the result is its value to the bit."""
    new, past, kv, group, prefix, _ = shape
    c = Case(new, past, kv=kv, group=group, hd=hd, page=32, dtype=dtype, prefix=prefix, seed=53)
    g = torch.Generator().manual_seed(54)
    c.q.zero_()
    c.q[..., 0] = q * times
    c.k.zero_()
    c.k[..., 0] = times * (55000 + 10000 * torch.rand(c.k.shape[:3], generator=g) * (1 if q < 0 else -5))
    want, at = torch.zeros(c.n_tok, c.heads, hd, dtype=dtype), 0
    for b, n in enumerate(new):
        first = c.prefix_ids[0] if prefix else int(c.table[b, 0])
        c.k[first, :, 0, 0] = times * (50000.0 if q < 0 else 60000.0)
        want[at:at + n] = c.v[first, :, 0].repeat_interleave(group, 0)
        at += n
    assert torch.equal(c.call().cpu(), want)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hd", [64, 80, 128])
def test_a_decoded_token_behind_a_prefix_is_exact_to_its_rounding(hd, dtype):
    """However many share the prefix, the weights are not rounded: nearly all results are the
    exact ones' roundings. fp32 errors of a few 2^-20 (of rows that cancel, of more than |o|)
    pass one of fp16's borders, 2^-10 apart, once in a hundred times, and bf16's once in a
    thousand; weights off by a third of a step on average would every fourth time."""
    for n in (4, 40):
        c = Case([1] * n, [7 * i for i in range(n)], kv=2, group=2, hd=hd, page=16, dtype=dtype, prefix=300, seed=61)
        want, _ = c.expected()
        other = (c.call().cpu() != want.to(dtype)).double().mean().item()
        assert other < 0.04, other


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("new", [[1, 1, 2], [1] * 20, [40, 25]])
def test_infinities_around_a_prefixs_end(new, dtype):
    """Behind the prefix's last token anything may lie; a visible infinity makes its channel of
    every row one, or NaN (a weight's remainder times it has any sign), and no other."""
    c = Case(new, [5 * i % 50 for i in range(len(new))], kv=2, group=2, hd=64, page=32, dtype=dtype, prefix=75, seed=62)
    want = c.call().cpu()
    last = c.prefix_ids[-1]
    for cache in (c.k, c.v):
        cache[last, :, 11:] = float("nan")
    assert torch.equal(c.call().cpu(), want)
    c.v[last, 1, 9, 33] = float("inf")
    got = c.call().cpu()
    assert not torch.isfinite(got[:, 2:, 33]).any()
    got[:, 2:, 33] = want[:, 2:, 33]
    # (That token's other channels are added apart from the rest: same bounds, other order.)
    u = torch.finfo(dtype).eps / 2
    ref = want.double()
    assert ((got.double() - ref).abs() <= 2 * u * ref.abs() + (2 * u if dtype != F else 2.0**-15) * 4).all()


WIDTHS = [
    # new, past, kv, group, page, prefix
    ([1, 1, 1], [5, 0, 70], 2, 2, 16, 333),  # a prefix for few rows
    ([1] * 40, list(range(40)), 1, 3, 32, 333),  # its pass for many, next to each sequence's own
    ([90, 41], [0, 7], 1, 2, 16, 100),  # before many rows of each
    ([20], [5000], 1, 1, 64, 0),  # a row tile's keys in parts, joined
    ([40, 3, 1], [2500, 4000, 900], 2, 1, 16, 0),  # next to sequences of few rows
    ([1] * 24, list(range(24)), 1, 1, 32, 3000),  # a prefix's keys in parts
]


@pytest.mark.parametrize("hd", [8, 40, 64, 80, 96, 128, 136, 256])
@pytest.mark.parametrize("shape", WIDTHS, ids=[str(i) for i in range(len(WIDTHS))])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_widths_behind_prefixes_and_in_parts(dtype, shape, hd):
    new, past, kv, group, page, prefix = shape
    Case(new, past, kv=kv, group=group, hd=hd, page=page, dtype=dtype, prefix=prefix, seed=71).check()


@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_a_compiled_caller(dtype):
    """A compiler's trace steps around the functions: same results, same writes, every time."""
    c = Case([1, 2], [5, 20], kv=1, group=2, hd=64, page=16, dtype=dtype, prefix=20, seed=72)
    cos, sin = torch.ones(64, 32, device=DEV), torch.zeros(64, 32, device=DEV)
    qkv = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(73)).to(dtype).to(DEV)
    more = dict(prefix_pages=torch.tensor(c.prefix_ids, dtype=torch.int32, device=DEV), prefix_len=20)
    u = torch.rand(3, generator=torch.Generator().manual_seed(74)).to(DEV)

    def step(qkv, k, v, table, lengths, starts):
        q = paged_append(qkv * 2, cos, sin, k, v, table, lengths, starts, prefix_len=20)
        o = paged_attention(q, k, v, table, lengths, starts, **more) + 1
        return o, sample_tokens(o.flatten(1), u, temperature=0.7, top_k=5) * 2

    got = []
    compiled = torch.compile(step, backend="eager")
    for fn in (step, compiled, compiled):
        k, v = c.k.to(DEV), c.v.to(DEV)
        with torch.no_grad():
            got.append((*fn(qkv, k, v, c.table.to(DEV), c.lengths.to(DEV), c.starts.to(DEV)), k, v))
    assert all(torch.equal(a, b) for some in zip(*got) for a, b in zip(some, some[1:]))


def _many(dtype, new, past, **kw):
    return Case(new, past, kv=1, group=1, hd=64, page=16, dtype=dtype, seed=81, **kw)


@pytest.mark.parametrize("dtype", [BF, F])
def test_more_sequences_than_lanes(dtype):
    """Of many rows each, evenly and raggedly; and thousands of single tokens, shared out."""
    _many(dtype, [20] * 70, [3 * i for i in range(70)]).check()
    _many(dtype, [20, 1, 33, 0, 130] * 30, [i for i in range(150)]).check()
    _many(dtype, [20, 1, 33, 0, 130] * 15, [i for i in range(75)], prefix=50).check()
    c = _many(dtype, [1] * 3000, [i % 60 for i in range(3000)])
    want = c.call()
    c.check(want)
    c.check(c.call(packed=True))


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("prefix", [0, 50])
@pytest.mark.parametrize("rows", [3, 200])
def test_rows_of_no_sequence_at_all(rows, prefix, dtype):
    c = _many(dtype, [rows, 0, 0], [40, 3, 900], prefix=prefix)
    q = c.q.to(DEV)
    for at in (0, 1, rows):
        c.starts = torch.full((4,), at, dtype=torch.int32)
        assert (c.call() == 0).all()
        out = torch.full_like(q, 3.0)
        c.call(out=out)
        assert (out == 3).all()
    k, v = c.k.to(DEV), c.v.to(DEV)
    ones = torch.ones(1000, 32, device=DEV)
    qkv = torch.randn(rows, 3, 64, device=DEV).to(dtype)
    got = paged_append(qkv, ones, ones, k, v, c.table.to(DEV), c.lengths.to(DEV), c.starts.to(DEV))
    assert (got == 0).all() and torch.equal(k.cpu(), c.k) and torch.equal(v.cpu(), c.v)

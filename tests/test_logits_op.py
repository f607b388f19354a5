"""Penalties, biases and masks on logits on the GPU against float64.

Tolerances. Penalties are computed in fp64 and rounded to fp32, the bias is added in fp32 and
the result rounded to the logits' dtype: 2^-24 of the penalised logit, 2^-24 of the sum, and
eps / 2 of the result."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a HIP device", allow_module_level=True)

from switchyard import _lib  # noqa: E402
from switchyard.logits_op import adjust_logits, pack_allowed  # noqa: E402
from switchyard.sample_op import sample_tokens  # noqa: E402

DEV = "cuda"
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _expected(x, tokens=None, lengths=None, prompts=None, r=1.0, p=0.0, f=0.0, bias=None, allowed=None):
    """Row by row; (result, tolerance)."""
    y = x.double().clone()
    b, v = x.shape
    row = lambda s, i: float(s[i]) if torch.is_tensor(s) else float(s)  # noqa: E731
    for i in range(b):
        if tokens is None:
            continue
        n = tokens.shape[1] if lengths is None else max(0, min(int(lengths[i]), tokens.shape[1]))
        first = 0 if prompts is None else int(prompts[i])
        hist = tokens[i, :n].tolist()
        for t in {t for t in hist if 0 <= t < v}:
            z = float(y[i, t])
            z = z / row(r, i) if z > 0 else z * row(r, i)
            said = sum(1 for j, h in enumerate(hist) if h == t and j >= first)
            if said:
                z -= row(f, i) * said + row(p, i)
            y[i, t] = z
    u = torch.finfo(x.dtype).eps / 2
    tol = y.abs() * 2.0**-24
    if bias is not None:
        y = y + bias.double()
        tol = tol + y.abs() * 2.0**-24
    tol = (tol + u * (y.abs() + tol)).nan_to_num(0.0, 0.0, 0.0)
    if x.dtype == HF:
        tol = tol + torch.finfo(HF).smallest_normal * u
    if allowed is not None:
        y = y.masked_fill(~allowed, -math.inf)
    return y, tol


def _check(got, want):
    y, tol = want
    got = got.cpu().double()
    fine = torch.isfinite(y)
    assert torch.equal(got[~fine].nan_to_num(7.0), y[~fine].nan_to_num(7.0))
    assert ((got - y).abs()[fine] <= tol[fine]).all()


def _cuda(**kw):
    return {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in kw.items()}


def _case(b, v, length, dtype, seed, per_row=False):
    g = _gen(seed)
    x = (3 * torch.randn(b, v, generator=g)).to(dtype)
    tokens = (v * torch.rand(b, length, generator=g) ** 3).long().clamp(max=v - 1)
    lengths = torch.randint(0, length + 1, (b,), generator=g, dtype=torch.int32)
    lengths[0] = length
    prompts = (lengths * torch.rand(b, generator=g)).int()
    if per_row:
        s = [0.5 + torch.rand(b, generator=g), torch.randn(b, generator=g), torch.randn(b, generator=g)]
    else:
        s = [1.3, 0.7, -0.2]
    return x, tokens, lengths, prompts, s


def _run(x, tokens, lengths, prompts, s, **more):
    return adjust_logits(x.to(DEV), tokens.to(DEV), **_cuda(
        lengths=lengths, prompt_lengths=prompts, repetition_penalty=s[0], presence_penalty=s[1], frequency_penalty=s[2],
        **more))


SHAPES = [(2, 5000, 9000), (1, 1, 1), (2, 7, 5), (3, 33, 64), (5, 1000, 300), (2, 1023, 9), (1, 1025, 2000), (4, 4097, 77), (9, 50257, 500),
          (130, 300, 40), (2, 131072, 3000)]


@pytest.mark.parametrize("b,v,length", SHAPES)
@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("per_row", [False, True])
def test_penalties(b, v, length, dtype, per_row):
    x, tokens, lengths, prompts, s = _case(b, v, length, dtype, b + v, per_row)
    want = _expected(x, tokens, lengths, prompts, *s)
    got = _run(x, tokens, lengths, prompts, s)
    assert got.dtype == dtype and got.shape == (b, v)
    _check(got, want)
    assert torch.equal(_run(x, tokens.int(), lengths, prompts, s), got)


@pytest.mark.parametrize("b,v", [(1, 1), (3, 31), (2, 33), (4, 1001), (7, 4099), (2, 50257)])
@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_biases_and_masks(b, v, dtype):
    g = _gen(v)
    x, tokens, lengths, prompts, s = _case(b, v, 20, dtype, v)
    rows = torch.rand(b, v, generator=g) < 0.4
    rows[0] = False  # a row that allows nothing
    if b > 1:
        rows[1] = True
    whole = torch.rand(v, generator=g) < 0.5
    wide, narrow = torch.randn(b, v, generator=g), torch.randn(v, generator=g).to(dtype)
    for bias in (None, wide, narrow, narrow.float(), wide.to(dtype)):
        for keep in (None, rows, whole):
            want = _expected(x, tokens, lengths, prompts, *s, bias=bias, allowed=keep)
            forms = [None] if keep is None else [keep.to(DEV), pack_allowed(keep.to(DEV))]
            for m in forms:
                _check(_run(x, tokens, lengths, prompts, s, bias=bias, allowed=m), want)
            if keep is not None:
                got = adjust_logits(x.to(DEV), bias=None if bias is None else bias.to(DEV), allowed=forms[1])
                _check(got, _expected(x, bias=bias, allowed=keep))


@pytest.mark.parametrize("dtype", [BF, F])
def test_in_place_and_strided_rows(dtype):
    x, tokens, lengths, prompts, s = _case(6, 5001, 100, dtype, 1)
    keep = torch.rand(6, 5001, generator=_gen(2)) < 0.7
    for allowed in (None, keep):
        want = _run(x, tokens, lengths, prompts, s, allowed=allowed)
        y = x.to(DEV)
        before = y._version
        assert _run(y, tokens, lengths, prompts, s, allowed=allowed, out=y) is y
        assert torch.equal(y, want) and y._version > before
        wide = torch.full((6, 6000), 7.0, dtype=dtype, device=DEV)
        wide[:, 3:5004] = x.to(DEV)
        view = wide[:, 3:5004]
        assert torch.equal(_run(view, tokens, lengths, prompts, s, allowed=allowed), want)
        _run(view, tokens, lengths, prompts, s, allowed=allowed, out=view)
        assert torch.equal(view, want) and (wide[:, :3] == 7).all() and (wide[:, 5004:] == 7).all()
        halves = torch.full((6, 2, 5001), 7.0, dtype=dtype, device=DEV)  # rows between the logits'
        halves[:, 0] = x.to(DEV)
        _run(halves[:, 0], tokens, lengths, prompts, s, allowed=allowed, out=halves[:, 1])
        assert torch.equal(halves[:, 0].cpu(), x) and torch.equal(halves[:, 1], want)
        with pytest.raises(RuntimeError, match="sy_adjust"):
            adjust_logits(wide[:, :5001], out=wide[:, 1:5002])
        with pytest.raises(RuntimeError, match="sy_adjust"):
            adjust_logits(wide[:5, :5001], out=wide[1:, :5001])
        turned = x.to(DEV).t().contiguous().t()
        assert torch.equal(_run(turned, tokens, lengths, prompts, s, allowed=allowed), want)
        assert torch.equal(_run(x, tokens.t().contiguous().t(), lengths, prompts, s, allowed=allowed), want)


def test_histories_of_any_content():
    x = torch.tensor([[2.0, -2.0, 0.0, -math.inf, math.inf, math.nan, 1.0, 1.0]] * 5)
    tokens = torch.tensor([[0, 1, 2, 3, 4, 5, 0, 0], [-1, 8, 2**40, -(2**40), 6, 6, 6, 6]] + [[6] * 8] * 3)
    lengths = torch.tensor([8, 8, 0, -3, 100], dtype=torch.int32)
    prompts = torch.tensor([6, 4, 0, 0, 200], dtype=torch.int32)
    for s in ((2.0, 0.5, 0.25), (1.0, 0.0, 0.0), (1.0, 1.0, 0.0)):
        _check(_run(x, tokens, lengths, prompts, s), _expected(x, tokens, lengths, prompts, *s))
    # No history at all, and one of no columns.
    assert torch.equal(adjust_logits(x.to(DEV)).cpu().nan_to_num(9.0), x.nan_to_num(9.0))
    got = adjust_logits(x.to(DEV), tokens[:, :0].to(DEV), repetition_penalty=3.0)
    assert torch.equal(got.cpu().nan_to_num(9.0), x.nan_to_num(9.0))
    assert adjust_logits(x[:0].to(DEV)).shape == (0, 8)


def test_a_shared_history_and_settings_by_broadcast():
    x, tokens, lengths, prompts, s = _case(4, 900, 50, F, 5)
    one = tokens[:1].expand(4, 50)
    want = _run(x, one.contiguous(), lengths, prompts, s)
    got = adjust_logits(x.to(DEV), tokens[:1].to(DEV).expand(4, 50), **_cuda(
        lengths=lengths, prompt_lengths=prompts, repetition_penalty=torch.tensor([1.3]).to(DEV).expand(4),
        presence_penalty=0.7, frequency_penalty=-0.2))
    assert (got - want).abs().max().item() <= 2.0**-20  # (1.3 as fp32 there)
    bias = torch.randn(1, 900, device=DEV)
    assert torch.equal(adjust_logits(x.to(DEV), bias=bias.expand(4, 900)), adjust_logits(x.to(DEV), bias=bias[0]))


def test_masked_rows_and_sampling():
    x = torch.randn(3, 100, device=DEV)
    keep = torch.zeros(3, 100, dtype=torch.bool)
    keep[0, 41] = keep[1, 99] = True
    y = adjust_logits(x, allowed=pack_allowed(keep).to(DEV))
    assert sample_tokens(y, torch.full((3,), 0.5, device=DEV)).tolist() == [41, 99, -1]


def test_another_stream_a_graph_and_the_python_path(monkeypatch):
    x, tokens, lengths, prompts, s = _case(5, 3001, 60, BF, 9)
    a = _cuda(x=x, tokens=tokens, lengths=lengths, prompts=prompts)
    call = lambda: adjust_logits(a["x"], a["tokens"], lengths=a["lengths"], prompt_lengths=a["prompts"],  # noqa: E731
                                 repetition_penalty=1.3, presence_penalty=0.7, frequency_penalty=-0.2)
    want = call()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = call()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = call()
    for i in range(3):
        a["lengths"].fill_(10 * i)
        a["tokens"].copy_(torch.randint(0, 3001, (5, 60), device=DEV))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, call())
    want = call()
    bias, keep = torch.randn(5, 3001, device=DEV), torch.rand(3001, device=DEV) < 0.5
    full = adjust_logits(a["x"], bias=bias, allowed=keep)
    monkeypatch.setattr(_lib, "ordinary", lambda *t: False)
    assert torch.equal(call(), want) and torch.equal(adjust_logits(a["x"], bias=bias, allowed=keep), full)


def test_gradients_are_refused():
    x = torch.randn(2, 10, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        adjust_logits(x)
    with torch.no_grad():
        adjust_logits(x)

"""Head norms with the rotation on the GPU, forward, backward and into a paged cache, against
float64.

Tolerances. A head's sum of squares is a chain of at most 16 fp32 additions a lane and 5 over
the lanes, the root halves its error, and r, the gain and the rotation add a few roundings:
under 2^-19 of the head's largest output. The gradient has one more such sum: under 2^-18 of
r max |g e| (1 + max u^2). Outputs are rounded once. Gains' gradients: a sum of n products in
fp32, at most n 2^-24 of the sum of their sizes."""

from __future__ import annotations

import gc
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a HIP device", allow_module_level=True)

from oracle.reference import dtype_floor, rel_l2  # noqa: E402
from switchyard import _lib, rope_op  # noqa: E402
from switchyard.cache_op import paged_append  # noqa: E402
from switchyard.rope_op import qk_norm_rope  # noqa: E402

DEV = "cuda"
BF, HF, F = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-6


def _rand(*shape, dtype, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _tables(t, hd):
    ang = torch.arange(t, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(hd // 2, dtype=torch.float64) * 2 / hd)
    return ang.cos().float(), ang.sin().float()


def _heads(x, gain, cos, sin):
    """fp64 ``x [..., hd]``, angles that broadcast over it."""
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gain
    lo, hi = y.chunk(2, -1)
    return torch.cat((lo * cos - hi * sin, lo * sin + hi * cos), -1)


def _by_formula(qkv, gq, gk, cos, sin, heads, kv):
    t = qkv.shape[1]
    q, k, v = qkv.transpose(1, 2).split([heads, kv, kv], 1)
    c, s = cos[:t].double(), sin[:t].double()
    return _heads(q, gq, c, s), _heads(k, gk, c, s), v


SHAPES = [  # b, t, heads, kv, hd
    (1, 1, 1, 1, 8), (2, 5, 3, 1, 16), (1, 33, 4, 2, 24), (3, 7, 6, 3, 40), (2, 130, 2, 2, 64), (1, 17, 5, 1, 72),
    (2, 9, 3, 3, 80), (1, 65, 12, 4, 96), (2, 40, 4, 4, 128), (1, 11, 2, 1, 248), (1, 300, 9, 3, 256), (5, 3, 48, 1, 64),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype,gains", [(BF, BF), (HF, HF), (F, F), (BF, F), (HF, F)])
def test_forward_and_backward(shape, dtype, gains):
    b, t, heads, kv, hd = shape
    qkv = _rand(b, t, heads + 2 * kv, hd, dtype=dtype, seed=1)
    gq, gk = ((1 + 0.5 * _rand(hd, dtype=F, seed=s)).to(gains) for s in (2, 3))
    cos, sin = _tables(t + 3, hd)
    grads = [_rand(b, h, t, hd, dtype=dtype, seed=4 + i) for i, h in enumerate((heads, kv, kv))]
    x, a, c = (z.to(DEV).requires_grad_() for z in (qkv, gq, gk))
    outs = qk_norm_rope(x, a, c, cos.to(DEV), sin.to(DEV), kv_heads=kv, eps=EPS)
    got = torch.autograd.grad(outs, (x, a, c), [g.to(DEV) for g in grads])
    x6, a6, c6 = (z.double().requires_grad_() for z in (qkv, gq, gk))
    want = _by_formula(x6, a6, c6, cos, sin, heads, kv)
    want_grads = torch.autograd.grad(want, (x6, a6, c6), [g.double() for g in grads])
    u = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(HF).smallest_normal * u if dtype == HF else 0.0
    for o, w in zip(outs, want):
        w = w.detach()
        tol = u * w.abs() + 2.0**-19 * w.abs().amax(-1, keepdim=True) * (1 + u) + tiny
        assert o.dtype == dtype and o.shape == w.shape and o.is_contiguous()
        assert ((o.detach().cpu().double() - w).abs() <= tol).all()
    assert torch.equal(outs[2].detach().cpu(), qkv[:, :, heads + kv:].transpose(1, 2))
    # dx, head by head
    dx, wx = got[0].cpu().double(), want_grads[0]
    assert got[0].dtype == dtype and got[0].shape == qkv.shape
    r = torch.rsqrt(qkv.double().square().mean(-1, keepdim=True) + EPS)
    top = qkv.double().mul(r).square().amax(-1, keepdim=True)
    e = torch.cat([g.double().transpose(1, 2) for g in grads], 2).abs()
    e = e + torch.cat(e.chunk(2, -1)[::-1], -1)  # at least the turned-back gradient
    gain = torch.stack([gq.double().abs().amax()] * heads + [gk.double().abs().amax()] * kv + [torch.ones(()).double()] * kv)
    size = r * e.amax(-1, keepdim=True) * gain[:, None] * (1 + top)
    assert ((dx - wx).abs() <= u * wx.abs() + 2.0**-18 * size * (1 + u) + tiny).all()
    n = b * t * max(heads, kv)
    ug = torch.finfo(gains).eps / 2
    for i, h0, h1 in ((1, 0, heads), (2, heads, heads + kv)):
        xs = qkv.double()[:, :, h0:h1]
        us = xs * torch.rsqrt(xs.square().mean(-1, keepdim=True) + EPS)
        size = (e[:, :, h0:h1] * us.abs()).sum((0, 1, 2))
        assert got[i].dtype == gains
        assert ((got[i].cpu().double() - want_grads[i]).abs()
                <= ug * want_grads[i].abs() + (n + 60) * 2.0**-24 * size * (1 + ug)).all()


def test_training_sizes_are_within_the_rounding_floor():
    for dtype, b, t, heads, kv, hd in ((BF, 2, 1500, 16, 16, 128), (F, 3, 701, 12, 4, 96), (HF, 1, 3000, 8, 2, 80)):
        qkv = _rand(b, t, heads + 2 * kv, hd, dtype=dtype, seed=1)
        gq, gk = ((1 + 0.3 * _rand(hd, dtype=F, seed=s)).to(dtype) for s in (2, 3))
        cos, sin = _tables(t, hd)
        grads = [_rand(b, h, t, hd, dtype=dtype, seed=4 + i) for i, h in enumerate((heads, kv, kv))]
        x, a, c = (z.to(DEV).requires_grad_() for z in (qkv, gq, gk))
        outs = qk_norm_rope(x, a, c, cos.to(DEV), sin.to(DEV), kv_heads=kv, eps=EPS)
        got = (*outs, *torch.autograd.grad(outs, (x, a, c), [g.to(DEV) for g in grads]))
        x6, a6, c6 = (z.double().requires_grad_() for z in (qkv, gq, gk))
        want = _by_formula(x6, a6, c6, cos, sin, heads, kv)
        want = (*want, *torch.autograd.grad(want, (x6, a6, c6), [g.double() for g in grads]))
        for o, w in zip(got, want):
            o, w = o.detach().cpu(), w.detach()
            floor = 1e-6 if dtype == F else 1.10 * dtype_floor(w, dtype)
            if o.ndim == 1 and dtype != F:  # few values: their own roundings, not the average one
                floor = torch.finfo(dtype).eps / 2
            assert rel_l2(o, w) <= floor


def test_against_differences():
    qkv = _rand(1, 3, 5, 16, dtype=torch.float64, seed=1)
    a, c = (1 + 0.3 * _rand(16, dtype=torch.float64, seed=s) for s in (2, 3))
    cos, sin = _tables(3, 16)
    grads = [_rand(1, h, 3, 16, dtype=torch.float64, seed=4 + i) for i, h in enumerate((3, 1, 1))]

    def loss(q, x, y):
        return sum((o * g).sum() for o, g in zip(_by_formula(q, x, y, cos, sin, 3, 1), grads)).item()

    xs = [z.float().to(DEV).requires_grad_() for z in (qkv, a, c)]
    outs = qk_norm_rope(*xs, cos.to(DEV), sin.to(DEV), kv_heads=1, eps=EPS)
    got = torch.autograd.grad(outs, xs, [g.float().to(DEV) for g in grads])
    base = [z.float().double() for z in (qkv, a, c)]
    for i in range(3):
        flat = base[i].view(-1)
        for j in range(0, flat.numel(), 7):
            h, old = 1e-5, flat[j].item()
            flat[j] = old + h
            up = loss(*base)
            flat[j] = old - h
            down = loss(*base)
            flat[j] = old
            # differences of a smooth function: h^2 of its third derivative (below 100 here) and
            # fp64's rounding over h; the kernel's own 2^-18
            assert abs(got[i].view(-1)[j].item() - (up - down) / (2 * h)) <= 1e-4


def test_strided_gradients_inputs_and_unused_outputs():
    b, t, heads, kv, hd = 2, 19, 4, 2, 64
    qkv = _rand(b, t, 8, hd, dtype=BF, seed=1).to(DEV)
    gq, gk = ((1 + 0.3 * _rand(hd, dtype=F, seed=s)).to(DEV) for s in (2, 3))
    cos, sin = (z.to(DEV) for z in _tables(t, hd))
    grads = [_rand(b, h, t, hd, dtype=BF, seed=4 + i).to(DEV) for i, h in enumerate((heads, kv, kv))]

    def run(x, gs):
        x = x.detach().requires_grad_()
        a, c = gq.clone().requires_grad_(), gk.clone().requires_grad_()
        outs = qk_norm_rope(x, a, c, cos, sin, kv_heads=kv, eps=EPS)
        return (*outs, *torch.autograd.grad([o for o, g in zip(outs, gs) if g is not None], (x, a, c),
                                            [g for g in gs if g is not None], allow_unused=True))

    want = run(qkv, grads)
    by_token = [g.transpose(1, 2).contiguous().transpose(1, 2) for g in grads]
    by_channel = [g.transpose(2, 3).contiguous().transpose(2, 3) for g in grads]
    wide = torch.empty(b, t, 8, 3 * hd, device=DEV, dtype=BF)
    wide[..., 5:5 + hd] = qkv
    for x, gs in ((qkv, by_token), (qkv, by_channel), (wide[..., 5:5 + hd], grads), (qkv.transpose(1, 2).contiguous().transpose(1, 2), grads)):
        for o, w in zip(run(x, gs), want):
            assert torch.equal(o, w)
    shared = torch.ones(1, 1, 1, 1, device=DEV, dtype=BF)
    same = [shared.expand(b, h, t, hd) for h in (heads, kv, kv)]
    for o, w in zip(run(qkv, same), run(qkv, [g.contiguous() for g in same])):
        assert torch.equal(o, w)
    for i in range(3):
        only = [g if j == i else None for j, g in enumerate(grads)]
        zeros = [g if j == i else torch.zeros_like(g) for j, g in enumerate(grads)]
        for o, w in zip(run(qkv, only), run(qkv, zeros)):
            assert torch.equal(o, w)


def test_second_derivatives_and_transforms():
    qkv = _rand(2, 4, 6, 16, dtype=F, seed=1).to(DEV).requires_grad_()
    gq, gk = ((1 + 0.3 * _rand(16, dtype=F, seed=s)).to(DEV).requires_grad_() for s in (2, 3))
    cos, sin = (z.to(DEV) for z in _tables(4, 16))
    gs = [_rand(2, 2, 4, 16, dtype=F, seed=4 + i).to(DEV).requires_grad_() for i in range(3)]

    def second(f):
        outs = f(qkv, gq, gk)
        first = torch.autograd.grad(outs, (qkv, gq, gk), gs, create_graph=True)
        return (*first, *torch.autograd.grad(sum(x.square().sum() for x in first), (qkv, gq, gk, gs[0], gs[1])))

    got = second(lambda *x: qk_norm_rope(*x, cos, sin, eps=EPS))
    want = second(lambda *x: rope_op._by_operations(*x, cos, sin, 2, 2, EPS))
    for o, w in zip(got, want):
        assert rel_l2(o.detach().cpu(), w.detach().cpu().double()) <= 1e-5  # two fp32 evaluations
    outs = torch.func.vmap(lambda x: qk_norm_rope(x, gq, gk, cos, sin, eps=EPS))(qkv.detach()[:, None])
    for o, w in zip(outs, qk_norm_rope(qkv.detach(), gq, gk, cos, sin, eps=EPS)):
        assert rel_l2(o[:, 0].detach().cpu(), w.detach().cpu().double()) <= 1e-6


def test_nothing_in_and_the_usual_layouts():
    cos, sin = (z.to(DEV) for z in _tables(9, 32))
    g = torch.ones(32, device=DEV)
    for shape in ((0, 5, 3, 32), (2, 0, 3, 32)):
        q, k, v = qk_norm_rope(torch.empty(shape, device=DEV), g, g, cos, sin)
        assert q.shape == k.shape == v.shape == (shape[0], 1, shape[1], 32)
    x = _rand(2, 9, 6, 32, dtype=BF, seed=1).to(DEV)
    want = qk_norm_rope(x, g, g, cos, sin)
    for o, w in zip(qk_norm_rope(x, g, g, cos[:, None], sin[:, None], kv_heads=2), want):  # as the decoder's tables
        assert torch.equal(o, w)
    zero = qk_norm_rope(torch.zeros_like(x), g, g, cos, sin)
    assert all((o == 0).all() for o in zero)
    bad = x.clone()
    bad[0, 3, 1, 5], bad[1, 2, 0, 0] = math.nan, math.inf  # a head's own alone
    q, k, v = qk_norm_rope(bad, g, g, cos, sin)
    nan = q.isnan().any(-1)
    assert nan.sum().item() == 2 and nan[0, 1, 3] and nan[1, 0, 2]
    assert torch.equal(q[~nan], want[0][~nan]) and torch.equal(k, want[1])


def test_replays_of_a_captured_training_step():
    x = _rand(2, 50, 12, 64, dtype=BF, seed=1).to(DEV).requires_grad_()
    gq, gk = ((1 + 0.3 * _rand(64, dtype=BF, seed=s)).to(DEV).requires_grad_() for s in (2, 3))
    cos, sin = (z.to(DEV) for z in _tables(50, 64))
    gs = [_rand(2, 4, 50, 64, dtype=BF, seed=4 + i).to(DEV) for i in range(3)]

    def step():
        outs = qk_norm_rope(x, gq, gk, cos, sin, eps=EPS)
        return (*(o.detach() for o in outs), *torch.autograd.grad(outs, (x, gq, gk), gs))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = step()
    for i in range(3):
        with torch.no_grad():
            x.copy_(_rand(2, 50, 12, 64, dtype=BF, seed=20 + i))
        g.replay()
        torch.cuda.synchronize()
        for o, w in zip(held, step()):
            assert torch.equal(o, w)


def test_a_captured_backward_next_to_an_eager_graph_of_its_leaves_is_refused():
    x = _rand(2, 30, 6, 32, dtype=BF, seed=1).to(DEV).requires_grad_()
    gq, gk = ((1 + 0.3 * _rand(32, dtype=BF, seed=s)).to(DEV).requires_grad_() for s in (2, 3))
    cos, sin = (z.to(DEV) for z in _tables(30, 32))

    def step():
        outs = qk_norm_rope(x, gq, gk, cos, sin, eps=EPS)
        return torch.autograd.grad(outs, (x, gq, gk), [torch.ones_like(o) for o in outs])

    want = step()
    alive = qk_norm_rope(x, gq, gk, cos, sin, eps=EPS)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured while an eager graph"):
        with torch.cuda.graph(g):
            step()
    torch.cuda.synchronize()
    for o, w in zip(step(), want):
        assert torch.equal(o, w)
    del alive, g
    gc.collect()  # (the exception's frames hold the refused step's)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = step()
    for _ in range(2):
        g.replay()
        torch.cuda.synchronize()
        for o, w in zip(held, want):
            assert torch.equal(o, w)


# -------------------------------------------------------------- into the cache


def _append(new, past, kv, group, hd, page, dtype, gains, seed=0, **more):
    heads, n_tok = kv * group, sum(new)
    g = torch.Generator().manual_seed(seed)
    need = [max(1, -(-(n + p) // page)) for n, p in zip(new, past)]
    ids = torch.randperm(sum(need) + 2, generator=g).tolist()
    table, at = [], 0
    for n in need:
        table.append(ids[at:at + n] + [0] * (max(need) - n))
        at += n
    k, v = (torch.randn(sum(need) + 2, kv, page, hd, generator=g).to(dtype) for _ in range(2))
    qkv = torch.randn(n_tok, heads + 2 * kv, hd, generator=g).to(dtype)
    gq, gk = ((1 + 0.5 * torch.randn(hd, generator=g)).to(gains) for _ in range(2))
    lengths = torch.tensor([n + p for n, p in zip(new, past)], dtype=torch.int32)
    starts = torch.tensor([0, *new], dtype=torch.int32).cumsum(0, dtype=torch.int32)
    offset = more.get("prefix_len", 0)
    cos, sin = _tables(int(lengths.max()) + offset, hd)
    kd, vd = k.to(DEV), v.to(DEV)
    q = paged_append(qkv.to(DEV), cos.to(DEV), sin.to(DEV), kd, vd, torch.tensor(table, dtype=torch.int32).to(DEV),
                     lengths.to(DEV), starts.to(DEV), q_gain=gq.to(DEV), k_gain=gk.to(DEV), eps=EPS, **more)
    wq, wk, wv = torch.zeros(n_tok, heads, hd, dtype=torch.float64), k.double(), v.double()
    at = 0
    for b, (n, p) in enumerate(zip(new, past)):
        for i in range(n):
            x, pos = qkv[at + i].double(), p + i
            c, s = cos[pos + offset].double(), sin[pos + offset].double()
            page_id, slot = table[b][pos // page], pos % page
            wq[at + i] = _heads(x[:heads], gq.double(), c, s)
            wk[page_id, :, slot] = _heads(x[heads:heads + kv], gk.double(), c, s)
            wv[page_id, :, slot] = x[heads + kv:]
        at += n
    return (q, kd, vd), (wq, wk, wv)


@pytest.mark.parametrize("new,past,kv,group,hd,page", [
    ([1], [0], 1, 1, 8, 1), ([1, 1, 1], [0, 31, 32], 2, 2, 128, 16), ([5, 0, 9], [4, 12, 0], 3, 3, 80, 16),
    ([17, 2, 40], [15, 0, 130], 2, 2, 96, 8), ([3], [60], 1, 4, 72, 16), ([2, 33], [7, 9], 4, 8, 64, 32),
    ([1, 6], [50, 3], 2, 1, 248, 4), ([12], [0], 2, 1, 256, 64)])
@pytest.mark.parametrize("dtype,gains", [(BF, BF), (HF, F), (F, F)])
@pytest.mark.parametrize("prefix", [0, 37])
def test_append(new, past, kv, group, hd, page, dtype, gains, prefix):
    got, want = _append(new, past, kv, group, hd, page, dtype, gains, prefix_len=prefix)
    u = torch.finfo(dtype).eps / 2
    for o, w in zip(got, want):
        tol = u * w.abs() + 2.0**-19 * w.abs().amax(-1, keepdim=True) * (1 + u) + (2.0**-24 * u if dtype == HF else 0.0)
        assert ((o.cpu().double() - w).abs() <= tol).all()
    assert torch.equal(got[2].cpu().double(), want[2])  # values are moved


def test_append_agrees_with_the_training_form_bit_for_bit():
    """What a model has cached is what its forward computes."""
    for dtype, hd in ((BF, 128), (HF, 72), (F, 64), (F, 256)):
        qkv = _rand(1, 20, 6, hd, dtype=dtype, seed=1).to(DEV)
        gq, gk = ((1 + 0.3 * _rand(hd, dtype=dtype, seed=s)).to(DEV) for s in (2, 3))
        cos, sin = (z.to(DEV) for z in _tables(20, hd))
        q, k, v = qk_norm_rope(qkv, gq, gk, cos, sin, eps=EPS)
        kc, vc = torch.zeros(2, 2, 16, hd, device=DEV, dtype=dtype), torch.zeros(2, 2, 16, hd, device=DEV, dtype=dtype)
        table, n = torch.tensor([[1, 0]], dtype=torch.int32, device=DEV), torch.tensor([20], dtype=torch.int32, device=DEV)
        got = paged_append(qkv[0], cos, sin, kc, vc, table, n, q_gain=gq, k_gain=gk, eps=EPS)
        rows = lambda c: torch.cat((c[1], c[0]), 1)[:, :20]  # noqa: E731
        assert torch.equal(got.transpose(0, 1), q[0]) and torch.equal(rows(kc), k[0]) and torch.equal(rows(vc), v[0])


def test_append_of_odd_rows_and_without_a_place(monkeypatch):
    hd, dtype = 64, BF
    cos, sin = (z.to(DEV) for z in _tables(8, hd))
    gq, gk = ((1 + 0.3 * _rand(hd, dtype=dtype, seed=s)).to(DEV) for s in (2, 3))
    table, n = torch.tensor([[0, 99]], dtype=torch.int32, device=DEV), torch.tensor([6], dtype=torch.int32, device=DEV)
    wide = _rand(6, 5, 150, dtype=dtype, seed=4).to(DEV)
    odd = wide[:, :, 3:3 + hd]
    outs = []
    for x in (odd.contiguous(), odd, odd.transpose(0, 1).contiguous().transpose(0, 1), odd.transpose(1, 2).contiguous().transpose(1, 2)):
        k, v = torch.zeros(1, 1, 4, hd, device=DEV, dtype=dtype), torch.zeros(1, 1, 4, hd, device=DEV, dtype=dtype)
        outs.append((paged_append(x, cos, sin, k, v, table, n, q_gain=gq, k_gain=gk, eps=EPS), k, v))
    for o in outs:
        assert torch.isfinite(o[0][:4]).all() and o[0][4:].isnan().all()  # the second page is none
        assert all(torch.equal(x.nan_to_num(5.0), y.nan_to_num(5.0)) for x, y in zip(o, outs[0]))
    k, v = torch.zeros(1, 1, 4, hd, device=DEV, dtype=dtype), torch.zeros(1, 1, 4, hd, device=DEV, dtype=dtype)
    monkeypatch.setattr(_lib, "ordinary", lambda *t: False)
    q = paged_append(odd, cos, sin, k, v, table, n, q_gain=gq, k_gain=gk, eps=EPS)
    assert all(torch.equal(x.nan_to_num(5.0), y.nan_to_num(5.0)) for x, y in zip((q, k, v), outs[0]))


def test_rows_of_no_sequence_stay():
    hd = 32
    cos, sin = (z.to(DEV) for z in _tables(8, hd))
    g = torch.ones(hd, device=DEV)
    k, v = (torch.zeros(2, 1, 4, hd, device=DEV) for _ in range(2))
    table = torch.tensor([[0], [1]], dtype=torch.int32, device=DEV)
    n, starts = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([2, 1], [1, 3, 4]))
    x = _rand(6, 4, hd, dtype=F, seed=1).to(DEV)
    q = paged_append(x, cos, sin, k, v, table, n, starts, q_gain=g, k_gain=g)
    assert (q[[0, 4, 5]] == 0).all() and (q[1:4] != 0).any()
    out = torch.full((6, 2, hd), 9.0, device=DEV)
    paged_append(x, cos, sin, k, v, table, n, starts, q_gain=g, k_gain=g, out=out)
    assert (out[[0, 4, 5]] == 9).all() and torch.equal(out[1:4], q[1:4])


@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 8), (1, 3, 4, 2, 64), (1, 17, 5, 1, 72), (2, 9, 3, 3, 80), (1, 1, 2, 1, 128),
                                   (2, 130, 2, 2, 64)], ids=str)
@pytest.mark.parametrize("dtype,gains", [(BF, BF), (HF, F), (F, F)])
def test_an_eps_of_zero(shape, dtype, gains, monkeypatch):
    """Places behind the last token hold no head: nothing of theirs is in the gains' gradients."""
    monkeypatch.setitem(globals(), "EPS", 0.0)  # (the oracle's and the calls' alike)
    test_forward_and_backward(shape, dtype, gains)


def test_no_kv_heads_are_refused():
    x, g = torch.zeros(1, 2, 6, 16, device=DEV, dtype=BF), torch.ones(16, device=DEV)
    cos, sin = (z.to(DEV) for z in _tables(2, 16))
    for kv in (0, -1, 3):
        with pytest.raises(ValueError, match="no queries"):
            qk_norm_rope(x, g, g, cos, sin, kv_heads=kv)


def test_second_derivatives_of_strided_inputs():
    """Of rows and gains that the kernels take copies of."""
    qkv = _rand(2, 4, 6, 16, dtype=F, seed=1).to(DEV)
    gains = (1 + 0.3 * _rand(16, 2, dtype=F, seed=2)).to(DEV)
    cos, sin = (z.to(DEV) for z in _tables(4, 16))
    gs = [_rand(2, 2, 4, 16, dtype=F, seed=4 + i).to(DEV) for i in range(3)]
    wide, off = torch.zeros(2, 4, 6, 40, device=DEV), torch.zeros(2 * 4 * 6 * 16 + 1, device=DEV)
    wide[..., 5:21], off[1:] = qkv, qkv.flatten()

    def second(x, a, c):
        x, a, c = (z.detach().requires_grad_() for z in (x, a, c))
        first = torch.autograd.grad(qk_norm_rope(x, a, c, cos, sin, eps=EPS), (x, a, c), gs, create_graph=True)
        return (*first, *torch.autograd.grad(sum(y.square().sum() for y in first), (x, a, c)))

    want = second(qkv, gains[:, 0].contiguous(), gains[:, 1].contiguous())
    for x in (wide[..., 5:21], off[1:].view(2, 4, 6, 16)):
        for o, w in zip(second(x, gains[:, 0], gains[:, 1]), want):
            assert rel_l2(o.detach().cpu(), w.detach().cpu().double()) <= 1e-5  # two fp32 evaluations


def test_strided_inputs_that_change_after_the_forward():
    """As for dense ones: autograd says so instead of taking other numbers."""
    cos, sin = (z.to(DEV) for z in _tables(4, 16))
    for dense in (True, False):
        x = _rand(2, 4, 6, 40, dtype=F, seed=1).to(DEV).requires_grad_()
        y = x[..., 5:21].clone() if dense else (x * 1.0)[..., 5:21]
        g = torch.ones(16, device=DEV, requires_grad=True)
        outs = qk_norm_rope(y, g, g, cos, sin)
        with torch.no_grad():
            y.mul_(2.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(outs, (x, g), [torch.ones_like(o) for o in outs])


@pytest.mark.parametrize("shape,dtype", [((3, 5500, 2, 1, 128), BF), ((1, 4099, 2, 1, 256), F), ((1, 131100, 1, 1, 8), HF)], ids=str)
def test_more_tokens_than_workgroups_at_once(shape, dtype):
    """Over 2048 groups of tokens each workgroup has a second one."""
    test_forward_and_backward(shape, dtype, dtype)


def test_bad_gains_of_an_append_are_refused(monkeypatch):
    hd = 32
    cos, sin = (z.to(DEV) for z in _tables(8, hd))
    k, v = (torch.zeros(2, 1, 4, hd, device=DEV, dtype=BF) for _ in range(2))
    table, n = torch.zeros(1, 2, dtype=torch.int32, device=DEV), torch.full((1,), 3, dtype=torch.int32, device=DEV)
    g = torch.ones(hd, device=DEV, dtype=BF)

    def call(**kw):
        return paged_append(_rand(3, 4, hd, dtype=BF, seed=1).to(DEV), cos, sin, k, v, table, n, **kw)

    for native in (True, False):
        if not native:
            monkeypatch.setattr(_lib, "ordinary", lambda *t: False)
        call(q_gain=g, k_gain=g)
        before = k.clone(), v.clone()
        for kw, what in ((dict(q_gain=g), "go together"), (dict(k_gain=g), "go together"),
                         (dict(q_gain=g[:16], k_gain=g), "q_gain must be"), (dict(q_gain=g, k_gain=g[:16]), "k_gain must be"),
                         (dict(q_gain=g.half(), k_gain=g.half()), "q_gain must be"),
                         (dict(q_gain=g, k_gain=g.float()), "k_gain must be"),
                         (dict(q_gain=g.cpu(), k_gain=g.cpu()), "q_gain must be"),
                         (dict(q_gain=g[:, None], k_gain=g), "q_gain must be")):
            with pytest.raises(ValueError, match=what):
                call(**kw)
        assert torch.equal(k, before[0]) and torch.equal(v, before[1])

"""Projections with 4-bit weights on the GPU against float64.

Tolerances. Products of x and 1 + c / 16 are exact in fp32. A group's sum is off by at most
(group + 40) 2^-23 of A = sum |x| (1 + c / 16) + (1 + z / 16) sum |x| (an addition each, the
matrix instruction's inner ones cut off instead of rounded), and sums over groups by (groups +
8) 2^-24 of what they add up. fp32 rows are three bf16 numbers, so three times the additions,
but of products with c - z: A = sum |x| |c - z|. The output is rounded once: eps / 2 of the
value."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a HIP device", allow_module_level=True)

from oracle.reference import dtype_floor, rel_l2  # noqa: E402
from switchyard import _lib  # noqa: E402
from switchyard.quant_op import Linear4, Weight4, linear4, quantize4  # noqa: E402

DEV = "cuda"
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _codes(n, k, group, dtype, zeros, seed):
    g = _gen(seed)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    shape = (n, -(-k // group))
    scales = (0.01 + 0.02 * torch.rand(shape, generator=g)).to(dtype)
    z = torch.randint(0, 16, shape, generator=g, dtype=torch.uint8) if zeros else None
    padded = torch.nn.functional.pad(codes, (0, k % 2))
    return codes, padded[:, 0::2] | padded[:, 1::2] << 4, scales, z


def _check(x, codes, scales, zeros, group, got):
    x6, s6 = x.cpu().double(), scales.double()
    n, k = codes.shape
    z6 = torch.full(scales.shape, 8.0, dtype=torch.float64) if zeros is None else zeros.double()
    out = torch.zeros(x6.shape[0], n, dtype=torch.float64)
    off = torch.zeros_like(out)
    planes = 3 if x.dtype == F else 1
    total = torch.zeros_like(out)
    for g in range(scales.shape[1]):
        at = slice(g * group, min(k, (g + 1) * group))
        xs, c = x6[:, at], codes[:, at].double()
        part = xs @ (c - z6[:, g:g + 1]).T * s6[:, g]
        if x.dtype == F:
            a = s6[:, g].abs() * (xs.abs() @ (c - z6[:, g:g + 1]).abs().T)
        else:
            a = 16 * s6[:, g].abs() * (xs.abs() @ (1 + c / 16).T + xs.abs().sum(1, keepdim=True) * (1 + z6[:, g] / 16))
        out += part
        off += a * planes * (group + 40) * 2.0**-23
        total += part.abs()
    off += total * (scales.shape[1] + 8) * 2.0**-24
    u = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal if x.dtype == HF else 0.0  # (fp16's small numbers have a fixed step)
    tol = off + u * (out.abs() + off) + tiny * u
    diff = (got.cpu().double() - out).abs()
    assert (diff <= tol).all(), (diff / tol.clamp_min(1e-300)).max().item()
    if x6.shape[0] * n > 200 and out.abs().max() > 2.0**-14:  # (below, fp16's own steps are what is off)
        assert rel_l2(got.cpu(), out) <= (5e-7 if x.dtype == F else 1.10 * dtype_floor(out, x.dtype))


SIZES = [(1, 16, 128), (1, 1, 1), (3, 17, 33), (16, 64, 256), (17, 100, 130), (5, 777, 1001), (33, 48, 640), (64, 130, 96),
         (65, 33, 2048), (130, 200, 257), (300, 70, 384), (2, 1030, 4096), (1, 16400, 128), (6, 16390, 200), (12, 80, 2300), (13, 16385, 136), (20, 8201, 300), (690, 780, 2049),
         (40, 8195, 150), (25, 8200, 4101), (600, 80, 200), (513, 130, 7), (9, 33, 5),
         (700, 3900, 140), (130, 10300, 260), (70, 10250, 380), (65, 2600, 5), (700, 3900, 144), (130, 10300, 264),
         (70, 10250, 384), (340, 5530, 1000), (340, 5530, 1001), (525, 7530, 8), (512, 2048, 1104), (178, 5187, 103),
         (1030, 5000, 520), (18, 4213, 1458), (49, 6261, 560), (15, 20100, 1002),
         (525, 7530, 70), (340, 5530, 290), (45, 12200, 136), (41, 19200, 257),
         (2, 100, 300), (2, 100, 301), (7, 100, 300), (8, 5000, 300), (12, 5000, 301), (6, 24600, 130), (3, 16000, 3900),
         (5, 16000, 3901), (2, 16000, 5200)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype,zeros", [(BF, False), (BF, True), (HF, True), (F, False), (F, True)])
def test_product(m, n, k, group, dtype, zeros):
    codes, packed, scales, z = _codes(n, k, group, dtype, zeros, seed=n + k)
    x = torch.randn(m, k, generator=_gen(m)).to(dtype)
    w = Weight4.from_codes(packed.to(DEV), scales.to(DEV), None if z is None else z.to(DEV), in_features=k, group=group)
    got = linear4(x.to(DEV), w)
    assert got.shape == (m, n) and got.dtype == dtype
    _check(x, codes, scales, z, group, got)
    c, s, zz = w.codes()
    assert torch.equal(c.cpu(), codes) and torch.equal(s.cpu(), scales)
    assert (zz is None) == (z is None) and (z is None or torch.equal(zz.cpu(), z))


def test_activations_that_share_a_sign_and_large_zero_points():
    """Where the two sums of a group nearly cancel."""
    codes, packed, scales, z = _codes(96, 512, 128, BF, True, seed=3)
    z = (z.int() + 12).to(torch.uint8)  # past the codes' range
    x = (100.0 + torch.randn(20, 512, generator=_gen(4))).to(BF)
    w = Weight4.from_codes(packed.to(DEV), scales.to(DEV), z.to(DEV), in_features=512, group=128)
    _check(x, codes, scales, z, 128, linear4(x.to(DEV), w))


@pytest.mark.parametrize("dtype,size", [(HF, 1e-6), (HF, 3e-7), (HF, 60000.0), (BF, 1e-36), (BF, 1e36), (F, 1e-25), (F, 1e30)])
@pytest.mark.parametrize("m", [3, 12, 30, 200])
def test_tiny_and_huge_activations(m, dtype, size):
    """fp16 activations below its normal numbers; sums far from 1."""
    n, k = 2600, 200
    codes, packed, scales, z = _codes(n, k, 32, dtype, True, seed=9)
    if dtype == HF:  # outputs among fp16's normal numbers
        scales = scales / 256 if size > 1 else scales * 4096
    x = (size * (torch.rand(m, k, generator=_gen(10)) - 0.5)).to(dtype)
    w = Weight4.from_codes(packed.to(DEV), scales.to(DEV), z.to(DEV), in_features=k, group=32)
    _check(x, codes, scales, z, 32, linear4(x.to(DEV), w))


def test_rows_of_any_shape_start_and_stride():
    codes, packed, scales, _ = _codes(40, 130, 64, BF, False, seed=5)
    w = Weight4.from_codes(packed.to(DEV), scales.to(DEV), in_features=130, group=64)
    x = torch.randn(6, 130, generator=_gen(6)).to(BF)
    want = linear4(x.to(DEV), w)
    wide = torch.full((6, 200), float("nan"), dtype=BF)
    wide[:, 7:137] = x
    assert torch.equal(linear4(wide.to(DEV)[:, 7:137], w), want)
    assert torch.equal(linear4(x.to(DEV).t().contiguous().t(), w), want)
    assert torch.equal(linear4(x.to(DEV).view(2, 3, 130), w), want.view(2, 3, 40))
    assert torch.equal(linear4(x.to(DEV)[:1].expand(4, 130), w), want[:1].expand(4, 40))
    assert torch.equal(linear4(x.to(DEV)[0], w), want[0])
    codes, packed, scales, z = _codes(6000, 264, 32, BF, True, seed=8)  # rows that go straight to LDS, or do not
    many = Weight4.from_codes(packed.to(DEV), scales.to(DEV), z.to(DEV), in_features=264, group=32)
    y = torch.randn(300, 264, generator=_gen(9)).to(BF)
    for start in (8, 7, 10):
        at = torch.full((300, 280), float("nan"), dtype=BF)
        at[:, start:start + 264] = y
        _check(y, codes, scales, z, 32, linear4(at.to(DEV)[:, start:start + 264], many))
    assert linear4(x.to(DEV)[:0], w).shape == (0, 40)
    assert linear4(torch.empty(3, 0, 130, dtype=BF, device=DEV), w).shape == (3, 0, 40)


@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_rows_with_infinities_do_not_touch_others(dtype):
    codes, packed, scales, _ = _codes(64, 256, 64, dtype, False, seed=7)
    w = Weight4.from_codes(packed.to(DEV), scales.to(DEV), in_features=256, group=64)
    x = torch.randn(20, 256, generator=_gen(8)).to(dtype)
    bad = x.clone()
    bad[3, 100], bad[11, 5], bad[17, 255] = math.inf, math.nan, -math.inf
    got, want = linear4(bad.to(DEV), w), linear4(x.to(DEV), w)
    rows = [i for i in range(20) if i not in (3, 11, 17)]
    assert got[[3, 11, 17]].isnan().all() and torch.equal(got[rows], want[rows])


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("n,k,group", [(5, 64, 32), (33, 200, 64), (16, 129, 128), (1, 1, 32), (70, 512, 128)])
def test_quantized_weights_are_the_nearest(n, k, group, symmetric, dtype):
    w = torch.randn(n, k, generator=_gen(n)).to(dtype)
    w[0, :group] = 0.0  # a group of zeros
    q = quantize4(w.to(DEV), group, symmetric=symmetric)
    c, s, z = (None if t is None else t.cpu() for t in q.codes())
    of = torch.arange(k) // group
    w6, s6 = w.double(), s.double()
    z6 = torch.full(s.shape, 8.0, dtype=torch.float64) if z is None else z.double()
    for g in range(s.shape[1]):
        part = w6[:, g * group:(g + 1) * group]
        top = part.abs().amax(1) / 7 if symmetric else (part.amax(1).clamp_min(0) - part.amin(1).clamp_max(0)) / 15
        assert ((s6[:, g] - top).abs() <= torch.finfo(dtype).eps / 2 * top + 2.0**-24 * top).all()
    # Nearest to the kept scale, but for quotients within 2^-23 of a half and ends of the range.
    best = (w6 / s6[:, of].clamp_min(1e-300)).clamp(-100, 100) + z6[:, of]
    near = best.clamp(1 if symmetric else 0, 15)
    live = s6[:, of] > 0
    assert ((c.double() - near).abs()[live] <= 0.5 + 1e-5).all()
    assert (c[~live] == 8 if symmetric else c[~live] == z6[:, of][~live]).all()
    assert torch.equal(q.dequantize().cpu().double(), ((c.double() - z6[:, of]) * s6[:, of]).float().double())


def test_the_module_its_state_and_autocast():
    torch.manual_seed(0)
    lin = torch.nn.Linear(200, 96, bias=False, device=DEV)
    m = Linear4.from_linear(lin, 32, symmetric=False)
    x = torch.randn(7, 200, device=DEV)
    want = m(x)
    assert torch.equal(want, linear4(x, m.weight4))
    other = Linear4(quantize4(torch.randn(96, 200, device=DEV), 32, symmetric=False))
    other.load_state_dict(m.state_dict())
    assert torch.equal(other(x), want)
    half = Linear4(quantize4(lin.weight.detach().bfloat16(), 32))
    with torch.autocast("cuda", dtype=BF):
        assert torch.equal(half(x), half(x.bfloat16()))
        assert m(x).dtype == BF and torch.equal(m(x), want.bfloat16())  # fp32 scales: fp32 inside
    with pytest.raises(ValueError, match="dtype"):
        half(x)
    with pytest.raises(ValueError, match="bias"):
        Linear4.from_linear(torch.nn.Linear(8, 8, device=DEV))


def test_gradients_and_tangents_are_refused():
    w = quantize4(torch.randn(32, 64, device=DEV))
    x = torch.randn(3, 64, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        linear4(x, w)
    with torch.no_grad():
        linear4(x, w)
    import torch.autograd.forward_ad as fwad

    with fwad.dual_level(), pytest.raises(RuntimeError, match="tangents"):
        linear4(fwad.make_dual(x.detach(), torch.ones_like(x)), w)


def test_another_stream_a_graph_and_two_calls_at_once():
    w = quantize4(torch.randn(512, 1024, device=DEV).bfloat16())
    x = torch.randn(9, 1024, device=DEV).bfloat16()
    want = linear4(x, w)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(linear4(x, w))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = linear4(x, w)
    for i in range(3):
        x.copy_(torch.randn(9, 1024, device=DEV).bfloat16())
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, linear4(x, w))


def test_the_python_path_gives_the_same(monkeypatch):
    w = quantize4(torch.randn(80, 100, device=DEV), 32, symmetric=False)
    x = torch.randn(4, 100, device=DEV)
    want = linear4(x, w)
    monkeypatch.setattr(_lib, "ordinary", lambda *t: False)
    assert torch.equal(linear4(x, w), want) and torch.equal(linear4(x.t().contiguous().t(), w), want)


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_weights_that_are_no_numbers_show(group, symmetric, dtype):
    """A group with one is NaN: in its scale, its weights and the products; the others are as without it."""
    n, k = 40, 300
    w = torch.randn(n, k, generator=_gen(1)).to(dtype)
    bad = w.clone()
    bad[1, 70], bad[2, 130], bad[3, 299] = math.nan, math.inf, -math.inf
    bad[4, :group], bad[5, 9], bad[5, 11] = math.nan, math.inf, -math.inf
    hit = torch.zeros(n, -(-k // group), dtype=torch.bool)
    for row, col in ((1, 70), (2, 130), (3, 299), (4, 0), (5, 9)):
        hit[row, col // group] = True
    q, p = quantize4(bad.to(DEV), group, symmetric=symmetric), quantize4(w.to(DEV), group, symmetric=symmetric)
    of = torch.arange(k) // group
    (c, s, z), (wc, ws, wz) = q.codes(), p.codes()
    assert torch.equal(s.isnan().cpu(), hit) and torch.equal(s[~hit.to(DEV)], ws[~hit.to(DEV)])
    assert torch.equal(c.cpu()[~hit[:, of]], wc.cpu()[~hit[:, of]])
    assert z is None or torch.equal(z.cpu()[~hit], wz.cpu()[~hit])
    assert torch.equal(q.dequantize().isnan().cpu(), hit[:, of])
    for m in (3, 20, 300):
        x = torch.randn(m, k, generator=_gen(m)).to(dtype).to(DEV)
        got, want = linear4(x, q), linear4(x, p)
        assert got[:, 1:6].isnan().all() and torch.equal(got[:, 6:], want[:, 6:]) and torch.equal(got[:, 0], want[:, 0])


@pytest.mark.parametrize("dtype,step", [(HF, 2.0**-24), (BF, 2.0**-133), (F, 2.0**-149)])
@pytest.mark.parametrize("symmetric", [True, False])
def test_small_weights_fit_the_scale_that_is_kept(dtype, step, symmetric):
    """Groups whose scale is a few of the type's last steps: rounded down it would leave the ends
    out of the codes' reach, or all of the group where it is 0."""
    n, group = 250, 32
    top = torch.arange(1, n + 1, dtype=torch.float64)
    w = top[:, None] * (2 * torch.rand(n, 64, generator=_gen(2), dtype=torch.float64) - 1)
    w[:, 0], w[:, 1], w[:, 40] = top, -top, top  # both ends; the second group's top alone
    w = (w.round() * step).to(dtype)
    assert (w.double()[:, 0] == top * step).all()
    q = quantize4(w.to(DEV), group, symmetric=symmetric)
    c, s, z = (None if t is None else t.cpu().double() for t in q.codes())
    of = torch.arange(64) // group
    w6, z = w.double(), torch.full_like(s, 8.0) if z is None else z
    assert (s > 0).all()
    off = (w6 / s[:, of] - (c - z[:, of])).abs()
    if symmetric:
        # 0.5 where nothing is cut off; quotients are fp32's, 2^-24 of at most 7.5.
        assert off.max() <= 0.5 + 1e-5 and c.min() >= 1
    else:
        # A zero point is up to half a step off, and the range up to half a step past 15.
        assert off.max() <= 1.0 + 1e-5
    for g in range(2):  # no larger than one of the type's steps over what fits
        part = w6[:, g * group:(g + 1) * group]
        fits = part.abs().amax(1) / 7 if symmetric else (part.amax(1).clamp_min(0) - part.amin(1).clamp_max(0)) / 15
        # (quotients of up to 34 steps: the type has all of them)
        assert (s[:, g] <= fits + step).all() and (s[:, g] >= fits - step / 2 * (1 + 1e-5)).all()


@pytest.mark.parametrize("dtype", [BF, F])
def test_a_range_past_the_largest_number(dtype):
    """max - min of finite weights may be none."""
    w = torch.randn(8, 64, generator=_gen(3)) * 1e37
    w[:, 3], w[:, 7] = 3e38, -3e38
    w[1, :32] = w[1, :32].abs().clamp_max(3e38)
    w = w.to(dtype)
    q = quantize4(w.to(DEV), 32, symmetric=False)
    c, s, z = (t.cpu().double() for t in q.codes())
    of = torch.arange(64) // 32
    assert torch.isfinite(s).all()
    top = (w.double().amax() - w.double().amin()) / 15  # of every row's first group but the second's
    assert ((s[2:, 0] - top).abs() <= (torch.finfo(dtype).eps / 2 + 2.0**-22) * top).all()
    best = w.double() / s[:, of] + z[:, of]
    assert ((c - best.clamp(0, 15)).abs() <= 0.5 + 1e-5).all() and (best >= -0.55).all() and (best <= 15.55).all()


def test_projections_that_are_more_than_their_weights_are_refused():
    class Twice(torch.nn.Linear):
        def forward(self, x):
            return 2 * super().forward(x)

    def plain():
        return torch.nn.Linear(64, 48, bias=False, device=DEV)

    hooked, before, own = plain(), plain(), plain()
    hooked.register_forward_hook(lambda m, a, y: 2 * y)
    before.register_forward_pre_hook(lambda m, a: (2 * a[0],))
    own.forward = lambda x: x[..., :48]
    for m in (hooked, before, own, Twice(64, 48, bias=False, device=DEV), torch.nn.Bilinear(4, 4, 8, bias=False, device=DEV)):
        with pytest.raises(ValueError, match="has no 4-bit form"):
            Linear4.from_linear(m)
    scaled = torch.nn.utils.parametrizations.weight_norm(plain())  # its weight is computed, its product the usual one
    assert torch.equal(Linear4.from_linear(scaled).weight4.dequantize(), quantize4(scaled.weight).dequantize())


@pytest.mark.parametrize("m,n,k", [(4100, 64, 100), (8201, 64, 2048)])
def test_more_fp32_rows_than_a_launch(m, n, k):
    test_product(m, n, k, 64, F, True)


def test_more_rows_than_a_launch():
    test_product(4101, 16, 128, 64, BF, True)
    test_product(4101, 16, 128, 64, HF, False)

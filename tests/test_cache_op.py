"""The paged cache on the GPU: the append with its rotation, and attention over the pages
and over a shared prefix, against float64.

Tolerances. A stored value is off by at most u = eps / 2 of its dtype, relative. The
rotation is two fp32 products and a sum before that: at most 3 2^-24 of |x cos| + |y sin|.
For an attention row with weights p and values v let A = sum p |v|. A score is off by at
most e = (hd + 4) 2^-24 max_j scale sum |q k_j|, a weight by a factor of 1 +- (2 e + 2^-20)
(own and normaliser, and the exponential), sums over n keys by (n + 64) 2^-24 A, and 16-bit
weights are rounded once more before the second product: u A. All of it is relative to the
exact result's |o|, or to A where rows cancel.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a HIP device", allow_module_level=True)

from switchyard.cache_op import paged_append, paged_attention  # noqa: E402

DEV = "cuda"
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


class Case:
    """Sequences with ``new`` rows and ``past`` earlier tokens each, in pages anywhere in a
    cache of random values."""

    def __init__(self, new, past, *, kv, group, hd, page, dtype, prefix=0, seed=0, spare=2):
        g = _gen(seed)
        self.new, self.past, self.kv, self.heads, self.hd, self.page = new, past, kv, kv * group, hd, page
        self.dtype, self.prefix, self.b, self.n_tok = dtype, prefix, len(new), sum(new)
        need = [max(1, -(-(n + p) // page)) for n, p in zip(new, past)]
        shared = -(-prefix // page)
        total = sum(need) + shared + spare
        ids = torch.randperm(total, generator=g).tolist()
        self.prefix_ids, at, table = ids[:shared], shared, []
        for n in need:
            table.append(ids[at:at + n] + [0] * (max(need) - n))
            at += n
        self.table = torch.tensor(table, dtype=torch.int32)
        self.k = torch.randn(total, kv, page, hd, generator=g).to(dtype)
        self.v = torch.randn(total, kv, page, hd, generator=g).to(dtype)
        self.q = (1.5 * torch.randn(self.n_tok, self.heads, hd, generator=g)).to(dtype)
        self.lengths = torch.tensor([n + p for n, p in zip(new, past)], dtype=torch.int32)
        self.starts = torch.tensor([0, *new], dtype=torch.int32).cumsum(0, dtype=torch.int32)

    def rows(self, cache, b, own):
        """The first ``own`` tokens of sequence b behind the prefix, float64 [n, kv, hd]."""
        out = []
        for ids, n in ((self.prefix_ids, self.prefix), (self.table[b].tolist(), own)):
            for j in range(n):
                out.append(cache[ids[j // self.page], :, j % self.page])
        return torch.stack(out).double() if out else torch.zeros(0, self.kv, self.hd, dtype=torch.float64)

    def expected(self, scale=None):
        """The rows' results and what they may be off by."""
        scale = self.hd**-0.5 if scale is None else scale
        u = torch.finfo(self.dtype).eps / 2
        out = torch.zeros(self.n_tok, self.heads, self.hd, dtype=torch.float64)
        tol = torch.zeros_like(out)
        at = 0
        for b in range(self.b):
            n, length = self.new[b], int(self.lengths[b])
            k, v = self.rows(self.k, b, max(length, 0)), self.rows(self.v, b, max(length, 0))
            for i in range(n):
                see = max(0, length - n + i + 1) + self.prefix
                if see == 0:
                    continue
                qi = self.q[at + i].double().view(self.kv, -1, self.hd)
                kk, vv = k[:see].transpose(0, 1), v[:see].transpose(0, 1)
                s = qi @ kk.transpose(1, 2) * scale
                p = torch.softmax(s, -1)
                o, a = p @ vv, p @ vv.abs()
                e = (self.hd + 4) * 2.0**-24 * (qi.abs() @ kk.abs().transpose(1, 2) * scale).amax(-1, keepdim=True)
                rel = 2 * e + 2.0**-20 + (see + 64) * 2.0**-24
                t = u * o.abs() + a * (rel + (u if self.dtype != F else 0.0)) * (1 + u)
                out[at + i], tol[at + i] = o.reshape(self.heads, self.hd), t.reshape(self.heads, self.hd)
            at += n
        return out, tol

    def call(self, fn=paged_attention, q=None, **more):
        if self.prefix:
            more.setdefault("prefix_pages", torch.tensor(self.prefix_ids, dtype=torch.int32, device=DEV))
            more.setdefault("prefix_len", self.prefix)
        starts = None if len(set(self.new)) == 1 and not more.pop("packed", False) else self.starts.to(DEV)
        return fn(self.q.to(DEV) if q is None else q, self.k.to(DEV), self.v.to(DEV), self.table.to(DEV),
                  self.lengths.to(DEV), starts, **more)

    def check(self, got=None, **more):
        got = self.call(**more) if got is None else got
        want, tol = self.expected()
        assert got.dtype == self.dtype and got.shape == want.shape
        diff = (got.cpu().double() - want).abs()
        assert torch.isfinite(got).all() and (diff <= tol).all(), (diff / tol.clamp_min(1e-30)).max().item()


SHAPES = [
    # new, past, kv, group, hd, page
    ([1], [0], 1, 1, 64, 16),  # one token that sees itself
    ([1, 1, 1], [0, 31, 32], 2, 1, 128, 16),  # at the edges of a tile
    ([1] * 5, [3, 63, 64, 200, 1000], 2, 4, 64, 64),
    ([1, 1], [700, 40], 1, 16, 128, 32),  # a full group of rows
    ([1, 1], [257, 5], 1, 20, 64, 16),  # more rows than a group
    ([3, 1, 7], [0, 100, 33], 3, 3, 80, 16),
    ([17, 2, 40], [15, 0, 130], 2, 2, 96, 8),
    ([65, 129], [0, 77], 2, 1, 128, 64),
    ([5, 0, 9], [4, 12, 0], 2, 2, 64, 16),  # a sequence without new rows
    ([1, 1], [300, 20], 2, 2, 256, 16),
    ([33, 20], [64, 0], 1, 2, 256, 128),
    ([1, 6], [50, 3], 2, 1, 8, 1),  # the narrowest head, one token a page
    ([70], [900], 4, 1, 64, 16),
    ([1] * 70, [7 * i for i in range(70)], 1, 2, 64, 16),  # more sequences than lanes
    ([2] * 130, [i for i in range(130)], 1, 1, 32, 16),
]


@pytest.mark.parametrize("shape", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_attention(shape, dtype):
    new, past, kv, group, hd, page = shape
    Case(new, past, kv=kv, group=group, hd=hd, page=page, dtype=dtype, seed=1).check()


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("prefix", [1, 40, 64, 333])
@pytest.mark.parametrize("shape", [([1, 1, 1], [5, 0, 70], 2, 1, 64, 16), ([1] * 40, list(range(40)), 1, 3, 128, 32),
                                   ([4, 0, 30], [10, 3, 0], 2, 2, 64, 16), ([1], [9], 2, 2, 128, 16),
                                   ([90, 41], [0, 7], 1, 2, 64, 16)])
def test_attention_behind_a_shared_prefix(shape, prefix, dtype):
    new, past, kv, group, hd, page = shape
    Case(new, past, kv=kv, group=group, hd=hd, page=page, dtype=dtype, prefix=prefix, seed=2).check()


def test_one_long_sequence_is_shared_by_many_waves():
    """Partial results of one row from hundreds of waves, next to short sequences."""
    Case([1, 1, 1], [20000, 3, 500], kv=1, group=2, hd=64, page=64, dtype=BF, seed=3).check()
    Case([2], [20000], kv=1, group=2, hd=64, page=64, dtype=F, seed=3).check()


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("new", [[1, 9, 40], [1, 1, 1], [70, 5, 66]])
def test_what_rows_do_not_see_does_not_matter(new, bad, dtype):
    """Infinities and NaN in slots behind a sequence's end, in pages of nobody, and in keys
    and values of later tokens."""
    c = Case(new, [30, 3, 0], kv=2, group=2, hd=64, page=16, dtype=dtype, seed=4)
    want = c.call().cpu()
    used = torch.zeros(c.k.shape[0], c.page, dtype=torch.bool)
    for b in range(c.b):
        for j in range(int(c.lengths[b])):
            used[c.table[b, j // c.page], j % c.page] = True
    for cache in (c.k, c.v):
        cache.transpose(1, 2)[~used] = bad
    assert torch.equal(c.call().cpu(), want)
    at = 0
    for b, n in enumerate(new):  # the last new token of each sequence: earlier rows must not change
        j = int(c.lengths[b]) - 1
        c.k[c.table[b, j // c.page], :, j % c.page, 3] = bad
        c.v[c.table[b, j // c.page], :, j % c.page, 5:7] = bad
        at += n
    got, at = c.call().cpu(), 0
    for n in new:
        # The other products of the row's tile are formed one by one here: same bounds, other order.
        ref, rows = want[at:at + n - 1].double(), got[at:at + n - 1].double()
        assert torch.isfinite(rows).all()
        u = torch.finfo(dtype).eps / 2
        assert ((rows - ref).abs() <= 2 * u * ref.abs() + (2 * u if dtype != F else 2.0**-15) * 4).all()
        at += n


def test_rows_that_see_nothing_are_zero():
    c = Case([2, 3, 1], [4, 0, 0], kv=2, group=1, hd=64, page=16, dtype=BF, seed=5)
    c.lengths = torch.tensor([6, 1, 0], dtype=torch.int32)  # fewer tokens than rows; none
    got = c.call()
    c.check(got)
    assert (got[2:4] == 0).all() and (got[5] == 0).all() and (got[4] != 0).any()


def test_bad_pages_and_lengths_hold_nothing():
    c = Case([1, 1], [60, 40], kv=2, group=2, hd=64, page=16, dtype=BF, seed=6)
    whole = c.call().cpu()
    table = c.table.clone()
    table[0, 1], table[1, 2] = -7, c.k.shape[0]
    got = paged_attention(c.q.to(DEV), c.k.to(DEV), c.v.to(DEV), table.to(DEV), c.lengths.to(DEV)).cpu()
    for b, hole in ((0, 1), (1, 2)):
        keep = [j for j in range(int(c.lengths[b])) if j // c.page != hole]
        k, v = (c.rows(x, b, int(c.lengths[b]))[keep].transpose(0, 1) for x in (c.k, c.v))
        p = torch.softmax(c.q[b].double().view(2, 2, 64) @ k.transpose(1, 2) / 8, -1)
        assert ((p @ v).view(4, 64) - got[b].double()).abs().max() <= 2 * 2.0**-8 * 4
    # a length past the table's row: all that the row holds is seen
    c.lengths = torch.tensor([1 << 30, 41], dtype=torch.int32)
    big = c.call().cpu()
    c.lengths = torch.tensor([64, 41], dtype=torch.int32)
    assert torch.equal(big, c.call().cpu()) and torch.equal(big[1], whole[1])


@pytest.mark.parametrize("n", [3, 30])
def test_tokens_past_the_capacity(n):
    """The last new tokens have no room: they are not cached, and a row sees what is there."""
    c = Case([n, n], [64 - n, 10], kv=2, group=2, hd=64, page=16, dtype=BF, seed=27)
    cos, sin = _tables(128, 64)
    qkv = torch.randn(2 * n, 8, 64, generator=_gen(28)).to(BF).to(DEV)
    c.lengths[0] = 66  # two more than the row of the table holds
    k, v = c.k.to(DEV), c.v.to(DEV)
    q = paged_append(qkv, cos, sin, k, v, c.table.to(DEV), c.lengths.to(DEV))
    lost = torch.zeros(2 * n, dtype=torch.bool)
    lost[n - 2:n] = True
    assert torch.equal(torch.isnan(q).any(-1).any(-1).cpu(), lost)
    want = qkv[:n, 6:].cpu()
    for i in range(n - 2):  # positions 66 - n + i
        j = 66 - n + i
        assert torch.equal(v[c.table[0, j // 16], :, j % 16].cpu(), want[i])
    c.k, c.v, c.q = k.cpu(), v.cpu(), torch.nan_to_num(q).cpu()
    got = c.call().cpu().double()
    for i in range(n):
        see = min(66 - n + i + 1, 64)
        kk, vv = (c.rows(x, 0, 64)[:see].transpose(0, 1) for x in (c.k, c.v))
        p = torch.softmax(c.q[i].double().view(2, 2, 64) @ kk.transpose(1, 2) / 8, -1)
        assert ((p @ vv).view(4, 64) - got[i]).abs().max() <= 2 * 2.0**-8 * 4


@pytest.mark.parametrize("op", ["attend", "prefix"])
def test_rows_behind_the_last_sequence(op):
    c = Case([3, 2], [10, 4], kv=2, group=2, hd=64, page=16, dtype=BF, prefix=20 if op == "prefix" else 0, seed=7)
    pad = torch.full((4, c.heads, c.hd), 7.0, dtype=BF)
    q = torch.cat((pad[:1], c.q, pad)).to(DEV)
    c.starts = c.starts + 1
    got = c.call(q=q)
    c.check(got[1:6])
    assert (got[0] == 0).all() and (got[6:] == 0).all()
    out = torch.full_like(q, 3.0)
    assert c.call(q=q, out=out) is out
    assert torch.equal(out[1:6], got[1:6]) and (out[0] == 3).all() and (out[6:] == 3).all()


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("prefix", [0, 40])
@pytest.mark.parametrize("new", [[1] * 3, [5] * 70, [70, 3, 1], [200, 130, 1]])
def test_the_queries_as_out(new, prefix, dtype):
    past = [(900, 33, 0, 5)[i % 4] for i in range(len(new))]
    c = Case(new, past, kv=2, group=2, hd=64, page=16, dtype=dtype, prefix=prefix, seed=9)
    q = c.q.to(DEV)
    got = c.call(q=q, out=q)
    assert got is q
    assert torch.equal(got, c.call())
    c.check(got=got)


def test_strides_and_orders_of_the_caches_and_queries():
    c = Case([1, 4], [50, 9], kv=2, group=2, hd=64, page=16, dtype=HF, seed=8)
    want = c.call()
    both = torch.stack((c.k, c.v), 1).to(DEV)  # one tensor [pages, 2, kv, page, hd]
    turned = [x.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) for x in (c.k, c.v)]  # token-major pages
    wide = torch.zeros(5, 9, 64, dtype=HF, device=DEV)
    wide[:, 2:6] = c.q.to(DEV)
    odd = torch.zeros(5 * 4 * 64 + 1, dtype=HF, device=DEV)[1:].view(5, 4, 64)  # rows of no 16-byte start
    odd.copy_(c.q)
    wide_table = torch.zeros(2, c.table.shape[1] + 3, dtype=torch.int32, device=DEV)
    wide_table[:, :c.table.shape[1]] = c.table
    rest = (c.lengths.to(DEV), c.starts.to(DEV))
    for q, k, v, t in ((c.q.to(DEV), both[:, 0], both[:, 1], c.table.to(DEV)), (c.q.to(DEV), *turned, c.table.to(DEV)),
                       (wide[:, 2:6], c.k.to(DEV), c.v.to(DEV), wide_table[:, :c.table.shape[1]]),
                       (odd, c.k.to(DEV), c.v.to(DEV), c.table.to(DEV))):
        assert torch.equal(paged_attention(q, k, v, t, *rest), want)
    assert torch.equal(paged_attention(c.q.to(DEV), c.k.to(DEV), c.v.to(DEV), c.table.to(DEV), *rest, scale=0.125), want)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("prefix", [0, 100])
@pytest.mark.parametrize("new", [[30, 10, 30, 10, 20, 40], [3, 1, 3, 1, 2, 4], [200, 1, 3, 1, 2, 4]])
def test_starts_out_of_order(new, prefix, dtype):
    """Results are then undefined; the caches stay as they are, and so does the call after."""
    c = Case(new, [900] * 6, kv=2, group=1, hd=64, page=16, dtype=dtype, prefix=prefix, seed=22)
    k, v, q = c.k.to(DEV), c.v.to(DEV), c.q.to(DEV)
    more = dict(prefix_pages=torch.tensor(c.prefix_ids, dtype=torch.int32, device=DEV), prefix_len=prefix)
    bad = torch.tensor([0, c.n_tok] * 3 + [0], dtype=torch.int32, device=DEV)
    paged_attention(q, k, v, c.table.to(DEV), c.lengths.to(DEV), bad, **(more if prefix else {}))
    assert torch.equal(k.cpu(), c.k) and torch.equal(v.cpu(), c.v) and torch.equal(q.cpu(), c.q)
    c.check()


def test_a_cache_past_32_bit_offsets():
    """Pages whose elements lie behind 2^32 bytes and 2^31 elements."""
    pages, kv, page, hd = 140000, 2, 64, 128
    k = torch.empty(pages, kv, page, hd, dtype=BF, device=DEV)
    v = torch.empty_like(k)
    c = Case([1, 2], [100, 30], kv=kv, group=2, hd=hd, page=page, dtype=BF, seed=9)
    far = pages - 1 - torch.arange(c.k.shape[0])
    k[far.to(DEV)], v[far.to(DEV)] = c.k.to(DEV), c.v.to(DEV)
    table = far[c.table.long()].int().to(DEV)
    got = paged_attention(c.q.to(DEV), k, v, table, c.lengths.to(DEV), c.starts.to(DEV))
    assert torch.equal(got, c.call())
    c.check(got)


# ------------------------------------------------------------------------ append


def _tables(n, hd):
    ang = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(hd // 2, dtype=torch.float64) * 2 / hd)
    return ang.cos().float().to(DEV), ang.sin().float().to(DEV)


def _append_expected(c, qkv, cos, sin, offset=0):
    cos, sin = cos.cpu().double(), sin.cpu().double()
    half = c.hd // 2
    x = qkv.cpu().double()
    out, tol = x.clone(), torch.zeros_like(x)
    k, v = c.k.double(), c.v.double()
    at = 0
    for b, n in enumerate(c.new):
        for i in range(n):
            j = int(c.lengths[b]) - n + i
            r = x[at + i, :c.heads + c.kv]
            lo, hi = r[:, :half], r[:, half:]
            co, si = cos[j + offset], sin[j + offset]
            out[at + i, :c.heads + c.kv] = torch.cat((lo * co - hi * si, lo * si + hi * co), -1)
            a = torch.cat(((lo * co).abs() + (hi * si).abs(), (lo * si).abs() + (hi * co).abs()), -1)
            tol[at + i, :c.heads + c.kv] = 3 * 2.0**-24 * a
            k[c.table[b, j // c.page], :, j % c.page] = out[at + i, c.heads:c.heads + c.kv]
            v[c.table[b, j // c.page], :, j % c.page] = x[at + i, c.heads + c.kv:]
        at += n
    return out, tol, k, v


@pytest.mark.parametrize("shape", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_append(shape, dtype):
    new, past, kv, group, hd, page = shape
    c = Case(new, past, kv=kv, group=group, hd=hd, page=page, dtype=dtype, seed=11)
    cos, sin = _tables(1030, hd)
    qkv = torch.randn(c.n_tok, c.heads + 2 * kv, hd, generator=_gen(12)).to(dtype).to(DEV)
    k, v = c.k.to(DEV), c.v.to(DEV)
    starts = None if len(set(new)) == 1 else c.starts.to(DEV)
    q = paged_append(qkv, cos, sin, k, v, c.table.to(DEV), c.lengths.to(DEV), starts)
    want, tol, wk, wv = _append_expected(c, qkv, cos, sin)
    u = torch.finfo(dtype).eps / 2

    def close(got, ref, t):
        small = torch.finfo(dtype).smallest_normal  # fp16 results may be subnormal
        assert ((got.cpu().double() - ref).abs() <= u * ref.abs() * (1 + 2.0**-20) + t * 1.01 + u * small).all()

    close(q, want[:, :c.heads], tol[:, :c.heads])
    # The cache: unchanged rows exactly, new ones to their rounding (3 2^-24 of at most |x| + |y| <= 12).
    close(k, wk, torch.tensor(3 * 2.0**-24 * 12))
    assert torch.equal(v.cpu(), wv.to(dtype))
    touched = (wk != c.k.double()).any(-1)
    assert torch.equal(k.cpu()[~touched], c.k[~touched])


@pytest.mark.parametrize("dtype", [BF, F])
def test_append_takes_any_rows(dtype):
    """Columns of a wider projection, rows of no 16- or 8-byte start, a turned projection, a
    given output, a prefix in front, padded rows."""
    c = Case([3, 2], [10, 4], kv=2, group=2, hd=64, page=16, dtype=dtype, seed=13)
    cos, sin = _tables(64, 64)
    base = torch.randn(8, 8, 64, generator=_gen(14)).to(dtype).to(DEV)
    rest = (c.table.to(DEV), c.lengths.to(DEV), (c.starts + 1).to(DEV))
    want = None
    wide = torch.zeros(8, 11, 64, dtype=dtype, device=DEV)
    wide[:, 1:9] = base
    turned = base.transpose(0, 1).contiguous().transpose(0, 1)
    across = base.transpose(1, 2).contiguous().transpose(1, 2)
    views = [base, wide[:, 1:9], turned, across]
    for shift in (1, 2, 4):
        x = torch.zeros(8 * 8 * 64 + shift, dtype=dtype, device=DEV)[shift:].view(8, 8, 64)
        x.copy_(base)
        views.append(x)
    for x in views:
        k, v = c.k.to(DEV), c.v.to(DEV)
        q = paged_append(x, cos[:, None], sin[:, None], k, v, *rest, prefix_len=37)
        assert (q[0] == 0).all() and (q[6:] == 0).all()
        out = torch.full_like(q, 5.0)
        assert paged_append(x, cos, sin, k, v, *rest, prefix_len=37, out=out) is out
        assert torch.equal(out[1:6], q[1:6]) and (out[0] == 5).all() and (out[6:] == 5).all()
        want = (q, k, v) if want is None else want
        assert all(torch.equal(a, b) for a, b in zip((q, k, v), want))
    ref, _, _, _ = _append_expected(c, base[1:6], cos, sin, offset=37)
    assert (q[1:6].cpu().double() - ref[:, :c.heads]).abs().max() <= 2 * 2.0**-8 * 8


def test_tokens_with_no_place():
    c = Case([2, 2, 2, 3], [20, 62, 0, 0], kv=1, group=2, hd=64, page=16, dtype=BF, seed=15)
    cos, sin = _tables(63, 64)  # the second sequence's last position is off the tables
    qkv = torch.randn(9, 4, 64, generator=_gen(16)).to(BF).to(DEV)
    table = c.table.clone()
    table[0, 1], table[2, 0] = 1 << 20, -1
    lengths = c.lengths.clone()
    lengths[3] = 2  # three rows, two tokens
    k, v = c.k.to(DEV), c.v.to(DEV)
    q = paged_append(qkv, cos, sin, k, v, table.to(DEV), lengths.to(DEV), c.starts.to(DEV))
    lost = torch.tensor([True, True, False, True, True, True, True, False, False])
    assert torch.equal(torch.isnan(q).all(-1).all(-1).cpu(), lost)
    assert torch.equal(torch.isnan(q).any(-1).any(-1).cpu(), lost)
    kept = torch.zeros(k.shape[0], 16, dtype=torch.bool)
    for b, j in ((1, 62), (3, 0), (3, 1)):
        kept[c.table[b, j // 16], j % 16] = True
    changed = (k.cpu() != c.k).any(-1).any(1)
    assert torch.equal(changed, kept) and torch.equal((v.cpu() != c.v).any(-1).any(1), kept)


# --------------------------------------------------------------- streams and graphs


def test_a_captured_step_follows_lengths_and_tables():
    """Append and attention captured once, replayed for other tokens, lengths and pages, with
    eager work in between; two graphs of the same call do not disturb one another."""
    c = Case([1, 1, 1], [200, 3, 77], kv=2, group=2, hd=64, page=16, dtype=BF, prefix=50, seed=17)
    cos, sin = _tables(512, 64)
    table, lengths = c.table.to(DEV), c.lengths.to(DEV)
    pre = torch.tensor(c.prefix_ids, dtype=torch.int32, device=DEV)
    qkv = torch.randn(3, 8, 64, generator=_gen(18)).to(BF).to(DEV)
    k, v = c.k.to(DEV), c.v.to(DEV)

    def step():
        q = paged_append(qkv, cos, sin, k, v, table, lengths, prefix_len=50)
        return paged_attention(q, k, v, table, lengths, prefix_pages=pre, prefix_len=50)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for turn in range(4):
        lengths.copy_(torch.tensor([201 - 7 * turn, 4 + turn, 78 - 20 * turn], dtype=torch.int32))
        qkv.copy_(torch.randn(3, 8, 64, generator=_gen(20 + turn)).to(BF))
        table.copy_((c.table + turn) % c.k.shape[0])  # other pages, still one sequence's each
        want = step().clone()
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("prefix", [0, 40])
def test_a_captured_ragged_call_follows_starts(prefix, dtype):
    """How the packed rows divide among the sequences is read when the call is replayed: many
    rows of one, few of all, none of some, rows of no sequence."""
    c = Case([60, 37, 3, 40], [100, 0, 900, 33], kv=2, group=2, hd=64, page=16, dtype=dtype, prefix=prefix, seed=21)
    q, k, v, table = c.q.to(DEV), c.k.to(DEV), c.v.to(DEV), c.table.to(DEV)
    starts, lengths = c.starts.to(DEV), c.lengths.to(DEV)
    more = dict(prefix_pages=torch.tensor(c.prefix_ids, dtype=torch.int32, device=DEV), prefix_len=prefix)
    out = torch.zeros_like(q)

    def call(to=None):
        return paged_attention(q, k, v, table, lengths, starts, out=to, **(more if prefix else {}))

    call(out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(out)
    for new, lens in (([60, 37, 3, 40], None), ([1, 1, 1, 137], [160, 1, 903, 139]), ([0, 0, 140, 0], [1, 0, 903, 2]),
                      ([8, 8, 8, 8], [160, 37, 8, 64]), ([30, 0, 2, 90], [31, 5, 800, 73])):
        starts.copy_(torch.tensor([0, *new], dtype=torch.int32).cumsum(0, dtype=torch.int32))
        lengths.copy_(c.lengths if lens is None else torch.tensor(lens, dtype=torch.int32))
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        want = call()
        rows = sum(new)
        assert torch.equal(out[:rows], want[:rows]) and (out[rows:] == 7).all() and (want[rows:] == 0).all()
        if lens is None:
            c.check(got=want)


def test_calls_on_two_streams_at_once():
    c = Case([1] * 8, [500 * i for i in range(8)], kv=2, group=2, hd=128, page=64, dtype=BF, seed=22)
    d = Case([40, 30], [800, 20], kv=2, group=2, hd=128, page=64, dtype=BF, seed=23)
    wants = [c.call(), d.call()]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    args = []
    for x in (c, d):
        args.append((x.q.to(DEV), x.k.to(DEV), x.v.to(DEV), x.table.to(DEV), x.lengths.to(DEV), x.starts.to(DEV)))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged_attention(*args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, got[i][0]) for o in got[i])
        assert (got[i][0].float() - wants[i].float()).abs().max() <= 2 * 2.0**-8 * 4


def test_a_mode_sees_the_call():
    """Inside a function mode the Python path makes the same call."""
    from torch.overrides import TorchFunctionMode

    class Mode(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    c = Case([1, 3], [50, 9], kv=2, group=2, hd=64, page=16, dtype=BF, prefix=20, seed=24)
    cos, sin = _tables(128, 64)
    qkv = torch.randn(4, 8, 64, generator=_gen(25)).to(BF).to(DEV)

    def step():
        k, v = c.k.to(DEV), c.v.to(DEV)
        q = paged_append(qkv, cos, sin, k, v, c.table.to(DEV), c.lengths.to(DEV), c.starts.to(DEV), prefix_len=20)
        return c.call(q=q), k, v

    want = step()
    with Mode():
        got = step()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_autograd_is_refused():
    c = Case([1], [5], kv=1, group=1, hd=64, page=16, dtype=F, seed=26)
    q = c.q.to(DEV).requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        c.call(q=q)
    with torch.no_grad():
        c.call(q=q)

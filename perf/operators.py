"""What generating with the decoder costs: each case is one call through a public entry
point of ``switchyard.cache_op`` or ``switchyard.sample_op``.

  append   the rotary positions of a fused QKV projection, its keys and values into
           the pages of a cache
  attend   attention of the new tokens over the pages
  prefix   the same for sequences that continue one prompt, whose pages they share
  sample   tokens from logits by temperature, top-k, top-p and min-p

``run`` computes a case with elementary torch operations while ``own`` is false, and
through the framework's entry points where it is true. ``exact`` gives the same outputs
in float64 from the operators' definitions.
"""

from __future__ import annotations

import math
import pathlib
import random
import sys

import numpy as np
import torch

_PKG = pathlib.Path(__file__).resolve().parent.parent / "blackwell-switchyard_amd"
if str(_PKG) not in sys.path:
    sys.path.insert(0, str(_PKG))

own = False

DEV = "cuda"
THETA = 10000.0
ONE = 1 << 44  # sampling weights are fractions of the largest in units of 2^-44
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # One decoded token of eight sequences of the 1.3B decoder: a launch's latency.
        dict(name="append_decode", kind="append", b=8, new=1, past=4000, heads=16, kv=16, hd=128, page=64,
             dtype="bf16", ragged=1),
        # Its prompts: four of up to 2048 tokens, none of them full pages.
        dict(name="append_prompts", kind="append", b=4, new=2048, past=0, heads=16, kv=16, hd=128, page=64,
             dtype="bf16", ragged=2),
        # The small decoder in fp32, four sequences within its 512 positions.
        dict(name="decode_small", kind="attend", b=4, new=1, past=500, heads=8, kv=8, hd=64, page=16,
             dtype="fp32", ragged=3),
        # The first tokens of eight short chats with the 1.3B decoder: two launches and little else.
        dict(name="decode_few", kind="attend", b=8, new=1, past=300, heads=16, kv=16, hd=128, page=64,
             dtype="bf16", ragged=10),
        # A serving batch of the 1.3B decoder, one token each, contexts of any length up to its 4096.
        dict(name="decode_batch", kind="attend", b=32, new=1, past=4095, heads=16, kv=16, hd=128, page=64,
             dtype="bf16", ragged=4),
        # Two long documents, grouped heads: few rows, a long axis.
        dict(name="decode_long", kind="attend", b=2, new=1, past=131000, heads=32, kv=4, hd=128, page=64,
             dtype="fp16", ragged=5),
        # The 1.3B decoder's prompts attending to themselves.
        dict(name="prompts", kind="attend", b=4, new=2048, past=0, heads=16, kv=16, hd=128, page=64,
             dtype="bf16", ragged=6),
        # Prompts taken in pieces next to sequences that decode: some of the batch brings up to 777 tokens
        # on top of a long past, the rest one; small pages, heads of 64.
        dict(name="pieces", kind="attend", b=12, new=777, past=9000, heads=24, kv=8, hd=64, page=16,
             dtype="fp16", ragged=7, mixed=True),
        # 64 answers to one prompt of 4096 tokens, each some way on.
        dict(name="prefix_answers", kind="prefix", b=64, new=1, past=255, prefix=4096, heads=16, kv=16, hd=128,
             page=64, dtype="bf16", ragged=8),
        # A long document in common, grouped heads, a ragged last page of it.
        dict(name="prefix_document", kind="prefix", b=16, new=1, past=1023, prefix=30011, heads=32, kv=8, hd=128,
             page=32, dtype="fp16", ragged=9),
        # Eight sequences over the 1.3B decoder's vocabulary with the usual settings.
        dict(name="sample_few", kind="sample", b=8, vocab=32000, dtype="bf16", temperature=0.8, top_k=50,
             top_p=0.95, min_p=0.0, per_row=False, banned=0.0),
        # A serving batch, every row with settings of its own, an odd vocabulary, some tokens ruled out.
        dict(name="sample_batch", kind="sample", b=256, vocab=50257, dtype="fp32", temperature=0.9, top_k=0,
             top_p=0.9, min_p=0.02, per_row=True, banned=0.1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "prefix", "prefix", "sample", "sample"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "sample":
        return dict(kind=kind, b=_log(rng, 1, 256), vocab=_log(rng, 300, 50257), dtype=dtype,
                    temperature=rng.choice([0.5, 0.7, 1.0, 1.3]), top_k=rng.choice([0, 0, 1, 20, 50, 400]),
                    top_p=rng.choice([1.0, 0.95, 0.9, 0.6]), min_p=rng.choice([0.0, 0.0, 0.05]),
                    per_row=rng.random() < 0.5, banned=rng.choice([0.0, 0.0, 0.3]))
    hd = rng.choice([64, 64, 128, 128, 128, 32, 80, 96, 256])
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    group = rng.choice([1, 1, 2, 3, 4, 8] if kv < 16 else [1, 1, 2])
    c = dict(kind=kind, heads=kv * group, kv=kv, hd=hd, page=rng.choice([16, 16, 32, 64, 128]), dtype=dtype,
             ragged=rng.randint(1, 1 << 30))
    if kind == "append":
        c.update(b=_log(rng, 1, 64), new=rng.choice([1, 1, _log(rng, 2, 2048)]), past=_log(rng, 1, 2000))
        while c["b"] * c["new"] * (c["heads"] + 2 * kv) * hd * _SIZE[dtype] > 9.0e7:
            c["b"], c["new"] = max(1, c["b"] // 2), max(1, c["new"] - c["new"] // 3)
        while c["b"] * c["past"] * kv * hd * _SIZE[dtype] > 2.0e8:
            c["past"] //= 2
        return c
    if kind == "prefix":
        c.update(b=_log(rng, 2, 64), new=rng.choice([1, 1, 1, rng.randint(2, 9)]), past=_log(rng, 1, 1023),
                 prefix=_log(rng, 100, 30000))
    elif rng.random() < 0.6:
        c.update(b=_log(rng, 1, 64), new=1, past=_log(rng, 1, 60000))
    else:
        c.update(b=_log(rng, 1, 16), new=_log(rng, 2, 2048), past=rng.choice([0, _log(rng, 1, 8000)]),
                 mixed=rng.random() < 0.5)
    # No more keys and values, nor products, than the largest listed cases have.
    while c["b"] * (c["past"] + c["new"] + c.get("prefix", 0)) * kv * hd * _SIZE[dtype] * 2 > 1.0e9:
        c["b"] = max(1, c["b"] // 2)
        c["past"] -= c["past"] // 4
        if "prefix" in c:
            c["prefix"] -= c["prefix"] // 4
    while work(c)["flops"] > (3.0e10 if dtype != "fp32" else 4.0e9):
        c["new"] = max(1, c["new"] // 2)
        c["past"] -= c["past"] // 4
        if "prefix" in c:
            c["prefix"] -= c["prefix"] // 4
    return c


# ------------------------------------------------------------------ inputs


def _counts(c):
    """New tokens and earlier tokens of every sequence: of the case, not of the seed."""
    rng = random.Random(c["ragged"])
    new, past = [], []
    for i in range(c["b"]):
        if c["new"] == 1 or (c.get("mixed") and i % 3):
            new.append(1)
        else:
            new.append(c["new"] if i == 0 else rng.randint((c["new"] + 1) // 2, c["new"]))
        past.append(c["past"] if i == 0 else rng.randint(c["past"] // 8, c["past"]))
    return new, past


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _ints(x):
    return torch.tensor(x, device=DEV, dtype=torch.int32)


def _pages(c, seed):
    """The page table, with every sequence's pages anywhere in the cache, and the prefix's
    pages; a few pages are nobody's."""
    new, past = _counts(c)
    page = c["page"]
    need = [-(-(n + p) // page) for n, p in zip(new, past)]
    shared = -(-c.get("prefix", 0) // page)
    total = sum(need) + shared + 3
    ids = list(range(total))
    random.Random(seed).shuffle(ids)
    table, at = [], shared
    for n in need:
        table.append(ids[at:at + n] + [0] * (max(need) - n))
        at += n
    return table, ids[:shared], total


def _settings(c, seed):
    """The sampling settings: numbers, or one of each for every row."""
    t, k, p, m = c["temperature"], c["top_k"], c["top_p"], c["min_p"]
    if not c["per_row"]:
        return t, k, p, m
    r, b = random.Random(seed), c["b"]
    f = lambda x: torch.tensor(x, device=DEV, dtype=torch.float32)  # noqa: E731
    return (f([t * r.uniform(0.7, 1.3) for _ in range(b)]), _ints([k * r.randint(0, 2) for _ in range(b)]),
            f([min(1.0, p * r.uniform(0.8, 1.2)) for _ in range(b)]), f([m * r.uniform(0.0, 2.0) for _ in range(b)]))


def prepare(case, seed):
    c, g = case, _gen(seed)
    dt = _DT[c["dtype"]]
    if c["kind"] == "sample":
        # Logits as a decoder's are: most of them far down, a few candidates ahead.
        x = 2.0 * torch.randn(c["b"], c["vocab"], device=DEV, generator=g)
        x[:, torch.randint(0, c["vocab"], (12,), device=DEV, generator=g)] += 5.0
        if c["banned"]:
            x[torch.rand(x.shape, device=DEV, generator=g) < c["banned"]] = -math.inf
        return {"case": c, "logits": x.to(dt), "u": torch.rand(c["b"], device=DEV, generator=g),
                "settings": _settings(c, seed)}
    new, past = _counts(c)
    table, shared, total = _pages(c, seed)
    tok, kv, hd = sum(new), c["kv"], c["hd"]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, dtype=dt, generator=g)

    s = {"case": c, "k": normal(total, kv, c["page"], hd), "v": normal(total, kv, c["page"], hd),
         "table": _ints(table), "lengths": _ints([n + p for n, p in zip(new, past)]),
         # One token of each sequence needs no list of where they start.
         "starts": None if c["new"] == 1 else _ints(starts)}
    if c["kind"] == "append":
        s["qkv"] = normal(tok, c["heads"] + 2 * kv, hd)
        inv = THETA ** (-torch.arange(hd // 2, device=DEV, dtype=torch.float64) * 2.0 / hd)
        ang = torch.arange(max(n + p for n, p in zip(new, past)), device=DEV, dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    else:
        s["q"] = 1.5 * normal(tok, c["heads"], hd)
        if c["kind"] == "prefix":
            s["prefix"] = _ints(shared)
    return s


# --------------------------------------------------------------- the calls


def run(state):
    with torch.no_grad():
        return (_run_own if own else _run_plain)(state)


def _run_own(s):
    c = s["case"]
    if c["kind"] == "sample":
        from switchyard.sample_op import sample_tokens

        t, k, p, m = s["settings"]
        return {"tokens": sample_tokens(s["logits"], s["u"], temperature=t, top_k=k, top_p=p, min_p=m)}
    from switchyard.cache_op import paged_append, paged_attention

    if c["kind"] == "append":
        q = paged_append(s["qkv"], s["cos"], s["sin"], s["k"], s["v"], s["table"], s["lengths"], s["starts"])
        return {"q": q, "k": s["k"], "v": s["v"]}
    more = {} if c["kind"] == "attend" else {"prefix_pages": s["prefix"], "prefix_len": c["prefix"]}
    return {"out": paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], s["starts"], **more)}


def _run_plain(s):
    c = s["case"]
    if c["kind"] == "sample":
        return {"tokens": _plain_sample(s["logits"], s["u"], *s["settings"])}
    if c["kind"] == "append":
        return _plain_append(s)
    new, past = _counts(c)
    at, outs = 0, []
    for b, (n, p) in enumerate(zip(new, past)):
        k, v = _plain_gather(s, b, n + p)
        outs.append(_plain_attend(s["q"][at:at + n], k, v, p + c.get("prefix", 0)))
        at += n
    return {"out": torch.cat(outs)}


def _plain_append(s):
    c = s["case"]
    new, past = _counts(c)
    tok = torch.cat([torch.arange(p, p + n, device=DEV) for n, p in zip(new, past)])
    seq = torch.cat([torch.full((n,), b, device=DEV) for b, n in enumerate(new)])
    page = s["table"].long()[seq, tok // c["page"]]
    slot = tok % c["page"]
    q, k, v = s["qkv"].split([c["heads"], c["kv"], c["kv"]], dim=1)

    def turn(x):
        lo, hi = x.float().chunk(2, dim=-1)
        cos, sin = s["cos"][tok][:, None], s["sin"][tok][:, None]
        return torch.cat((lo * cos - hi * sin, lo * sin + hi * cos), dim=-1).to(x.dtype)

    s["k"][page, :, slot] = turn(k)
    s["v"][page, :, slot] = v
    return {"q": turn(q), "k": s["k"], "v": s["v"]}


def _plain_gather(s, b, n):
    """Keys and values of sequence ``b`` behind those of the prefix, ``[keys, kv, hd]``."""
    c = s["case"]
    parts = [(s["table"][b], n)]
    if c["kind"] == "prefix":
        parts.insert(0, (s["prefix"], c["prefix"]))
    got = []
    for x in (s["k"], s["v"]):
        rows = [x[ids[:-(-m // c["page"])].long()].transpose(1, 2).reshape(-1, c["kv"], c["hd"])[:m]
                for ids, m in parts]
        got.append(torch.cat(rows).float())
    return got


def _plain_attend(q, k, v, first):
    """``q [n, heads, hd]``, the first of its tokens at position ``first`` of the keys."""
    n, heads, hd = q.shape
    kv, keys = k.shape[1], k.shape[0]
    qh = q.float().view(n, kv, heads // kv, hd).permute(1, 2, 0, 3).reshape(kv, -1, hd)
    s = (qh @ k.permute(1, 2, 0).contiguous()).view(kv, heads // kv, n, keys) * hd**-0.5
    if n > 1:
        at = torch.arange(n, device=DEV)[:, None] + first
        s = s.masked_fill(torch.arange(keys, device=DEV)[None] > at, -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    o = e.view(kv, -1, keys) @ v.permute(1, 0, 2).contiguous()
    o = o.view(kv, -1, n, hd) / e.sum(-1, keepdim=True)
    return o.permute(2, 0, 1, 3).reshape(n, heads, hd).to(q.dtype)


def _column(x):
    """A setting as a column of doubles."""
    return x.double()[:, None] if torch.is_tensor(x) else x


def _plain_sample(logits, u, temperature, top_k, top_p, min_p):
    n = logits.shape[1]
    x = logits.double()
    e = torch.exp((x - x.amax(-1, keepdim=True)) / _column(temperature))
    w = torch.round(e * ONE).long()
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    sorted_w = w.gather(1, order)
    rank = torch.arange(n, device=DEV)[None]
    k = top_k.long()[:, None] if torch.is_tensor(top_k) else torch.tensor([[top_k]], device=DEV)
    keep = (rank < k) | (k <= 0)
    sorted_w = sorted_w * keep
    before = sorted_w.cumsum(-1) - sorted_w
    total = sorted_w.sum(-1, keepdim=True).double()
    keep = keep & ((rank == 0) | (before.double() < _column(top_p) * total))
    kept = torch.zeros_like(keep).scatter(1, order, keep) & (e >= _column(min_p))
    w = w * kept
    cum = w.cumsum(-1)
    r = (u.double()[:, None] * cum[:, -1:].double()).long()
    last = torch.where(w > 0, rank, -1).amax(-1)
    return torch.minimum((cum <= r).sum(-1), last)


# -------------------------------------------------------- what is expected


def work(case):
    c = case
    if c["kind"] == "sample":
        # The logits once; a weight, its comparisons and its sums for each.
        n = c["b"] * c["vocab"]
        return {"bytes": n * _SIZE[c["dtype"]] + 12 * c["b"], "flops": 8 * n}
    new, past = _counts(c)
    size, tok = _SIZE[c["dtype"]], sum(new)
    if c["kind"] == "append":
        # The projection in, the queries and the cache's rows out, the tables' rows.
        rows = c["heads"] + 2 * c["kv"]
        return {"bytes": tok * (2 * rows * c["hd"] * size + 4 * c["hd"]),
                "flops": 3 * tok * (c["heads"] + c["kv"]) * c["hd"]}
    keys = sum(n + p for n, p in zip(new, past)) + c.get("prefix", 0)
    seen = sum(n * (p + c.get("prefix", 0)) + n * (n + 1) // 2 for n, p in zip(new, past))
    return {"bytes": 2 * size * c["hd"] * (keys * c["kv"] + tok * c["heads"]),
            "flops": 4 * c["hd"] * c["heads"] * seen}


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "sample":
        return {"tokens": _exact_sample(s)}
    new, past = _counts(c)
    page = c["page"]

    def rows(x, ids, n):  # the first n rows that a list of pages holds
        j = torch.arange(n, device=DEV)
        return x[ids.long()[j // page], :, j % page]

    at = 0
    if c["kind"] == "append":
        k, v = s["k"].double(), s["v"].double()
        q = torch.empty(sum(new), c["heads"], c["hd"], device=DEV, dtype=torch.float64)
        half = c["hd"] // 2
        for b, (n, p) in enumerate(zip(new, past)):
            x = s["qkv"][at:at + n].double()
            z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous())
            turn = torch.complex(s["cos"][p:p + n].double(), s["sin"][p:p + n].double())[:, None]
            z = z * turn
            z = torch.cat((z.real, z.imag), dim=-1)
            q[at:at + n] = z[:, :c["heads"]]
            j = torch.arange(p, p + n, device=DEV)
            ids = s["table"][b].long()[j // page]
            k[ids, :, j % page] = z[:, c["heads"]:c["heads"] + c["kv"]]
            v[ids, :, j % page] = x[:, c["heads"] + c["kv"]:]
            at += n
        return {"q": q, "k": k, "v": v}
    out = torch.empty(sum(new), c["heads"], c["hd"], device=DEV, dtype=torch.float64)
    group = c["heads"] // c["kv"]
    for b, (n, p) in enumerate(zip(new, past)):
        kk, vv = rows(s["k"], s["table"][b], n + p).double(), rows(s["v"], s["table"][b], n + p).double()
        if c["kind"] == "prefix":
            kk = torch.cat((rows(s["k"], s["prefix"], c["prefix"]).double(), kk))
            vv = torch.cat((rows(s["v"], s["prefix"], c["prefix"]).double(), vv))
        hidden = torch.ones(n, kk.shape[0], device=DEV, dtype=torch.bool).triu(kk.shape[0] - n + 1)
        for h in range(c["heads"]):
            kh, vh = kk[:, h // group], vv[:, h // group]
            a = (s["q"][at:at + n, h].double() @ kh.T) / math.sqrt(c["hd"])
            out[at:at + n, h] = torch.softmax(a.masked_fill(hidden, -math.inf), dim=-1) @ vh
        at += n
    return {"out": out}


def _exact_sample(s):
    """Row by row on the host: candidates in order of their logits, then the draw in order
    of their indices, in whole numbers."""
    x = s["logits"].double().cpu().numpy()
    u = s["u"].double().cpu().numpy()
    per = [v.double().cpu().numpy() if torch.is_tensor(v) else np.full(len(x), float(v)) for v in s["settings"]]
    tokens = []
    for row, r, t, k, p, m in zip(x, u, *per):
        e = np.exp((row - row.max()) / t)
        w = np.rint(e * ONE).astype(np.int64)
        first = np.argsort(-row, kind="stable")
        if k >= 1:
            first = first[:int(k)]
        ws = w[first]
        before = np.concatenate(([0], np.cumsum(ws)[:-1]))
        enough = before >= p * float(ws.sum())
        enough[0] = False
        first = first[~enough]
        chosen = np.sort(first[e[first] >= m])
        cum = np.cumsum(w[chosen])
        i = int(np.searchsorted(cum, int(r * float(cum[-1])), side="right"))
        tokens.append(int(chosen[min(i, np.flatnonzero(w[chosen])[-1])]))
    return torch.tensor(tokens, device=DEV)

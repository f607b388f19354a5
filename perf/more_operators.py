"""What a decoder with normalised heads costs to train, and what its steps cost to serve from
4-bit weights and to steer: each case is one call, or one forward + backward, through a
public entry point of ``switchyard.rope_op``, ``switchyard.cache_op``,
``switchyard.quant_op`` or ``switchyard.logits_op``.

  rope     RMSNorm of every query and key head with the rotation to its position, and the
           split of the fused projection into attention's layout; trained
  append   the same norms and rotation on the way into the pages of a cache
  linear4  a projection with 4-bit weights, a scale (and a zero point) for each group
  adjust   penalties for tokens that were there before, biases and a grammar's mask on logits

``run`` computes a case with elementary torch operations while ``own`` is false, and
through the framework's entry points where it is true. ``exact`` gives the same outputs
in float64 from the operators' definitions.
"""

from __future__ import annotations

import math
import pathlib
import random
import sys

import torch

_PKG = pathlib.Path(__file__).resolve().parent.parent / "blackwell-switchyard_amd"
if str(_PKG) not in sys.path:
    sys.path.insert(0, str(_PKG))

own = False

DEV = "cuda"
THETA = 10000.0
EPS = 1e-6
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # The fused QKV projection of the 1.3B decoder for one token: a launch and 6 MB.
        dict(name="linear4_one", kind="linear4", m=1, n=6144, k=2048, group=64, zeros=False, dtype="bf16"),
        # Its LM head for eight sequences.
        dict(name="linear4_head", kind="linear4", m=8, n=32000, k=2048, group=128, zeros=False, dtype="bf16"),
        # Its gate and up projection for a serving batch, with zero points.
        dict(name="linear4_up", kind="linear4", m=32, n=11264, k=2048, group=64, zeros=True, dtype="fp16"),
        # A wide model's feed-forward, sixteen sequences: the weights' bytes are all that counts.
        dict(name="linear4_wide", kind="linear4", m=16, n=28672, k=8192, group=128, zeros=True, dtype="bf16"),
        # Odd everything in fp32: rows of no multiple of anything, a last group that is not full.
        dict(name="linear4_odd", kind="linear4", m=5, n=1407, k=2001, group=32, zeros=True, dtype="fp32"),
        # A prompt of 2048 tokens through the 1.3B decoder's down projection.
        dict(name="linear4_prompt", kind="linear4", m=2048, n=2048, k=5632, group=64, zeros=False, dtype="bf16"),
        # Eight chats over the 1.3B decoder's vocabulary, a penalty on what was said before.
        dict(name="adjust_few", kind="adjust", b=8, vocab=32000, past=4000, dtype="bf16", repetition=1.1,
             presence=0.0, frequency=0.0, per_row=False, bias="", allowed=0.0, ragged=1),
        # A serving batch, every row with settings of its own, an odd vocabulary, biases and a
        # grammar that leaves a third of the tokens.
        dict(name="adjust_batch", kind="adjust", b=256, vocab=50257, past=1500, dtype="fp32", repetition=1.2,
             presence=0.4, frequency=0.2, per_row=True, bias="shared", allowed=0.3, ragged=2),
        # One decoded token of eight sequences of the 1.3B decoder.
        dict(name="append_decode", kind="append", b=8, new=1, past=4000, heads=16, kv=16, hd=128, page=64,
             dtype="bf16", ragged=3),
        # Prompts of grouped heads of 64, small pages, none of them full.
        dict(name="append_prompts", kind="append", b=5, new=1777, past=300, heads=32, kv=4, hd=64, page=16,
             dtype="fp16", ragged=4),
        # The 1.3B decoder's training step: four sequences of 2048 tokens, forward and backward.
        dict(name="rope_train", kind="rope", b=4, t=2048, heads=16, kv=16, hd=128, dtype="bf16"),
        # Grouped heads of 96 in fp32, odd sizes.
        dict(name="rope_grouped", kind="rope", b=3, t=701, heads=12, kv=4, hd=96, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear4", "linear4", "linear4", "adjust", "adjust", "append", "rope", "rope"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "linear4":
        c = dict(kind=kind, m=rng.choice([1, _log(rng, 1, 16), _log(rng, 1, 64), _log(rng, 16, 2048)]),
                 n=_log(rng, 64, 32000), k=_log(rng, 64, 8192), group=rng.choice([32, 64, 128]),
                 zeros=rng.random() < 0.5, dtype=dtype)
        if rng.random() < 0.6:  # sizes as models mostly have them
            c["n"], c["k"] = -(-c["n"] // 64) * 64, -(-c["k"] // 64) * 64
        # fp32 counts for more: its products have three parts.
        while c["m"] * c["n"] * c["k"] > (2.3e10 if dtype != "fp32" else 4.0e9):
            c["m"] -= c["m"] // 3
        return c
    if kind == "adjust":
        c = dict(kind=kind, b=_log(rng, 1, 256), vocab=_log(rng, 300, 131072), past=_log(rng, 1, 16000), dtype=dtype,
                 repetition=rng.choice([1.0, 1.1, 1.3, 0.9]), presence=rng.choice([0.0, 0.5, -0.3]),
                 frequency=rng.choice([0.0, 0.2]), per_row=rng.random() < 0.5,
                 bias=rng.choice(["", "", "shared", "rows"]), allowed=rng.choice([0.0, 0.0, 0.5, 0.01]),
                 ragged=rng.randint(1, 1 << 30))
        while c["b"] * c["vocab"] > 1.2e7:
            c["b"] -= c["b"] // 3
        while c["b"] * c["past"] > 4.0e5:
            c["past"] -= c["past"] // 3
        return c
    hd = rng.choice([64, 64, 128, 128, 128, 32, 80, 96, 256])
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    group = rng.choice([1, 1, 2, 3, 4, 8] if kv < 16 else [1, 1, 2])
    c = dict(kind=kind, heads=kv * group, kv=kv, hd=hd, dtype=dtype)
    row = (kv * group + 2 * kv) * hd * _SIZE[dtype]
    if kind == "rope":
        c.update(b=_log(rng, 1, 16), t=_log(rng, 1, 4096))
        while c["b"] * c["t"] * row > 1.0e8:
            c["b"], c["t"] = max(1, c["b"] // 2), max(1, c["t"] - c["t"] // 3)
        return c
    c.update(b=_log(rng, 1, 64), new=rng.choice([1, 1, _log(rng, 2, 2048)]), past=_log(rng, 1, 2000),
             page=rng.choice([16, 16, 32, 64, 128]), ragged=rng.randint(1, 1 << 30))
    while c["b"] * c["new"] * row > 6.0e7:
        c["b"], c["new"] = max(1, c["b"] // 2), max(1, c["new"] - c["new"] // 3)
    while c["b"] * c["past"] * kv * hd * _SIZE[dtype] > 2.0e8:
        c["past"] //= 2
    return c


# ------------------------------------------------------------------ inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _ints(x):
    return torch.tensor(x, device=DEV, dtype=torch.int32)


def _counts(c):
    """New tokens and earlier tokens of every sequence: of the case, not of the seed."""
    rng = random.Random(c["ragged"])
    new = [c["new"] if i == 0 else rng.randint((c["new"] + 1) // 2, c["new"]) for i in range(c["b"])]
    past = [c["past"] if i == 0 else rng.randint(c["past"] // 8, c["past"]) for i in range(c["b"])]
    return new, past


def _angles(positions, hd):
    inv = THETA ** (-torch.arange(hd // 2, device=DEV, dtype=torch.float64) * 2.0 / hd)
    ang = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def _gains(c, g):
    """Learned gains: near one, a few channels far off."""
    return [(1.0 + 0.3 * torch.randn(c["hd"], device=DEV, generator=g)).to(_DT[c["dtype"]]) for _ in range(2)]


def prepare(case, seed):
    return {"linear4": _prepare_linear4, "adjust": _prepare_adjust, "append": _prepare_append,
            "rope": _prepare_rope}[case["kind"]](case, _gen(seed), seed)


def _prepare_linear4(c, g, seed):
    m, n, k, group, dt = c["m"], c["n"], c["k"], c["group"], _DT[c["dtype"]]
    groups = -(-k // group)
    # Activations with a few channels that are much larger, as a decoder's are; codes as a
    # normal distribution rounds to them, two to a byte, the even column in the low half.
    x = torch.randn(m, k, device=DEV, generator=g)
    x[:, torch.randint(0, k, (max(1, k // 256),), device=DEV, generator=g)] *= 12.0
    half = -(-k // 2)
    lo, hi = ((torch.randn(n, half, device=DEV, generator=g, dtype=torch.bfloat16) * 2.9 + 7.5).round().clamp(0, 15)
              .to(torch.uint8) for _ in range(2))
    s = {"case": c, "x": x.to(dt), "codes": lo | (hi << 4),
         "scales": (0.006 + 0.006 * torch.rand(n, groups, device=DEV, generator=g)).to(dt),
         "zeros": torch.randint(5, 11, (n, groups), device=DEV, generator=g, dtype=torch.uint8) if c["zeros"] else None}
    if own:  # a program lays its weights out when it loads them
        from switchyard.quant_op import Weight4

        s["weight"] = Weight4.from_codes(s["codes"], s["scales"], s["zeros"], in_features=k, group=group)
    return s


def _prepare_adjust(c, g, seed):
    b, v, r = c["b"], c["vocab"], random.Random(seed)
    x = 2.0 * torch.randn(b, v, device=DEV, generator=g)
    x[:, torch.randint(0, v, (12,), device=DEV, generator=g)] += 5.0
    # Tokens as text has them: a few of them often, most of them hardly ever. The last third
    # of a history was generated.
    at = torch.rand(b, c["past"], device=DEV, generator=g, dtype=torch.float64)
    tokens = (v * at**3).long().clamp(max=v - 1)
    rng = random.Random(c["ragged"])
    lengths = [c["past"] if i == 0 else rng.randint(c["past"] // 8, c["past"]) for i in range(b)]
    names = ("repetition", "presence", "frequency")
    settings = [c[n] for n in names]
    if c["per_row"]:
        settings = [torch.tensor([1.0 + (c[n] - 1.0) * r.uniform(0.2, 1.8) if n == "repetition" else c[n] * r.uniform(0, 2)
                                  for _ in range(b)], device=DEV) for n in names]
    bias = None
    if c["bias"]:
        bias = torch.randn(*([v] if c["bias"] == "shared" else [b, v]), device=DEV, generator=g)
        bias = bias * (torch.rand(bias.shape, device=DEV, generator=g) < 0.02)
    bits = None
    if c["allowed"]:
        # A grammar's mask: bit i of word j stands for token 32 j + i.
        words = -(-v // 32)
        keep = torch.rand(b, words, 32, device=DEV, generator=g) < c["allowed"]
        bits = (keep.long() << torch.arange(32, device=DEV)).sum(-1)
        bits = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
    return {"case": c, "logits": x.to(_DT[c["dtype"]]), "tokens": tokens, "lengths": _ints(lengths),
            "prompts": _ints([2 * n // 3 for n in lengths]), "settings": settings, "bias": bias, "bits": bits}


def _prepare_append(c, g, seed):
    new, past = _counts(c)
    page, dt = c["page"], _DT[c["dtype"]]
    need = [-(-(n + p) // page) for n, p in zip(new, past)]
    total = sum(need) + 3
    ids = list(range(total))  # every sequence's pages lie anywhere in the cache
    random.Random(seed).shuffle(ids)
    table, starts = [], [0]
    for n in need:
        table.append(ids[:n] + [0] * (max(need) - n))
        ids = ids[n:]
    for n in new:
        starts.append(starts[-1] + n)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, dtype=dt, generator=g)

    cos, sin = _angles(max(n + p for n, p in zip(new, past)), c["hd"])
    return {"case": c, "k": normal(total, c["kv"], page, c["hd"]), "v": normal(total, c["kv"], page, c["hd"]),
            "qkv": normal(sum(new), c["heads"] + 2 * c["kv"], c["hd"]), "gains": _gains(c, g), "cos": cos, "sin": sin,
            "table": _ints(table), "lengths": _ints([n + p for n, p in zip(new, past)]),
            # One token of each sequence needs no list of where they start.
            "starts": None if c["new"] == 1 else _ints(starts)}


def _prepare_rope(c, g, seed):
    b, t, hd, dt = c["b"], c["t"], c["hd"], _DT[c["dtype"]]
    cos, sin = _angles(t, hd)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, dtype=dt, generator=g)

    return {"case": c, "qkv": normal(b, t, c["heads"] + 2 * c["kv"], hd).requires_grad_(True),
            "gains": [x.requires_grad_(True) for x in _gains(c, g)], "cos": cos, "sin": sin,
            "grads": [normal(b, h, t, hd) for h in (c["heads"], c["kv"], c["kv"])]}


# --------------------------------------------------------------- the calls


def run(state):
    kind = state["case"]["kind"]
    if kind == "rope":
        return _rope_train(state)
    with torch.no_grad():
        if own:
            return {"linear4": _own_linear4, "adjust": _own_adjust, "append": _own_append}[kind](state)
        return {"linear4": _plain_linear4, "adjust": _plain_adjust, "append": _plain_append}[kind](state)


def _own_linear4(s):
    from switchyard.quant_op import linear4

    return {"out": linear4(s["x"], s["weight"])}


def _own_adjust(s):
    from switchyard.logits_op import adjust_logits

    r, p, f = s["settings"]
    return {"logits": adjust_logits(s["logits"], s["tokens"], lengths=s["lengths"], prompt_lengths=s["prompts"],
                                    repetition_penalty=r, presence_penalty=p, frequency_penalty=f, bias=s["bias"],
                                    allowed=s["bits"])}


def _own_append(s):
    from switchyard.cache_op import paged_append

    q = paged_append(s["qkv"], s["cos"], s["sin"], s["k"], s["v"], s["table"], s["lengths"], s["starts"],
                     q_gain=s["gains"][0], k_gain=s["gains"][1], eps=EPS)
    return {"q": q, "k": s["k"], "v": s["v"]}


def _rope_train(s):
    c = s["case"]
    if own:
        from switchyard.rope_op import qk_norm_rope

        outs = qk_norm_rope(s["qkv"], *s["gains"], s["cos"], s["sin"], kv_heads=c["kv"], eps=EPS)
    else:
        outs = _plain_rope(s["qkv"], *s["gains"], s["cos"], s["sin"], c["heads"], c["kv"])
    grads = torch.autograd.grad(outs, [s["qkv"], *s["gains"]], s["grads"])
    return {"q": outs[0].detach(), "k": outs[1].detach(), "v": outs[2].detach(), "dqkv": grads[0], "dq_gain": grads[1],
            "dk_gain": grads[2]}


def _plain_linear4(s):
    c = s["case"]
    codes = torch.stack((s["codes"] & 15, s["codes"] >> 4), -1).view(c["n"], -1)[:, :c["k"]].float()
    of = torch.arange(c["k"], device=DEV) // c["group"]
    zero = 8.0 if s["zeros"] is None else s["zeros"].float()[:, of]
    w = (codes - zero) * s["scales"].float()[:, of]
    return {"out": (s["x"].float() @ w.T).to(s["x"].dtype)}


def _rows(x):
    """A setting as a column."""
    return x[:, None] if torch.is_tensor(x) else x


def _plain_adjust(s):
    c, x = s["case"], s["logits"].float()
    r, p, f = (_rows(v) for v in s["settings"])
    at = torch.arange(c["past"], device=DEV)[None]
    there = at < s["lengths"][:, None]
    count = torch.zeros(x.shape, device=DEV)
    count.scatter_add_(1, s["tokens"], (there & (at >= s["prompts"][:, None])).float())
    seen = torch.zeros(x.shape, device=DEV)
    seen.scatter_add_(1, s["tokens"], there.float())
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - f * count - p * (count > 0)
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["bits"] is not None:
        keep = (s["bits"][:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
        x = x.masked_fill(keep.view(c["b"], -1)[:, :c["vocab"]] == 0, -math.inf)
    return {"logits": x.to(s["logits"].dtype)}


def _plain_norm(x, gain):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gain.float()


def _plain_turn(x, cos, sin):
    lo, hi = x.chunk(2, dim=-1)
    return torch.cat((lo * cos - hi * sin, lo * sin + hi * cos), dim=-1)


def _plain_rope(qkv, q_gain, k_gain, cos, sin, heads, kv):
    q, k, v = qkv.transpose(1, 2).split([heads, kv, kv], dim=1)
    q = _plain_turn(_plain_norm(q, q_gain), cos, sin).to(qkv.dtype)
    k = _plain_turn(_plain_norm(k, k_gain), cos, sin).to(qkv.dtype)
    return q, k, v.contiguous()


def _plain_append(s):
    c = s["case"]
    tok = torch.arange(s["qkv"].shape[0], device=DEV)
    starts = torch.arange(c["b"] + 1, device=DEV) if s["starts"] is None else s["starts"].long()
    seq = torch.searchsorted(starts, tok, right=True) - 1
    at = s["lengths"].long()[seq] - starts[seq + 1] + tok
    page, slot = s["table"].long()[seq, at // c["page"]], at % c["page"]
    q, k, v = s["qkv"].split([c["heads"], c["kv"], c["kv"]], dim=1)
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    s["k"][page, :, slot] = _plain_turn(_plain_norm(k, s["gains"][1]), cos, sin).to(k.dtype)
    s["v"][page, :, slot] = v
    return {"q": _plain_turn(_plain_norm(q, s["gains"][0]), cos, sin).to(q.dtype), "k": s["k"], "v": s["v"]}


# -------------------------------------------------------- what is expected


def work(case):
    c, size = case, _SIZE[case["dtype"]]
    if c["kind"] == "linear4":
        groups = -(-c["k"] // c["group"])
        # Activations in and out, half a byte a weight, a scale (and a zero point's byte) a group.
        return {"bytes": c["m"] * (c["n"] + c["k"]) * size + c["n"] * c["k"] // 2
                + c["n"] * groups * (size + (1 if c["zeros"] else 0)), "flops": 2 * c["m"] * c["n"] * c["k"]}
    if c["kind"] == "adjust":
        # Logits in and out, the histories, biases and masks once.
        rng = random.Random(c["ragged"])
        past = sum(c["past"] if i == 0 else rng.randint(c["past"] // 8, c["past"]) for i in range(c["b"]))
        bias = {"": 0, "shared": 4 * c["vocab"], "rows": 4 * c["b"] * c["vocab"]}[c["bias"]]
        bits = 4 * c["b"] * -(-c["vocab"] // 32) if c["allowed"] else 0
        return {"bytes": 2 * size * c["b"] * c["vocab"] + 8 * past + bias + bits, "flops": 4 * c["b"] * c["vocab"]}
    rows = c["heads"] + 2 * c["kv"]
    turned = c["heads"] + c["kv"]
    if c["kind"] == "append":
        # The projection in, the queries and the cache's rows out, the tables' rows.
        tok = sum(_counts(c)[0])
        return {"bytes": tok * (2 * rows * c["hd"] * size + 4 * c["hd"]), "flops": 7 * tok * turned * c["hd"]}
    # Forward: the projection in, its parts out. Backward: their gradients and the heads that
    # were normalised in, the projection's gradient out.
    tok = c["b"] * c["t"]
    return {"bytes": tok * (4 * rows + turned) * c["hd"] * size + 2 * 4 * c["t"] * c["hd"],
            "flops": 22 * tok * turned * c["hd"]}


def exact(case, seed):
    s = prepare(case, seed)
    return {"linear4": _exact_linear4, "adjust": _exact_adjust, "append": _exact_append,
            "rope": _exact_rope}[case["kind"]](case, s)


def _exact_linear4(c, s):
    """Group by group: the sum of a group's products with whole numbers, then its scale."""
    out = torch.zeros(c["m"], c["n"], device=DEV, dtype=torch.float64)
    x = s["x"].double()
    q = torch.empty(c["n"], 2 * s["codes"].shape[1], device=DEV, dtype=torch.int8)
    q[:, 0::2] = s["codes"] % 16
    q[:, 1::2] = s["codes"] // 16
    for g in range(s["scales"].shape[1]):
        lo, hi = g * c["group"], min(c["k"], (g + 1) * c["group"])
        z = 8 if s["zeros"] is None else s["zeros"][:, g:g + 1].to(torch.int8)
        out += (x[:, lo:hi] @ (q[:, lo:hi] - z).double().T.contiguous()) * s["scales"][:, g].double()
    return {"out": out}


def _exact_adjust(c, s):
    """Row by row, by counting each token's occurrences."""
    x = s["logits"].double()
    lengths, prompts = s["lengths"].tolist(), s["prompts"].tolist()
    # The settings are fp32 numbers where they are tensors, and the numbers given elsewhere.
    r, p, f = ([float(v)] * c["b"] if not torch.is_tensor(v) else v.double().tolist() for v in s["settings"])
    for i in range(c["b"]):
        whole = torch.bincount(s["tokens"][i, :lengths[i]], minlength=c["vocab"])
        said = torch.bincount(s["tokens"][i, prompts[i]:lengths[i]], minlength=c["vocab"])
        seen = whole.nonzero()[:, 0]
        y = x[i, seen]
        x[i, seen] = y * torch.where(y > 0, 1.0 / r[i], r[i]) - f[i] * said[seen] - p[i] * said[seen].clamp(max=1)
    if s["bias"] is not None:
        x += s["bias"].double()
    if s["bits"] is not None:
        v = torch.arange(c["vocab"], device=DEV)
        word = s["bits"].long()[:, v // 32] & 0xFFFFFFFF
        x[(word // (2 ** (v % 32))) % 2 == 0] = -math.inf
    return {"logits": x}


def _exact_heads(x, gain, turn):
    """Norm and rotation of heads ``[..., hd]`` in float64: pairs of channels as complex
    numbers, turned by the complex numbers ``turn``."""
    y = x * gain / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS)
    half = x.shape[-1] // 2
    z = torch.complex(y[..., :half].contiguous(), y[..., half:].contiguous()) * turn
    return torch.cat((z.real, z.imag), dim=-1)


def _exact_append(c, s):
    new, past = _counts(c)
    k, v = s["k"].double(), s["v"].double()
    gq, gk = (g.double() for g in s["gains"])
    q = torch.empty(sum(new), c["heads"], c["hd"], device=DEV, dtype=torch.float64)
    at, last = 0, c["heads"] + c["kv"]
    for b, (n, p) in enumerate(zip(new, past)):
        x = s["qkv"][at:at + n].double()
        turn = torch.complex(s["cos"][p:p + n].double(), s["sin"][p:p + n].double())[:, None]
        j = torch.arange(p, p + n, device=DEV)
        ids = s["table"][b].long()[j // c["page"]]
        q[at:at + n] = _exact_heads(x[:, :c["heads"]], gq, turn)
        k[ids, :, j % c["page"]] = _exact_heads(x[:, c["heads"]:last], gk, turn)
        v[ids, :, j % c["page"]] = x[:, last:]
        at += n
    return {"q": q, "k": k, "v": v}


def _exact_rope(c, s):
    """Forward as above; backward by the formulas, the turned gradient first: with y the
    gradient turned back, r = 1/rms and u = r x, dgain = sum y u and
    dx = r (gain y - u mean(gain y u))."""
    turn = torch.complex(s["cos"][:c["t"]].double(), s["sin"][:c["t"]].double())
    x = s["qkv"].detach().double()
    cuts = [0, c["heads"], c["heads"] + c["kv"], c["heads"] + 2 * c["kv"]]
    outs, dx, dg = [], torch.empty_like(x), []
    for i in range(3):
        xi, di = x[:, :, cuts[i]:cuts[i + 1]].transpose(1, 2), s["grads"][i].double()
        if i == 2:
            outs.append(xi.contiguous())
            dx[:, :, cuts[i]:cuts[i + 1]] = di.transpose(1, 2)
            continue
        gain, half = s["gains"][i].detach().double(), c["hd"] // 2
        outs.append(_exact_heads(xi, gain, turn))
        z = torch.complex(di[..., :half].contiguous(), di[..., half:].contiguous()) * turn.conj()
        y = torch.cat((z.real, z.imag), dim=-1)
        r = 1.0 / torch.sqrt((xi * xi).sum(-1, keepdim=True) / c["hd"] + EPS)
        u = r * xi
        dg.append((y * u).sum((0, 1, 2)))
        y = y * gain
        dx[:, :, cuts[i]:cuts[i + 1]] = (r * (y - u * (y * u).mean(-1, keepdim=True))).transpose(1, 2)
    return {"q": outs[0], "k": outs[1], "v": outs[2], "dqkv": dx, "dq_gain": dg[0], "dk_gain": dg[1]}

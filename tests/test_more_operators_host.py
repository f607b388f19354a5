"""Head norms, 4-bit projections and adjusted logits without a GPU: what they refuse, and the
decoder's head norms operation by operation."""

from __future__ import annotations

import ctypes

import pytest
import torch

from switchyard import _lib
from switchyard.cache_op import paged_append
from switchyard.logits_op import adjust_logits, pack_allowed
from switchyard.model import ModelConfig, Transformer
from switchyard.quant_op import Linear4, Weight4, linear4, quantize4
from switchyard.rope_op import qk_norm_rope

OK, NULL, SHAPE, DTYPE, WORKSPACE, STRIDE = 0, -1, -2, -3, -4, -5
FAKE = 0x1000  # never dereferenced: every call below fails validation first
BF, F = _lib.SY_BF16, _lib.SY_F32


def _norm(fn="sy_qk_norm_rope", strides=None, **kw):
    a = dict(qkv=FAKE, q_gain=FAKE, k_gain=FAKE, cos=FAKE, sin=FAKE, q=FAKE, k=FAKE, v=FAKE, dqkv=FAKE, dgq=FAKE, dgk=FAKE,
             ws=FAKE, ws_bytes=1 << 40, n_tok=12, seq=6, heads=4, kv=2, hd=64, dtype=BF, gains=BF)
    a.update(kw)
    lib, sizes = _lib.lib(), (a["n_tok"], a["seq"], a["heads"], a["kv"], a["hd"], a["dtype"], a["gains"], 1e-6, None)
    head = (a["qkv"], a["q_gain"], a["k_gain"], a["cos"], a["sin"], a["q"], a["k"], a["v"])
    if fn == "sy_qk_norm_rope":
        return lib.sy_qk_norm_rope(*head, *sizes)
    s = (ctypes.c_int64 * 9)(*(strides or [768, 64, 128] * 3))
    return lib.sy_qk_norm_rope_bwd(*head, s, a["dqkv"], a["dgq"], a["dgk"], a["ws"], a["ws_bytes"], *sizes)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=5), DTYPE), (dict(gains=_lib.SY_F16), DTYPE), (dict(n_tok=-6), SHAPE), (dict(n_tok=13), SHAPE),
    (dict(seq=0), SHAPE), (dict(heads=0), SHAPE), (dict(kv=0), SHAPE), (dict(heads=1 << 16), SHAPE), (dict(hd=60), SHAPE),
    (dict(hd=0), SHAPE), (dict(hd=264), SHAPE), (dict(qkv=None), NULL), (dict(q_gain=None), NULL), (dict(k_gain=None), NULL),
    (dict(cos=None), NULL), (dict(sin=None), NULL), (dict(v=None), NULL), (dict(qkv=FAKE + 8), SHAPE), (dict(k=FAKE + 2), SHAPE)])
def test_a_bad_head_norm_is_refused(change, code):
    assert _norm(**change) == code
    assert _norm("sy_qk_norm_rope_bwd", **change) == code


def test_other_bad_head_norms_are_refused():
    bwd = "sy_qk_norm_rope_bwd"
    for name in ("dqkv", "dgq", "dgk"):
        assert _norm(bwd, **{name: None}) == NULL
    assert _norm(bwd, dqkv=FAKE + 4) == SHAPE
    assert _norm(bwd, strides=[768, 64, 128] * 2 + [768, 60, 128]) == STRIDE
    assert _norm(bwd, strides=[-768, 64, 128] * 3) == STRIDE
    assert _norm(bwd, ws=None) == WORKSPACE and _norm(bwd, ws_bytes=8) == WORKSPACE
    lib = _lib.lib()
    assert lib.sy_qk_norm_rope_bwd_bytes(12, 4, 2, 64, BF) >= 2 * 64 * 4
    assert lib.sy_qk_norm_rope_bwd_bytes(12, 4, 2, 60, BF) == SHAPE and lib.sy_qk_norm_rope_bwd_bytes(12, 4, 2, 64, 9) == DTYPE
    assert lib.sy_qk_norm_rope_bwd_bytes(0, 4, 2, 64, BF) == 0
    none = dict(n_tok=0, qkv=None, q_gain=None, k_gain=None, cos=None, sin=None, q=None, k=None, v=None)
    assert _norm(**none) == OK and _norm(bwd, ws=None, **none) == OK


def test_a_bad_normalised_append_is_refused():
    lib = _lib.lib()

    def call(qkv=FAKE, tok=512, head=64, gq=FAKE, gk=FAKE, gains=BF, dtype=BF, c=None):
        c = c or _lib.Paged(FAKE, FAKE, FAKE, FAKE, None, 2 * 16 * 64, 16 * 64, 64, 4, 3, 3, 10, 4, 16, 4, 2, 64, dtype)
        return lib.sy_paged_append_norm(ctypes.byref(c), qkv, tok, head, gq, gk, gains, 1e-6, FAKE, FAKE, 8, 0, FAKE, 0, None)

    assert call(gq=None) == NULL and call(gk=None) == NULL and call(qkv=None) == NULL
    assert call(gains=_lib.SY_F16) == DTYPE and call(dtype=7) == DTYPE
    assert call(qkv=FAKE + 4) == SHAPE and call(tok=510) == STRIDE and call(head=62) == STRIDE
    assert lib.sy_paged_append_norm(None, FAKE, 512, 64, FAKE, FAKE, BF, 1e-6, FAKE, FAKE, 8, 0, FAKE, 0, None) == NULL


def _adjust(n_rows=3, vocab=100, row_stride=100, out_stride=100, dtype=BF, logits=FAKE, out=FAKE, **kw):
    how = _lib.Adjusting(1.1, 0.0, 0.0, tokens_bytes=8, **kw) if "tokens_bytes" not in kw else _lib.Adjusting(1.1, 0.0, 0.0, **kw)
    return _lib.lib().sy_adjust(logits, out, ctypes.byref(how), n_rows, vocab, row_stride, out_stride, dtype, None)


def test_bad_adjustments_are_refused():
    assert _lib.lib().sy_adjust(FAKE, FAKE, None, 3, 100, 100, 100, BF, None) == NULL
    assert _adjust(dtype=9) == DTYPE and _adjust(bias=FAKE, bias_dtype=_lib.SY_F16) == DTYPE
    assert _adjust(n_rows=-1) == SHAPE and _adjust(vocab=0) == SHAPE and _adjust(vocab=(1 << 30) + 1) == SHAPE
    assert _adjust(n_tokens=-1) == SHAPE and _adjust(tokens_bytes=2) == SHAPE and _adjust(mask_kind=3) == SHAPE
    assert _adjust(row_stride=-1) == STRIDE and _adjust(out_stride=99) == STRIDE and _adjust(mask_stride=-1) == STRIDE
    assert _adjust(bias_stride=-1) == STRIDE and _adjust(tokens_stride=-1) == STRIDE
    assert _adjust(logits=None) == NULL and _adjust(out=None) == NULL and _adjust(mask_kind=1) == NULL
    assert _adjust(n_tokens=4) == NULL
    assert _adjust(n_rows=0, logits=None, out=None) == OK


@pytest.mark.parametrize("size,dtype", [(2, BF), (4, F)])
def test_adjusted_rows_are_in_place_or_apart(size, dtype):
    for off, kw in [(1, {}), (299, {}), (-299, {}), (100, {}), (0, dict(out_stride=101)), (0, dict(row_stride=0)),
                    (10, dict(n_rows=1)), (99, dict(row_stride=250, out_stride=250)),
                    (151, dict(row_stride=250, out_stride=250)), (350, dict(row_stride=0, out_stride=200, logits=FAKE + 500 * size))]:
        assert _adjust(out=FAKE + size * off, dtype=dtype, **kw) == STRIDE, (off, kw)


def test_bad_4_bit_weights_are_refused():
    lib = _lib.lib()

    def product(x=FAKE, stride=64, tiles=FAKE, scales=FAKE, zeros=None, out=FAKE, m=3, n=16, k=64, group=32, dtype=BF):
        return lib.sy_linear4(x, stride, tiles, scales, zeros, out, m, n, k, group, dtype, None)

    def pack(codes=FAKE, scales=FAKE, zeros=None, tiles=FAKE, to=FAKE, zeros_to=None, n=16, k=64, group=32, dtype=BF):
        return lib.sy_pack4(codes, scales, zeros, tiles, to, zeros_to, n, k, group, dtype, None)

    def quantize(w=FAKE, stride=64, codes=FAKE, scales=FAKE, n=16, k=64, group=32, dtype=BF):
        return lib.sy_quantize4(w, stride, codes, scales, None, n, k, group, dtype, None)

    for fn in (product, pack, quantize):
        assert fn(dtype=4) == DTYPE
        for bad in (dict(n=0), dict(k=0), dict(n=(1 << 24) + 1), dict(k=(1 << 24) + 1), dict(group=16), dict(group=48)):
            assert fn(**bad) == SHAPE
    assert product(m=-1) == SHAPE and product(m=1 << 31) == SHAPE and product(stride=-1) == STRIDE
    assert product(tiles=FAKE + 4) == SHAPE and product(scales=FAKE + 2) == SHAPE and product(zeros=FAKE + 1) == SHAPE
    assert product(x=None) == NULL and product(tiles=None) == NULL and product(scales=None) == NULL and product(out=None) == NULL
    assert product(m=0, x=None, tiles=None, scales=None, out=None) == OK
    assert pack(codes=None) == NULL and pack(scales=None) == NULL and pack(tiles=None) == NULL and pack(to=None) == NULL
    assert pack(zeros=FAKE) == NULL and pack(zeros_to=FAKE) == NULL and pack(tiles=FAKE + 8) == SHAPE
    assert quantize(w=None) == NULL and quantize(codes=None) == NULL and quantize(scales=None) == NULL
    assert quantize(stride=-1) == STRIDE


def test_bad_tensors_are_refused():
    t = torch.zeros
    with pytest.raises(ValueError, match="qkv must be"):
        qk_norm_rope(t(2, 3, 8), t(8), t(8), t(3, 4), t(3, 4))
    with pytest.raises(ValueError, match="kv_heads says"):
        qk_norm_rope(t(1, 2, 4, 8), t(8), t(8), t(3, 4), t(3, 4))
    with pytest.raises(ValueError, match="no queries"):
        qk_norm_rope(t(1, 2, 4, 8), t(8), t(8), t(3, 4), t(3, 4), kv_heads=2)
    with pytest.raises(ValueError, match="multiple of 8"):
        qk_norm_rope(t(1, 2, 3, 20), t(20), t(20), t(3, 10), t(3, 10))
    with pytest.raises(ValueError, match="dtype"):
        qk_norm_rope(t(1, 2, 3, 8).double(), t(8), t(8), t(3, 4), t(3, 4))
    with pytest.raises(ValueError, match="CUDA"):
        qk_norm_rope(t(1, 2, 3, 8), t(8), t(8), t(3, 4), t(3, 4))
    with pytest.raises(ValueError, match="CUDA"):
        adjust_logits(t(2, 8))
    with pytest.raises(ValueError, match=r"\[B, V\]"):
        adjust_logits(t(8))
    for bad in (0.0, -1.0, float("nan"), float("inf"), "x"):
        with pytest.raises(ValueError, match="repetition_penalty"):
            adjust_logits(t(2, 8), repetition_penalty=bad)
    with pytest.raises(ValueError, match="presence_penalty"):
        adjust_logits(t(2, 8), presence_penalty=float("nan"))
    with pytest.raises(ValueError, match="CUDA"):
        quantize4(t(16, 64))
    with pytest.raises(ValueError, match="group"):
        quantize4(t(16, 64), 48)
    with pytest.raises(ValueError, match=r"\[N, K\]"):
        quantize4(t(64))
    codes, scales = t(16, 32, dtype=torch.uint8), t(16, 2)
    for kw in (dict(in_features=66, group=32), dict(in_features=64, group=64), dict(in_features=64, group=33)):
        with pytest.raises(ValueError):
            Weight4.from_codes(codes, scales, **kw)
    with pytest.raises(ValueError, match="zeros"):
        Weight4.from_codes(codes, scales, t(16, 2), in_features=64, group=32)
    with pytest.raises(ValueError, match="uint8"):
        Weight4.from_codes(codes.int(), scales, in_features=64, group=32)
    with pytest.raises(ValueError, match="CUDA"):
        Weight4.from_codes(codes, scales, in_features=64, group=32)
    w = Weight4(t(1, 1, 64, 4, dtype=torch.int32), t(1, 1, 16, 4), None, 16, 64, 32)
    for x in (t(3, 63), t(3, 64).bfloat16(), t(3, 64)):
        with pytest.raises(ValueError):
            linear4(x, w)
    with pytest.raises(ValueError, match="tiles"):
        Weight4(t(1, 2, 64, 4, dtype=torch.int32), t(1, 1, 16, 4), None, 16, 64, 32)
    with pytest.raises(ValueError, match="scales"):
        Weight4(t(1, 1, 64, 4, dtype=torch.int32), t(1, 1, 16, 2), None, 16, 64, 32)
    with pytest.raises(ValueError, match="bias"):
        Linear4.from_linear(torch.nn.Linear(8, 8))


def test_gains_go_together():
    k, v = torch.zeros(2, 1, 4, 8), torch.zeros(2, 1, 4, 8)
    args = (torch.zeros(1, 3, 8), torch.zeros(4, 4), torch.zeros(4, 4), k, v, torch.zeros(1, 1, dtype=torch.int32),
            torch.ones(1, dtype=torch.int32))
    with pytest.raises(ValueError):  # (no CUDA device comes first or the gains: refused either way)
        paged_append(*args, q_gain=torch.ones(8))


def test_packed_masks():
    g = torch.Generator().manual_seed(0)
    for v in (1, 31, 32, 33, 100):
        keep = torch.rand(3, v, generator=g) < 0.5
        words = pack_allowed(keep)
        assert words.dtype == torch.int32 and words.shape == (3, -(-v // 32))
        bits = (words[:, :, None] >> torch.arange(32, dtype=torch.int32)) & 1
        assert torch.equal(bits.flatten(1)[:, :v].bool(), keep) and (bits.flatten(1)[:, v:] == 0).all()


def test_the_decoder_normalises_heads_on_the_cpu():
    torch.manual_seed(0)
    base = dict(vocab_size=50, d_model=32, n_layers=2, n_heads=2, d_ff=48, n_blocks=2, max_seq_len=16)
    plain, m = Transformer(ModelConfig(**base)), None
    torch.manual_seed(0)
    m = Transformer(ModelConfig(**base, qk_norm=True))
    assert all(torch.equal(p, dict(m.named_parameters())[n]) for n, p in plain.named_parameters())
    extra = set(dict(m.named_parameters())) - set(dict(plain.named_parameters()))
    assert extra == {f"layers.{i}.attn.{x}_norm.weight" for i in range(2) for x in "qk"}
    idx = torch.randint(0, 50, (2, 9))
    _, loss = m(idx, idx)
    loss.backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
    # A gain on one side is a gain on the other: scores see their product.
    with torch.no_grad():
        a = m.layers[0].attn
        want = m(idx)
        a.q_norm.weight.mul_(4.0)
        a.k_norm.weight.mul_(0.25)
        assert (m(idx) - want).abs().max() <= 1e-5 and (plain(idx) - want).abs().max() > 1e-4


def test_no_kv_heads_are_refused():
    with pytest.raises(ValueError, match="no queries"):
        qk_norm_rope(torch.zeros(1, 2, 6, 8), torch.ones(8), torch.ones(8), torch.zeros(3, 4), torch.zeros(3, 4), kv_heads=0)


def test_head_norms_of_another_type_than_the_projections_on_the_cpu():
    torch.manual_seed(0)
    cfg = ModelConfig(vocab_size=50, d_model=32, n_layers=2, n_heads=2, d_ff=48, n_blocks=2, max_seq_len=16, qk_norm=True)
    m = Transformer(cfg).bfloat16()
    idx = torch.randint(0, 50, (2, 9))
    want = m(idx)
    for layer in m.layers:
        layer.attn.q_norm.float()
        layer.attn.k_norm.float()
    got, loss = m(idx, idx)
    loss.backward()
    assert got.dtype == want.dtype and m.layers[0].attn.q_norm.weight.grad.dtype == torch.float32
    # The gains are one: the norms round less, by bf16's 2^-8 a few times a layer.
    assert (got - want).abs().max() <= 2.0**-4 * want.abs().max()

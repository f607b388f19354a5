"""Generation through normalised heads, 4-bit projections and adjusted logits together: the
decoder's own paths against its forward and against the operators one by one. fp32 models,
where two evaluations differ by the order of fp32 sums: logits of size ~1 to 1e-4."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a HIP device", allow_module_level=True)

from switchyard import _lib  # noqa: E402
from switchyard.logits_op import pack_allowed  # noqa: E402
from switchyard.model import DecodeState, ModelConfig, RMSNorm, Transformer  # noqa: E402
from switchyard.quant_op import Linear4  # noqa: E402
from switchyard.sample_op import sample_tokens  # noqa: E402


def _model(dtype=torch.float32, **kw):
    base = dict(vocab_size=300, d_model=128, n_layers=2, n_heads=2, d_ff=256, n_blocks=2, max_seq_len=128,
                residual="switchyard", qk_norm=True)
    torch.manual_seed(0)
    m = Transformer(ModelConfig(**{**base, **kw})).cuda()
    with torch.no_grad():
        for name, p in m.named_parameters():
            if name.startswith("attn_res") and name.endswith(".w"):
                p.normal_(std=0.3)
            elif "_norm" in name and "attn." in name:
                p.normal_(1.0, 0.3)
            elif p.ndim == 2:
                p.mul_(4.0)
    return m.to(dtype).eval()


def _tokens(*shape, seed=1):
    return torch.randint(0, 300, shape, generator=torch.Generator().manual_seed(seed)).cuda()


def _close(got, want):
    assert (got - want).abs().max().item() <= 1e-4 * max(1.0, want.abs().max().item())


@pytest.mark.parametrize("residual", ["standard", "switchyard"])
def test_pieces_of_a_sequence_give_the_forwards_logits(residual):
    m = _model(residual=residual)
    idx = _tokens(3, 90)
    want = m(idx).detach()
    state = DecodeState(m, 3, 100, page=16)
    at = 0
    for n in (40, 1, 1, 17, 31):
        got = m.decode(idx[:, at:at + n], state)
        at += n
        _close(got, want[:, at - 1])


def test_training_agrees_with_the_plain_operations(monkeypatch):
    m = _model().train()
    idx = _tokens(2, 33)

    def step():
        m.zero_grad()
        logits, loss = m(idx, idx)
        loss.backward()
        return logits.detach(), {n: p.grad.clone() for n, p in m.named_parameters()}

    calls = []
    real = _lib.native()

    class Spy:
        def __getattr__(self, name):
            calls.append(name)
            return getattr(real, name)

    monkeypatch.setattr(_lib, "native", lambda: Spy())
    got, grads = step()
    assert calls.count("qk_norm_rope") == 2 and "rope_qkv" not in calls
    monkeypatch.setattr(_lib, "native", lambda: real)
    monkeypatch.setattr(_lib, "ordinary", lambda *t: False)
    want, want_grads = step()
    _close(got, want)
    for n, g in grads.items():
        assert (g - want_grads[n]).norm() <= 1e-4 * want_grads[n].norm() + 1e-7, n


def test_norms_that_are_more_than_their_kernel():
    class Scaled(RMSNorm):
        def forward(self, x):
            return 2.0 * super().forward(x)

    m = _model()
    for layer in m.layers:
        other = Scaled(64, 1e-6).cuda()
        other.weight.data.copy_(layer.attn.q_norm.weight / 2)
        layer.attn.q_norm = other
    plain = _model()
    idx = _tokens(2, 20)
    want = plain(idx).detach()
    _close(m(idx).detach(), want)
    _close(m.decode(idx, DecodeState(m, 2, 30, page=16)), want[:, -1])
    assert plain.layers[0].attn.head_gains() is not None and m.layers[0].attn.head_gains() is None


@pytest.mark.parametrize("symmetric,group", [(True, 64), (False, 32)])
def test_a_quantized_decoder(symmetric, group):
    m, ref = _model(), _model()
    m.quantize4_(group, symmetric=symmetric)
    swapped = [n for n, x in m.named_modules() if isinstance(x, Linear4)]
    assert len(swapped) == 9 and "lm_head" in swapped and isinstance(m.embed, torch.nn.Embedding)
    ref.lm_head.weight = torch.nn.Parameter(ref.lm_head.weight.detach().clone())  # (it was the embedding's)
    with torch.no_grad():
        for n in swapped:
            ref.get_submodule(n).weight.copy_(m.get_submodule(n).weight4.dequantize())
        assert m.quantize4_(group) is m  # nothing is left to do
        idx = _tokens(3, 70)
        want = ref(idx)
        _close(m(idx), want)
        state = DecodeState(m, 3, 80, page=16)
        _close(m.decode(idx[:, :69], state), want[:, 68])
        _close(m.decode(idx[:, 69:], state), want[:, 69])
    with pytest.raises(RuntimeError, match="no backward"):
        m(idx)


def _plain_adjust(logits, history, n_prompt, r, p, f, bias, keep):
    y = logits.double().clone()
    for i, h in enumerate(history):
        for t in set(h):
            z = y[i, t].item()
            z = z / r if z > 0 else z * r
            said = h[n_prompt[i]:].count(t)
            y[i, t] = z - (f * said + p if said else 0.0)
    if bias is not None:
        y = y + bias.double()
    if keep is not None:
        y = y.masked_fill(~keep, -math.inf)
    return y.float()


@pytest.mark.parametrize("prefix", [0, 11])
def test_generation_under_control(prefix):
    """Token by token the same as the forward over everything so far, adjusted in float64: where
    the two best candidates are further apart than the two evaluations."""
    m = _model().quantize4_(64)
    rows = [_tokens(n, seed=10 + n) for n in (5, 17, 1)]
    pre = _tokens(prefix, seed=3) if prefix else None
    bias = torch.zeros(300, device="cuda")
    bias[7], bias[100:120] = 3.0, -2.0
    keep = torch.rand(300, generator=torch.Generator().manual_seed(5)) < 0.7
    steps = []

    def allowed(so_far):
        steps.append(so_far.shape[1])
        return None if so_far.shape[1] % 3 == 2 else pack_allowed(keep).cuda()

    got = m.generate(rows, 9, temperature=0.0, repetition_penalty=1.7, presence_penalty=0.5, frequency_penalty=0.25,
                     bias=bias, allowed=allowed, prefix=pre, page=16)
    assert steps == list(range(9)) and got.shape == (3, 9)
    history = [([] if pre is None else pre.tolist()) + r.tolist() for r in rows]
    n_prompt = [len(h) for h in history]
    sure = 0
    for i in range(9):
        logits = torch.stack([_logits(m, h) for h in history])
        want = _plain_adjust(logits.cpu(), history, n_prompt, 1.7, 0.5, 0.25, bias.cpu(), None if i % 3 == 2 else keep)
        top = want.topk(2, -1).values
        for b in range(3):
            if top[b, 0] - top[b, 1] > 1e-3:
                sure += 1
                assert got[b, i].item() == want[b].argmax().item()
            history[b].append(got[b, i].item())
    assert sure >= 20


@torch.no_grad()
def _logits(m, h):
    return m(torch.tensor([h], device="cuda"))[0, -1]


def test_per_row_penalties_and_a_mask_that_leaves_nothing():
    m = _model()
    prompts = _tokens(3, 6)
    keep = torch.ones(3, 300, dtype=torch.bool, device="cuda")
    keep[1] = False
    r = torch.tensor([1.0, 1.3, 2.0], device="cuda")
    got = m.generate(prompts, 5, temperature=0.0, repetition_penalty=r, allowed=keep)
    assert (got[1] == -1).all() and (got[[0, 2]] >= 0).all()
    plain = m.generate(prompts, 5, temperature=0.0)
    assert torch.equal(got[0], plain[0])
    assert torch.equal(m.generate(prompts, 5, temperature=0.0, repetition_penalty=1.0, presence_penalty=0.0), plain)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sixteen_bit_generation_runs_in_every_part(dtype):
    m = _model(dtype).quantize4_(128, symmetric=False)
    with torch.autocast("cuda", enabled=False):
        got = m.generate(_tokens(2, 30), 8, temperature=0.8, top_k=20, repetition_penalty=1.2,
                         u=torch.rand(8, 2, generator=torch.Generator().manual_seed(2)))
    assert got.shape == (2, 8) and ((got >= 0) & (got < 300)).all()


def test_a_quantized_decoder_under_autocast():
    m = _model().quantize4_(64)
    with torch.autocast("cuda", dtype=torch.bfloat16), torch.no_grad():
        state = DecodeState(m, 2, 40, page=16)
        assert state.k.dtype == torch.bfloat16
        idx = _tokens(2, 20)
        got = m.decode(idx, state)
        want = m(idx)[:, -1]
        assert got.dtype == want.dtype and (got - want).float().norm() <= 0.03 * want.float().norm()  # bf16 all the way
        assert m.generate(idx, 3, repetition_penalty=1.2).shape == (2, 3)


def test_a_captured_step_of_all_of_them():
    """Norm, rotation and append, attention, projections, penalties and sampling as one graph,
    replayed for tokens and lengths that change on the device."""
    from switchyard.logits_op import adjust_logits

    m = _model().quantize4_(64)
    idx = _tokens(2, 20)
    tokens = torch.full((2, 40), -1, dtype=torch.int64, device="cuda")
    tokens[:, :20] = idx
    n, prompts = (torch.full((2,), 20, dtype=torch.int32, device="cuda") for _ in range(2))
    u = torch.rand(2, generator=torch.Generator().manual_seed(4)).cuda()

    def step(state, last):
        logits = m.decode(last[:, None], state)
        y = adjust_logits(logits, tokens, lengths=n, prompt_lengths=prompts, repetition_penalty=1.5, frequency_penalty=0.5)
        return y, sample_tokens(y, u, temperature=0.9, top_k=40)

    def fresh():
        state = DecodeState(m, 2, 60, page=16)
        m.decode(idx[:, :-1], state)
        return state

    state, last = fresh(), idx[:, -1].clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(fresh(), last)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, drawn = step(state, last)
    state.lengths.fill_(19)  # (the capture has not run, but counted nothing either way)
    twin = fresh()
    for i in range(4):
        g.replay()
        torch.cuda.synchronize()
        want_y, want = step(twin, last.clone())
        assert torch.equal(drawn, want) and torch.equal(y, want_y)
        last.copy_(drawn)
        tokens[:, 20 + i] = drawn
        n += 1


def test_a_decoder_is_quantized_whole_or_not_at_all():
    m = _model()
    m.layers[1].mlp.down.register_forward_hook(lambda mod, a, y: 2 * y)
    with pytest.raises(ValueError, match="has no 4-bit form"):
        m.quantize4_()
    assert not any(isinstance(x, Linear4) for x in m.modules())


def test_gains_of_another_type_than_the_projections():
    """Every rounding is fp16's, 2^-11; some twenty a layer and as many a logit's terms, in two
    evaluations: under 2^-5 of the largest logit."""
    m = _model(dtype=torch.bfloat16, residual="standard")
    idx = _tokens(2, 20)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.float16):
        want = m(idx).float()
        got = m.decode(idx, DecodeState(m, 2, 30, page=16)).float()
    assert (got - want[:, -1]).abs().max() <= 2.0**-5 * want.abs().max()
    mixed = _model(dtype=torch.bfloat16)
    for layer in mixed.layers:
        layer.attn.q_norm.float()  # next to a k_norm in bf16
    with torch.no_grad():
        want = mixed(idx).float()
        got = mixed.decode(idx, DecodeState(mixed, 2, 30, page=16)).float()
    assert (got - want[:, -1]).abs().max() <= 2.0**-2 * want.abs().max()  # bf16's: 2^-8

"""Generation with the decoder: prompts, single tokens and a shared prefix through the paged
cache against the forward over the whole sequence. The model is fp32, where the two differ
by the order of fp32 sums: logits of size ~1 through two layers to 1e-4."""

from __future__ import annotations

import pytest
import torch

from switchyard.model import DecodeState, ModelConfig, Transformer

HAS_GPU = torch.cuda.is_available()
gpu = pytest.mark.gpu
needs = pytest.mark.skipif(not HAS_GPU, reason="needs a HIP device")


def _model(residual="switchyard", dev="cuda", **kw):
    base = dict(vocab_size=300, d_model=128, n_layers=2, n_heads=2, d_ff=256, n_blocks=2, max_seq_len=128,
                residual=residual)
    torch.manual_seed(0)
    m = Transformer(ModelConfig(**{**base, **kw})).to(dev)
    with torch.no_grad():
        for name, p in m.named_parameters():
            if name.startswith("attn_res") and name.endswith(".w"):
                p.normal_(std=0.3)
            elif p.ndim == 2:
                p.mul_(4.0)
    return m.eval()


def _tokens(*shape, seed=1):
    return torch.randint(0, 300, shape, generator=torch.Generator().manual_seed(seed))


def _close(got, want):
    assert (got - want).abs().max().item() <= 1e-4 * max(1.0, want.abs().max().item())


@gpu
@needs
@pytest.mark.parametrize("residual,sources", [("standard", "arena"), ("switchyard", "arena"), ("switchyard", "table"),
                                              ("switchyard", "stack"), ("attnres", "arena")])
def test_pieces_of_a_sequence_give_the_forwards_logits(residual, sources):
    m = _model(residual, sources=sources)
    idx = _tokens(3, 90).cuda()
    want = m(idx).detach()
    state = DecodeState(m, 3, 100, page=16)
    at = 0
    for n in (40, 1, 1, 17, 31):
        got = m.decode(idx[:, at:at + n], state)
        at += n
        _close(got, want[:, at - 1])
    assert state.lengths.tolist() == [90, 90, 90]
    state.reset()
    _close(m.decode(idx[:, :90], state), want[:, 89])


@gpu
@needs
def test_ragged_prompts_and_a_shared_prefix():
    m = _model()
    lens, prefix = [5, 33, 1, 20], _tokens(37, seed=2).cuda()
    rows = [_tokens(n, seed=10 + n).cuda() for n in lens]
    want = torch.stack([m(torch.cat((prefix, r))[None])[0, -1] for r in rows]).detach()
    state = DecodeState(m, 4, 40, page=16, prefix_len=37)
    with pytest.raises(ValueError, match="prefix"):
        m.decode(rows[0][None].expand(4, -1), state)
    last = m.decode(prefix, state, to_prefix=True)
    _close(last, m(prefix[None])[:, -1].detach())
    starts = torch.tensor([0, *lens]).cumsum(0).int().cuda()
    _close(m.decode(torch.cat(rows), state, starts), want)
    nxt = want.argmax(-1)
    got = m.decode(nxt[:, None], state)
    want = torch.stack([m(torch.cat((prefix, r, t[None]))[None])[0, -1] for r, t in zip(rows, nxt)]).detach()
    _close(got, want)


@gpu
@needs
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_generation(dtype):
    """Greedy tokens are the largest logits of the forward over what came before (in bf16 of
    nearly the largest), and the same numbers give the same tokens."""
    m = _model().to(dtype)
    lens, prefix = [3, 12, 7], _tokens(20, seed=3)
    rows = [_tokens(n, seed=20 + n) for n in lens]
    out = m.generate(rows, 9, temperature=0.0, prefix=prefix)
    assert out.shape == (3, 9) and out.dtype == torch.int64
    for r, o in zip(rows, out.cpu()):
        seq = torch.cat((prefix, r, o)).cuda()[None]
        logits = m(seq)[0, 19 + r.numel():-1].float()
        chosen = logits.gather(1, o.cuda()[:, None])[:, 0]
        slack = 1e-3 if dtype == torch.float32 else 0.15 * logits.std().item()
        assert (chosen >= logits.amax(-1) - slack).all()
    u = torch.rand(6, 3, generator=torch.Generator().manual_seed(4))
    a = m.generate(torch.stack([r[:3] for r in rows]), 6, temperature=0.8, top_k=40, top_p=0.9, u=u)
    b = m.generate([r[:3] for r in rows], 6, temperature=0.8, top_k=40, top_p=0.9, u=u)
    assert torch.equal(a, b) and (a >= 0).all()
    g = torch.Generator(device="cuda").manual_seed(5)
    assert m.generate(rows, 2, generator=g, min_p=torch.full((3,), 0.01, device="cuda")).shape == (3, 2)


@gpu
@needs
def test_a_captured_token_step():
    """One token of every sequence captured into a graph: sampling, the model, the lengths."""
    from switchyard.sample_op import sample_tokens

    m = _model()
    idx = _tokens(3, 20).cuda()
    u = torch.rand(8, 3, generator=torch.Generator().manual_seed(6)).cuda()

    def run(captured):
        state = DecodeState(m, 3, 60, page=16)
        logits, r, tokens = m.decode(idx, state).clone(), torch.zeros(3, device="cuda"), []

        def step():
            t = sample_tokens(logits, r, temperature=0.7, top_p=0.9)
            logits.copy_(m.decode(t[:, None], state))
            return t

        replay = step
        if captured:
            before = logits.clone()
            step()  # warm up, then back
            state.lengths.sub_(1), logits.copy_(before)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                held = step()

            def replay():
                g.replay()
                return held
        for i in range(8):
            r.copy_(u[i])
            tokens.append(replay().clone())
            torch.cuda.synchronize()
        return torch.stack(tokens), state.lengths.tolist()

    eager, captured = run(False), run(True)
    assert torch.equal(eager[0], captured[0]) and eager[1] == captured[1] == [28] * 3


@gpu
@needs
@pytest.mark.parametrize("residual", ["standard", "switchyard"])
def test_inference_mode_and_another_stream(residual):
    m = _model(residual)
    idx, u = _tokens(2, 9), torch.rand(4, 2, generator=torch.Generator().manual_seed(3))
    want = m.generate(idx, 4, u=u, top_p=0.9)
    with torch.inference_mode():
        assert torch.equal(m.generate(idx, 4, u=u, top_p=0.9), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = m.generate(idx, 4, u=u, top_p=0.9)
    side.synchronize()
    assert torch.equal(got, want)


@gpu
@needs
def test_what_does_not_fit_is_nan():
    m = _model("standard")
    state = DecodeState(m, 2, 16, page=16)
    assert torch.isfinite(m.decode(_tokens(2, 16).cuda(), state)).all()
    assert torch.isnan(m.decode(_tokens(2, 1).cuda(), state)).all()


@gpu
@needs
def test_a_model_of_nan():
    """Rows without a logit give -1, which is no token that the model could go on from."""
    m = _model("standard")
    with torch.no_grad():
        m.lm_head.weight.fill_(float("nan"))
    assert (m.generate(_tokens(2, 5), 3) == -1).all()
    assert torch.isnan(m(_tokens(1, 4).cuda())).all()


@gpu
@needs
def test_starts_past_the_tokens():
    """The logits of a sequence that ends past the tokens are some row's, not a read behind them."""
    m = _model("standard")
    state = DecodeState(m, 2, 16, page=16)
    starts = torch.tensor([0, 3, 90], dtype=torch.int32, device="cuda")
    idx = _tokens(8).cuda()
    got = m.decode(idx, state, starts)
    _close(got[:1], m(idx[None, :3])[:, -1])


def test_refusals():
    m = _model(dev="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        DecodeState(m, 2, 16)
    with pytest.raises(ValueError, match="max_seq_len"):
        DecodeState(m, 2, 100, prefix_len=29)
    with pytest.raises(ValueError, match="at least one token"):
        DecodeState(m, 0, 16)
    with pytest.raises(ValueError, match="power of two"):
        DecodeState(m, 2, 16, page=24)
    with pytest.raises(ValueError, match="multiple of 8"):
        DecodeState(_model(dev="cpu", d_model=120, n_heads=10), 2, 16)
    with pytest.raises(ValueError, match="at least one token"):
        m.generate([torch.zeros(0, dtype=torch.long)], 3)
    with pytest.raises(ValueError, match="n_new"):
        m.generate(_tokens(2, 4), 0)


@gpu
@needs
def test_refusals_of_a_state():
    m = _model()
    state = DecodeState(m, 2, 16, prefix_len=4)
    with pytest.raises(ValueError, match=r"\[4\]"):
        m.decode(_tokens(5).cuda(), state, to_prefix=True)
    m.decode(_tokens(4).cuda(), state, to_prefix=True)
    with pytest.raises(ValueError, match=r"\[2, n\]"):
        m.decode(_tokens(3, 2).cuda(), state)
    with pytest.raises(ValueError, match="starts"):
        m.decode(_tokens(3).cuda(), state, torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match=r"u must be"):
        m.generate(_tokens(2, 4), 3, u=torch.zeros(2, 2))
    before = state.lengths.tolist()
    with pytest.raises(ValueError, match="int32"):
        m.decode(_tokens(3).cuda(), state, torch.tensor([0, 1, 3], device="cuda"))
    with torch.autocast("cuda", dtype=torch.bfloat16), pytest.raises(ValueError, match="same dtype"):
        m.decode(_tokens(2, 3).cuda(), state)
    assert state.lengths.tolist() == before  # a refused call adds nothing

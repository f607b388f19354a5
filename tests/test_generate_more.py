"""What generating with the decoder refuses and takes besides the ordinary calls."""

from __future__ import annotations

import pytest
import torch

from switchyard.model import DecodeState

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a HIP device", allow_module_level=True)

from test_generate import _close, _model, _tokens  # noqa: E402


def test_another_prefix_needs_a_reset():
    """Tokens that attended to one prefix must not go on behind another."""
    m = _model()
    first, second, idx = _tokens(7, seed=1).cuda(), _tokens(7, seed=2).cuda(), _tokens(2, 5, seed=3).cuda()
    state = DecodeState(m, 2, 16, page=16, prefix_len=7)
    m.decode(second, state, to_prefix=True)
    m.decode(first, state, to_prefix=True)  # nothing stands behind it yet
    _close(m.decode(idx, state), m(torch.cat((first.expand(2, -1), idx), 1))[:, -1].detach())
    with pytest.raises(ValueError, match="reset"):
        m.decode(second, state, to_prefix=True)
    more = _tokens(2, 1, seed=4).cuda()
    _close(m.decode(more, state), m(torch.cat((first.expand(2, -1), idx, more), 1))[:, -1].detach())
    state.reset()
    m.decode(second, state, to_prefix=True)
    _close(m.decode(idx, state), m(torch.cat((second.expand(2, -1), idx), 1))[:, -1].detach())


def test_a_prefix_that_failed_is_no_prefix():
    m = _model()
    state = DecodeState(m, 2, 16, page=16, prefix_len=7)
    m.decode(_tokens(7).cuda(), state, to_prefix=True)
    hook = m.layers[1].mlp.register_forward_pre_hook(lambda *_: (_ for _ in ()).throw(RuntimeError("stop")))
    with pytest.raises(RuntimeError, match="stop"):
        m.decode(_tokens(7, seed=2).cuda(), state, to_prefix=True)
    hook.remove()
    with pytest.raises(ValueError, match="filled first"):
        m.decode(_tokens(2, 3).cuda(), state)


@pytest.mark.parametrize("residual", ["standard", "attnres", "switchyard"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_autocast(dtype, residual):
    """fp32 weights under autocast, as the forward takes them: no further from the fp32 logits
    than twice the forward is."""
    m = _model(residual)
    idx, prefix = _tokens(3, 33).cuda(), _tokens(20, seed=2).cuda()
    seq = torch.cat((prefix.expand(3, -1), idx), 1)
    with torch.no_grad():
        exact = m(seq)[:, [-2, -1]]
        with torch.autocast("cuda", dtype=dtype):
            near = m(seq)[:, [-2, -1]]
            state = DecodeState(m, 3, 40, page=16, prefix_len=20)
            m.decode(prefix, state, to_prefix=True)
            got = torch.stack((m.decode(idx[:, :-1], state), m.decode(idx[:, -1:], state)), 1)
            assert state.k.dtype == dtype and got.dtype == near.dtype
            assert (m.generate(idx, 4, prefix=prefix) >= 0).all()
        assert (got.float() - exact).norm() <= 2 * (near.float() - exact).norm()
        with pytest.raises(ValueError, match="same dtype"):  # a state of the other setting
            m.decode(idx[:, -1:], state)

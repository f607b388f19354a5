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

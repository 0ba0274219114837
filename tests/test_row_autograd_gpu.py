"""What the channel-last row operators (HIP) do under the parts of autograd that they do not compute."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _calls():
    from graspbalance_amd import fused_rows
    x, w, b = torch.randn(2, 40, 64, device=DEV), torch.randn(64, device=DEV), torch.randn(64, device=DEV)
    m, held = torch.randn(24, 64, device=DEV), fused_rows.Fp8Weight.quantize(torch.randn(24, 64, device=DEV))
    bias = torch.randn(24, device=DEV)
    return [("dropout x", x, lambda t: fused_rows.dropout(t, 0.5, (1, 2))),
            ("dropout residual", x, lambda t: fused_rows.dropout(x, 0.5, (1, 2), residual=t)),
            ("norm x", x, lambda t: fused_rows.group_norm_act(t, 4, w, b, act="gelu")),
            ("norm weight", w, lambda t: fused_rows.group_norm_act(x, 4, t, b)),
            ("norm weight in 16 bits", w.half(), lambda t: fused_rows.group_norm_act(x, 4, t, b)),
            ("norm bias", b, lambda t: fused_rows.group_norm_act(x, 4, None, t)),
            ("norm residual", x, lambda t: fused_rows.group_norm_act(x, 4, residual=t)),
            ("product x", x, lambda t: fused_rows.fp8_linear(t, m)), ("product kept", x, lambda t: fused_rows.fp8_linear(t, held)),
            ("product weight", m, lambda t: fused_rows.fp8_linear(x, t)),
            ("product bias", bias, lambda t: fused_rows.fp8_linear(x, held, t))]


@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_is_refused(grad_mode):
    """An operand with a tangent raises; without one - also inside a level - the call gives what it always gives."""
    for name, t, call in _calls():
        want = call(t)
        with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
            assert torch.equal(call(t), want), name
            with pytest.raises(NotImplementedError):
                call(forward_ad.make_dual(t, torch.ones_like(t)))
        assert torch.equal(call(t), want), name


def test_function_transforms_are_refused():
    for name, t, call in _calls():
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(call, (t,), (torch.ones_like(t),))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda v: call(v).sum())(t)
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(torch.stack([t, t]))

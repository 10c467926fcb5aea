"""Forward-mode derivatives through the step operators raise: there are none, and
a dropped tangent would be a wrong derivative.  On meta tensors, which run the
operators' autograd code without a device."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from conftest import load_pkg


def _calls():
    load_pkg()
    ops = torch.ops.gmdn
    x, w = torch.zeros(3, 8, device="meta"), torch.ones(8, device="meta")
    t = torch.zeros(3, dtype=torch.int64, device="meta")
    return {
        "x": (x, lambda d: ops.norm_fwd(d, None, w, None, 1e-5, True, True)[0]),
        "residual": (x, lambda d: ops.norm_fwd(x, d, w, None, 1e-5, False, True)[0]),
        "weight": (w, lambda d: ops.norm_fwd(x, None, d, None, 1e-5, True, True)[0]),
        "bias": (w, lambda d: ops.norm_fwd(x, None, w, d, 1e-5, True, True)[0]),
        "logits": (x, lambda d: ops.token_logprobs_fwd(d, t, True, 2, -100)[0]),
    }


@pytest.mark.parametrize("which", ["x", "residual", "weight", "bias", "logits"])
@pytest.mark.parametrize("grad", [False, True])
def test_a_tangent_is_refused(which, grad):
    p, call = _calls()[which]
    with torch.set_grad_enabled(grad), fw.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            call(fw.make_dual(p, torch.ones_like(p)))
        assert fw.unpack_dual(call(p)).tangent is None      # none given, none due
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(call, (p,), (torch.ones_like(p),))


@pytest.mark.parametrize("which", ["x", "logits"])
def test_a_tangent_on_a_cotangent_is_refused(which):
    """Forward over reverse: the gradient is linear in the cotangent."""
    p, call = _calls()[which]
    p = p.clone().requires_grad_(True)
    y = call(p)
    with fw.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.autograd.grad(y, p, fw.make_dual(torch.ones_like(y), torch.ones_like(y)))
    (g,) = torch.autograd.grad(call(p), p, torch.ones_like(y))
    assert g.shape == p.shape

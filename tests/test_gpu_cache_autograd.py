"""Autograd around the attention cache's operators on the GPU."""

import pytest
import torch
import torch.autograd.forward_ad as fw

pytestmark = pytest.mark.gpu


def _rotary_args():
    from spark_b200.rotary import rotary_frequencies

    g = torch.Generator(device="cuda").manual_seed(2)
    x, t = (torch.randn(2, 3, 4, 64, generator=g, device="cuda") for _ in range(2))
    return x, t, torch.randint(0, 90_000, (2, 3), generator=g, device="cuda"), rotary_frequencies(32)


@pytest.mark.parametrize("how", [dict(), dict(interleaved=False, offset=8, inverse=True, amplitude=1.3)])
def test_rotary_forward_mode(cuda_device, how):
    """The tangent is the rotated tangent, bit for bit, alone, under no_grad, beside a
    backward graph and through torch.func.jvp; the backward pass of a tangent too."""
    from spark_b200.rotary import rotary

    x, t, pos, f = _rotary_args()
    want, turned = rotary(x, pos, f, **how), rotary(t, pos, f, **how)
    with fw.dual_level():
        for leaf in (x, x.clone().requires_grad_()):
            y, dy = fw.unpack_dual(rotary(fw.make_dual(leaf, t), pos, f, **how))
            assert torch.equal(y, want) and torch.equal(dy, turned) and y.requires_grad == leaf.requires_grad
        gx, = torch.autograd.grad(y, leaf, t)
        back = dict(how, inverse=not how.get("inverse", False))
        assert torch.equal(gx, rotary(t, pos, f, **back))
        with torch.no_grad():
            assert torch.equal(fw.unpack_dual(rotary(fw.make_dual(x, t), pos, f, **how)).tangent, turned)
    y, dy = torch.func.jvp(lambda v: rotary(v, pos, f, **how), (x,), (t,))
    assert torch.equal(y, want) and torch.equal(dy, turned)
    double = x.clone().requires_grad_()
    g = t.clone().requires_grad_()
    gx, = torch.autograd.grad(rotary(double, pos, f, **how), double, g, create_graph=True)
    gg, = torch.autograd.grad(gx, g, x)
    assert torch.equal(gg, want)

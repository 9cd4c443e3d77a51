"""How the attention cache's operators answer torch's autograd, on meta tensors: what
is shared by every device lies above the kernels."""

import pytest
import torch
import torch.autograd.forward_ad as fw

META = torch.device("meta")


@pytest.fixture(scope="module")
def dsv4():
    from spark_b200 import ops

    return ops.load()


def _rotary_args(requires_grad=False):
    return (torch.empty(2, 3, 4, 128, device=META, requires_grad=requires_grad),
            torch.empty(2, 3, dtype=torch.int64, device=META), torch.empty(32, dtype=torch.float64, device=META))


def test_rotary_has_a_tangent(dsv4):
    x, pos, f = _rotary_args()
    with fw.dual_level():
        y = dsv4.rotary(fw.make_dual(x, torch.empty_like(x)), pos, f)
        primal, tangent = fw.unpack_dual(y)
        assert tangent is not None and tangent.shape == primal.shape == x.shape and not y.requires_grad
        x.requires_grad_()
        y = dsv4.rotary(fw.make_dual(x, torch.empty_like(x, requires_grad=True)), pos, f)
        assert fw.unpack_dual(y).tangent.requires_grad and fw.unpack_dual(y).primal.requires_grad
        assert fw.unpack_dual(dsv4.rotary(x, pos, f)).tangent is None
    y, t = torch.func.jvp(lambda v: dsv4.rotary(v, pos, f), (x.detach(),), (torch.empty_like(x).detach(),))
    assert y.shape == t.shape == x.shape

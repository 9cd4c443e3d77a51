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


def test_operators_without_a_gradient(cuda_device):
    """paged_attn, append and rotary_ refuse tensors that require a gradient, take them
    under no_grad and in inference mode, and give new versions to what they write."""
    from spark_b200 import kv_cache
    from spark_b200.rotary import rotary, rotary_

    x, t, pos, f = _rotary_args()
    pages = torch.randn(4, 16, 128, device="cuda").half()
    table = torch.tensor([[0, 2], [3, 1]], dtype=torch.int32, device="cuda")
    rows = torch.randn(2, 128, device="cuda").half()
    q = torch.randn(2, 8, 128, device="cuda").half()
    sink = torch.zeros(8, device="cuda")
    at = torch.tensor([20, 5], device="cuda")
    need = lambda v: v.clone().requires_grad_()  # noqa: E731
    for call in (lambda: rotary_(need(x), pos, f), lambda: rotary(x, pos, need(f)),
                 lambda: kv_cache.append(pages, need(rows), table, None, at),
                 lambda: kv_cache.append(need(pages), rows, table, None, at),
                 lambda: kv_cache.paged_attn(need(q), pages, table, None, at, sink, 0.1),
                 lambda: kv_cache.paged_attn(q, need(pages), table, None, at, sink, 0.1),
                 lambda: kv_cache.paged_attn(q, pages, table, None, at, need(sink), 0.1)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
        with torch.no_grad():
            call()
        with torch.inference_mode():
            call()
    want = kv_cache.paged_attn(q, pages, table, None, at, sink, 0.1)
    with torch.no_grad():
        assert torch.equal(kv_cache.paged_attn(need(q), pages, table, None, at, need(sink), 0.1), want)
    w = need(x)
    z = (x * w).sum()
    version = x._version
    rotary_(x, pos, f)
    assert x._version == version + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_a_cache_made_in_inference_mode(cuda_device):
    """It is written and read outside of inference mode as well."""
    from spark_b200 import _lib
    from spark_b200.kv_cache import PagedKVCache

    with torch.inference_mode():
        cache = PagedKVCache(2, 8, 3, 64, page_size=16, dim=128)
    ids, pos = torch.arange(2, device="cuda").int(), torch.tensor([3, 17], device="cuda").int()
    rows = torch.randn(2, 128, device="cuda").bfloat16()
    cache.reserve(ids, pos + 1)
    cache.append(1, rows, ids, pos)
    cache.fork(ids[1:], ids[1:] + 1)
    q = torch.randn(1, 4, 128, device="cuda").bfloat16()
    out = cache.attend(1, q, ids[1:] + 1, pos[1:], None, 0.1, window=1)
    assert torch.equal(out[0], rows[1:].expand(4, 128))               # the only visible row, copied by the fork
    cache.copy_pages(ids[:1], ids[:1] + 7)
    cache.free(ids[:1])
    assert cache.compact().tolist()[1:4] == [1, 2, 0]
    torch.cuda.synchronize()
    _lib.raise_on_device_error()

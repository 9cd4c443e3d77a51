"""Index tensors of the attention cache's operators on the GPU: the shapes they may
have, and that other orders of as many elements are refused."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_positions_and_ids_of_another_shape(cuda_device):
    from spark_b200 import kv_cache
    from spark_b200.rotary import rotary, rotary_, rotary_frequencies

    f = rotary_frequencies(64)
    x = torch.randn(2, 3, 4, 128, device="cuda")
    pos = torch.randint(0, 1000, (2, 3), device="cuda")
    want = rotary(x, pos, f)
    for good in (pos.flatten(), pos[:, None], pos[None], pos.t().contiguous().t(), pos.int()):
        assert torch.equal(rotary(x, good, f), want) and torch.equal(rotary_(x.clone(), good, f), want)
    for bad in (pos.t(), pos.t().contiguous(), pos.view(3, 2), pos[:, :1], pos[:1].expand(2, 3)[:, :2]):
        for op in (rotary, rotary_):
            for mode in (torch.enable_grad, torch.inference_mode):
                with mode(), pytest.raises(RuntimeError, match="positions"):
                    op(x, bad, f)
    pages = torch.randn(9, 16, 128, device="cuda").half()
    table = torch.randperm(8, device="cuda").int().view(4, 2)
    q, rows = torch.randn(6, 4, 128, device="cuda").half(), torch.randn(6, 128, device="cuda").half()
    at, seq = torch.tensor([3, 9, 31, 0, 17, 8], device="cuda"), torch.tensor([0, 1, 2, 3, 1, 0], device="cuda")
    sink = torch.randn(4, device="cuda")
    kv_cache.append(pages, rows, table, seq[:, None], at[None])
    out = kv_cache.paged_attn(q, pages, table, seq, at, sink, 0.1)
    assert torch.equal(kv_cache.paged_attn(q, pages, table, seq[None], at[:, None], sink[None], 0.1), out)
    for call in (lambda: kv_cache.append(pages, rows, table, seq, at.view(2, 3)),
                 lambda: kv_cache.append(pages, rows, table, seq.view(3, 2), at),
                 lambda: kv_cache.paged_attn(q, pages, table, seq, at.view(2, 3), sink, 0.1),
                 lambda: kv_cache.paged_attn(q, pages, table, seq.view(3, 2), at, sink, 0.1),
                 lambda: kv_cache.paged_attn(q, pages, table, seq, at, sink.view(2, 2), 0.1)):
        with pytest.raises(RuntimeError, match="must be of shape"):
            call()


def test_layers_that_overlap(cuda_device):
    """Layers apart by less than their pages, or pages by less than their layers, would be
    copied onto one another; nested layouts of either order are taken."""
    from spark_b200 import _lib, kv_cache

    base = torch.randn(4096, device="cuda").half()
    src, dst = (torch.tensor([v], dtype=torch.int32, device="cuda") for v in (0, 2))
    page = 4 * 8
    for strides in ((96, 32), (160, 40), (32, 96), (48, 160), (1000, 32)):      # three layers, three pages
        v = base.clone().as_strided((3, 3, 4, 8), (*strides, 8, 1))
        want = v.clone()
        want[:, 2] = want[:, 0]
        kv_cache.copy_pages(v, src, dst)
        torch.cuda.synchronize()
        _lib.raise_on_device_error()
        assert torch.equal(v, want)
    for strides in ((0, 32), (88, 32), (32, 64), (24, 96), (40, 104), (16, 32), (32, 0), (104, 40), (64, 32)):
        v = base.as_strided((3, 3, 4, 8), (*strides, 8, 1))
        for call in (lambda: kv_cache.copy_pages(v, src, dst),
                     lambda: kv_cache.compact(v, torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                                              torch.ones(3, dtype=torch.int32, device="cuda"))):
            with pytest.raises(RuntimeError, match="must not overlap"):
                call()
    one = base.clone().as_strided((3, 1, 4, 8), (page, 7, 8, 1))                # one page a layer
    kv_cache.copy_pages(one, src, src)

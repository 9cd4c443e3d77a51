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

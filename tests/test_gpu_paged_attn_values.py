"""Paged attention on values that are no ordinary numbers: NaN and infinities in
queries, keys and sinks, and pages that are missing, in rows that one block holds
whole and in rows joined from pieces.  The formula in float64 says where NaN belongs
(oracle/cache_oracle.py ``paged_attn``); everything else obeys its bound."""

import numpy as np
import pytest
import torch

from oracle import cache_oracle as C
from test_gpu_paged_attn import HALF, TINY, Cache

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")
LENS = [40, 3000, 64, 9001]  # whole, joined, whole, joined


def _check(out, q, kv_of, pos, sink, scale):
    with np.errstate(all="ignore"):
        ref, bound = C.paged_attn(q.double().cpu().numpy(), kv_of, pos, None if sink is None else sink.cpu().numpy(),
                                  scale, 0, 0, HALF[q.dtype], TINY[q.dtype])
    got = out.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    there = ~np.isnan(ref)
    assert np.all(np.abs(got - ref)[there] <= bound[there])


def _put(c, t, first, last, channel, value):
    """``value`` into one channel of keys first .. last - 1 of sequence t."""
    for j in range(first, last):
        c.pages[c.table[t, j // c.page].long(), j % c.page, channel] = value
    c.rows[t][first:last, channel] = value


def _attend(c, H, dtype, sink, change_q=None):
    from spark_b200 import kv_cache

    D = c.pages.shape[2]
    q = torch.randn(len(LENS), H, D, generator=c.g, device="cuda").to(dtype)
    if change_q is not None:
        change_q(q)
    s = torch.randn(H, generator=c.g, device="cuda") if sink else None
    pos = [n - 1 for n in LENS]
    out = kv_cache.paged_attn(q, c.pages, c.table, None, torch.tensor(pos, device="cuda"), s, D ** -0.5)
    torch.cuda.synchronize()
    _check(out, q, lambda t, keys: c.rows[t][keys], pos, s, D ** -0.5)
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,sink", [(64, True), (16, False)])
def test_nan_in_a_query(cuda_device, dtype, H, sink):
    """One head of every row has a NaN: all its scores are NaN, so is its output, whole
    or joined; the other heads are as they would be."""
    from spark_b200 import _lib

    def change(q):
        q[:, 3, 5] = NAN

    out = _attend(Cache(LENS, 64, 128, dtype, seed=H), H, dtype, sink, change)
    _lib.raise_on_device_error()
    assert torch.isnan(out[:, 3]).all() and torch.isfinite(out[:, 4:]).all()


@pytest.mark.parametrize("sink", [True, False])
@pytest.mark.parametrize("t,first,last", [(0, 0, 40), (1, 64, 128), (1, 0, 3000), (2, 63, 64), (3, 0, 1), (3, 4480, 4736),
                                          (3, 8960, 9001)])
def test_pages_of_nan(cuda_device, t, first, last, sink):
    c = Cache(LENS, 64, 512, torch.bfloat16, seed=first)
    _put(c, t, first, last, slice(None), NAN)
    out = _attend(c, 64, torch.bfloat16, sink)
    assert torch.isnan(out[t]).all()
    assert torch.isfinite(out[[x for x in range(4) if x != t]]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sink", [True, False])
@pytest.mark.parametrize("value", [INF, -INF])
@pytest.mark.parametrize("t,first,last", [(0, 7, 8), (0, 0, 40), (1, 64, 128), (1, 0, 3000), (2, 0, 64), (3, 4000, 5000),
                                          (3, 0, 9001)])
def test_infinite_keys(cuda_device, dtype, t, first, last, value, sink):
    """A score of +inf makes its head NaN; one of -inf has weight 0, and 0 x inf is NaN
    in the infinite channel.  Where every score is -inf the weights are 0 / 0, unless
    a sink keeps the denominator."""
    c = Cache(LENS, 64, 128, dtype, seed=last)
    _put(c, t, first, last, 9, value)
    out = _attend(c, 16, dtype, sink)
    assert torch.isnan(out[t, :, 9]).all() and torch.isfinite(out[[x for x in range(4) if x != t]]).all()


@pytest.mark.parametrize("sink", [None, 0.5, INF])
def test_rows_on_no_page_give_zeros(cuda_device, sink):
    """Nothing seen is told apart from scores of -inf: zeros and a latched error, whole or
    joined, also where only some pieces see nothing."""
    from spark_b200 import _lib, kv_cache

    c = Cache(LENS, 64, 128, torch.bfloat16, seed=2)
    c.table[0], c.table[1], c.table[3, 8:100] = -1, -1, -1
    q = torch.randn(len(LENS), 16, 128, generator=c.g, device="cuda").bfloat16()
    s = None if sink is None else torch.full((16,), sink, device="cuda")
    pos = [n - 1 for n in LENS]
    out = kv_cache.paged_attn(q, c.pages, c.table, None, torch.tensor(pos, device="cuda"), s, 0.1)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="cache sequence, position"):
        _lib.raise_on_device_error()
    assert torch.all(out[:2] == 0)
    if sink != INF:
        _check(out[2:], q[2:], lambda t, keys: c.rows[2 + t][keys if t == 0 else keys[(keys < 512) | (keys >= 6400)]],
               [63, 9000], s, 0.1)
    else:
        assert torch.all(out == 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nats,small", [(18, 1e-3), (22, 1e-4)])
@pytest.mark.parametrize("place", [0, 2050, 4000])
def test_a_dominating_key_of_small_values(cuda_device, dtype, nats, small, place):
    """One key far above thousands of others, with values so small that the others' tiny
    weights still make a part of the output.  In fp16 the largest weight is at least 2^9
    and the steps are 2^-24: a key loses 2^-34 of the largest weight at most."""
    from spark_b200 import _lib, kv_cache

    T, H, D, n = 300, 3, 128, 4001
    c = Cache([n], 64, D, dtype, seed=place)
    rows = torch.randn(n, D, generator=c.g, device="cuda") + 1.0
    rows[place] *= small
    rows[:, 0] = 0.0
    rows[place, 0] = 1.0
    rows = rows.to(dtype)
    for j in range(-(-n // 64)):
        part = rows[j * 64:(j + 1) * 64]
        c.pages[c.table[0, j].long(), : len(part)] = part
    q = torch.zeros(T, H, D, device="cuda")
    q[:, :, 0] = torch.tensor([nats, nats - 3.0, 1.0], device="cuda")
    q = q.to(dtype)
    pos = [n - 1 - (t % 3) if place < 4000 else n - 1 for t in range(T)]
    out = kv_cache.paged_attn(q, c.pages, c.table, torch.zeros(T, dtype=torch.int32, device="cuda"),
                              torch.tensor(pos, dtype=torch.int32, device="cuda"), None, 1.0)
    torch.cuda.synchronize()
    _lib.raise_on_device_error()
    kv = rows.double().cpu().numpy()
    ref, bound = C.paged_attn(q.double().cpu().numpy(), lambda t, keys: kv[keys], pos, None, 1.0, 0, 0, HALF[dtype],
                              TINY[dtype], TINY[dtype] * 2.0 ** -9)
    err = np.abs(out.double().cpu().numpy() - ref)
    assert np.all(err <= bound), (float((err / bound).max()), float(err.max()))


def test_rising_scores_in_fp16(cuda_device):
    """Scores that rise by two to forty in base 2 from chunk to chunk, and fall again: no
    weight passes fp16's range."""
    from spark_b200 import _lib, kv_cache

    D, H, n = 128, 64, 2500
    c = Cache([n, n], 64, D, torch.float16, seed=1)
    q = torch.zeros(2, H, D, device="cuda").half()
    q[:, :, 0] = torch.linspace(-20, 20, H, device="cuda").half()
    rows = torch.from_numpy(c.rows[0]).cuda()
    rows[:, 0] = torch.cat((torch.linspace(0, 30, 1500), torch.linspace(30, -30, 1000))).half().double().cuda()
    for t in range(2):
        for j in range(-(-n // 64)):
            part = rows[j * 64:(j + 1) * 64]
            c.pages[c.table[t, j].long(), : len(part)] = part.half()
    kv = rows.cpu().numpy()
    out = kv_cache.paged_attn(q, c.pages, c.table, None, torch.tensor([n - 1, 63], device="cuda"), None, 1.0)
    torch.cuda.synchronize()
    _lib.raise_on_device_error()
    ref, bound = C.paged_attn(q.double().cpu().numpy(), lambda t, keys: kv[keys], [n - 1, 63], None, 1.0, 0, 0,
                              HALF[torch.float16], TINY[torch.float16], TINY[torch.float16] * 2.0 ** -9)
    err = np.abs(out.double().cpu().numpy() - ref)
    assert np.all(err <= bound), (float((err / bound).max()), float(err.max()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [200, 2000])
def test_the_error_of_a_dominating_weight_cancels(cuda_device, dtype, n):
    """A key that takes nearly all of the weight, behind the one that set the running max,
    so that its own weight is no power of two (as many rows as leave each to one block).  Weights p_j (1 + d_j) summed as rounded
    give sum p_j (1 + d_j) kv_j / sum p_j (1 + d_j) = out + sum d_j p_j (kv_j - out) to
    first order: half a step of sum p_j |kv_j - out|, not of sum p_j |kv_j|, then the
    output's half step and 3e-4 of sum p |kv| + |out| for scores and exponentials in
    32 bits (cache_oracle.paged_attn)."""
    from spark_b200 import _lib, kv_cache

    D, H = 128, 64
    c = Cache([n], 64, D, dtype, seed=n)
    rows = torch.randn(n, D, generator=c.g, device="cuda")
    rows[:, 0], rows[0, 0], rows[150, 0] = -5.0, 0.0, 1.0
    rows = rows.to(dtype)
    for j in range(-(-n // 64)):
        part = rows[j * 64:(j + 1) * 64]
        c.pages[c.table[0, j].long(), : len(part)] = part
    q = torch.zeros(300, H, D, device="cuda")
    q[:, :, 0] = torch.linspace(3, 4, H, device="cuda")
    q = q.to(dtype)
    where = torch.zeros(300, dtype=torch.int32, device="cuda"), torch.full((300,), n - 1, dtype=torch.int32, device="cuda")
    out = kv_cache.paged_attn(q, c.pages, c.table, *where, None, 1.0)
    torch.cuda.synchronize()
    _lib.raise_on_device_error()
    kv = rows.double().cpu().numpy()
    z = q[0].double().cpu().numpy() @ kv.T
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    ref = p @ kv
    apart = np.stack([p[h] @ np.abs(kv - ref[h]) for h in range(H)])
    bound = 1.02 * HALF[dtype] * apart + HALF[dtype] * np.abs(ref) + 3e-4 * (p @ np.abs(kv) + np.abs(ref)) + TINY[dtype]
    err = np.abs(out.double().cpu().numpy() - ref)
    assert np.all(err <= bound), (float((err / bound).max()), int((err > bound).sum()))

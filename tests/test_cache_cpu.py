"""The attention cache's operators on the CPU: frequencies, refusals of the C ABI
(every call returns before a CUDA call), schemas and output shapes of the torch
ops, and the oracle the GPU tests compare against."""

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import cache_oracle as C

OPS = ["rotary", "rotary_", "cache_append", "cache_reserve", "cache_free", "cache_fork", "cache_compact",
       "cache_copy", "paged_attn"]
P = ctypes.c_void_p(0x10000)


@pytest.fixture(scope="module")
def lib():
    from spark_b200 import _lib

    return _lib.load()


@pytest.fixture(scope="module")
def dsv4():
    from spark_b200 import ops

    return ops.load()


def test_ops_are_registered_and_have_shapes_on_meta(dsv4):
    for name in OPS:
        assert getattr(dsv4, name).default._schema.name == f"dsv4moe::{name}"
    m = torch.device("meta")
    x = torch.empty(2, 3, 64, 512, dtype=torch.bfloat16, device=m)
    pos, f = torch.empty(2, 3, dtype=torch.int64, device=m), torch.empty(32, dtype=torch.float64, device=m)
    assert dsv4.rotary(x, pos, f).shape == x.shape
    pages = torch.empty(9, 64, 512, dtype=torch.bfloat16, device=m)
    table, refs = torch.empty(4, 8, dtype=torch.int32, device=m), torch.empty(9, dtype=torch.int32, device=m)
    q = torch.empty(4, 64, 512, dtype=torch.bfloat16, device=m)
    o = dsv4.paged_attn(q, pages, table, None, pos[0, :1].expand(4), None, 0.04, 128, 4)
    assert o.shape == q.shape and o.dtype == q.dtype
    assert dsv4.cache_compact(pages, table, refs).shape == refs.shape
    assert dsv4.cache_free(table, refs[:4], refs, refs[:2]) is None


def test_rotary_frequencies():
    from spark_b200.rotary import rotary_frequencies

    f = rotary_frequencies(64, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (32,)
    assert f[0] == 1.0 and abs(float(f[31]) - 10000.0 ** (-62 / 64)) < 1e-18
    assert torch.equal(rotary_frequencies(64, scaling="linear", factor=4, device="cpu"), f / 4)
    y = rotary_frequencies(64, scaling="yarn", factor=16, original_len=65536, device="cpu")
    turns = 65536 * f / (2 * math.pi)
    ratio = y / f
    assert torch.all(ratio[turns > 64] == 1) and torch.all((ratio[turns < 0.5] - 1 / 16).abs() < 1e-15)
    assert torch.all(ratio[1:] <= ratio[:-1])  # the blend falls over the pair index
    assert rotary_frequencies(2, device="cpu").tolist() == [1.0]
    for bad in (dict(rot=63), dict(rot=0), dict(rot=64, scaling="x"), dict(rot=64, base=1.0),
                dict(rot=64, scaling="linear", factor=0.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad, device="cpu")


def test_rotary_refusals(lib):
    from spark_b200 import _lib

    ll3 = ctypes.c_longlong * 3
    st = ll3(512, 512, 512)

    def call(x=P, y=P, dtype=0, pos=P, freqs=P, B=1, S=1, H=1, D=512, rot=64, offset=448, xs=st, ys=st):
        return lib.dsv4_rotary(x, y, dtype, pos, 0, freqs, B, S, H, D, rot, offset, 1, 0, 1.0, xs, ys, None)

    for bad in (dict(B=-1), dict(S=-1), dict(H=-1), dict(D=0), dict(rot=63), dict(rot=-2), dict(offset=449),
                dict(offset=-1), dict(x=None), dict(y=None), dict(pos=None), dict(freqs=None), dict(xs=None),
                dict(ys=ll3(512, 512, 1024)), dict(offset=2 ** 31 - 1)):
        assert call(**bad) == _lib.ERR_ARG, bad
    for bad in (dict(dtype=3), dict(dtype=-1), dict(D=8192, rot=4098, offset=0), dict(D=(1 << 20) + 8)):
        assert call(**bad) == _lib.ERR_UNSUPPORTED, bad
    for empty in (dict(B=0), dict(S=0), dict(H=0)):
        assert call(**empty) == _lib.OK


def test_append_refusals(lib):
    from spark_b200 import _lib

    def call(rows=P, dtype=0, T=1, D=512, pages=P, n_pages=4, page=64, stride=64 * 512, table=P, n_seqs=2,
             max_pages=2, pos=P, freqs=P, rot=64, offset=448):
        return lib.dsv4_cache_append(rows, 512, dtype, T, D, pages, n_pages, page, stride, table, n_seqs, max_pages,
                                     None, pos, 0, freqs, rot, offset, 1, 1.0, None)

    for bad in (dict(T=-1), dict(rows=None), dict(pages=None), dict(table=None), dict(pos=None), dict(freqs=None),
                dict(n_pages=0), dict(page=0), dict(n_seqs=0), dict(max_pages=0), dict(rot=65), dict(offset=500)):
        assert call(**bad) == _lib.ERR_ARG, bad
    for bad in (dict(dtype=2), dict(D=516, offset=0), dict(stride=64 * 512 + 4), dict(pages=ctypes.c_void_p(0x10008)),
                dict(page=8192), dict(max_pages=1 << 21), dict(D=1024, rot=514, offset=0), dict(max_pages=1 << 20, page=4096)):
        assert call(**bad) == _lib.ERR_UNSUPPORTED, bad
    assert call(T=0, rows=None) == _lib.OK


def test_page_operation_refusals(lib):
    from spark_b200 import _lib

    big = 1 << 30

    def reserve(table=P, lens=P, refs=P, n_seqs=4, max_pages=8, n_pages=16, page=64, seqs=P, new=P, n=2, ws=P, wsb=big):
        return lib.dsv4_cache_reserve(table, lens, refs, n_seqs, max_pages, n_pages, page, seqs, new, n, ws, wsb, None)

    for bad in (dict(table=None), dict(lens=None), dict(refs=None), dict(seqs=None), dict(new=None), dict(n=-1),
                dict(n_seqs=0), dict(max_pages=0), dict(n_pages=0), dict(page=0)):
        assert reserve(**bad) == _lib.ERR_ARG, bad
    need = lib.dsv4_cache_reserve_workspace_bytes(2, 4, 16)
    assert need == 4 * (4 + 3 + 16)
    assert reserve(wsb=need - 1) == _lib.ERR_WORKSPACE and reserve(ws=None) == _lib.ERR_WORKSPACE
    assert reserve(n=0) == _lib.OK and lib.dsv4_cache_reserve_workspace_bytes(-1, 4, 16) == -1

    def free(table=P, lens=P, refs=P, n_seqs=4, n=1, seqs=P):
        return lib.dsv4_cache_free(table, lens, refs, n_seqs, 8, 16, seqs, n, None)

    for bad in (dict(table=None), dict(lens=None), dict(refs=None), dict(seqs=None), dict(n=-1), dict(n_seqs=0)):
        assert free(**bad) == _lib.ERR_ARG, bad
    assert free(n=0) == _lib.OK

    def fork(pages=P, layers=2, D=512, ls=1 << 24, ps=64 * 512, parents=P, children=P, n=2, ws=P, wsb=big):
        return lib.dsv4_cache_fork(pages, layers, D, ls, ps, P, P, P, 4, 8, 16, 64, parents, children, None, n, ws, wsb,
                                   None)

    for bad in (dict(pages=None), dict(layers=0), dict(D=0), dict(parents=None), dict(children=None), dict(n=-1)):
        assert fork(**bad) == _lib.ERR_ARG, bad
    for bad in (dict(D=510), dict(ls=(1 << 24) + 1), dict(ps=64 * 512 + 4), dict(pages=ctypes.c_void_p(0x10008))):
        assert fork(**bad) == _lib.ERR_UNSUPPORTED, bad
    assert fork(wsb=4 * (4 + 6) - 1) == _lib.ERR_WORKSPACE and fork(n=0) == _lib.OK

    def compact(pages=P, map_=P, ws=P, wsb=big, n_pages=16):
        return lib.dsv4_cache_compact(pages, 2, 512, 1 << 24, 64 * 512, P, P, 4, 8, n_pages, 64, map_, ws, wsb, None)

    assert compact(pages=None) == compact(map_=None) == compact(n_pages=0) == _lib.ERR_ARG
    assert compact(wsb=4 * 17 - 1) == _lib.ERR_WORKSPACE

    def copy(pages=P, src=P, dst=P, n=2):
        return lib.dsv4_cache_copy(pages, 2, 512, 1 << 24, 64 * 512, 16, 64, src, dst, n, None)

    assert copy(pages=None) == copy(src=None) == copy(dst=None) == copy(n=-1) == _lib.ERR_ARG
    assert copy(n=0) == _lib.OK


def test_paged_attn_refusals(lib):
    from spark_b200 import _lib

    def call(q=P, qt=64 * 512, qh=512, dtype=0, T=2, H=64, D=512, pages=P, n_pages=16, page=64, stride=64 * 512, table=P,
             n_seqs=4, max_pages=8, pos=P, window=0, first=0, out=P, ws=P, wsb=1 << 40):
        return lib.dsv4_paged_attn(q, qt, qh, dtype, T, H, D, pages, n_pages, page, stride, table, n_seqs, max_pages,
                                   None, pos, 0, None, 0.05, window, first, out, ws, wsb, None)

    for bad in (dict(q=None), dict(pages=None), dict(table=None), dict(pos=None), dict(out=None), dict(T=-1),
                dict(H=0), dict(D=0), dict(n_pages=0), dict(page=0), dict(n_seqs=0), dict(max_pages=0),
                dict(window=-1), dict(first=-1), dict(q=ctypes.c_void_p(0x10008)), dict(out=ctypes.c_void_p(0x10002)),
                dict(qt=64 * 512 + 4), dict(qh=516), dict(qh=8), dict(stride=8)):
        assert call(**bad) == _lib.ERR_ARG, bad
    for bad in (dict(H=129), dict(D=64), dict(D=384), dict(page=8), dict(page=48), dict(page=8192), dict(dtype=2),
                dict(stride=64 * 512 + 4), dict(pages=ctypes.c_void_p(0x10008))):
        assert call(**bad) == _lib.ERR_UNSUPPORTED, bad
    need = lib.dsv4_paged_attn_workspace_bytes(2, 64, 512, 64, 8)
    assert need > 0 and call(wsb=need - 1) == _lib.ERR_WORKSPACE and call(ws=None) == _lib.ERR_WORKSPACE
    assert call(T=0, q=None) == _lib.OK
    assert lib.dsv4_paged_attn_workspace_bytes(2, 129, 512, 64, 8) == -1


def test_torch_ops_refuse_cpu_tensors(dsv4):
    x = torch.zeros(2, 4, 64)
    with pytest.raises(NotImplementedError):
        dsv4.rotary(x, torch.zeros(2, dtype=torch.int32), torch.ones(8, dtype=torch.float64))


def test_oracle_rotary_inverse_is_the_transpose():
    g = np.random.default_rng(0)
    f = 10000.0 ** (-np.arange(8) / 8)
    x, y, pos = g.standard_normal((5, 3, 40)), g.standard_normal((5, 3, 40)), g.integers(0, 10 ** 6, 5)
    for inter in (True, False):
        a = C.rotary(x, pos, f, 10, inter)
        assert abs((a * y).sum() - (x * C.rotary(y, pos, f, 10, inter, inverse=True)).sum()) < 1e-9
        assert np.allclose(C.rotary(a, pos, f, 10, inter, inverse=True), x, atol=1e-9)
        assert np.array_equal(a[..., :10], x[..., :10]) and np.array_equal(a[..., 26:], x[..., 26:])


def test_oracle_pool_keeps_counts():
    pool = C.Pool([[-1] * 4 for _ in range(6)], [0] * 6, [0] * 10, 4)
    pool.reserve([0, 2], [9, 4])
    assert pool.table[0][:3] == [0, 1, 2] and pool.table[2][0] == 3
    pool.fork([0, 0], [1, 3], None)
    assert pool.refs[:6] == [3, 3, 1, 1, 1, 1] and pool.table[1][:3] == [0, 1, 4]
    pool.free([0, 2])
    assert pool.refs[:6] == [2, 2, 0, 0, 1, 1]
    assert pool.compact()[:6] == [0, 1, -1, -1, 2, 3] and pool.table[3][:3] == [0, 1, 3]
    pool.reserve([4, 5], [16, 12])
    assert pool.short and pool.lens[4] == 0
    assert C.visible(9, 3, 2).tolist() == [0, 1, 7, 8, 9] and C.visible(2, 5, 2).tolist() == [0, 1, 2]


def test_index_tensors_of_another_shape_are_refused(dsv4):
    """As many elements in another order are no positions: those of a transposed batch
    would turn tokens by other tokens' positions.  Axes of one entry say nothing, and a
    flat vector has one order only."""
    m = torch.device("meta")

    def ints(*shape):
        return torch.empty(*shape, dtype=torch.int64, device=m)

    f = torch.empty(32, dtype=torch.float64, device=m)
    x = torch.empty(2, 3, 4, 128, device=m)
    for op in (dsv4.rotary, dsv4.rotary_):
        for good in ((2, 3), (6,), (2, 1, 3), (1, 6)):
            op(x, ints(*good), f)
        for bad in ((3, 2), (1, 3, 2), (2, 3, 2), (5,), (2,)):
            with pytest.raises(RuntimeError, match="positions"):
                op(x, ints(*bad), f)
        op(x[0, 0], ints(1)[0], f)
        op(x[:0], ints(0, 3), f)
        five = torch.empty(2, 3, 4, 5, 128, device=m)
        op(five, ints(2, 3, 4), f)
        for bad in ((6, 4), (2, 12), (4, 3, 2)):
            with pytest.raises(RuntimeError, match="positions"):
                op(five, ints(*bad), f)
    pages, table = torch.empty(9, 16, 128, dtype=torch.bfloat16, device=m), torch.empty(8, 8, dtype=torch.int32, device=m)
    q, rows = torch.empty(6, 4, 128, dtype=torch.bfloat16, device=m), torch.empty(6, 128, dtype=torch.bfloat16, device=m)

    def attend(seq=None, pos=ints(6), sink=None):
        return dsv4.paged_attn(q, pages, table, seq, pos, sink, 0.1)

    def append(seq=None, pos=ints(6)):
        return dsv4.cache_append(pages, rows, table, seq, pos)

    for call in (attend, append):
        for good in (dict(), dict(pos=ints(6, 1)), dict(seq=ints(6)), dict(seq=ints(1, 6))):
            call(**good)
        for bad in (dict(pos=ints(2, 3)), dict(pos=ints(7)), dict(seq=ints(3, 2)), dict(seq=ints(5))):
            with pytest.raises(RuntimeError, match="positions|seq_ids"):
                call(**bad)
    attend(sink=torch.empty(4, device=m))
    for bad in ((2, 2), (3,), (4, 4)):
        with pytest.raises(RuntimeError, match="attn_sink"):
            attend(sink=torch.empty(*bad, device=m))


def test_sizes_at_the_end_of_32_bits_are_refused(lib):
    """The page operations step through lists, sequences and pages by up to a block's
    threads in 32 bits: a step past the end must not wrap, or the loop never ends."""
    from spark_b200 import _lib

    big, most, huge = 1 << 62, 2 ** 31 - 1, 2 ** 31 - 4096

    def reserve(n_seqs=4, n_pages=16, n=2):
        return lib.dsv4_cache_reserve(P, P, P, n_seqs, 8, n_pages, 64, P, P, n, P, big, None)

    def free(n_seqs=4, n_pages=16, n=2):
        return lib.dsv4_cache_free(P, P, P, n_seqs, 8, n_pages, P, n, None)

    def fork(n_seqs=4, n_pages=16, n=2):
        return lib.dsv4_cache_fork(P, 1, 512, 1 << 24, 64 * 512, P, P, P, n_seqs, 8, n_pages, 64, P, P, None, n, P, big, None)

    def compact(n_seqs=4, n_pages=16):
        return lib.dsv4_cache_compact(P, 1, 512, 1 << 24, 64 * 512, P, P, n_seqs, 8, n_pages, 64, P, P, big, None)

    def copy(n_pages=16, n=2):
        return lib.dsv4_cache_copy(P, 1, 512, 1 << 24, 64 * 512, n_pages, 64, P, P, n, None)

    def append(n_seqs=4, n_pages=16, T=2):
        return lib.dsv4_cache_append(P, 512, 0, T, 512, P, n_pages, 64, 64 * 512, P, n_seqs, 8, None, P, 0, None, 0, 0, 1,
                                     1.0, None)

    for call, names in ((reserve, ("n_seqs", "n_pages", "n")), (free, ("n_seqs", "n_pages", "n")),
                        (fork, ("n_seqs", "n_pages", "n")), (compact, ("n_seqs", "n_pages")), (copy, ("n_pages", "n")),
                        (append, ("n_seqs", "n_pages", "T"))):
        for name in names:
            for size in (most, huge):
                assert call(**{name: size}) == _lib.ERR_UNSUPPORTED, (call.__name__, name, size)

"""GPU parity of the page operations with lists (oracle/cache_oracle.py ``Pool``):
tables, lengths, holder counts and page contents are equal, whatever the order of
the calls; refused entries, too few pages, and a captured graph."""

import numpy as np
import pytest
import torch

from oracle import cache_oracle as C

pytestmark = pytest.mark.gpu


def _ints(v):
    return torch.tensor(list(v), dtype=torch.int32, device="cuda")


class Both:
    """The device's cache and the oracle's, and the same calls on both."""

    def __init__(self, seqs, most, pool, page, layers=2, D=16, seed=0, pages_first=False):
        self.page = page
        g = torch.Generator(device="cuda").manual_seed(seed)
        shape = (pool, layers, page, D) if pages_first else (layers, pool, page, D)
        data = torch.randn(*shape, generator=g, device="cuda").bfloat16()
        self.pages = data.transpose(0, 1) if pages_first else data
        self.table = torch.full((seqs, most), -1, dtype=torch.int32, device="cuda")
        self.lens, self.refs = _ints([0] * seqs), _ints([0] * pool)
        self.ref = C.Pool(self.table.tolist(), [0] * seqs, [0] * pool, page, self.pages.float().cpu().numpy())

    def same(self, bad=False, short=False):
        from spark_b200 import _lib

        torch.cuda.synchronize()
        if bad or short:
            with pytest.raises(RuntimeError, match="out of free pages" if short else "cache sequence, position"):
                _lib.raise_on_device_error()
        else:
            _lib.raise_on_device_error()
        assert self.ref.bad == bad and self.ref.short == short
        self.ref.bad = self.ref.short = False
        assert self.table.tolist() == self.ref.table and self.lens.tolist() == self.ref.lens
        assert self.refs.tolist() == self.ref.refs
        assert np.array_equal(self.pages.float().cpu().numpy(), self.ref.pages)

    def reserve(self, seqs, lens, **k):
        from spark_b200 import kv_cache

        kv_cache.reserve(self.table, self.lens, self.refs, _ints(seqs), _ints(lens), self.page)
        self.ref.reserve(seqs, lens)
        self.same(**k)

    def free(self, seqs, **k):
        from spark_b200 import kv_cache

        kv_cache.free(self.table, self.lens, self.refs, _ints(seqs))
        self.ref.free(seqs)
        self.same(**k)

    def fork(self, a, b, lens=None, **k):
        from spark_b200 import kv_cache

        kv_cache.fork(self.pages, self.table, self.lens, self.refs, _ints(a), _ints(b),
                      None if lens is None else _ints(lens))
        self.ref.fork(a, b, lens)
        self.same(**k)

    def compact(self, **k):
        from spark_b200 import kv_cache

        got = kv_cache.compact(self.pages, self.table, self.refs)
        assert got.tolist() == self.ref.compact()
        self.same(**k)


@pytest.mark.parametrize("pages_first", [False, True])
@pytest.mark.parametrize("page", [1, 16, 24])
def test_a_run_of_operations(cuda_device, page, pages_first):
    c = Both(9, 7, 40, page, seed=page, pages_first=pages_first)
    c.reserve([0, 3, -1, 5], [2 * page + 1, 7 * page, 5, 1])
    c.reserve([3, 0, 7], [page, 3 * page + 2 if page > 2 else 4, 0])  # one shrinks (keeps its room), one grows
    c.fork([0, 0, 3, -1, 5], [1, 2, 4, 6, -1])
    c.fork([3, 3], [6, 7], [page + page // 2, 0])
    c.reserve([1, 2], [5 * page, 4 * page])
    c.free([0, 5, -3])
    c.compact()
    c.compact()                                                       # nothing left to move
    c.free([3, 1, 3])                                                 # the same sequence twice
    c.compact()
    c.free(range(9))
    assert c.refs.tolist() == [0] * 40
    c.compact()
    c.reserve(range(9), [1] * 9)


def test_refused_entries_and_too_few_pages(cuda_device):
    c = Both(6, 4, 10, 16)
    c.reserve([0, 0, 6, 1, 2], [20, 40, 5, 65, -1], bad=True)         # named again, no such sequence, too long, negative
    c.reserve([1, 2, 3], [64, 64, 17], short=True)                    # ten pages, two held, ten asked
    c.reserve([1, 2], [64, 64])                                       # exactly all
    c.reserve([3], [1], short=True)
    c.fork([0], [3], short=True)                                      # no page for the part-filled one
    c.fork([1], [3])                                                  # full pages need none
    c.fork([1, 0, 7, 0, 2, 2], [2, 6, 4, 5, 4, 4], [16, 16, 16, 21, 32, 32], bad=True)
    c.free([6, 1], bad=True)
    c.reserve([5], [2 ** 31 - 1], bad=True)


def test_64_bit_ids_do_not_wrap(cuda_device):
    """2^32 is no sequence, not sequence 0; 2^32 + 5 no length of 5."""
    from spark_b200 import _lib, kv_cache

    c = Both(4, 4, 12, 16)
    c.reserve([0, 1], [20, 30])
    before = c.table.clone(), c.lens.clone(), c.refs.clone()
    big = torch.tensor([2 ** 32, 2 ** 32 + 1], device="cuda")
    small = torch.tensor([2, 3], device="cuda")
    for call in (lambda: kv_cache.reserve(c.table, c.lens, c.refs, big, small, 16),
                 lambda: kv_cache.reserve(c.table, c.lens, c.refs, small, big, 16),
                 lambda: kv_cache.free(c.table, c.lens, c.refs, big),
                 lambda: kv_cache.fork(c.pages, c.table, c.lens, c.refs, big, small),
                 lambda: kv_cache.fork(c.pages, c.table, c.lens, c.refs, torch.tensor([0, 1], device="cuda"), big),
                 lambda: kv_cache.copy_pages(c.pages, big, small)):
        call()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="cache sequence, position"):
            _lib.raise_on_device_error()
        assert torch.equal(c.table, before[0]) and torch.equal(c.lens, before[1]) and torch.equal(c.refs, before[2])
    kv_cache.free(c.table, c.lens, c.refs, torch.tensor([-2 ** 40], device="cuda"))  # padding
    c.same()


@pytest.mark.parametrize("seqs", [1500, 2600])  # claims in shared memory, in the workspace
def test_many_sequences_and_pages(cuda_device, seqs):
    rng = np.random.default_rng(5)
    c = Both(seqs, 20, 30000, 16, layers=1, D=8)
    every = rng.permutation(seqs).tolist()
    c.reserve(every, rng.integers(0, 20 * 16 // 2, seqs).tolist())
    c.free(every[:700])
    c.reserve(every[:300] + every[:1], rng.integers(0, 20 * 16, 301).tolist(), bad=True)
    c.fork([every[0]] * 200 + every[701:900], every[300:699])
    c.compact()
    c.reserve(every, [160] * seqs)


def test_few_long_sequences(cuda_device):
    c = Both(5, 1500, 5000, 16, layers=1, D=8)
    c.reserve([3, 1], [16 * 1400 + 3, 16 * 131])
    c.reserve([0, 1, 4], [16 * 33, 16 * 700, 16 * 1500])
    c.free([3])
    c.fork([4, 1], [2, 3])
    c.compact()


def test_pages_larger_than_a_copy_part(cuda_device):
    c = Both(5, 3, 12, 128, layers=3, D=264)                          # 66 KB a page
    c.reserve([0, 1, 2], [130, 384, 100])
    c.fork([0, 2], [3, 4])
    c.free([0, 1])
    c.compact()


def test_copy_pages(cuda_device):
    from spark_b200 import _lib, kv_cache

    g = torch.Generator(device="cuda").manual_seed(1)
    pages = torch.randn(3, 12, 16, 40, generator=g, device="cuda").half()
    want = pages.clone()
    kv_cache.copy_pages(pages, _ints([0, 3, -1, 7, 0]), _ints([5, 6, 2, -1, 11]))
    want[:, [5, 6, 11]] = want[:, [0, 3, 0]]
    torch.cuda.synchronize()
    _lib.raise_on_device_error()
    assert torch.equal(pages, want)
    # chains, swaps, a target twice, out of range: reported, the rest is copied
    kv_cache.copy_pages(pages, _ints([0, 1, 4, 8, 9, 10, 12, 2]), _ints([1, 2, 3, 3, 10, 9, 0, 12]))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="cache sequence, position"):
        _lib.raise_on_device_error()
    want[:, 3] = want[:, 4]
    assert torch.equal(pages, want)
    one = pages[0].clone()
    kv_cache.copy_pages(one, _ints([]), _ints([]))
    kv_cache.copy_pages(one, _ints([1]).long(), _ints([1]).long())
    assert torch.equal(one, pages[0])
    for bad in (lambda: kv_cache.copy_pages(pages, _ints([1]), _ints([1, 2])),
                lambda: kv_cache.copy_pages(pages.float(), _ints([1]), _ints([2])),
                lambda: kv_cache.copy_pages(pages[..., :20], _ints([1]), _ints([2])),
                lambda: kv_cache.copy_pages(pages, torch.tensor([1]), torch.tensor([2]))):
        with pytest.raises(RuntimeError):
            bad()


def test_a_captured_step_follows_the_tables(cuda_device):
    """reserve + fork + free + compact in a graph, replayed on other inputs."""
    from spark_b200 import _lib, kv_cache

    c = Both(6, 5, 24, 16)
    seqs, lens, a, b, drop = _ints([0, 1]), _ints([1, 1]), _ints([0]), _ints([2]), _ints([-1])
    c.reserve([3], [40])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # first launches outside the capture, on nothing
        none = _ints([-1])
        kv_cache.reserve(c.table, c.lens, c.refs, none, none, 16)
        kv_cache.fork(c.pages, c.table, c.lens, c.refs, none, none)
        kv_cache.free(c.table, c.lens, c.refs, none)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv_cache.reserve(c.table, c.lens, c.refs, seqs, lens, 16)
        kv_cache.fork(c.pages, c.table, c.lens, c.refs, a, b)
        kv_cache.free(c.table, c.lens, c.refs, drop)
        moved = kv_cache.compact(c.pages, c.table, c.refs)
    for s, n, p, q, d in (([0, 1], [20, 3], [0], [2], [-1]), ([1, 0], [33, 41], [1], [4], [3]), ([5, -1], [9, 1], [2], [3], [0])):
        for t, v in ((seqs, s), (lens, n), (a, p), (b, q), (drop, d)):
            t.copy_(_ints(v))
        graph.replay()
        c.ref.reserve(s, n)
        c.ref.fork(p, q)
        c.ref.free(d)
        assert moved.tolist() == c.ref.compact()
        c.same()
    del graph
    _lib.raise_on_device_error()


def test_argument_checks(cuda_device):
    from spark_b200 import kv_cache

    c = Both(4, 4, 8, 16)
    ok = c.table, c.lens, c.refs
    for bad in (lambda: kv_cache.reserve(c.table.long(), c.lens, c.refs, _ints([0]), _ints([1]), 16),
                lambda: kv_cache.reserve(c.table.t(), c.lens, c.refs, _ints([0]), _ints([1]), 16),
                lambda: kv_cache.reserve(c.table, c.lens[:3], c.refs, _ints([0]), _ints([1]), 16),
                lambda: kv_cache.reserve(*ok, _ints([0]), _ints([1, 2]), 16),
                lambda: kv_cache.reserve(*ok, _ints([0]), _ints([1]), 0),
                lambda: kv_cache.reserve(*ok, _ints([0]), torch.ones(1, device="cuda"), 16),
                lambda: kv_cache.free(*ok, torch.tensor([0], dtype=torch.int32)),
                lambda: kv_cache.fork(c.pages, c.table, c.lens, c.refs[:4], _ints([0]), _ints([1])),
                lambda: kv_cache.fork(c.pages, *ok, _ints([0]), _ints([1]), _ints([1, 2])),
                lambda: kv_cache.compact(c.pages[:, :4], c.table, c.refs),
                lambda: kv_cache.compact(c.pages.cpu(), c.table, c.refs)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            bad()
    kv_cache.free(*ok, _ints([]))
    kv_cache.reserve(*ok, _ints([]), _ints([]), 16)
    c.same()


@pytest.mark.parametrize("n,layers", [(3001, 11), (17000, 3)])  # a part of the layers per block, all of them
def test_many_copies(cuda_device, n, layers):
    from spark_b200 import _lib, kv_cache

    g = torch.Generator(device="cuda").manual_seed(n)
    pages = torch.randn(layers, 2 * n + 5, 2, 16, generator=g, device="cuda").bfloat16()
    order = torch.randperm(2 * n + 5, generator=g, device="cuda").int()
    src, dst = order[:n].clone(), order[n:2 * n].clone()
    src[7], dst[11] = -1, src[40]                                     # padding; another entry's source
    live = torch.ones(n, dtype=torch.bool, device="cuda")
    live[7] = live[11] = False
    want = pages.clone()
    want[:, dst[live].long()] = want[:, src[live].long()]
    kv_cache.copy_pages(pages, src, dst)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="cache sequence, position"):
        _lib.raise_on_device_error()
    assert torch.equal(pages, want)

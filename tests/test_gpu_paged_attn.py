"""GPU parity of the attention over the paged cache with float64 softmax attention
(oracle/cache_oracle.py ``paged_attn``, which derives the error bound): head counts,
head dims, page sizes, lengths around the chunk borders, windows and first tokens,
hidden rows full of NaN, missing pages, padding, strides, streams and graphs."""

import numpy as np
import pytest
import torch

from oracle import cache_oracle as C

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


class Cache:
    """Sequences of the given lengths on shuffled pages; every row that no sequence
    sees is NaN."""

    def __init__(self, lens, page, D, dtype, seed=0, spare=5):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.page = page
        need = [-(-n // page) for n in lens]
        pool = sum(need) + spare
        order = torch.randperm(pool, generator=g, device="cuda").int()
        self.table = torch.full((len(lens), max(need + [1]) + 1), -1, dtype=torch.int32, device="cuda")
        self.pages = torch.full((pool, page, D), float("nan"), dtype=dtype, device="cuda")
        self.rows, at = [], 0
        for s, n in enumerate(lens):
            self.table[s, : need[s]] = order[at:at + need[s]]
            r = torch.randn(n, D, generator=g, device="cuda").to(dtype)
            for j in range(need[s]):
                part = r[j * page:(j + 1) * page]
                self.pages[order[at + j].long(), : len(part)] = part
            self.rows.append(r.double().cpu().numpy())
            at += need[s]
        self.g = g


def _check(out, q, kv_of, pos, sink, scale, window, first):
    ref, bound = C.paged_attn(q.double().cpu().numpy(), kv_of, pos, None if sink is None else sink.cpu().numpy(), scale,
                              window, first, HALF[q.dtype], TINY[q.dtype])
    got = out.double().cpu().numpy()
    assert np.isfinite(got).all()
    err = np.abs(got - ref)
    assert np.all(err <= bound), (float((err / (bound + 1e-300)).max()), float(err.max()))


def _run(lens, H, D, page, dtype, *, window=0, first=0, sink=True, seed=0, index=torch.int32, q_scale=2.0):
    from spark_b200 import _lib, kv_cache

    c = Cache(lens, page, D, dtype, seed)
    T = len(lens)
    q = (q_scale * torch.randn(T, H, D, generator=c.g, device="cuda")).to(dtype)
    s = torch.randn(H, generator=c.g, device="cuda") if sink else None
    pos = [n - 1 for n in lens]
    p = torch.tensor(pos, dtype=index, device="cuda")
    scale = D ** -0.5
    out = kv_cache.paged_attn(q, c.pages, c.table, torch.arange(T, dtype=index, device="cuda"), p, s, scale,
                              window=window, first=first)
    torch.cuda.synchronize()
    _lib.raise_on_device_error()
    assert out.shape == q.shape and out.dtype == dtype
    _check(out, q, lambda t, keys: c.rows[t][keys], pos, s, scale, window, first)
    for t, n in enumerate(lens):
        if n == 0:
            assert torch.all(out[t] == 0)
    again = kv_cache.paged_attn(q, c.pages, c.table, None, p, s, scale, window=window, first=first)
    assert torch.equal(out, again)  # the same bits in every run


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,D,page", [(64, 512, 64), (16, 512, 16), (5, 256, 32), (32, 128, 128), (64, 256, 256),
                                      (1, 128, 16), (96, 512, 64), (128, 128, 64), (33, 512, 1024)])
def test_heads_dims_and_pages(cuda_device, dtype, H, D, page):
    _run([1, 130, 517, 64], H, D, page, dtype, seed=H + D)


@pytest.mark.parametrize("lens", [[1], [2], [127], [128], [129], [255, 256, 257], [0, 5, 0, 0, 300, 0], [0], [4000],
                                  [1] * 200, [700, 1, 3000, 1, 1, 129] * 3])
def test_lengths(cuda_device, lens):
    _run(lens, 64, 512, 64, torch.bfloat16, seed=len(lens))


@pytest.mark.parametrize("window,first", [(1, 0), (1, 1), (128, 4), (100, 0), (100, 130), (1000, 1), (5, 10000), (129, 128)])
@pytest.mark.parametrize("H,page", [(64, 64), (16, 16)])
def test_window_and_first_tokens(cuda_device, window, first, H, page):
    _run([1, 5, 128, 131, 400, 2000], H, 512, page, torch.bfloat16, window=window, first=first, seed=window)


@pytest.mark.parametrize("D,H", [(512, 64), (128, 16)])
def test_without_sink_and_with_large_scores(cuda_device, D, H):
    _run([1, 300, 1000], H, D, 64, torch.bfloat16, sink=False, index=torch.int64)
    _run([1, 300, 1000], H, D, 64, torch.float16, sink=False, q_scale=15.0)


def test_rising_scores_rescale_the_running_sums(cuda_device):
    """Keys whose scores rise by hundreds from chunk to chunk, and fall again."""
    from spark_b200 import _lib, kv_cache

    D, H, page, n = 128, 64, 64, 1500
    c = Cache([n], page, D, torch.bfloat16)
    q = torch.zeros(1, H, D, device="cuda").bfloat16()
    q[0, :, 0] = torch.linspace(-3, 3, H, device="cuda").bfloat16()
    ramp = torch.cat((torch.linspace(0, 30, 900), torch.linspace(30, -30, 600))).bfloat16().cuda()
    rows = torch.from_numpy(c.rows[0]).cuda()
    rows[:, 0] = ramp.double()
    for j in range(-(-n // page)):
        part = rows[j * page:(j + 1) * page]
        c.pages[c.table[0, j].long(), : len(part)] = part.bfloat16()
    c.rows[0] = rows.cpu().numpy()
    out = kv_cache.paged_attn(q, c.pages, c.table, None, torch.tensor([n - 1], device="cuda"), None, 1.0)
    torch.cuda.synchronize()
    _lib.raise_on_device_error()
    _check(out, q, lambda t, keys: c.rows[0][keys], [n - 1], None, 1.0, 0, 0)


def test_rows_of_one_sequence_padding_and_order(cuda_device):
    """Drafted tokens and a prompt's piece: several rows per sequence, in any order,
    between padding rows."""
    from spark_b200 import _lib, kv_cache

    c = Cache([400, 90, 260], 32, 512, torch.bfloat16, seed=3)
    seq = [2, 0, -1, 0, 1, 2, 2, 0, 1, -7, 0]
    pos = [259, 0, 17, 399, 89, 3, 258, 127, -1, -1, 128]
    q = torch.randn(len(seq), 64, 512, generator=c.g, device="cuda").bfloat16()
    sink = torch.randn(64, generator=c.g, device="cuda")
    out = kv_cache.paged_attn(q, c.pages, c.table, torch.tensor(seq, device="cuda"), torch.tensor(pos, device="cuda").int(),
                              sink, 0.05, window=150, first=2)
    torch.cuda.synchronize()
    _lib.raise_on_device_error()
    live = [p if s >= 0 else -1 for s, p in zip(seq, pos)]
    _check(out, q, lambda t, keys: c.rows[seq[t]][keys], live, sink, 0.05, 150, 2)
    for t, p in enumerate(live):
        if p < 0:
            assert torch.all(out[t] == 0)
    prompt = torch.arange(300, device="cuda")
    q = torch.randn(300, 16, 512, generator=c.g, device="cuda").bfloat16()
    out = kv_cache.paged_attn(q, c.pages, c.table, torch.zeros(300, dtype=torch.int64, device="cuda"), prompt, None, 0.05)
    _check(out, q, lambda t, keys: c.rows[0][keys], list(range(300)), None, 0.05, 0, 0)


@pytest.mark.parametrize("H,window", [(16, 0), (100, 60)])
def test_more_rows_than_threads(cuda_device, H, window):
    """Several rows per thread where the shares are worked out, padding among them, and
    rows of two head groups."""
    from spark_b200 import _lib, kv_cache

    c = Cache([300, 1, 77, 200], 16, 128, torch.bfloat16, seed=12)
    rng = np.random.default_rng(1)
    seq = rng.integers(-1, 4, 900)
    pos = np.array([-1 if s < 0 else int(rng.integers(0, len(c.rows[s]))) for s in seq])
    q = torch.randn(900, H, 128, generator=c.g, device="cuda").bfloat16()
    out = kv_cache.paged_attn(q, c.pages, c.table, torch.from_numpy(seq).cuda(), torch.from_numpy(pos).cuda(), None, 0.1,
                              window=window)
    torch.cuda.synchronize()
    _lib.raise_on_device_error()
    _check(out, q, lambda t, keys: c.rows[seq[t]][keys], pos.tolist(), None, 0.1, window, 0)
    assert torch.all(out[torch.from_numpy(pos < 0).cuda()] == 0)


def test_missing_pages_are_left_out_and_reported(cuda_device):
    from spark_b200 import _lib, kv_cache

    c = Cache([500, 100], 64, 512, torch.bfloat16, seed=4)
    q = torch.randn(2, 64, 512, generator=c.g, device="cuda").bfloat16()
    pos = torch.tensor([499, 99], device="cuda")
    good = c.table.clone()
    for page in (-1, c.pages.shape[0], 2 ** 31 - 1):
        c.table.copy_(good)
        c.table[0, 3] = page
        out = kv_cache.paged_attn(q, c.pages, c.table, None, pos, None, 0.05)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="cache sequence, position"):
            _lib.raise_on_device_error()

        def kv_of(t, keys):
            return c.rows[t][keys if t else keys[(keys < 192) | (keys >= 256)]]

        _check(out, q, kv_of, [499, 99], None, 0.05, 0, 0)
    c.table.copy_(good)
    for seq, p in (([0, 2], [499, 99]), ([0, 1], [499, 64 * c.table.shape[1]]), ([0, 1], [499, 2 ** 40])):
        out = kv_cache.paged_attn(q, c.pages, c.table, torch.tensor(seq, device="cuda"), torch.tensor(p, device="cuda"),
                                  None, 0.05)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="cache sequence, position"):
            _lib.raise_on_device_error()
        _check(out[:1], q[:1], lambda t, keys: c.rows[t][keys], [499], None, 0.05, 0, 0)
        assert torch.all(out[1] == 0)


def test_visible_infinities_and_nan_stay_in_their_row(cuda_device):
    from spark_b200 import kv_cache

    c = Cache([200, 200, 200], 64, 512, torch.bfloat16, seed=5)
    q = torch.randn(3, 64, 512, generator=c.g, device="cuda").bfloat16()
    c.pages[c.table[1, 1].long(), 5, 7] = float("nan")
    out = kv_cache.paged_attn(q, c.pages, c.table, None, torch.tensor([199, 199, 199], device="cuda"), None, 0.05)
    assert torch.isnan(out[1]).all()
    _check(out[::2], q[::2], lambda t, keys: c.rows[2 * t][keys], [199, 199], None, 0.05, 0, 0)


def test_extreme_sinks(cuda_device):
    """A sink of +inf takes all the weight, one of -inf none, in whole rows and in rows
    joined from pieces."""
    from spark_b200 import kv_cache

    c = Cache([40, 3000], 64, 512, torch.bfloat16, seed=7)
    q = torch.randn(2, 64, 512, generator=c.g, device="cuda").bfloat16()
    sink = torch.randn(64, generator=c.g, device="cuda")
    sink[3], sink[5], sink[6], sink[7] = float("inf"), float("-inf"), 200.0, -200.0
    pos = torch.tensor([39, 2999], device="cuda")
    out = kv_cache.paged_attn(q, c.pages, c.table, None, pos, sink, 0.05)
    assert torch.all(out[:, 3] == 0)
    keep = [h for h in range(64) if h != 3]
    _check(out[:, keep], q[:, keep], lambda t, keys: c.rows[t][keys], [39, 2999], sink[keep], 0.05, 0, 0)


def test_strides_and_layouts(cuda_device):
    from spark_b200 import kv_cache

    c = Cache([150, 40, 333], 32, 256, torch.float16, seed=6)
    pos = torch.tensor([149, 39, 332], device="cuda")
    base = torch.randn(12, 3, 264, generator=c.g, device="cuda").half()
    q = base[:, :, :256].transpose(0, 1)                                 # [3, 12, 256], heads outermost in memory
    want = kv_cache.paged_attn(q.contiguous(), c.pages, c.table, None, pos, None, 0.06)
    _check(want, q, lambda t, keys: c.rows[t][keys], pos.tolist(), None, 0.06, 0, 0)
    fused = torch.randn(3, 12 * 256 + 512, generator=c.g, device="cuda").half()
    part = fused[:, 512:].view(3, 12, 256)
    part.copy_(q)
    odd = torch.randn(3, 12, 257, generator=c.g, device="cuda").half()[..., 1:]
    odd.copy_(q)
    mixed = torch.full((c.pages.shape[0], 2, 32, 256), float("nan"), device="cuda").half()
    mixed[:, 1] = c.pages
    for x, pages in ((q, c.pages), (part, c.pages), (odd, c.pages), (q, mixed[:, 1]), (part, mixed[:, 1])):
        assert torch.equal(kv_cache.paged_attn(x, pages, c.table, None, pos, None, 0.06), want)
    none = kv_cache.paged_attn(q[:0], c.pages, c.table, None, pos[:0], None, 0.06)
    assert none.shape == (0, 12, 256)


def test_offsets_beyond_32_bits(cuda_device):
    from spark_b200 import kv_cache

    n_pages = 70000                                                      # 2.3e9 elements, 4.6 GB
    pages = torch.empty(n_pages, 64, 512, dtype=torch.bfloat16, device="cuda")
    table = torch.tensor([[n_pages - 1, 3, n_pages - 2]], dtype=torch.int32, device="cuda")
    rows = torch.randn(180, 512, device="cuda").bfloat16()
    pos = torch.arange(180, device="cuda")
    kv_cache.append(pages, rows, table, torch.zeros_like(pos), pos)
    assert torch.equal(pages[n_pages - 1], rows[:64])
    q = torch.randn(1, 64, 512, device="cuda").bfloat16()
    out = kv_cache.paged_attn(q, pages, table, None, pos[-1:], None, 0.05)
    kv = rows.double().cpu().numpy()
    _check(out, q, lambda t, keys: kv[keys], [179], None, 0.05, 0, 0)


def test_streams_and_graphs(cuda_device):
    """Two calls at once on two streams, and two captured graphs whose lengths change
    between replays."""
    from spark_b200 import _lib, kv_cache

    c = Cache([900, 77, 2000, 500], 64, 512, torch.bfloat16, seed=8)
    q = torch.randn(4, 64, 512, generator=c.g, device="cuda").bfloat16()
    pos = torch.tensor([899, 76, 1999, 499], dtype=torch.int32, device="cuda")
    want = kv_cache.paged_attn(q, c.pages, c.table, None, pos, None, 0.05)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(5):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(kv_cache.paged_attn(q, c.pages, c.table, None, pos, None, 0.05))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, kv_cache.paged_attn(q, c.pages, c.table, None, pos, None, 0.05)))
    for new in ([0, 0, 0, 0], [899, -1, 127, 128], [500, 76, 1999, 3]):
        pos.copy_(torch.tensor(new))
        for g, o in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, o in graphs:
            _check(o, q, lambda t, keys: c.rows[t][keys], new, None, 0.05, 0, 0)
    del graphs
    _lib.raise_on_device_error()


def test_raw_c_abi_and_mixed_index_types(cuda_device):
    """The C entry with a caller's workspace gives the op's bytes; sequence ids and
    positions of different widths are compared in the wider one."""
    from spark_b200 import _lib, kv_cache

    c = Cache([700, 33], 64, 512, torch.bfloat16, seed=9)
    q = torch.randn(3, 64, 512, generator=c.g, device="cuda").bfloat16()
    seq, pos = torch.tensor([1, 0, 0], device="cuda"), torch.tensor([32, 699, 5], device="cuda")
    want = kv_cache.paged_attn(q, c.pages, c.table, seq, pos, None, 0.05)
    lib = _lib.load()
    need = int(lib.dsv4_paged_attn_workspace_bytes(3, 64, 512, 64, c.table.shape[1]))
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    _lib.check(lib.dsv4_paged_attn(q.data_ptr(), 64 * 512, 512, 0, 3, 64, 512, c.pages.data_ptr(), c.pages.shape[0], 64,
                                   64 * 512, c.table.data_ptr(), 2, c.table.shape[1], seq.data_ptr(), pos.data_ptr(), 1,
                                   None, 0.05, 0, 0, out.data_ptr(), ws.data_ptr(), need, _lib.stream_ptr()),
               "dsv4_paged_attn")
    assert torch.equal(out, want)
    for s, p in ((seq.int(), pos), (seq, pos.int())):
        assert torch.equal(kv_cache.paged_attn(q, c.pages, c.table, s, p, None, 0.05), want)
    torch.cuda.synchronize()
    _lib.raise_on_device_error()
    wrapped = seq + torch.tensor([0, 2 ** 32, 0], device="cuda")
    out = kv_cache.paged_attn(q, c.pages, c.table, wrapped, pos.int(), None, 0.05)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="cache sequence, position"):
        _lib.raise_on_device_error()
    assert torch.all(out[1] == 0) and torch.equal(out[::2], want[::2])


def test_argument_checks(cuda_device):
    from spark_b200 import kv_cache

    c = Cache([100, 50], 64, 512, torch.bfloat16)
    q = torch.randn(2, 64, 512, device="cuda").bfloat16()
    pos = torch.tensor([99, 49], device="cuda")

    def call(q=q, pages=c.pages, table=c.table, seq=None, pos=pos, sink=None, **k):
        return kv_cache.paged_attn(q, pages, table, seq, pos, sink, 0.05, **k)

    call()
    for bad in (dict(q=q.half()), dict(q=q.float(), pages=c.pages.float()), dict(q=q[..., :256]), dict(q=q[0]),
                dict(pages=c.pages[:, :48]), dict(pages=c.pages[:, :, :64], q=q[..., :64]), dict(table=c.table.long()),
                dict(pos=pos[:1]), dict(pos=pos.float()), dict(seq=pos[:1]), dict(sink=torch.zeros(3, device="cuda")),
                dict(window=-1), dict(first=-1), dict(q=torch.cat((q, q)), pos=torch.cat((pos, pos))),
                dict(q=torch.cat((q, q, q), 1)), dict(pos=pos.cpu()), dict(q=q.cpu()),
                dict(pages=c.pages.repeat(1, 1, 2)[..., :640], q=torch.cat((q, q), 2)[..., :640])):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call(**bad)


def test_a_decode_loop(cuda_device):
    """The operators as they are used together: prompts are appended, steps reserve,
    rotate, append, attend and turn the output back, a sequence is forked, another
    freed, the pool moved together; beside it the same rows on plain tensors."""
    from spark_b200 import _lib
    from spark_b200.attention import sparse_attn
    from spark_b200.kv_cache import PagedKVCache
    from spark_b200.rotary import rotary, rotary_, rotary_frequencies

    g = torch.Generator(device="cuda").manual_seed(11)
    f = rotary_frequencies(64, scaling="yarn", factor=16, original_len=65536)
    cache = PagedKVCache(2, 40, 6, 700, page_size=64)
    sink = torch.randn(64, generator=g, device="cuda")
    scale = 512 ** -0.5
    plain = {}                                                            # sequence -> [rows of layer 0, of layer 1]

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    def add(seqs, counts):
        start = [plain[s][0].shape[0] if s in plain else 0 for s in seqs]
        cache.reserve(ints(seqs), ints([a + n for a, n in zip(start, counts)]))
        sid = ints([s for s, n in zip(seqs, counts) for _ in range(n)])
        pos = torch.cat([torch.arange(a, a + n) for a, n in zip(start, counts)]).int().cuda()
        for layer in range(2):
            rows = torch.randn(len(sid), 512, generator=g, device="cuda").bfloat16()
            cache.append(layer, rows, sid, pos, f)
            turned = rotary(rows[:, None], pos, f)[:, 0]                  # the same kernel arithmetic, other path
            for s in seqs:
                have = plain.setdefault(s, [torch.empty(0, 512, device="cuda").bfloat16() for _ in range(2)])
                have[layer] = torch.cat((have[layer], turned[sid == s]))

    def attend(seqs, window=0, first=0):
        pos = [plain[s][0].shape[0] - 1 for s in seqs]
        for layer in range(2):
            q = torch.randn(len(seqs), 64, 512, generator=g, device="cuda").bfloat16()
            rotary_(q, ints(pos), f)
            out = cache.attend(layer, q, ints(seqs), ints(pos), sink, scale, window=window, first=first)
            _check(out, q, lambda t, keys: plain[seqs[t]][layer][keys.tolist()].double().cpu().numpy(), pos, sink, scale,
                   window, first)
            for t, s in enumerate(seqs):                                  # and the unpaged kernel on the same rows
                kv = plain[s][layer][None]
                keys = torch.from_numpy(C.visible(pos[t], window, first)).int().cuda()[None, None]
                other = sparse_attn(q[t][None, None], kv, sink, keys, scale)[0, 0]
                # two kernels, each within 1% RMS of the formula
                assert (out[t].float() - other.float()).norm() <= 2e-2 * other.float().norm()
            back = rotary_(out.clone(), ints(pos), f, inverse=True)
            assert back.shape == out.shape

    add([0, 2, 3], [200, 64, 130])
    attend([3, 0, 2])
    for _ in range(3):
        add([0, 2, 3], [1, 1, 1])
        attend([0, 2, 3], window=128, first=4)
    cache.fork(ints([0, 3]), ints([1, 4]))
    plain[1], plain[4] = [r.clone() for r in plain[0]], [r.clone() for r in plain[3]]
    add([0, 1, 4], [1, 2, 60])                                            # both sides write behind the fork
    attend([0, 1, 2, 3, 4])
    cache.free(ints([0, 2]))
    del plain[0], plain[2]
    used = int((cache.page_refs > 0).sum())
    cache.compact()
    assert int((cache.page_refs[:used] > 0).sum()) == used and int(cache.page_refs[used:].sum()) == 0
    attend([1, 3, 4])
    add([5, 1], [300, 1])
    attend([5, 4, 3, 1])
    torch.cuda.synchronize()
    _lib.raise_on_device_error()

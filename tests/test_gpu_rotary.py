"""GPU parity of the rotary positions and of the cache append against float64
(oracle/cache_oracle.py, whose ``rotary_bound`` derives the tolerance): layouts,
types, strides, odd sizes, far positions, in place, the gradient, padding and
refused rows."""

import numpy as np
import pytest
import torch

from oracle import cache_oracle as C

pytestmark = pytest.mark.gpu

TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}


def _freqs(rot):
    from spark_b200.rotary import rotary_frequencies

    return rotary_frequencies(rot, scaling="yarn", factor=16, original_len=65536)


def _check(y, x, pos, f, offset, inter, inverse=False, amplitude=1.0):
    assert y.dtype == x.dtype and y.shape == x.shape
    x64, y64 = x.double().cpu().numpy(), y.double().cpu().numpy()
    ref = C.rotary(x64, pos.cpu().numpy(), f.cpu().numpy(), offset, inter, inverse, amplitude)
    bound = C.rotary_bound(x64, ref, f.cpu().numpy(), offset, inter, torch.finfo(x.dtype).eps, TINY[x.dtype], amplitude)
    err = np.abs(y64 - ref)
    assert np.all(err <= bound), (float((err - bound).max()), float(err.max()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("shape,rot,offset", [
    ((1, 1, 64, 512), 64, 448),    # a decode step's queries
    ((3, 7, 5, 512), 64, 448),
    ((2, 33, 3, 128), 128, 0),     # the whole head
    ((1, 70, 1, 64), 32, 16),      # channels on both sides
    ((2, 3, 2, 24), 6, 5),         # nothing aligned
    ((1, 300, 2, 130), 130, 0),    # pairs and no packs
    ((1, 2, 3, 8), 0, 0),          # nothing rotated
    ((1, 3, 1, 4096), 4096, 0),
])
def test_rotary(cuda_device, dtype, inter, shape, rot, offset):
    from spark_b200.rotary import rotary, rotary_

    g = torch.Generator(device="cuda").manual_seed(rot + shape[1])
    x = torch.randn(*shape, generator=g, device="cuda").to(dtype)
    pos = torch.randint(0, 1_000_000, shape[:2], generator=g, device="cuda")
    f = _freqs(rot) if rot else torch.zeros(0, dtype=torch.float64, device="cuda")
    for inverse, amplitude in ((False, 1.0), (True, 1.25)):
        y = rotary(x, pos, f, interleaved=inter, offset=offset, inverse=inverse, amplitude=amplitude)
        _check(y, x, pos, f, offset, inter, inverse, amplitude)
        z = x.clone()
        assert rotary_(z, pos.int(), f, interleaved=inter, offset=offset, inverse=inverse, amplitude=amplitude) is z
        assert torch.equal(z, y)


def test_rotary_keeps_the_other_channels_bits(cuda_device):
    from spark_b200.rotary import rotary

    x = torch.randint(-32768, 32767, (4, 3, 128), dtype=torch.int16, device="cuda").view(torch.bfloat16)
    y = rotary(x, torch.arange(4, device="cuda"), _freqs(64), offset=32)
    a, b = x.view(torch.int16), y.view(torch.int16)
    assert torch.equal(a[..., :32], b[..., :32]) and torch.equal(a[..., 96:], b[..., 96:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rotary_strides(cuda_device, dtype):
    from spark_b200.rotary import rotary, rotary_

    g = torch.Generator(device="cuda").manual_seed(3)
    f = _freqs(64)
    base = torch.randn(2, 5, 9, 200, generator=g, device="cuda").to(dtype)
    pos = torch.randint(0, 5000, (2, 9), generator=g, device="cuda")
    for x in (base.transpose(1, 2)[..., 8:136], base.transpose(1, 2)[..., 3:131]):  # [2, 9, 5, 128], aligned or not
        _check(rotary(x, pos, f), x, pos, f, 64, True)
        whole = base.clone()
        part = whole.transpose(1, 2)[..., 8:136]
        ref = rotary(part, pos, f, interleaved=False)
        rotary_(part, pos, f, interleaved=False)
        assert torch.equal(part, ref)
        assert torch.equal(whole[..., :8], base[..., :8]) and torch.equal(whole[..., 136:], base[..., 136:])
    x = base.permute(0, 2, 3, 1)[..., :4]                        # the last dimension strided
    f2 = _freqs(4)
    _check(rotary(x, pos, f2), x, pos, f2, 0, True)
    one = base[0, 0, 0, :64].expand(2, 9, 5, 64)                 # a broadcast input
    _check(rotary(one, pos, f), one.contiguous(), pos, f, 0, True)
    five = torch.randn(2, 3, 4, 2, 64, generator=g, device="cuda").to(dtype)
    p5 = torch.randint(0, 100, (2, 3, 4), generator=g, device="cuda")
    _check(rotary(five, p5, f), five, p5, f, 0, True)
    two = five[0, 0, 0]
    _check(rotary(two, p5[0, 0, 0], f), two, p5[0, 0, 0], f, 0, True)
    assert rotary(five[:0], p5[:0], f).shape == (0, 3, 4, 2, 64)


def test_rotary_gradient(cuda_device):
    from spark_b200.rotary import rotary

    g = torch.Generator(device="cuda").manual_seed(4)
    f = _freqs(32)
    pos = torch.randint(0, 100_000, (2, 5), generator=g, device="cuda")
    x = torch.randn(2, 5, 3, 48, generator=g, device="cuda", requires_grad=True)
    for inter in (True, False):
        w = torch.randn(2, 5, 3, 48, generator=g, device="cuda")
        y = rotary(x, pos, f, interleaved=inter, offset=8, amplitude=1.1)
        gx, = torch.autograd.grad(y, x, w)
        _check(gx, w, pos, f, 8, inter, inverse=True, amplitude=1.1)  # the formula's
        # against differences: the map is linear, so they are exact but for rounding
        d = torch.randn(2, 5, 3, 48, generator=g, device="cuda")
        with torch.no_grad():
            diff = (rotary(x + d, pos, f, interleaved=inter, offset=8, amplitude=1.1).double()
                    - rotary(x - d, pos, f, interleaved=inter, offset=8, amplitude=1.1).double()) / 2
        a, b = (diff * w.double()).sum().item(), (gx.double() * d.double()).sum().item()
        # 1440 products; each side off by at most 1e-6 (|x| + |d|) |w| per entry, of magnitude below 10 x 5
        assert abs(a - b) <= 1440 * 1e-6 * 50
    # a gradient of strides 0, a broadcast input, and a second use of one leaf
    leaf = torch.randn(48, generator=g, device="cuda", requires_grad=True)
    rotary(leaf.expand(2, 5, 3, 48), pos, f, offset=8).sum().backward()
    ref = C.rotary(np.ones((2, 5, 3, 48)), pos.cpu().numpy(), f.cpu().numpy(), 8, True, True).sum((0, 1, 2))
    assert np.abs(leaf.grad.double().cpu().numpy() - ref).max() <= 30 * 2e-6 * 2  # 30 terms of at most 2
    gg = torch.randn(2, 5, 3, 48, generator=g, device="cuda")
    y = rotary(rotary(x, pos, f), pos, f, inverse=True)
    gx, = torch.autograd.grad(y, x, gg)
    # two rotations each way: 4e-7 (|a| + |b|) twice, below 8 each
    assert (gx - gg).abs().max().item() <= 2 * 4e-7 * 16


def test_rotary_and_its_gradient_in_a_graph(cuda_device):
    from spark_b200.rotary import rotary

    f = _freqs(64)
    x = torch.randn(3, 5, 2, 64, device="cuda", requires_grad=True)
    w = torch.randn(3, 5, 2, 64, device="cuda")
    pos = torch.randint(0, 1000, (3, 5), device="cuda")

    def step():
        y = rotary(x, pos, f)
        return y.detach(), torch.autograd.grad(y, x, w)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, gx = step()
    for p in (7, 99_000):
        pos.fill_(p)
        graph.replay()
        torch.cuda.synchronize()
        _check(y, x.detach(), pos, f, 0, True)
        _check(gx, w, pos, f, 0, True, inverse=True)


def test_rotary_refusals(cuda_device):
    from spark_b200.rotary import rotary, rotary_

    f = _freqs(64)
    x = torch.randn(3, 4, 128, device="cuda")
    pos = torch.arange(3, device="cuda")
    for bad in (lambda: rotary(x, pos[:2], f), lambda: rotary(x, pos.float(), f), lambda: rotary(x, pos, f.float()),
                lambda: rotary(x, pos.cpu(), f), lambda: rotary(x, pos, f.cpu()), lambda: rotary(x.double(), pos, f),
                lambda: rotary(x, pos, f, offset=65), lambda: rotary(x, pos, f, offset=-1),
                lambda: rotary(x[..., :60], pos, f), lambda: rotary(x[0, 0], pos[0], f),
                lambda: rotary_(x[..., ::2], pos, _freqs(32)), lambda: rotary_(x[:1].expand(3, 4, 128), pos, f),
                lambda: rotary_(x.clone().requires_grad_(), pos, f),
                lambda: rotary(x, pos, _freqs(64).expand(2, 32))):
        with pytest.raises(RuntimeError):
            bad()


def _pool(rng, seqs, most, page, D, dtype, layers=None):
    n = seqs * most + 3
    order = torch.from_numpy(rng.permutation(n)[: seqs * most].reshape(seqs, most).astype(np.int32)).cuda()
    shape = (n, page, D) if layers is None else (layers, n, page, D)
    return order, torch.full(shape, 7.0, dtype=dtype, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,D,page,rot,inter", [
    (1, 512, 64, 64, True), (3, 512, 16, 64, False), (37, 128, 32, 128, True), (200, 256, 64, 0, True),
    (19, 40, 5, 6, False), (8, 512, 1, 512, True),
])
def test_append(cuda_device, dtype, T, D, page, rot, inter):
    from spark_b200 import _lib, kv_cache

    rng = np.random.default_rng(T + D)
    seqs, most = 5, 12
    table, pages = _pool(rng, seqs, most, page, D, dtype)
    places = rng.permutation(seqs * most * page)[:T]
    seq, pos = torch.from_numpy(places // (most * page)).cuda(), torch.from_numpy(places % (most * page)).cuda()
    rows = torch.randn(T, D, device="cuda").to(dtype)
    f = _freqs(rot) if rot else None
    want = pages.clone()
    at = table.long()[seq, pos // page], pos % page
    for s, p, r in ((seq.int(), pos.int(), rows), (seq, pos, torch.cat((rows[:, :1], rows, rows), 1)[:, 1:D + 1])):
        pages.fill_(7.0)
        kv_cache.append(pages, r, table, s, p, f, interleaved=inter)
        torch.cuda.synchronize()
        _lib.raise_on_device_error()
        if rot:
            _check(pages[at][:, None], rows[:, None], pos, f, D - rot, inter)
        else:
            assert torch.equal(pages[at], rows)
        want[at] = pages[at]
        assert torch.equal(pages, want)  # everything else as it was


def test_append_padding_bad_rows_and_other_layouts(cuda_device):
    from spark_b200 import _lib, kv_cache

    rng = np.random.default_rng(0)
    table, pages = _pool(rng, 3, 4, 16, 128, torch.bfloat16)
    table[1, 2:] = -1
    rows = torch.randn(6, 128, device="cuda").bfloat16()
    seq = torch.tensor([0, -1, 1, 2, 0, 1], device="cuda")
    pos = torch.tensor([5, 3, -1, 63, 6, 31], device="cuda")
    kv_cache.append(pages, rows, table, seq, pos)
    torch.cuda.synchronize()
    _lib.raise_on_device_error()  # padding is no error
    want = torch.full_like(pages, 7.0)
    for i in (0, 3, 4, 5):
        want[table[seq[i], pos[i] // 16].long(), pos[i] % 16] = rows[i]
    assert torch.equal(pages, want)
    for s, p in ((3, 0), (1, 32), (0, 64), (2 ** 40, 0), (0, 2 ** 40), (0, 2 ** 31 - 1)):
        kv_cache.append(pages, rows[:1], table, torch.tensor([s], device="cuda"), torch.tensor([p], device="cuda"))
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="cache sequence, position"):
            _lib.raise_on_device_error()
    assert torch.equal(pages, want)
    bad = table.clone()
    bad[0, 0] = pages.shape[0]
    kv_cache.append(pages, rows[:1], bad, None, torch.zeros(1, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="cache sequence, position"):
        _lib.raise_on_device_error()
    # one layer of [P, L, page, D]: a page stride that skips the other layers
    mixed = torch.full((pages.shape[0], 3, 16, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    kv_cache.append(mixed[:, 1], rows, table, seq, pos)
    torch.cuda.synchronize()
    _lib.raise_on_device_error()
    assert torch.equal(mixed[:, 1], want) and torch.all(mixed[:, 0] == 7) and torch.all(mixed[:, 2] == 7)
    kv_cache.append(pages, rows[:0], table, seq[:0], pos[:0])
    for bad_call in (lambda: kv_cache.append(pages, rows.half(), table, seq, pos),
                     lambda: kv_cache.append(pages, rows[:, :64], table, seq, pos),
                     lambda: kv_cache.append(pages, rows, table, seq[:3], pos),
                     lambda: kv_cache.append(pages, rows, table.long(), seq, pos),
                     lambda: kv_cache.append(pages, rows, table, None, pos),       # six rows, three sequences
                     lambda: kv_cache.append(pages.float(), rows.float(), table, seq, pos),
                     lambda: kv_cache.append(pages[:, ::2], rows, table, seq, pos),
                     lambda: kv_cache.append(pages[:, :, :120], rows[:, :120], table, seq, pos),
                     lambda: kv_cache.append(pages, rows, table, seq.cpu(), pos)):
        with pytest.raises(RuntimeError):
            bad_call()

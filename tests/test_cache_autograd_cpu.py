"""How the attention cache's operators answer torch's autograd, on meta tensors: what
is shared by every device lies above the kernels."""

import contextlib

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


def _calls(op, made=contextlib.nullcontext):
    """Every operator that writes: the call, and the tensors it writes, which come into
    being under ``made``."""
    def ints(*shape):
        return torch.empty(*shape, dtype=torch.int32, device=META)

    def bf16(*shape):
        return torch.empty(*shape, dtype=torch.bfloat16, device=META)

    with made():
        x = _rotary_args()[0]
        pages, table, lens, refs = bf16(2, 9, 16, 64), ints(4, 8), ints(4), ints(9)
        layer = pages[0]
    _, pos, f = _rotary_args()
    rows, ids, f16 = bf16(2, 64), ints(2), torch.empty(16, dtype=torch.float64, device=META)
    return {
        "rotary_": (lambda: op.rotary_(x, pos, f), [x]),
        "cache_append": (lambda: op.cache_append(layer, rows, table, ids, ids, f16), [pages]),
        "cache_reserve": (lambda: op.cache_reserve(table, lens, refs, ids, ids, 16), [table, lens, refs]),
        "cache_free": (lambda: op.cache_free(table, lens, refs, ids), [table, lens, refs]),
        "cache_fork": (lambda: op.cache_fork(pages, table, lens, refs, ids, ids), [pages, table, lens, refs]),
        "cache_compact": (lambda: op.cache_compact(pages, table, refs), [pages, table, refs]),
        "cache_copy": (lambda: op.cache_copy(pages, ids, ids), [pages]),
    }


WRITING = ["rotary_", "cache_append", "cache_reserve", "cache_free", "cache_fork", "cache_compact", "cache_copy"]


@pytest.mark.parametrize("name", WRITING)
def test_what_is_written_gets_a_new_version(dsv4, name):
    """Also through a view (a layer of the pages), under no_grad and in inference mode, as
    torch's own in-place operators do; what is only read keeps its version."""
    call, written = _calls(dsv4)[name]
    for mode in (torch.enable_grad, torch.no_grad, torch.inference_mode):
        before = [t._version for t in written]
        with mode():
            call()
        assert [t._version for t in written] == [v + 1 for v in before]
    with torch.inference_mode():
        _calls(dsv4)[name][0]()  # on inference tensors, which have no version


def test_a_tensor_turned_in_place_is_refused_by_an_earlier_backward(dsv4):
    x, pos, f = _rotary_args()
    w = torch.empty_like(x, requires_grad=True)
    z = (x * w).sum()
    dsv4.rotary_(x, pos, f)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    y = dsv4.rotary(w, pos, f).sum()
    pos.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def _attn_args():
    return {"q": torch.empty(3, 16, 128, dtype=torch.bfloat16, device=META),
            "pages": torch.empty(9, 16, 128, dtype=torch.bfloat16, device=META),
            "table": torch.empty(4, 8, dtype=torch.int32, device=META),
            "seq": torch.empty(3, dtype=torch.int32, device=META), "pos": torch.empty(3, dtype=torch.int32, device=META),
            "sink": torch.empty(16, device=META)}


def _refused(call, tensors):
    """Refused where one of the tensors requires a gradient or has a tangent; not under
    no_grad, nor where none does."""
    call(tensors)
    for name, t in tensors.items():
        if not t.is_floating_point():
            continue
        needs = dict(tensors, **{name: t.clone().requires_grad_()})
        with pytest.raises(RuntimeError, match="no gradient"):
            call(needs)
        with torch.no_grad():
            call(needs)
        with fw.dual_level():
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(RuntimeError, match="no gradient"):
                    call(dict(tensors, **{name: fw.make_dual(t.clone(), torch.empty_like(t))}))


def test_operators_without_a_gradient_refuse_one(dsv4):
    _refused(lambda a: dsv4.paged_attn(a["q"], a["pages"], a["table"], a["seq"], a["pos"], a["sink"], 0.1), _attn_args())
    a = _attn_args()
    a["rows"], a["f"] = torch.empty(3, 128, dtype=torch.bfloat16, device=META), torch.empty(32, dtype=torch.float64, device=META)
    del a["q"], a["sink"]
    _refused(lambda a: dsv4.cache_append(a["pages"], a["rows"], a["table"], a["seq"], a["pos"], a["f"]), a)
    x, pos, f = _rotary_args()
    _refused(lambda a: dsv4.rotary_(a["x"], pos, a["f"]), {"x": x, "f": f})
    _refused(lambda a: dsv4.rotary(x, pos, a["f"]), {"f": f})
    ids, lens, refs = (torch.empty(n, dtype=torch.int32, device=META) for n in (2, 4, 9))
    table, pages = _attn_args()["table"], {"pages": _attn_args()["pages"]}
    _refused(lambda a: dsv4.cache_fork(a["pages"], table, lens, refs, ids, ids), pages)
    _refused(lambda a: dsv4.cache_compact(a["pages"], table, refs), pages)
    _refused(lambda a: dsv4.cache_copy(a["pages"], ids, ids), pages)


@pytest.mark.parametrize("name", WRITING)
def test_tensors_made_in_inference_mode_are_written_outside_of_it(dsv4, name):
    """A cache made in inference mode has no versions to raise; beside ordinary ids and
    positions it is written outside of inference mode too."""
    call, written = _calls(dsv4, torch.inference_mode)[name]
    assert all(t.is_inference() for t in written)
    with torch.no_grad():
        call()
    call()

"""Rows of logits: what can be checked of their entry points without a GPU."""
import copy
import ctypes as C
import pickle

import pytest
import torch

from gan_amd import _abi
from gan_amd import logits as L

P = C.c_void_p(4096)      # never read: every call that is given it is refused on its sizes


def test_a_teachers_rows_are_three_tensors():
    """The temperature that the log-sum-exp was taken at goes along, but is not one of them."""
    values, index, lse = torch.randn(4, 2), torch.zeros(4, 2, dtype=torch.int32), torch.randn(4)
    top = L.TopRows(values, index, lse, 2.0)
    assert len(top) == 3 and all(a is b for a, b in zip(top, (values, index, lse)))
    assert all(torch.is_tensor(v) for v in tuple(top))
    v, i, s = top
    assert v is top.values and i is top.index and s is top.lse and top.temperature == 2.0
    assert L.TopRows(values, index, lse).temperature is None and L.TopRows(values, index, None).lse is None
    assert L.TopRows(values=values, index=index, lse=lse, temperature=0.5).temperature == 0.5
    moved = top._replace(index=index + 1)
    assert type(moved) is L.TopRows and moved.temperature == 2.0 and moved.values is values and int(moved.index[0, 0]) == 1
    assert top._replace(temperature=3.0).temperature == 3.0 and top.temperature == 2.0
    with pytest.raises(ValueError):
        top._replace(places=index)
    for other in (copy.copy(top), copy.deepcopy(top), pickle.loads(pickle.dumps(top))):
        assert type(other) is L.TopRows and other.temperature == 2.0 and torch.equal(other.lse, lse)


@pytest.mark.parametrize("seen", ["slice", "expanded", "dense"])
@pytest.mark.parametrize("copy_of", ["dense", "by columns", "wider", "none"])
def test_a_copy_of_saved_logits_has_strides_of_its_own(monkeypatch, seen, copy_of):
    """The backward pass passes the kernel what a hook on saved tensors hands back, with that tensor's strides.  (What would be
    launched is looked at instead.)"""
    rows, width, wide = 6, 5, 12
    launched = []
    monkeypatch.setattr(L, "_rows_of", lambda t, what: (t.size(0), t.size(1), t.stride(0), 0))
    monkeypatch.setattr(L, "_call", lambda name, device, *args, meta=None: launched.append((name, args[0]._obj)) if name == "aig_distill_rows" else None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    whole = torch.randn(rows, wide).requires_grad_(True)
    x = whole[:, :width] if seen == "slice" else whole[:1, :width].expand(rows, width) if seen == "expanded" else whole[:, :width].contiguous()
    top = L.TopRows(torch.randn(rows, 2), torch.zeros(rows, 2, dtype=torch.int32), torch.zeros(rows), 1.0)
    handed = {}

    def unpack(t):
        if not t.is_floating_point() or t.shape != (rows, width):
            return t if copy_of == "none" else t.clone()
        if copy_of == "dense":
            t = t.clone(memory_format=torch.contiguous_format)
        elif copy_of == "by columns":
            t = t.t().contiguous().t()
        elif copy_of == "wider":
            t = torch.cat([t, torch.zeros(rows, 3)], dim=1)[:, :width]
        handed["x"] = t
        return t

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        loss = L.distill_loss(x, top, reduction="none")
    loss.backward(torch.ones(rows))
    (_, forth), (_, back) = launched
    assert forth.ld == x.stride(0) and forth.logits == x.data_ptr()
    t = handed["x"]
    if copy_of == "by columns":          # rows whose logits are apart are laid out anew
        assert back.logits != t.data_ptr() and back.ld == width
    else:
        assert back.logits == t.data_ptr() and back.ld == t.stride(0)
    assert (back.rows, back.width, back.m) == (rows, width, 2)
    assert forth.logits == x.data_ptr() and forth.ld == x.stride(0)        # (what was kept stays what it was)


@pytest.mark.parametrize("change", [lambda t: t.bfloat16(), lambda t: t[:-1].clone(), lambda t: t[:, :-1].clone()])
def test_saved_tensors_that_come_back_as_others_are_refused(monkeypatch, change):
    monkeypatch.setattr(L, "_rows_of", lambda t, what: (t.size(0), t.size(1), t.stride(0), 0))
    monkeypatch.setattr(L, "_call", lambda *args, **kw: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    x, values = torch.randn(6, 5, requires_grad=True), torch.randn(6, 2)
    top = L.TopRows(values, torch.zeros(6, 2, dtype=torch.int32), torch.zeros(6), 1.0)
    for shape in ((6, 5), (6, 2)):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: change(t) if t.is_floating_point() and t.shape == shape else t):
            loss = L.distill_loss(x, top, reduction="none")
        with pytest.raises(_abi.AigAbiError, match="saved (logits|values) must be"):
            loss.backward(torch.ones(6))


@pytest.mark.parametrize("rows", [(1 << 26) - 3, (1 << 26) - 1])
def test_rows_that_round_up_to_a_launch_too_large(rows):
    """64 lanes a row and four rows a workgroup: 2^32 threads and more are not launched."""
    how = _abi.Sampling(temperature=1.0, top_p=1.0)
    lib = _abi.lib()
    assert lib.aig_sample_rows(rows, 600, 600, 0, P, None, None, C.byref(how), 1, P, P, None) == -4
    assert lib.aig_top_rows(rows, 600, 600, 0, P, None, 4, 1.0, P, P, P, None) == -4
    a = _abi.Distill(rows=rows, width=600, ld=600, m=2, dtype=0, temperature=1.0, scale=1.0, logits=4096, values=4096, index=4096)
    assert lib.aig_distill_rows(C.byref(a), P, None, 0, None, 0, None) == -4


@pytest.mark.parametrize("rows,width,forth", [(600_000_000, 5, True), (2 ** 31 - 1, 2, True), (300_000_000, 9, True), (2 ** 31 - 1, 1, False)])
def test_windows_that_take_a_launch_too_large(rows, width, forth):
    """Fewer than 2^32 places, but a power of two of lanes a row (four of every row for the table's gradient)."""
    a = _abi.ScoreWindowsArg(rows=rows, width=width, nodes=5, kinds=2, classes=3, cand=4096, cls=4096, row_kind=4096, by_kind=4096, kind_start=4096)
    lib = _abi.lib()
    if forth:
        assert lib.aig_class_scores(C.byref(a), P, P, None) == -4
    if rows > (1 << 30):
        assert lib.aig_class_scores_bwd(C.byref(a), P, P, P, 1 << 50, None) == -4

"""Rows of logits: what can be checked of their entry points without a GPU."""
import copy
import pickle

import pytest
import torch

from gan_amd import logits as L


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

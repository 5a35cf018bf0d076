"""Checks of the learning operators' arguments (bundlesdf_amd/learn_ops.py) that need no GPU."""
import pytest
import torch

from bundlesdf_amd import learn_ops as L
from bundlesdf_amd import lib


def test_what_a_new_state_overlaps():
    line = torch.zeros(100)
    a = line[10:34].view(4, 6)

    def clear(x):
        return L._clear_of(a.data_ptr(), a.data_ptr() + 96, 6, x, x.data_ptr(), x.stride(0))

    assert clear(a) and clear(line[34:58].view(4, 6)) and clear(line[0:10].view(2, 5)) and clear(line[:0].view(0, 6))
    for lo in (5, 9, 11, 33):
        assert not clear(line[lo:lo + 24].view(4, 6)), lo
    assert not clear(line[10:34].view(6, 4)) and not clear(line[33:34].view(1, 1)) and not clear(a.view(torch.int32)) and not clear(a[:, :5])
    assert clear(line[34:35].view(1, 1)) and clear(line[9:10].view(1, 1))
    assert not clear(line.view(4, 25)[:, :2]) and not clear(line[8:9].view(1, 1).expand(4, 1).as_strided((4, 1), (1, 1)))
    assert clear(line[8:9].view(1, 1).expand(4, 6)[:, :1])                                # one element for every row


def test_steps_are_judged_before_anything_is_made_of_them():
    for steps in (0, -1, 33, 10 ** 12):
        with pytest.raises(lib.NofError, match='steps'):
            L.orthogonalize(torch.zeros(4, 6), steps=steps)
    with pytest.raises(lib.NofError, match='triple'):
        L.orthogonalize(torch.zeros(4, 6), coefficients=())

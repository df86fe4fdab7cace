"""Numbers that stand for positions and rows are whole ones: a fraction is refused, not cut."""

import numpy as np
import pytest
import torch

import kotodama_amd


class _Stop(Exception):
    pass


@pytest.fixture
def taken(monkeypatch):
    """What reaches the calls, in place of them."""
    seen = []

    class Native:
        def attention(self, *a):
            seen.append(a[7])
            raise _Stop

        def embedding(self, *a):
            seen.append(a[3])
            raise _Stop

    monkeypatch.setattr(kotodama_amd.lmops, "native", Native())
    return seen


def test_q_start_is_a_whole_number(taken):
    t = torch.empty(1, 1, 4, 64)
    for bad in (1.5, 2.0, np.float32(3), "4"):
        with pytest.raises(TypeError):
            kotodama_amd.attention(t, t, t, q_start=bad)
    assert taken == []
    for good in (3, np.int64(3)):
        with pytest.raises(_Stop):
            kotodama_amd.attention(t, t, t, q_start=good)
    assert taken == [3, 3]


def test_padding_idx_is_a_whole_number(taken):
    ids, w = torch.zeros(3, dtype=torch.int64), torch.empty(5, 8)
    for bad in (0.5, 2.0, "1"):
        with pytest.raises(TypeError):
            kotodama_amd.embedding(ids, w, padding_idx=bad)
    assert taken == []
    for good, row in ((2, 2), (np.int32(-1), 4)):
        with pytest.raises(_Stop):
            kotodama_amd.embedding(ids, w, padding_idx=good)
        assert taken[-1] == row and type(taken[-1]) is int

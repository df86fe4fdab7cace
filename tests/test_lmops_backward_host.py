"""What the language-model operators' registered backward ops refuse, on the
CPU: gradients and saved results that do not fit the call's sizes and types
never reach the C calls, which take the sizes from q, k and ids."""

import contextlib

import pytest
import torch

from kotodama_amd import _capi, lmops

BF, FP = torch.bfloat16, torch.float32


@pytest.fixture
def launches(monkeypatch):
    """The backward calls that would have been launched, with CPU tensors let through."""
    calls = []
    monkeypatch.setattr(lmops, "_require_device", lambda *tensors: torch.device("cpu"))
    monkeypatch.setattr(lmops, "_DeviceStream", lambda device: contextlib.nullcontext(0))
    for name in ("attention", "qk_norm_rope", "embedding"):
        monkeypatch.setattr(_capi, f"{name}_workspace_size", lambda *a: 4)
        monkeypatch.setattr(_capi, f"{name}_bwd", lambda *a, name=name: calls.append(name))
    return calls


def _t(shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


def _attention(out=(2, 4, 5, 64), lse=(2, 4, 5), go=(2, 4, 5, 64), gl=None, odt=BF, ldt=FP, gdt=BF):
    q, k = _t((2, 4, 5, 64)), _t((2, 2, 7, 64))
    return lmops.attention_bwd_op(q, k, k.clone(), _t(out, odt), _t(lse, ldt), _t(go, gdt),
                                  None if gl is None else _t(gl, FP), True, 0.1, None, None, 0)


def test_attention_backward_refusals(launches):
    _attention()
    _attention(gl=(2, 4, 5), gdt=FP)
    assert launches == ["attention"] * 2
    for kw in (dict(out=(2, 4, 4, 64)), dict(out=(2, 4, 5, 32)), dict(out=(5, 64)), dict(lse=(4,)), dict(lse=(2, 5, 4)),
               dict(lse=(2, 4, 5, 1)), dict(go=(2, 4, 1, 64)), dict(go=(1, 4, 5, 64)), dict(go=(2, 4, 5)),
               dict(gl=(2, 4, 4)), dict(gl=(1,))):
        with pytest.raises(ValueError, match="attention_bwd"):
            _attention(**kw)
    for kw in (dict(ldt=BF), dict(ldt=torch.float64), dict(odt=FP), dict(odt=torch.float16)):
        with pytest.raises(TypeError, match="attention_bwd"):
            _attention(**kw)
    assert launches == ["attention"] * 2


def _qk(gq=(2, 4, 5, 64), gk=(2, 2, 5, 64)):
    w, tab = _t((64,)), _t((9, 64))
    return lmops.qk_norm_rope_bwd_op(_t((2, 4, 5, 64)), _t((2, 2, 5, 64)), w, w.clone(), tab, tab.clone(), None, 1e-5,
                                     _t(gq), _t(gk))


def test_qk_norm_rope_backward_refusals(launches):
    _qk()
    assert launches == ["qk_norm_rope"]
    for kw in (dict(gq=(2, 4, 4, 64)), dict(gq=(2, 2, 5, 64)), dict(gq=(64,)), dict(gk=(2, 2, 5, 32)), dict(gk=(1, 2, 5, 64))):
        with pytest.raises(ValueError, match="qk_norm_rope_bwd"):
            _qk(**kw)
    assert launches == ["qk_norm_rope"]


def _embedding(ids=(4, 25), go=(4, 25, 8), rows=30, pad=-1, dtype=torch.int64, gdt=BF):
    return lmops.embedding_bwd_op(torch.zeros(ids, dtype=dtype), _t(go, gdt), rows, 1.0, pad)


def test_embedding_backward_refusals(launches):
    _embedding()
    _embedding(ids=(), go=(8,))
    assert launches == ["embedding"] * 2
    for kw in (dict(go=(10, 8)), dict(go=(100, 8)), dict(go=(4, 26, 8)), dict(go=(4, 25)), dict(go=(4, 25, 0)),
               dict(ids=(), go=()), dict(rows=-1), dict(pad=-2), dict(pad=30)):
        with pytest.raises(ValueError, match="embedding_bwd"):
            _embedding(**kw)
    for kw in (dict(dtype=torch.int16), dict(gdt=torch.float16)):
        with pytest.raises(TypeError):
            _embedding(**kw)
    # a row that 32 bits do not count (its one element read over and over)
    wide = torch.zeros((1,), dtype=BF).expand(1, 1 << 31)
    with pytest.raises(ValueError, match="2\\^31"):
        lmops._embedding_bwd_impl(torch.zeros(1, dtype=torch.int64), wide, 1, 1.0, -1)
    assert launches == ["embedding"] * 2

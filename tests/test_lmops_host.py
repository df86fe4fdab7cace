"""The language-model operators' checks of arguments, on the CPU: what the
Python layer and the C ABI refuse, before anything reaches a GPU."""

import ctypes

import pytest
import torch

import kotodama_amd
from kotodama_amd import _capi, lmops

FAKE = 0x7F0000000000  # never dereferenced: argument checks run first
BF, F32 = _capi.DTYPE_BF16, _capi.DTYPE_F32


def _st(b, h, t):
    return (ctypes.c_int64 * 3)(b, h, t)


@pytest.mark.parametrize("call", [
    lambda t: kotodama_amd.attention(t(2, 2, 4, 64), t(2, 2, 4, 64), t(2, 2, 4, 64)),
    lambda t: kotodama_amd.qk_norm_rope(t(2, 2, 4, 64), t(2, 2, 4, 64), t(64), t(64), t(4, 64).detach(),
                                        t(4, 64).detach(), 1e-5),
    lambda t: kotodama_amd.embedding(torch.zeros(3, dtype=torch.int64), t(5, 8)),
])
@pytest.mark.parametrize("grad", [False, True])
def test_cpu_tensors_raise(call, grad):
    with pytest.raises(RuntimeError, match="no CPU path"):
        call(lambda *s: torch.ones(s, dtype=torch.bfloat16, requires_grad=grad))


def _attn(q=(2, 4, 5, 64), k=(2, 2, 7, 64), v=None, dt=torch.bfloat16, kdt=None, lens=None, start=None):
    t = lambda s, d: torch.empty(s, dtype=d)  # noqa: E731
    lmops._check_attention(t(q, dt), t(k, kdt or dt), t(v or k, dt), lens, start)


def test_attention_refusals():
    _attn()
    for kw in (dict(q=(2, 4, 64)), dict(v=(2, 2, 6, 64)), dict(q=(3, 4, 5, 64)), dict(q=(2, 4, 5, 32)),
               dict(q=(2, 3, 5, 64)), dict(k=(2, 0, 7, 64)), dict(q=(2, 4, 5, 68), k=(2, 2, 7, 68)),
               dict(q=(2, 4, 5, 136), k=(2, 2, 7, 136)), dict(lens=torch.zeros(3, dtype=torch.int32)),
               dict(start=torch.zeros((2, 1), dtype=torch.int64))):
        with pytest.raises(ValueError, match="attention"):
            _attn(**kw)
    for kw in (dict(dt=torch.float16), dict(dt=torch.float64), dict(kdt=torch.float32), dict(lens=torch.zeros(2)),
               dict(start=torch.zeros(2, dtype=torch.int16))):
        with pytest.raises(TypeError):
            _attn(**kw)
    t = torch.empty(1, 1, 1, 64)
    with pytest.raises(ValueError, match="q_start"):
        kotodama_amd.attention(t, t, t, q_start=1 << 41)
    for scale in (0.0, -0.5, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            kotodama_amd.attention(t, t, t, scale=scale)
    with pytest.raises(TypeError, match="kv_lens"):
        kotodama_amd.attention(t, t, t, kv_lens=[1])


def test_sizes_over_32_bits_are_refused():
    lmops._check_sizes("x", torch.empty((2**31 - 1, 2), device="meta"), torch.empty((), device="meta"))
    with pytest.raises(ValueError, match="2\\^31"):
        lmops._check_sizes("x", torch.empty((1, 2**31), device="meta"))


def test_qk_norm_rope_refusals():
    def check(q=(2, 4, 5, 64), k=(2, 2, 5, 64), w=(64,), cos=(9, 64), sin=None, dt=torch.bfloat16, tdt=None, pos=None,
              wdt=None):
        t = lambda s, d: torch.empty(s, dtype=d)  # noqa: E731
        lmops._check_qk(t(q, dt), t(k, dt), t(w, wdt or dt), t(w, dt), t(cos, tdt or dt), t(sin or cos, tdt or dt), pos)

    check()
    check(tdt=torch.float32)
    check(pos=torch.zeros(5, dtype=torch.int32))
    for kw in (dict(k=(2, 2, 6, 64)), dict(q=(2, 5, 64)), dict(w=(63,)), dict(cos=(9, 32)), dict(sin=(8, 64)),
               dict(cos=(4, 64)), dict(q=(2, 4, 5, 63), k=(2, 2, 5, 63), w=(63,), cos=(9, 63)),
               dict(q=(2, 4, 5, 258), k=(2, 2, 5, 258), w=(258,), cos=(9, 258)),
               dict(pos=torch.zeros((3, 5), dtype=torch.int64)), dict(pos=torch.zeros(4, dtype=torch.int64))):
        with pytest.raises(ValueError, match="qk_norm_rope"):
            check(**kw)
    for kw in (dict(dt=torch.float16), dict(wdt=torch.float32), dict(tdt=torch.float64),
               dict(dt=torch.float32, tdt=torch.bfloat16), dict(pos=torch.zeros(5))):
        with pytest.raises(TypeError):
            check(**kw)
    leaf = torch.ones(4, 64, requires_grad=True)
    with pytest.raises(NotImplementedError, match="no gradient"):
        kotodama_amd.qk_norm_rope(torch.ones(1, 1, 4, 64), torch.ones(1, 1, 4, 64), torch.ones(64), torch.ones(64),
                                  leaf, leaf, 1e-5)


def test_embedding_refusals():
    ids = torch.zeros(3, dtype=torch.int64)
    lmops._check_embedding(ids, torch.ones(5, 8), -1)
    for args in ((ids, torch.ones(5), -1), (ids, torch.ones(5, 0), -1)):
        with pytest.raises(ValueError, match="embedding"):
            lmops._check_embedding(*args)
    for args in ((ids.float(), torch.ones(5, 8), -1), (ids, torch.ones(5, 8, dtype=torch.float16), -1),
                 (ids.to(torch.int16), torch.ones(5, 8), -1)):
        with pytest.raises(TypeError):
            lmops._check_embedding(*args)
    for pad in (5, -6):
        with pytest.raises(ValueError, match="padding_idx"):
            kotodama_amd.embedding(ids, torch.ones(5, 8), padding_idx=pad)


def attention_fwd(b=2, h=4, hk=2, tq=5, tk=7, d=64, dt=BF, causal=1, scale=0.1, q=FAKE, st=None, index=0, out=FAKE,
                  lens=None):
    st = _st(*(st or (4096, 64, 256)))
    return _capi.lib().attnres_attention_fwd(q, st, FAKE, st, FAKE, st, b, h, hk, tq, tk, d, dt, causal, scale, lens,
                                             None, index, 0, out, st, None, None, 0, None)


def test_attention_abi_refusals():
    assert attention_fwd(b=0) == _capi.OK  # nothing to do: returns before any HIP call
    assert attention_fwd(tq=0) == _capi.OK
    for kw in (dict(b=-1), dict(h=3), dict(hk=0), dict(tq=-1), dict(dt=5), dict(causal=2), dict(scale=float("nan")), dict(scale=0.0),
               dict(scale=-1.0), dict(scale=3e38), dict(q=None), dict(out=None), dict(index=7)):
        assert attention_fwd(**kw) == _capi.ERR_ARG, kw
    for kw in (dict(d=4), dict(d=68), dict(d=136), dict(tk=1 << 31), dict(b=1 << 20, tq=1 << 20),
               dict(h=8194, hk=2), dict(st=(4096, 64, 1 << 24))):
        assert attention_fwd(**kw) == _capi.ERR_UNSUPPORTED, kw
    for kw in (dict(q=FAKE + 8), dict(st=(4096, 64, 257)), dict(lens=FAKE + 2), dict(lens=FAKE + 4, index=1)):
        assert attention_fwd(**kw) == _capi.ERR_ALIGN, kw


def test_attention_backward_abi_refusals():
    def bwd(lse=FAKE, ws=FAKE, nbytes=1 << 30, dk=FAKE, b=2):
        st = _st(4096, 64, 256)
        return _capi.lib().attnres_attention_bwd(
            FAKE, st, FAKE, st, FAKE, st, FAKE, st, FAKE, st, lse, None, b, 4, 2, 5, 7, 64, BF, 1, 0.1, None, None, 0, 0,
            FAKE, st, dk, st, FAKE, st, ws, nbytes, None)

    assert bwd(b=0) == _capi.OK
    assert bwd(lse=None) == _capi.ERR_ARG
    assert bwd(ws=None) == _capi.ERR_ARG
    assert bwd(nbytes=8) == _capi.ERR_ARG
    assert bwd(dk=None) == _capi.ERR_ARG
    assert bwd(ws=FAKE + 4) == _capi.ERR_ALIGN
    with pytest.raises(_capi.AttnResError, match="head_dim 300"):
        _capi.attention_workspace_size(1, 1, 1, 1, 1, 300, BF, 1)


def test_qk_norm_rope_abi_refusals():
    def fwd(b=2, t=5, d=64, dt=BF, tdt=BF, q=FAKE, w=FAKE, cos=FAKE, ld=64, eps=1e-5, pos=None, index=0, rows=9):
        st = _st(4096, 64, 256)
        return _capi.lib().attnres_qk_norm_rope_fwd(q, st, FAKE, st, b, 4, 2, t, d, dt, w, FAKE, cos, ld, FAKE, ld, rows,
                                                    tdt, pos, index, 0, 1, eps, FAKE, st, None, st, None)

    assert fwd(b=0) == _capi.OK
    assert fwd(t=0) == _capi.OK
    for kw in (dict(b=-1), dict(dt=9), dict(tdt=9), dict(dt=F32, tdt=BF), dict(q=None), dict(w=None), dict(cos=None),
               dict(ld=63), dict(eps=-1.0), dict(eps=float("nan")), dict(index=3), dict()):  # k_out is NULL in all
        assert fwd(**kw) == _capi.ERR_ARG, kw
    for kw in (dict(d=3), dict(d=258), dict(b=1 << 20, t=1 << 20)):
        assert fwd(**kw) == _capi.ERR_UNSUPPORTED, kw
    for kw in (dict(q=FAKE + 1), dict(cos=FAKE + 1), dict(pos=FAKE + 2)):
        assert fwd(**kw) == _capi.ERR_ALIGN, kw


def test_embedding_abi_refusals():
    def fwd(ids=FAKE, n=5, rows=9, hidden=64, ld=64, dt=BF, scale=1.0, out=FAKE, index=1):
        return _capi.lib().attnres_embedding_fwd(ids, index, n, FAKE, ld, rows, hidden, dt, scale, out, None)

    def bwd(g=FAKE, rows=9, ld=64, pad=-1, ws=FAKE, nbytes=1 << 30, dw=FAKE):
        return _capi.lib().attnres_embedding_bwd(FAKE, 1, 5, g, ld, rows, 64, BF, 1.0, pad, dw, ws, nbytes, None)

    assert fwd(n=0) == _capi.OK
    for kw in (dict(ids=None), dict(n=-1), dict(hidden=0), dict(ld=63), dict(dt=4), dict(scale=float("inf")),
               dict(out=None), dict(index=2)):
        assert fwd(**kw) == _capi.ERR_ARG, kw
    assert fwd(n=1 << 31) == _capi.ERR_UNSUPPORTED
    assert fwd(hidden=1 << 24, ld=1 << 24) == _capi.ERR_UNSUPPORTED
    assert fwd(ids=FAKE + 4) == _capi.ERR_ALIGN
    assert fwd(out=FAKE + 1) == _capi.ERR_ALIGN
    assert bwd(rows=0) == _capi.OK
    for kw in (dict(g=None), dict(ld=63), dict(pad=-2), dict(ws=None), dict(nbytes=100), dict(dw=None)):
        assert bwd(**kw) == _capi.ERR_ARG, kw
    assert bwd(ws=FAKE + 8) == _capi.ERR_ALIGN
    assert _capi.embedding_workspace_size(0, 0, 8) >= 0

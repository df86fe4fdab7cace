"""The paged-cache operators' checks of arguments, on the CPU: what the Python layer
and the C ABI refuse, before anything reaches a GPU."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import kotodama_amd
from kotodama_amd import _capi, lmstep, paged

FAKE = 0x7F0000000000  # never dereferenced: argument checks run first
BF, F32 = _capi.DTYPE_BF16, _capi.DTYPE_F32
I32, I64 = torch.int32, torch.int64


def _z(*s, dtype=I32):
    return torch.zeros(s, dtype=dtype)


def _b(*s, dtype=torch.bfloat16):
    return torch.ones(s, dtype=dtype)


CALLS = {
    "slots": lambda: kotodama_amd.paged_slots(_z(2, 4), _z(2), _z(2), _z(9), _z(1), 16, 5),
    "release": lambda: kotodama_amd.paged_release(_z(2, 4), _z(2), _z(2), _z(9), _z(1), 16),
    "write": lambda: kotodama_amd.paged_write(_b(5, 2, 64), _b(5, 2, 64), _b(3, 2, 16, 64), _b(3, 2, 16, 64), _z(5)),
    "attention": lambda: kotodama_amd.paged_attention(_b(5, 4, 64), _b(3, 2, 16, 64), _b(3, 2, 16, 64), _z(2, 4), _z(2),
                                                      _z(3)),
    "verify": lambda: kotodama_amd.verify_drafts(_b(5, 9), _z(5, dtype=I64), _z(3), torch.zeros(5, 2)),
}


@pytest.mark.parametrize("op", CALLS)
def test_cpu_tensors_raise(op):
    with pytest.raises(RuntimeError, match="no CPU path"):
        CALLS[op]()


def test_slots_refusals():
    def check(table=None, held=None, new=None, free=None, count=None, page=16, tokens=5):
        table = _z(2, 4) if table is None else table
        kotodama_amd.paged_slots(table, _z(2) if held is None else held, _z(2) if new is None else new,
                                 _z(9) if free is None else free, _z(1) if count is None else count, page, tokens)

    def slots_check(**kw):
        args = dict(table=_z(2, 4), held=_z(2), new=_z(2), free=_z(9), count=_z(1), page=16)
        args.update(kw)
        paged._check_slots("paged_slots", args["table"], args["held"], "new", args["new"], args["free"], args["count"],
                           args["page"])

    slots_check()
    slots_check(held=_z(2, dtype=I64), page=65536)
    for kw in (dict(table=_z(8)), dict(table=_z(4, 2).t()), dict(table=_z(1, 4).expand(2, 4)), dict(held=_z(3)),
               dict(new=_z(2, 1)), dict(free=_z(3, 3)), dict(free=_z(18)[::2]), dict(count=_z(2)), dict(page=8),
               dict(page=24), dict(page=1 << 17), dict(table=_z(2, 1 << 15), page=65536)):
        with pytest.raises(ValueError, match="paged_slots"):
            slots_check(**kw)
    for kw in (dict(table=_z(2, 4, dtype=I64)), dict(held=torch.zeros(2)), dict(new=_z(2, dtype=torch.int16)),
               dict(free=_z(9, dtype=I64)), dict(count=_z(1, dtype=I64))):
        with pytest.raises(TypeError, match="paged_slots"):
            slots_check(**kw)
    for tokens in (-1, (1 << 30) + 1):
        with pytest.raises(ValueError, match="num_tokens"):
            check(tokens=tokens)
    with pytest.raises(TypeError):
        check(tokens=5.0)
    for page in (0, 15, 48, 1 << 17):
        with pytest.raises(ValueError, match="page size"):
            check(page=page)
    with pytest.raises(TypeError):
        check(page=16.0)


def test_write_refusals():
    def check(k=(5, 2, 64), v=None, kc=(3, 2, 16, 64), vc=None, slots=None, dt=torch.bfloat16, cdt=None):
        paged._check_write(_b(*k, dtype=dt), _b(*(v or k), dtype=dt), _b(*kc, dtype=cdt or dt),
                           _b(*(vc or kc), dtype=cdt or dt), _z(5) if slots is None else slots)

    check()
    check(dt=torch.float32, slots=_z(5, dtype=I64))
    check(k=(5, 2, 8), kc=(0, 2, 16, 8))
    for kw in (dict(k=(5, 128)), dict(v=(5, 2, 32)), dict(k=(5, 3, 64)), dict(k=(5, 2, 32)), dict(kc=(3, 2, 64)),
               dict(vc=(4, 2, 16, 64)), dict(kc=(3, 0, 16, 64), k=(5, 0, 64)), dict(kc=(3, 2, 24, 64)),
               dict(kc=(3, 2, 8, 64)), dict(kc=(3, 2, 16, 68), k=(5, 2, 68)), dict(kc=(3, 2, 16, 136), k=(5, 2, 136)),
               dict(slots=_z(4)), dict(slots=_z(5, 1))):
        with pytest.raises(ValueError, match="paged_write"):
            check(**kw)
    for kw in (dict(dt=torch.float16), dict(cdt=torch.float32), dict(slots=torch.zeros(5))):
        with pytest.raises(TypeError):
            check(**kw)
    # a cache that would have to be copied
    c = _b(3, 2, 16, 72)[..., :64]
    paged._check_cache_memory("paged_write", c, c)
    for c in (_b(3, 2, 16, 128)[..., ::2], _b(3, 2, 16, 68)[..., :64], _b(1 + 3 * 2 * 16 * 64)[1:].view(3, 2, 16, 64)):
        with pytest.raises(ValueError, match="16-byte"):
            paged._check_cache_memory("paged_write", c, c)


def test_attention_refusals():
    def check(q=(5, 4, 64), kc=(3, 2, 16, 64), table=None, lens=None, starts="three", dt=torch.bfloat16, qdt=None):
        starts = _z(3) if starts == "three" else starts
        paged._check_paged_attention(_b(*q, dtype=qdt or dt), _b(*kc, dtype=dt), _b(*kc, dtype=dt),
                                     _z(2, 4) if table is None else table, _z(2) if lens is None else lens, starts)

    check()
    check(q=(2, 4, 64), starts=None)
    check(lens=_z(2, dtype=I64), starts=_z(3, dtype=I64))
    for kw in (dict(q=(5, 64)), dict(q=(5, 4, 32)), dict(q=(5, 3, 64)), dict(q=(5, 0, 64)), dict(table=_z(8)),
               dict(lens=_z(3)), dict(starts=_z(2)), dict(starts=None), dict(table=_z(2, 1 << 27)),
               dict(kc=(3, 2, 16, 132), q=(5, 4, 132)), dict(kc=(3, 2, 20, 64))):
        with pytest.raises(ValueError, match="paged_attention"):
            check(**kw)
    for kw in (dict(dt=torch.float16), dict(qdt=torch.float32), dict(table=_z(2, 4, dtype=I64)),
               dict(lens=torch.zeros(2)), dict(starts=torch.zeros(3))):
        with pytest.raises(TypeError):
            check(**kw)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            kotodama_amd.paged_attention(_b(2, 4, 64), _b(3, 2, 16, 64), _b(3, 2, 16, 64), _z(2, 4), _z(2), scale=scale)


def test_verify_refusals():
    def check(logits=(5, 9), ids=None, starts=None, u=None, q=None, t=1.0, dt=torch.bfloat16):
        paged._check_verify(_b(*logits, dtype=dt), _z(5, dtype=I64) if ids is None else ids,
                            _z(3) if starts is None else starts, torch.zeros(5, 2) if u is None else u, q, t)

    check()
    check(q=_b(5, 9, dtype=torch.float32), t=0.0, ids=_z(5))
    for kw in (dict(logits=(5,)), dict(logits=(5, 0)), dict(ids=_z(4)), dict(starts=_z(0)), dict(starts=_z(3, 1)),
               dict(u=torch.zeros(5)), dict(u=torch.zeros(4, 2)), dict(q=_b(5, 8)), dict(t=-1.0), dict(t=float("nan")),
               dict(t=float("inf")), dict(t=1e-9)):
        with pytest.raises(ValueError, match="verify_drafts"):
            check(**kw)
    for kw in (dict(dt=torch.float16), dict(ids=torch.zeros(5)), dict(starts=torch.zeros(3)),
               dict(u=torch.zeros(5, 2, dtype=torch.float64)), dict(q=_b(5, 9, dtype=torch.float16))):
        with pytest.raises(TypeError):
            check(**kw)
    with pytest.raises(ValueError, match="2\\^21"):
        paged._check_verify(torch.empty((1, (1 << 21) + 1), device="meta"), _z(1), _z(2), torch.zeros(1, 2), None, 1.0)


def test_derivatives_are_refused():
    leaf = _b(5, 2, 64).requires_grad_(True)
    cache = _b(3, 2, 16, 64)
    logits = _b(5, 9).requires_grad_(True)
    calls = [lambda k, x: kotodama_amd.paged_write(k, k.detach(), cache, cache, _z(5)),
             lambda k, x: kotodama_amd.paged_attention(k, cache, cache, _z(2, 4), _z(2), _z(3)),
             lambda k, x: kotodama_amd.verify_drafts(x, _z(5), _z(3), torch.zeros(5, 2))]
    for call in calls:
        with pytest.raises(NotImplementedError, match="no gradient"):
            call(leaf, logits)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
            call(leaf, logits)
        with forward_ad.dual_level(), torch.no_grad(), pytest.raises(NotImplementedError, match="forward"):
            call(*(forward_ad.make_dual(t.detach(), t.detach()) for t in (leaf, logits)))


def _st(*v):
    return (ctypes.c_int64 * len(v))(*v)


def test_slots_abi_refusals():
    def slots(seqs=2, width=4, ld=4, held=FAKE, hd=0, free=FAKE, nfree=9, count=FAKE, page=16, tokens=5, out=FAKE,
              table=FAKE):
        return _capi.lib().attnres_paged_slots(table, ld, seqs, width, held, hd, FAKE, 0, free, nfree, count, page,
                                               tokens, out, FAKE, FAKE, FAKE, FAKE, None)

    def release(**kw):
        a = dict(seqs=2, width=4, held=FAKE, free=FAKE, page=16, out=FAKE)
        a.update(kw)
        return _capi.lib().attnres_paged_release(FAKE, 4, a["seqs"], a["width"], a["held"], 0, FAKE, 0, a["free"], 9,
                                                 FAKE, a["page"], a["out"], None)

    for kw in (dict(seqs=-1), dict(width=-1), dict(ld=3), dict(held=None), dict(hd=4), dict(free=None), dict(nfree=-1),
               dict(count=None), dict(tokens=-1), dict(out=None), dict(table=None)):
        assert slots(**kw) == _capi.ERR_ARG, kw
    for kw in (dict(page=8), dict(page=24), dict(page=1 << 17), dict(page=0), dict(page=-16), dict(tokens=1 << 31),
               dict(width=1 << 27), dict(seqs=(1 << 20) + 1)):
        assert slots(**kw) == _capi.ERR_UNSUPPORTED, kw
    for kw in (dict(held=FAKE + 2), dict(held=FAKE + 4, hd=1), dict(free=FAKE + 2), dict(count=FAKE + 1),
               dict(out=FAKE + 2)):
        assert slots(**kw) == _capi.ERR_ALIGN, kw
    for kw in (dict(seqs=-1), dict(held=None), dict(free=None), dict(out=None)):
        assert release(**kw) == _capi.ERR_ARG, kw
    assert release(page=12) == _capi.ERR_UNSUPPORTED


def test_write_abi_refusals():
    def write(k=FAKE, st=(128, 64), n=5, hk=2, d=64, dt=BF, kc=FAKE, cst=(2048, 1024, 64), pages=3, page=16,
              slots=FAKE, sd=0):
        return _capi.lib().attnres_paged_write(k, _st(*st), FAKE, _st(*st), n, hk, d, dt, kc, _st(*cst), FAKE,
                                               _st(*cst), pages, page, slots, sd, None)

    assert write(n=0) == _capi.OK  # nothing to do: returns before any HIP call
    assert write(pages=0) == _capi.OK
    for kw in (dict(k=None), dict(n=-1), dict(hk=0), dict(dt=7), dict(kc=None), dict(pages=-1), dict(slots=None),
               dict(sd=5), dict(cst=(2048, -1024, 64)), dict(cst=(0, 1024, 64)), dict(cst=(2048, 0, 64)),
               dict(cst=(2048, 1024, 0))):
        assert write(**kw) == _capi.ERR_ARG, kw
    for kw in (dict(d=4), dict(d=68), dict(d=136), dict(page=8), dict(page=48), dict(cst=(2048, 1024, 1 << 28)),
               dict(hk=(1 << 14) + 1), dict(n=1 << 31)):
        assert write(**kw) == _capi.ERR_UNSUPPORTED, kw
    for kw in (dict(k=FAKE + 8), dict(st=(129, 64)), dict(kc=FAKE + 4), dict(cst=(2048, 1025, 64)),
               dict(slots=FAKE + 2)):
        assert write(**kw) == _capi.ERR_ALIGN, kw


def test_attention_abi_refusals():
    def fwd(q=FAKE, qst=(256, 64), kc=FAKE, cst=(2048, 1024, 64), n=5, seqs=2, h=4, hk=2, d=64, dt=BF, pages=3, page=16,
            table=FAKE, ld=4, width=4, lens=FAKE, ld_=0, starts=FAKE, scale=0.1, out=FAKE, lse=None):
        return _capi.lib().attnres_paged_attention_fwd(
            q, _st(*qst), kc, _st(*cst), FAKE, _st(*cst), n, seqs, h, hk, d, dt, pages, page, table, ld, width, lens,
            ld_, starts, 0, scale, out, _st(*qst), lse, None, 0, None)

    assert fwd(n=0) == _capi.OK
    for kw in (dict(n=-1), dict(seqs=-1), dict(h=3), dict(hk=0), dict(h=0), dict(dt=9), dict(width=-1), dict(q=None),
               dict(kc=None), dict(table=None), dict(ld=3), dict(lens=None), dict(ld_=3), dict(scale=0.0),
               dict(scale=float("nan")), dict(scale=3e38), dict(out=None), dict(pages=-1), dict(starts=None)):
        assert fwd(**kw) == _capi.ERR_ARG, kw
    for kw in (dict(d=4), dict(d=12), dict(d=136), dict(page=20), dict(page=8), dict(width=1 << 27, ld=1 << 27),
               dict(h=8194), dict(seqs=(1 << 20) + 1), dict(n=(1 << 29) + 1), dict(cst=(2048, 1024, 1 << 27))):
        assert fwd(**kw) == _capi.ERR_UNSUPPORTED, kw
    for kw in (dict(q=FAKE + 8), dict(qst=(257, 64)), dict(kc=FAKE + 2), dict(cst=(2049, 1024, 64)),
               dict(table=FAKE + 2), dict(lens=FAKE + 1), dict(starts=FAKE + 2), dict(lse=FAKE + 2)):
        assert fwd(**kw) == _capi.ERR_ALIGN, kw
    with pytest.raises(_capi.AttnResError, match="head_dim 300"):
        _capi.paged_attention_workspace_size(5, 2, 4, 2, 300, BF, 4, 16)


def test_verify_abi_refusals():
    def verify(logits=FAKE, ld=9, ldt=BF, q=None, qdt=BF, rows=5, vocab=9, ids=FAKE, idt=1, starts=FAKE, seqs=2, u=FAKE,
               t=1.0, out=FAKE, counts=FAKE, ws=FAKE, nbytes=1 << 20):
        return _capi.lib().attnres_verify_drafts(logits, ld, ldt, q, ld, qdt, rows, vocab, ids, idt, starts, 0, seqs, u,
                                                 t, out, counts, ws, nbytes, None)

    assert verify(rows=0, seqs=0) == _capi.OK
    for kw in (dict(logits=None), dict(ld=8), dict(ldt=4), dict(q=FAKE, qdt=4), dict(rows=-1), dict(vocab=0),
               dict(ids=None), dict(idt=2), dict(starts=None), dict(seqs=-1), dict(u=None), dict(t=-1.0),
               dict(t=float("nan")), dict(t=1e-9), dict(out=None), dict(counts=None), dict(ws=None), dict(nbytes=8)):
        assert verify(**kw) == _capi.ERR_ARG, kw
    for kw in (dict(vocab=(1 << 21) + 1, ld=1 << 22), dict(rows=(1 << 24) + 1), dict(seqs=(1 << 20) + 1)):
        assert verify(**kw) == _capi.ERR_UNSUPPORTED, kw
    for kw in (dict(logits=FAKE + 1), dict(ids=FAKE + 4), dict(starts=FAKE + 2), dict(u=FAKE + 2), dict(out=FAKE + 4),
               dict(counts=FAKE + 2), dict(ws=FAKE + 8), dict(q=FAKE + 1)):
        assert verify(**kw) == _capi.ERR_ALIGN, kw


def test_cache_and_model_refusals():
    c = lmstep.LMConfig("t", 64, 2, 4, 2, 16, 96, vocab_size=128, attn_res_n_blocks=2, batch=2, seq=40)
    model = lmstep.LanguageModel(c, "cpu", torch.float32)
    cache = model.new_cache(5, 3, page_size=16)
    assert cache.kv.shape == (2, 2, 5, 2, 16, 16) and cache.block_table.shape == (3, 2)  # two whole pages of 40 tokens
    assert cache.free_pages.tolist() == [4, 3, 2, 1, 0] and cache.free_count.tolist() == [5]
    with pytest.raises(ValueError, match="rope tables"):
        model.new_cache(5, 3, max_tokens=64)
    for kw in (dict(page_size=16, max_tokens=20), dict(page_size=64)):
        with pytest.raises(ValueError, match="whole pages"):
            model.new_cache(5, 3, **kw)
    with pytest.raises(ValueError, match="page size"):
        model.new_cache(5, 3, page_size=24, max_tokens=24)

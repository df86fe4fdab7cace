"""paged_attention on the GPU where its workspace holds another call's notes: only the
call's own parts are joined.  Results are within the bounds of oracle/lm_oracle.py."""

import math

import pytest
import torch

import kotodama_amd
from kotodama_amd import _capi, paged
from kotodama_amd.ops import dtype_code
from oracle import paged_oracle as PO

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
BF, FP = torch.bfloat16, torch.float32


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _starts(new):
    at = [0]
    for n in new:
        at.append(at[-1] + n)
    return at


class Calls:
    """Calls of one size, in one workspace: ``tokens`` packed rows, and pages for the sequences of any of them."""

    def __init__(self, seed, tokens, seqs, capacity, h, hk, d, dtype, page=64):
        g = torch.Generator(device=DEV).manual_seed(seed)
        m = capacity // page
        self.k, self.v = (torch.randn((seqs * m + 1, hk, page, d), generator=g, device=DEV).to(dtype) for _ in "kv")
        self.table = torch.randperm(seqs * m + 1, generator=g, device=DEV)[:seqs * m].reshape(seqs, m).int()
        self.q = (torch.randn((tokens, h, d), generator=g, device=DEV) * 1.5).to(dtype)
        self.size = (tokens, seqs, h, hk, d, dtype_code(dtype), m, page)
        nbytes = _capi.paged_attention_workspace_size(*self.size)
        self.ws = torch.zeros(nbytes // 4, dtype=torch.int32, device=DEV)

    def leave_notes(self):
        """The whole workspace, its end the notes, as notes of two parts of a tile that the call has."""
        tokens, _, h, hk = self.size[:4]
        note = _ints([0, 0, tokens * (h // hk), 0, 2, 0, hk, hk])
        self.ws.copy_(note.repeat(self.ws.numel() // 8 + 1)[-self.ws.numel():])

    def __call__(self, lens, starts):
        tokens, seqs, h, hk, d, code, m, page = self.size
        out = torch.full_like(self.q, 7.0)
        lse = torch.full((tokens, h), 7.0, device=DEV)
        with paged._DeviceStream(DEV) as stream:
            _capi.paged_attention_fwd(self.q.data_ptr(), paged._i64x2(h * d, d), self.k.data_ptr(),
                                      paged._cache_strides(self.k), self.v.data_ptr(), paged._cache_strides(self.v),
                                      tokens, seqs, h, hk, d, code, self.k.shape[0], page, self.table.data_ptr(), m, m,
                                      lens.data_ptr(), _capi.INDEX_I32, starts.data_ptr(), _capi.INDEX_I32,
                                      1 / math.sqrt(d), out.data_ptr(), paged._i64x2(h * d, d), lse.data_ptr(),
                                      self.ws.data_ptr(), self.ws.numel() * 4, stream)
        return out, lse

    def check(self, out, lse, lens, starts):
        want, want_lse = PO.attention(self.q, self.k, self.v, self.table, lens, starts)
        for got, (value, bound) in ((out, want), (lse, want_lse)):
            same = got.double() == value
            over = torch.where(same, 0.0, (got.double() - value).abs() / bound.clamp_min(1e-300)).max().item()
            assert over <= 1.0, f"{over:.3g} times the bound"


# (new, lens, tokens, heads, kv_heads, capacity): the first ones have as many parts as a head has workgroups
CASES = [
    ([1184], [16384], 1184, 32, 8, 16384),
    ([592], [12288], 592, 64, 8, 16384),
    ([4416], [8192], 4416, 8, 4, 8192),
    ([361, 8], [15772, 9986], 2048, 32, 8, 16384),
    ([1, 1, 1, 1, 1, 1, 1, 512], [27069, 21578, 29456, 17002, 12234, 26756, 16454, 14283], 1280, 32, 8, 32768),
    ([1040], [16000], 1040, 32, 8, 16384),  # some workgroups left over
    ([2048], [2048], 2048, 32, 8, 16384),  # room for parts, none cut
    ([1], [16000], 1, 32, 8, 16384),  # few rows
    ([3, 1, 8], [9000, 0, 300], 12, 8, 4, 16384),
]


@pytest.mark.parametrize("new,lens,tokens,h,hk,capacity", CASES)
def test_a_workspace_that_holds_notes(new, lens, tokens, h, hk, capacity):
    print(f"paged_attention in a used workspace: new={new} lens={lens} tokens={tokens} {h}/{hk}", flush=True)
    calls = Calls(len(new), tokens, len(new), capacity, h, hk, 128, BF)
    calls.leave_notes()
    out, lse = calls(_ints(lens), _ints(_starts(new)))
    calls.check(out, lse, lens, _starts(new))
    again = calls(_ints(lens), _ints(_starts(new)))  # behind its own notes
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("tokens,h,hk,capacity,steps", [
    (1280, 32, 8, 32768, [
        ([1, 1024, 128, 1, 1, 1, 1, 1], [20762, 13180, 19533, 9062, 23415, 32197, 28307, 10153]),
        ([1, 1, 1, 1, 1, 1, 1, 512], [27069, 21578, 29456, 17002, 12234, 26756, 16454, 14283])]),
    (2048, 32, 8, 16384, [([1994, 1], [6876, 5980]), ([361, 8], [15772, 9986])]),
])
def test_one_call_behind_another(tokens, h, hk, capacity, steps, dtype):
    # the second of two steps joins nothing of the first, eager and in one graph
    seqs = len(steps[0][0])
    print(f"paged_attention, step after step: {tokens} tokens of {seqs} {dtype}", flush=True)
    calls = Calls(tokens, tokens, seqs, capacity, h, hk, 128, dtype)
    eager = []
    for new, lens in steps:
        out, lse = calls(_ints(lens), _ints(_starts(new)))
        calls.check(out, lse, lens, _starts(new))
        eager.append(out)
    lens, starts = _ints([0] * seqs), _ints([0] * (seqs + 1))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kotodama_amd.paged_attention(calls.q, calls.k, calls.v, calls.table, lens, starts)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kotodama_amd.paged_attention(calls.q, calls.k, calls.v, calls.table, lens, starts)
    for i in (0, 1, 0, 1, 1):
        new, n = steps[i]
        lens.copy_(_ints(n))
        starts.copy_(_ints(_starts(new)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, eager[i]), i

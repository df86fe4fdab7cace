"""verify_drafts on the GPU where its starts fall, in a workspace that held something else:
no sequence takes a token from rows that the call has not looked at."""

import pytest
import torch

from kotodama_amd import _capi, paged
from oracle import paged_oracle as PO

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("temperature", [0.0, 0.75])
@pytest.mark.parametrize("starts", [[0, 5, 3, 6, 4], [0, 9, 4], [0, 40, -3, 7, 9, 1], [0, 3, 9], [0, 0]])
def test_starts_that_fall(starts, temperature):
    g = torch.Generator(device=DEV).manual_seed(len(starts))
    n, v = 9, 5000
    seqs = len(starts) - 1
    logits = torch.randn((n, v), generator=g, device=DEV) * 2
    ids = logits.argmax(-1).roll(1)  # drafts that stay when greedy
    u = torch.rand((n, 2), generator=g, device=DEV) * 0.01
    s = torch.tensor(starts, dtype=torch.int32, device=DEV)
    ws = torch.full((_capi.verify_drafts_workspace_size(n, seqs, v) // 4,), 10**9, dtype=torch.int32, device=DEV)
    tokens, counts = torch.full((n,), 77, device=DEV), torch.full((seqs,), 77, dtype=torch.int32, device=DEV)
    print(f"verify_drafts, starts {starts}, temperature {temperature}", flush=True)
    with paged._DeviceStream(DEV) as stream:
        _capi.verify_drafts(logits.data_ptr(), v, _capi.DTYPE_F32, None, 0, _capi.DTYPE_F32, n, v, ids.data_ptr(),
                            _capi.INDEX_I64, s.data_ptr(), _capi.INDEX_I32, seqs, u.data_ptr(), temperature,
                            tokens.data_ptr(), counts.data_ptr(), ws.data_ptr(), ws.numel() * 4, stream)
    tokens, counts = tokens.tolist(), counts.tolist()
    last = min(max(starts[-1], 0), n)
    assert tokens[last:] == [-1] * (n - last)
    assert all(-1 <= t < v for t in tokens[:last])
    inside = [0] + [min(max(x, 0), last) for x in starts[1:]]
    for b, (lo, hi) in enumerate(zip(inside, inside[1:])):  # each sequence's number of tokens is that of its own rows
        want = PO.verify(logits, ids, [lo, max(lo, hi)], u, None, temperature)
        assert counts[b] == want[1][0], b
    assert tokens[0] == PO.verify(logits, ids, [0, last], u, None, temperature)[0][0] if starts[1] and last else True

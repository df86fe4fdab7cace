"""The language model of kotodama_amd.lmstep served from a paged cache: chunks of
prompts, single tokens and drafts of several sequences together, against the same
model behind its own cache, sequence by sequence.

Bar: both compute the same sums in other tilings: fp32, within 2e-4 of the largest logit (the bar of decoding
token by token against the whole sequence)."""

import pytest
import torch

from kotodama_amd import lmstep

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def _model(seq=96, seed=5, dtype=torch.float32):
    c = lmstep.LMConfig("t", 512, 3, 4, 2, 128, 384, vocab_size=1000, attn_res_n_blocks=2, batch=2, seq=seq)
    model = lmstep.LanguageModel(c, DEV, dtype=dtype, seed=seed)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    with torch.no_grad():  # routing away from uniform, norms away from one
        for name, p in model.named_parameters():
            if "res_query" in name:
                p.copy_((torch.randn(p.shape, generator=g, device=DEV) * 0.2).to(dtype))
            elif "norm" in name:
                p.add_((torch.randn(p.shape, generator=g, device=DEV) * 0.1).to(dtype))
    return c, model, g


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def test_chunks_and_single_tokens_of_several_sequences():
    c, model, g = _model()
    lens = [96, 33, 1, 64]
    ids = [torch.randint(0, 1000, (n,), generator=g, device=DEV) for n in lens]
    whole = [model.logits(s[None])[0][0] for s in ids]
    scale = max(w.abs().max().item() for w in whole)
    cache = model.new_cache(pages=20, sequences=5, page_size=16)
    assert cache.block_table.shape == (5, 6)
    done = [0] * 4
    for new in ([40, 0, 1, 16], [1, 33, 0, 7], [16, 0, 0, 1], [39, 0, 0, 40]):
        packed = torch.cat([s[d:d + n] for s, d, n in zip(ids, done, new)] + [torch.zeros(3, device=DEV).long()])
        step = cache.extend(_ints(new + [0]), len(packed))
        got = model.logits_paged(packed, cache, step)
        at = 0
        for i, n in enumerate(new):
            assert ((got[at:at + n] - whole[i][done[i]:done[i] + n]).abs() <= 2e-4 * scale).all(), (i, new)
            at += n
        if sum(new):
            rows = torch.tensor([0, at - 1], device=DEV)
            assert ((model.logits_paged(packed, cache, step, rows) - got[rows]).abs() <= 2e-4 * scale).all()
        done = [d + n for d, n in zip(done, new)]
    assert cache.lens.tolist() == lens + [0] and done == lens
    cache.keep(_ints([0] * 5))
    assert cache.free_count.tolist() == [20] and sorted(cache.free_pages.tolist()) == list(range(20))


def test_greedy_steps_with_drafts_are_greedy_decoding():
    c, model, g = _model(seq=64)
    prompts = [torch.randint(0, 1000, (n,), generator=g, device=DEV) for n in (7, 20, 1)]
    total = 24
    want = []
    for p in prompts:  # each alone, token by token
        out, past = model.logits(p[None])
        toks = [int(out[0, -1].argmax())]
        while len(toks) < total:
            out, past = model.logits(torch.tensor([[toks[-1]]], device=DEV), past)
            toks.append(int(out[0, -1].argmax()))
        want.append(toks)
    cache = model.new_cache(pages=12, sequences=3, page_size=16)
    n = [len(p) for p in prompts]
    packed = torch.cat(prompts)
    step = cache.extend(_ints(n), len(packed))
    ends = (step.q_starts[1:] - 1).long()
    first = model.logits_paged(packed, cache, step, ends).argmax(-1)
    got = [[int(t)] for t in first]
    round_ = 0
    while min(map(len, got)) < total:
        new, packed = [], []
        for i, toks in enumerate(got):
            k = min((round_ + i) % 5, total - len(toks))  # drafts: the right ones but for the last, or none
            drafts = want[i][len(toks):len(toks) + k]
            if k > 1 and round_ % 2:
                drafts[-1] = (drafts[-1] + 1) % 1000
            mine = [] if len(toks) >= total else [toks[-1]] + drafts
            new.append(len(mine))
            packed += mine
        before = cache.lens.tolist()
        packed = torch.tensor(packed + [0, 0], device=DEV)
        u = torch.zeros((len(packed), 2), device=DEV)
        tokens, counts = model.step_paged(packed, _ints(new), cache, u, temperature=0.0)
        at = 0
        for i, (k, m) in enumerate(zip(new, counts.tolist())):
            assert (m > 0) == (k > 0) and (tokens[at + m:at + k] == -1).all()
            got[i] += tokens[at:at + m].tolist()
            at += k
        assert cache.lens.tolist() == [b + m for b, m in zip(before, counts.tolist())]
        round_ += 1
    for i in range(3):
        assert got[i][:total] == want[i]


def test_a_refused_sequence_keeps_what_it_has():
    c, model, g = _model(seq=64, dtype=torch.bfloat16)
    cache = model.new_cache(pages=3, sequences=2, page_size=16)
    ids = torch.randint(0, 1000, (47,), generator=g, device=DEV)
    model.logits_paged(ids, cache, cache.extend(_ints([32, 15]), 47))
    u = torch.rand((4, 2), generator=g, device=DEV)
    tokens, counts = model.step_paged(ids[:4], _ints([2, 2]), cache, u)  # both need a page, none is free
    assert tokens.tolist() == [-1] * 4 and counts.tolist() == [0, 0] and cache.lens.tolist() == [32, 15]
    tokens, counts = model.step_paged(ids[:2], _ints([1, 1]), cache, u[:2])  # the second has room for one
    assert counts.tolist() == [0, 1] and int(tokens[0]) == -1 and 0 <= int(tokens[1]) < 1000
    assert cache.lens.tolist() == [32, 16] and cache.free_count.tolist() == [0]
    cache.keep(_ints([0, 16]))
    tokens, counts = model.step_paged(ids[:3], _ints([1, 2]), cache, u[:3])
    assert counts.tolist()[0] == 1 and counts.tolist()[1] >= 1


def test_a_captured_step_serves_like_the_eager_one():
    c, model, g = _model(seq=64)
    caches = [model.new_cache(pages=14, sequences=3, page_size=16) for _ in range(2)]
    prompt = torch.randint(0, 1000, (20,), generator=g, device=DEV)
    for cache in caches:
        model.logits_paged(prompt, cache, cache.extend(_ints([9, 4, 7]), 20))
    n = 8
    ids, new = torch.zeros(n, dtype=torch.int64, device=DEV), _ints([0, 0, 0])
    u, probs = torch.zeros((n, 2), device=DEV), torch.full((n, 1000), 1e-3, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        model.step_paged(ids, new, caches[0], u, probs)  # nothing new: loads what it calls
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = model.step_paged(ids, new, caches[0], u, probs)
    for i, some in enumerate(([1, 3, 2], [4, 0, 4], [1, 1, 1], [0, 0, 0], [2, 5, 1], [3, 4, 3])):  # the last: over n
        ids.copy_(torch.randint(0, 1000, (n,), generator=g, device=DEV))
        new.copy_(_ints(some))
        u.copy_(torch.rand((n, 2), generator=g, device=DEV))
        u[:, 0].mul_(0.01)  # so that drafts stay
        graph.replay()
        torch.cuda.synchronize()
        want = model.step_paged(ids, new, caches[1], u, probs)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i
        assert [m > 0 for m in got[1].tolist()] == [k > 0 and (i < 5 or b < 2) for b, k in enumerate(some)]
        for name in ("lens", "free_count", "free_pages", "block_table"):
            assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), (i, name)

"""A serving step with a chunk of a prompt among single tokens and drafts, as the
integration guide (the file read below) puts it together."""

import re
from pathlib import Path

import pytest
import torch

from kotodama_amd import lmstep, verify_drafts

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
ROOT = Path(__file__).resolve().parent.parent


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _guide():
    text = (ROOT / "INTEGRATION.md").read_text()
    (block,) = [b for b in re.findall(r"```python\n(.*?)```", text, re.S) if "logits[rows]" in b]
    return "\n".join(s for s in block.splitlines() if not s.startswith("rows, starts"))


def test_chunks_among_drafts_decode_greedily():
    # greedy decoding of each sequence alone, and of all together: the first has drafts, the second its prompt in
    # chunks (no token of it may be cut), the third single tokens, the fourth no room in its row of the table
    c = lmstep.LMConfig("t", 512, 2, 4, 2, 128, 384, vocab_size=500, attn_res_n_blocks=2, batch=2, seq=64)
    model = lmstep.LanguageModel(c, DEV, dtype=torch.float32, seed=3)
    g = torch.Generator(device=DEV).manual_seed(4)
    prompts = [torch.randint(0, 500, (n,), generator=g, device=DEV).tolist() for n in (6, 30, 1, 5)]
    want = []
    for p in prompts[:3]:
        out, past = model.logits(torch.tensor([p], device=DEV))
        tokens = [int(out[0, -1].argmax())]
        for _ in range(12):
            out, past = model.logits(torch.tensor([[tokens[-1]]], device=DEV), past)
            tokens.append(int(out[0, -1].argmax()))
        want.append(tokens)
    cache = model.new_cache(pages=16, sequences=4, page_size=16)
    cache.lens[3] = 64  # full: whatever it adds is refused
    got = [[], [], [], []]
    todo = [list(p) for p in prompts]
    for i in range(6):
        packed, new, rows, starts = [], [], [], [0]
        for s in range(4):
            if todo[s]:  # a chunk: a token is taken behind the prompt's last
                chunk, todo[s] = todo[s][:11], todo[s][11:]
                mine = [len(chunk) - 1]
            else:
                chunk = got[s][-1:]
                if s == 0:  # drafts: the right one, and in turn a wrong one
                    chunk = chunk + want[0][len(got[0]):len(got[0]) + 2]
                    chunk[-1] = (chunk[-1] + i % 2) % 500
                mine = list(range(len(chunk)))
            rows += [len(packed) + r for r in mine]
            starts.append(len(rows))
            packed += chunk
            new.append(len(chunk))
        ended = [not t for t in todo]
        packed.append(0)
        scope = dict(torch=torch, verify_drafts=verify_drafts, cache=cache, ids=torch.tensor(packed, device=DEV),
                     rows=torch.tensor(rows, device=DEV), starts=_ints(starts), new=_ints(new), temperature=0.0,
                     uniforms=torch.zeros((len(packed), 2), device=DEV), held=cache.lens.clone())
        scope["step"] = cache.extend(scope["new"], len(packed))
        scope["logits"] = model.logits_paged(scope["ids"], cache, scope["step"])
        exec(_guide(), scope)  # noqa: S102 - the repository's own guide
        tokens, counts = scope["tokens"].tolist(), scope["counts"].tolist()
        assert counts[3] == 0
        for s in range(3):
            if ended[s]:
                got[s] += tokens[starts[s]:starts[s] + counts[s]]
        assert cache.lens.tolist() == [len(p) - len(t) + max(0, len(o) - 1) for p, t, o in
                                       zip(prompts[:3], todo, got)] + [64], i
    assert len(got[0]) >= 6 and len(got[1]) == 4 and len(got[2]) == 6
    for s in range(3):
        assert got[s] == want[s][:len(got[s])], s

"""The serving loop of the integration guide (the file read below), behind its model: what
it does with the verification's answer, run on the CPU with one sequence refused."""

import re
from pathlib import Path

import torch

from kotodama_amd import PagedSlots

ROOT = Path(__file__).resolve().parent.parent


def test_the_guides_loop_gives_a_refused_sequence_nothing():
    text = (ROOT / "INTEGRATION.md").read_text()
    blocks = [b for b in re.findall(r"```python\n(.*?)```", text, re.S) if "cache.extend(" in b]
    assert len(blocks) == 1
    lines = blocks[0].splitlines()
    extend = next(i for i, s in enumerate(lines) if "cache.extend(" in s)
    verify = next(i for i, s in enumerate(lines) if "verify_drafts(" in s and "import" not in s)

    def ints(*v):
        return torch.tensor(v, dtype=torch.int32)

    # three sequences of 2, 2 and 1 new tokens, the second without room; a row of padding
    step = PagedSlots(ints(7, 8, -1, -1, 40, -1), ints(5, 6, 32, 33, 9, 0), ints(0, 2, 4, 5), ints(7, 0, 10), ints(0))

    class Cache:
        lens = ints(5, 32, 9)
        kept = None

        def extend(self, new, num_tokens):
            self.lens.copy_(torch.where(step.kv_lens > 0, step.kv_lens, self.lens))
            return step

        def keep(self, kept):
            self.kept = kept

    def verify_drafts(*args):
        return torch.tensor([11, 12, 21, 22, 31, -1]), ints(2, 2, 1)  # it knows of no refusal

    cache = Cache()
    names = ("logits", "ids", "uniforms", "draft_probs", "temperature", "new", "num_tokens")
    scope = dict(cache=cache, verify_drafts=verify_drafts, torch=torch, **dict.fromkeys(names))
    before = [s for s in lines[:extend + 1] if not s.startswith(("from ", "import ")) and "PagedCache(" not in s]
    exec("\n".join(before + lines[verify:]), scope)  # noqa: S102 - the repository's own guide
    assert scope["tokens"].tolist() == [11, 12, -1, -1, 31, -1]
    assert scope["counts"].tolist() == [2, 0, 1]
    assert cache.kept.tolist() == [7, 32, 10]

"""paged_attention's notes on the CPU: of every call of many rows each note is written
once, by the part that it is of or as one that none has, so that the join never reads
what an earlier call left in the workspace."""

import ctypes
import random
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
CUS, ROOM = 256, 1 << 16


@pytest.fixture(scope="module")
def notes(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    lib = tmp_path_factory.mktemp("notes") / "paged_notes.so"
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-Wno-unused-function", "-shared", "-fPIC",
                    f"-I{ROOT / 'kotodama_amd' / 'csrc'}", str(ROOT / "oracle" / "paged_notes.cpp"), "-o", str(lib)],
                   check=True)
    fn = ctypes.CDLL(str(lib)).paged_notes
    i32, i64, p64 = ctypes.c_int, ctypes.c_int64, ctypes.POINTER(ctypes.c_int64)
    fn.argtypes = [i32, i64, i32, i32, i32, i32, i32, i64, p64, p64, i32, ctypes.POINTER(ctypes.c_int32), i32, p64]
    written = (ctypes.c_int32 * ROOM)()

    def call(starts, lens, heads, kv_heads, dim=128, f32=False, capacity=32768, tokens=None, cut=-1):
        tokens = starts[-1] if tokens is None else tokens
        info = (i64 * 5)()
        rc = fn(CUS, tokens, len(lens), heads, kv_heads, dim, int(f32), capacity, (i64 * len(starts))(*starts),
                (i64 * max(1, len(lens)))(*lens), cut, written, ROOM, info)
        names = ("all", "parts", "slots", "used", "cut")
        return rc, dict(zip(names, info)), written[:info[2]]

    return call


def _starts(new):
    at = [0]
    for n in new:
        at.append(at[-1] + n)
    return at


# calls whose parts are as many as a head's workgroups, so that none is left over: (new, lens, tokens, heads, kv_heads)
FULL = [
    ([1184], [16384], 1184, 32, 8),
    ([592], [16384], 592, 64, 8),
    ([2368], [8192], 2368, 16, 8),
    ([4416], [65536], 4416, 8, 4),
    ([4736], [16384], 4736, 8, 8),
    ([361, 8], [15772, 9986], 2048, 32, 8),
    ([1, 1, 1, 1, 1, 1, 1, 512], [27069, 21578, 29456, 17002, 12234, 26756, 16454, 14283], 1280, 32, 8),
]


@pytest.mark.parametrize("new,lens,tokens,heads,kv_heads", FULL)
def test_notes_where_every_workgroup_has_a_part(notes, new, lens, tokens, heads, kv_heads):
    rc, info, written = notes(_starts(new), lens, heads, kv_heads, capacity=max(16384, max(lens)), tokens=tokens)
    assert rc == 0
    assert info["parts"] == info["all"] and 0 < info["used"] < info["slots"], info  # the case it stands for
    assert written == [1] * info["slots"]


@pytest.mark.parametrize("heads,kv_heads,dim,f32", [(32, 8, 128, False), (8, 4, 128, False), (64, 8, 64, False),
                                                    (24, 8, 96, True), (12, 12, 64, True), (7, 7, 128, False),
                                                    (96, 1, 128, True), (6, 3, 32, False)])
def test_every_note_is_written_once(notes, heads, kv_heads, dim, f32):
    rng = random.Random(heads * dim)
    seen = dict(few=0, split=0, full=0)
    for _ in range(400):
        tokens = int(256 * 2 ** rng.uniform(0, 6)) * 8 * 4 // max(1, heads // 4)
        seqs = rng.choice((1, 2, 3, 8, 40, 300))
        capacity = 64 * rng.choice((8, 9, 100, 512, 1024))
        cuts = sorted(rng.randint(0, tokens) for _ in range(seqs))
        kind = rng.random()
        if kind < 0.4:  # a chunk among single tokens, padding behind them
            cuts = _starts([1] * (seqs - 1) + [max(1, int((tokens - seqs) * rng.random()))])[1:]
        starts = [0] + cuts
        if kind > 0.9:  # starts that fall
            rng.shuffle(starts)
        lens = [rng.randint(0, capacity + 9) if rng.random() < 0.9 else rng.choice((-5, 0, 1 << 40))
                for _ in range(seqs)]
        for cut in range(-1, 8):
            rc, info, written = notes(starts, lens, heads, kv_heads, dim, f32, capacity, tokens, cut)
            assert rc == 0 or (rc == 1 and cut == -1) or (rc == 2 and cut > 0), (rc, cut)
            if rc == 1:  # few rows
                seen["few"] += 1
                break
            if rc == 0:
                assert written == [1] * info["slots"], (cut, info, starts, lens)
                seen["split"] += info["used"] > 0
                seen["full"] += info["used"] > 0 and info["parts"] == info["all"]
    assert seen["split"] > 100, seen

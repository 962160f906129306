"""The list of the beam selection's first pass, on the CPU: tests/c/beam_list.cpp walks a part of a row by the kernel's own rules
(moonshine_amd/csrc/beam_list.h).  Its length must stay within the room in shared memory whatever the logits are, and the part's K best must
come out in order, ties to the lowest id."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
LOWEST = {4: np.finfo(np.float32).min, 8: np.float32(-3.38953139e38)}    # 32-bit floats; bf16


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("beam_list") / "beam_list.so")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(HERE, "..", "moonshine_amd", "csrc"),
                    os.path.join(HERE, "c", "beam_list.cpp"), "-o", out], check=True)
    return C.CDLL(out)


def logits(kind, vocab, vec, rng):
    """vec 8: values that bf16 holds."""
    i = np.arange(vocab)
    if kind == "ascending":
        x = i * 0.01 - 300.0
    elif kind == "descending":
        x = 300.0 - i * 0.01
    elif kind == "random":
        x = 3 * rng.standard_normal(vocab)
    elif kind == "masked_first":          # every part begins with what a finite mask leaves out
        x = np.where(i % 5632 < 2048, float(LOWEST[vec]), 3 * rng.standard_normal(vocab))
    elif kind == "steps":                 # each chunk of 2048 two standard deviations above the one before
        x = rng.standard_normal(vocab) + 2.0 * (i // 2048)
    elif kind == "plateaus":              # ascending plateaus with ties across the chunks' borders
        x = (i // 1500).astype(np.float64)
    elif kind == "few_lanes":             # 5, 9 or 17 lanes far above the others, rising from chunk to chunk
        x = np.where((i // vec) % 64 < 17, i * 0.01, rng.standard_normal(vocab) - 50.0)
    x = x.astype(np.float32)
    return x if vec == 4 else (x.view(np.uint32) & 0xFFFF0000).view(np.float32)


@pytest.mark.parametrize("vec", [4, 8])
@pytest.mark.parametrize("K", [1, 2, 4, 5, 8, 9, 16])
@pytest.mark.parametrize("vocab, parts, off", [(32768, 6, 0), (32768, 12, 3), (70001, 16, 1), (20000, 1, 2), (9000, 2, 0), (2049, 1, 0), (100, 3, 1)])
def test_list_stays_in_its_room(lib, vec, K, vocab, parts, off):
    room = lib.beam_list_room()
    val, idx, longest = np.zeros(K, np.float32), np.zeros(K, np.int32), C.c_int()
    for kind in ("ascending", "descending", "random", "masked_first", "steps", "plateaus", "few_lanes"):
        x = logits(kind, vocab, vec, np.random.default_rng(K + vocab))
        nv = (vocab + off + vec - 1) // vec
        per = ((nv + parts - 1) // parts + 63) // 64 * 64
        for part in range(parts):
            lo, hi = max(0, part * per * vec - off), min(vocab, (part + 1) * per * vec - off)
            n = lib.beam_list_walk(x.ctypes.data_as(C.c_void_p), vocab, vec, off, parts, part, K, val.ctypes.data_as(C.c_void_p), idx.ctypes.data_as(C.c_void_p),
                                   C.byref(longest))
            assert longest.value <= room, (kind, part, longest.value, room)
            ids = np.arange(lo, max(lo, hi))
            want = ids[np.lexsort((ids, -x[ids]))][:K]
            assert n == len(want) and idx[:n].tolist() == want.tolist() and np.array_equal(val[:n], x[want]), (kind, part)


"""Beam selection over rows whose parts are several chunks long, with logits that rise, fall, are masked or tie from chunk to chunk: what
passes the bound of an earlier chunk is anything from nothing to whole chunks.  The oracle and the tolerance are those of
tests/test_gpu_serve_ops.py; the list's room is walked on the CPU by tests/test_beam_list.py."""
import numpy as np
import pytest
import torch

import serve_ref as ref
from moonshine_amd import ops
from test_beam_list import logits as structured
from test_gpu_serve_ops import TYPES, check_select, dev, gen, host

pytestmark = pytest.mark.gpu

KINDS = ["ascending", "descending", "random", "masked_first", "steps", "plateaus", "few_lanes"]


def rows(kind, count, vocab, dtype, seed):
    """Each row a little different; fp16 holds what bf16 does here but for the lowest value."""
    vec = 4 if dtype == "f32" else 8
    x = np.stack([np.roll(structured(kind, vocab, vec, gen(seed + r)), 3 * r if kind == "random" else 0) for r in range(count)])
    if dtype == "f16":
        x = np.maximum(x, np.float32(torch.finfo(torch.float16).min))
    return dev(x, TYPES[dtype])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("beams, vocab", [(1, 400000), (4, 400001), (8, 400003), (16, 140001)])
def test_select_over_parts_of_several_chunks(dtype, kind, beams, vocab):
    x = rows(kind, beams, vocab, dtype, beams).view(1, beams, vocab)
    scores = -np.cumsum(gen(beams).random((1, beams)) + 0.01, 1)
    finished = np.zeros((1, beams), bool)
    check_select(x, scores, finished, 2)
    if beams > 1:
        finished[0, 1] = True
        check_select(x, scores, finished, 2)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("batch, beams, vocab", [(256, 8, 32768), (128, 16, 32768), (256, 4, 50000)])
def test_select_of_full_batches(dtype, kind, batch, beams, vocab):
    """The engine's own size among them; every other entry is random, so that a list that runs over its room would show in its neighbours.
    Some of both kinds are compared with the oracle."""
    base = rows(kind, beams, vocab, dtype, 1)
    x = (3 * torch.randn((batch, beams, vocab), generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")).to(TYPES[dtype])
    x[::2] = base
    rng = gen(9)
    scores = -np.cumsum(rng.random((batch, beams)) + 0.01, 1)
    finished = rng.random((batch, beams)) < 0.1
    s, f = dev(scores.astype(np.float32)), dev(finished.astype(np.uint8))
    got = ops.beam_select(x, s, f, 2)
    assert int(got[1].min()) >= 0 and int(got[1].max()) < beams and int(got[2].min()) >= 0 and int(got[2].max()) < vocab
    for b in (0, 1, 2, 3, batch // 2, batch // 2 + 1, batch - 2, batch - 1):
        want = ref.beam_select(host(x[b:b + 1]), scores[b:b + 1].astype(np.float32), finished[b:b + 1], 2)
        (order, parent), = want[4]
        assert (np.abs(host(got[0][b]) - want[0][0]) <= 2.0 ** -19 + 2.0 ** -24 * np.abs(want[0][0])).all()
        if any(p - q <= 2.0 ** -19 and i != j for p, q, i, j in zip(order, order[1:], parent, parent[1:])):
            continue                                             # two beams' candidates closer than the sums are exact
        assert host(got[1][b]).tolist() == want[1][0].tolist() and host(got[2][b]).tolist() == want[2][0].tolist(), b
        assert host(got[3][b]).astype(bool).tolist() == want[3][0].tolist()

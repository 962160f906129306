"""Calls of the serving operators that their documentation allows and no other test makes: row ranges with rows before, between and behind them that are
no sequence's, outputs with the heads outside, the largest pages, tables that two graphs share, engine clips long enough for several key ranges."""
import numpy as np
import pytest
import torch

import serve_ref as ref
import test_gpu_parity as tp
from moonshine_amd import ops
from moonshine_amd.synth import make_audio
from test_gpu_beam_mxfp4 import check_logits
from test_gpu_serve_ops import TYPES, bound, dev, gen, host, i32, values

pytestmark = pytest.mark.gpu


def filled(rng, batch, n, heads, width, page):
    """A cache of `batch` sequences of n tokens in shuffled pages, with the values that it holds."""
    need = -(-n // page)
    cache = ops.kv4_cache(batch * need, heads, page, width)
    table = rng.permutation(batch * need).reshape(batch, need).astype(np.int32)
    t = np.arange(n)
    ks, vs = [], []
    for b in range(batch):
        k, v = values(rng, (n, heads, width)), values(rng, (n, heads, width))
        ops.kv4_write(cache, dev(k), dev(v), dev(table[b, t // page].astype(np.int64) * page + t % page))
        ks.append(ref.quantise(k))
        vs.append(ref.quantise(v))
    return cache, table, ks, vs


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n, starts, max_q, heads, kv_heads, width", [
    (90, [3, 5, 5, 16, 17], 4, 4, 2, 52),              # one range of keys; the third sequence has eleven rows, four of them count
    (3000, [2, 3, 3, 9, 10], 2, 4, 1, 64),             # several ranges, joined
    (2200, [7, 47, 47, 147, 148], 40, 2, 2, 40),       # tiles of 32 and ranges
    (8300, [1, 90, 90, 290, 291], 80, 8, 8, 32),       # the same, longer
])
@pytest.mark.parametrize("outside", [False, True])
def test_rows_of_no_sequence_stay(dtype, n, starts, max_q, heads, kv_heads, width, outside):
    """... in out, before, between (behind the first max_q of a sequence) and behind; `outside`: out and q with the heads outside."""
    rng = gen(n + width)
    batch, rows = len(starts) - 1, starts[-1] + 3
    cache, table, ks, vs = filled(rng, batch, n, kv_heads, width, 64)
    lens = [n, n // 2, n - 1, 33]
    x = values(rng, (rows, heads, width))
    q, out = dev(x, TYPES[dtype]), torch.full((rows, heads, width), 7.0, dtype=TYPES[dtype], device="cuda")
    if outside:
        q, out = q.transpose(0, 1).contiguous().transpose(0, 1), torch.full((heads, rows, width), 7.0, dtype=TYPES[dtype], device="cuda").transpose(0, 1)
    got, lse = ops.kv4_attention(q, cache, dev(table), i32(lens), q_start=i32(starts), max_q=max_q, return_lse=True, out=out)
    assert got.data_ptr() == out.data_ptr() and got.stride() == out.stride()
    free = np.ones(rows, bool)
    for b in range(batch):
        count = min(starts[b + 1] - starts[b], max_q)
        if count == 0:
            continue
        part = slice(starts[b], starts[b] + count)
        free[part] = False
        see = ref.visible(count, lens[b], True)
        want, want_lse, mass, top, spread = ref.attention(host(q[part]), ks[b][:lens[b]], vs[b][:lens[b]], see, width ** -0.5)
        tol, tol_lse = bound(dtype, width, lens[b], want, mass, top, spread)
        assert (np.abs(host(out[part]) - want) <= tol).all(), b
        live = see.any(1)
        assert (host(out[part])[~live] == 0).all() and (host(lse[part])[~live] == -np.inf).all()
        assert (np.abs(host(lse[part])[live] - want_lse[live]) <= tol_lse[live] + 2.0 ** -23 * np.abs(want_lse[live])).all()
    assert free.sum() > 3 and (host(out)[free] == 7.0).all()


def test_the_largest_pages():
    """One page of 65536 tokens a sequence."""
    rng = gen(5)
    page, width = 65536, 40
    cache = ops.kv4_cache(2, 1, page, width)
    table, lens = i32([[1], [0]]), [40000, 65536]
    held = []
    for b, n in enumerate(lens):
        k, v = values(rng, (n, 1, width)), values(rng, (n, 1, width))
        slots, used = ops.page_plan(table[b:b + 1].clone(), i32([n]), i32([n]), i32([0]), n + 2, i32([1 - b]), page)
        assert int(used) == 1 and slots[-2:].tolist() == [-1, -1] and int(slots[0]) == (1 - b) * page
        ops.kv4_write(cache, dev(k), dev(v), slots[:n].contiguous())
        held.append((ref.quantise(k), ref.quantise(v)))
    q = values(rng, (2, 3, width))
    out = ops.kv4_attention(dev(q), cache, table, i32(lens))
    for b, (k, v) in enumerate(held):
        want, _, mass, top, spread = ref.attention(q[b:b + 1].astype(np.float64), k, v, ref.visible(1, lens[b], True), width ** -0.5)
        assert (np.abs(host(out[b:b + 1]) - want) <= bound("f32", width, lens[b], want, mass, top, spread)[0]).all()


def test_graphs_of_calls_with_workspaces_replayed_in_turn():
    """Two captured calls that are split into ranges and two captured selections, over other inputs each: replayed in turn, alone and at once on two streams,
    each gives its eager result -- their workspaces are their own."""
    cache, table, _, _ = filled(gen(3), 4, 6000, 2, 64, 64)
    table, lens = dev(table), i32([6000, 300, 5999, 0])
    qs = [dev(values(gen(10 + i), (4, 8, 64)), torch.bfloat16) for i in range(2)]
    logits = [dev(values(gen(20 + i), (3, 5, 70001))) for i in range(2)]
    scores, finished = -torch.rand((3, 5), device="cuda"), torch.zeros((3, 5), dtype=torch.uint8, device="cuda")

    def call(i):
        return [*ops.kv4_attention(qs[i], cache, table, lens, return_lse=True), *ops.beam_select(logits[i], scores, finished, 2)]

    want = [call(0), call(1)]
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            outs.append(call(i))
        graphs.append(g)
    for turn in range(6):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        if turn % 2:
            for i in (0, 1, 0, 1):
                graphs[i].replay()
        else:
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
        eager = call(turn % 2)
        torch.cuda.synchronize()
        for a, b in zip(want[0] + want[1] + want[turn % 2], outs[0] + outs[1] + eager):
            assert torch.equal(a, b), turn


@pytest.mark.parametrize("arch, seconds", [("micro", [70, 30, 3]), ("micro", [180]), ("tiny", [45, 1])])
def test_mxfp4_over_clips_long_enough_for_several_key_ranges(tmp_path_factory, arch, seconds):
    e, w, cfg = tp._engine(tmp_path_factory, arch, 0)
    e.set_kv_dtype("mxfp4")
    check_logits(e, w, cfg, [make_audio(40 + i, 16000 * s) for i, s in enumerate(seconds)], 3)
    e.close()


def test_beams_over_long_clips(tmp_path_factory):
    """Four beams over clips of several key ranges: the same ids every time."""
    e, w, cfg = tp._engine(tmp_path_factory, "micro", 0)
    e.set_kv_dtype("mxfp4")
    e.set_beam_width(4)
    clips = [make_audio(80 + i, 16000 * s) for i, s in enumerate((60, 33))]
    got = e.transcribe_tokens(clips, forced_steps=6)
    again = e.transcribe_tokens(clips, forced_steps=6)
    assert got == again and all(len(t) == 7 and all(0 <= x < cfg.vocab for x in t) for t in got)
    e.close()

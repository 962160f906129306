"""The serving operators on the GPU (moonshine_amd/ops.py) against their 64-bit restatements (tests/serve_ref.py).

Tolerances of the attention, derived before the first run.  Inputs are the types' own values and the cache's exact values, so
  scores     d products and as many fp32 additions per 32 elements and term: |ds| <= (d + 40) 2^-24 * scale * sum |q_i k_i| (q's terms hold all
             of its 24 / 11 / 8 bits), and the multiplication by the scale, the exponent's argument and exp2: 2^-21 (1 + |s|)
  p          relative 2 ds, cut to two bf16 terms (each off by half a step: 2^-9 * 2^-9 = 2^-18 -> counted as 2^-17) or three (2^-26)
  sums       relative (tokens / 8 + 64) 2^-24: a lane adds tokens / 4 / waves values one after another, the matrix unit 32 at a time
  output     everything above times sum p |v|, and half a step of the output's type: eps / 2 of the value, of the smallest normal one below
             it (an fp16 output of 4e-9 becomes 0: its steps there are 2^-24, half of one is 2^-14 * eps / 2)
  underflow  p is held relative to the row's maximum in fp32 (and in bf16 terms of the same range): what is below 2^-126 of it, or a term of
             p that is, may become 0: 4 * 2^-126 a token times its |v| (a score 200 below the maximum has p = 1e-87)
"""
import numpy as np
import pytest
import torch

import serve_ref as ref
from moonshine_amd import ops
from moonshine_amd.hip_api import MshError

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def gen(seed):
    return np.random.default_rng(seed)


def dev(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t if dtype is None else t.to(dtype)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def host(t):
    return t.detach().cpu().double().numpy() if t.is_floating_point() else t.detach().cpu().numpy()


def values(rng, shape):
    """Rows as a model has them: channels and tokens of unlike size."""
    x = rng.standard_normal(shape) * np.exp(0.6 * rng.standard_normal((1,) + shape[1:])) * np.exp(0.3 * rng.standard_normal(shape[:-1] + (1,)))
    return x.astype(np.float32)


# ------------------------------------------------------------------ writing and reading
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows, heads, width, page", [(1, 1, 1, 32), (3, 2, 31, 32), (70, 3, 33, 64), (65, 8, 36, 32), (130, 8, 52, 128),
                                                      (40, 1, 64, 64), (37, 2, 96, 32), (33, 1, 100, 32), (64, 2, 128, 256), (9, 3, 160, 32),
                                                      (31, 1, 192, 32), (20, 1, 200, 64), (50, 2, 256, 32)])
def test_write_read_exact(dtype, rows, heads, width, page):
    """Bit for bit what the definition says, in any slots, and nothing but those slots changes."""
    rng = gen(rows * 1000 + width)
    k, v = dev(values(rng, (rows, heads, width)), TYPES[dtype]), dev(values(rng, (rows, heads, width)), TYPES[dtype])
    pages = -(-rows // page) + 2
    every = torch.from_numpy(rng.permutation(pages * page)).cuda()
    slots, others = every[:rows].contiguous(), every[rows:].contiguous()
    cache = ops.kv4_cache(pages, heads, page, width)
    ko, vo = dev(values(rng, (others.numel(), heads, width))), dev(values(rng, (others.numel(), heads, width)))
    ops.kv4_write(cache, ko, vo, others)
    before = ops.kv4_read(cache, others, width, torch.float32)
    ops.kv4_write(cache, k, v, slots)
    for got, x in zip(ops.kv4_read(cache, slots, width, torch.float32), (k, v)):
        assert np.array_equal(host(got), ref.quantise(host(x)))
    for a, b, x in zip(before, ops.kv4_read(cache, others, width, torch.float32), (ko, vo)):
        assert torch.equal(a, b) and np.array_equal(host(a), ref.quantise(host(x)))
    for a, b in zip(ops.kv4_read(cache, slots, width, torch.bfloat16), ops.kv4_read(cache, slots, width, torch.float32)):
        assert torch.equal(a.float(), b)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_write_every_tie_and_power(dtype):
    """All 4-bit borders at many powers of two, both signs: ties to the even code, the choice of the power at 1.75."""
    y = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.2495, 0.2505, 1.249, 1.251, 4.995, 5.01])
    rows = []
    for top in (3.5, 3.49, 4.0, 6.0, 6.98, 7.0, 7.5, 7.99):
        for p in (range(-110, 120, 7) if dtype != "f16" else range(-8, 12)):
            row = np.concatenate([y * np.sign(np.cos(np.arange(14.0) + p)), [top], np.zeros(17)])
            rows.append(np.ldexp(row, p))
    x = dev(np.array(rows, np.float32)[:, None, :], TYPES[dtype])
    cache = ops.kv4_cache(-(-len(rows) // 32), 1, 32, 32)
    slots = torch.arange(len(rows), device="cuda")
    ops.kv4_write(cache, x, -x, slots)
    k, v = ops.kv4_read(cache, slots, 32, torch.float32)
    assert np.array_equal(host(k), ref.quantise(host(x))) and np.array_equal(host(v), ref.quantise(-host(x)))


def test_write_special_values():
    x = np.zeros((6, 1, 40), np.float32)
    x[0, 0, :5] = [np.nan, 1.0, -3.0, np.nan, 0.5]
    x[1, 0, 33:36] = [np.inf, -np.inf, 1e30]
    x[2, 0] = 1e-40
    x[3, 0, 0] = np.finfo(np.float32).max
    x[4, 0, :4] = [2.0 ** -101, 2.0 ** -102, 2.0 ** -103, -2.0 ** -101]
    cache = ops.kv4_cache(1, 1, 32, 40)
    slots = torch.arange(6, device="cuda")
    ops.kv4_write(cache, dev(x), dev(x), slots)
    for got in ops.kv4_read(cache, slots, 40, torch.float32):
        assert np.isfinite(host(got)).all() and np.array_equal(host(got), ref.quantise(x))


def test_write_skips_slots_outside_and_takes_any_strides():
    rng = gen(3)
    rows, heads, width = 48, 3, 52
    big = dev(values(rng, (width, heads, 2 * rows)))
    k = big[:, :, ::2].permute(2, 1, 0)                      # element stride 6 * rows, row stride 2
    v = dev(values(rng, (rows, heads, 2, width + 3)))[:, :, 1, 1:-2]      # rows that start at odd addresses
    slots = torch.arange(rows, device="cuda") + 5
    slots[::7] = -1
    slots[3] = 96
    slots[4] = 1 << 40
    slots[5] = -(1 << 40)
    cache = ops.kv4_cache(3, heads, 32, width)
    guard = cache.clone()
    ops.kv4_write(cache, k, v, slots)
    live = host((slots >= 0) & (slots < 96))
    for got, x in zip(ops.kv4_read(cache, slots, width, torch.float32), (k, v)):
        assert np.array_equal(host(got), np.where(live[:, None, None], ref.quantise(host(x)), 0.0))
    other = torch.tensor([0, 1, 4, 5, 95], device="cuda")
    for got in ops.kv4_read(cache, other, width, torch.float32):
        assert not got.any()
    assert torch.equal(guard[2], cache[2])                   # slots 64..: none was named


def test_offsets_past_32_bits():
    """A cache of more than 4 GiB: pages at its far end, written, read and attended."""
    heads, width, page = 4, 256, 1024
    pages = (5 << 30) // (heads * page // 32 * 8704) + 1
    cache = ops.kv4_cache(pages, heads, page, width)
    assert cache.numel() > 5 << 30
    rng = gen(11)
    n = 70
    x = [values(rng, (n, heads, width)) for _ in range(2)]
    table = i32([[pages - 1, pages - 2]])
    slots = torch.arange(n, device="cuda") + (pages - 1) * page + 0
    ops.kv4_write(cache, dev(x[0]), dev(x[1]), slots)
    k, v = (host(t) for t in ops.kv4_read(cache, slots, width, torch.float32))
    assert np.array_equal(k, ref.quantise(x[0])) and np.array_equal(v, ref.quantise(x[1]))
    q = values(rng, (1, heads, width))
    out = ops.kv4_attention(dev(q), cache, table, i32([n]))
    want = ref.attention(q.astype(np.float64), k, v, ref.visible(1, n, True), width ** -0.5)[0]
    assert np.abs(host(out) - want).max() < 1e-4
    del cache


# ------------------------------------------------------------------ attention
VALUE_MOST = 256.0   # no |v| of values() comes near it


def bound(dtype, d, n_tokens, want, mass, top, spread):
    eps = torch.finfo(TYPES[dtype]).eps / 2
    ds = (d + 40) * 2.0 ** -24 * mass + 2.0 ** -21 * (1 + top)
    rel = 2 * ds + (2.0 ** -26 if dtype == "f32" else 2.0 ** -17) + (n_tokens / 8 + 64) * 2.0 ** -24
    return rel[..., None] * spread + eps * np.maximum(np.abs(want), torch.finfo(TYPES[dtype]).tiny) + n_tokens * 2.0 ** -124 * VALUE_MOST, ds + (n_tokens / 8 + 64) * 2.0 ** -24


def check_attention(dtype, heads, kv_heads, width, page, lengths, counts, causal=True, window=0, scale=None, spare=2, uniform=False,
                    fill=0xFF, seed=0, magnitude=1.0):
    """Sequences of `lengths` tokens and `counts` rows: packed rows with `spare` more behind, tables wider than needed, every byte of the
    cache that no token owns set to `fill`."""
    rng = gen(seed + 17 * width + len(lengths))
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + 2
    order = rng.permutation(pages)[:sum(need)]
    wide = max(need) + 1
    table = np.full((len(lengths), wide), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    cache = ops.kv4_cache(pages, kv_heads, page, width)
    cache.fill_(fill)
    scale = width ** -0.5 if scale is None else scale
    ks, vs = [], []
    for b, n in enumerate(lengths):
        k, v = values(rng, (n, kv_heads, width)) * magnitude, values(rng, (n, kv_heads, width))
        ks.append(ref.quantise(k))
        vs.append(ref.quantise(v))
        if n:
            t = np.arange(n)
            ops.kv4_write(cache, dev(k), dev(v), dev(table[b, t // page].astype(np.int64) * page + t % page))
    rows = sum(counts)
    total = rows + (0 if uniform else spare)
    q = dev(values(rng, (total, heads, width)), TYPES[dtype])
    out = torch.full((total, heads, width), 7.0, dtype=TYPES[dtype], device="cuda")
    starts = np.concatenate([[0], np.cumsum(counts)])
    got, lse = ops.kv4_attention(q, cache, dev(table), i32(lengths), q_start=None if uniform else i32(starts.tolist()), max_q=max(max(counts), 1),
                                 scale=scale, causal=causal, window=window, return_lse=True, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert torch.equal(out[rows:], torch.full_like(out[rows:], 7.0))          # rows of no sequence are left alone
    worst = 0.0
    for b, n in enumerate(lengths):
        if counts[b] == 0:
            continue
        part = slice(int(starts[b]), int(starts[b + 1]))
        see = ref.visible(counts[b], n, causal, window)
        want, want_lse, mass, top, spread = ref.attention(host(q[part]), ks[b], vs[b], see, scale)
        tol, tol_lse = bound(dtype, width, n, want, mass, top, spread)
        err = np.abs(host(out[part]) - want)
        assert np.isfinite(err).all()
        assert (err <= tol).all(), f"sequence {b}: {float((err / tol).max()):.2f} of the bound"
        worst = max(worst, float((err / tol).max()))
        empty = ~see.any(1)
        assert (host(out[part])[empty] == 0).all() and (host(lse[part])[empty] == -np.inf).all()
        assert (np.abs(host(lse[part])[~empty] - want_lse[~empty]) <= tol_lse[~empty] + 2.0 ** -23 * np.abs(want_lse[~empty])).all()
    return worst


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("heads, kv_heads, width, page", [(1, 1, 1, 32), (8, 8, 36, 32), (8, 8, 40, 32), (8, 8, 52, 64), (4, 2, 64, 32), (8, 4, 80, 32),
                                                          (6, 2, 96, 64), (16, 2, 128, 128), (3, 3, 130, 32), (4, 1, 160, 32), (2, 2, 192, 32),
                                                          (3, 1, 224, 32), (8, 2, 256, 64)])
def test_attention_single_tokens(dtype, heads, kv_heads, width, page):
    """One row a sequence; lengths of zero and one, at and around the ends of blocks and pages."""
    lengths = [0, 1, 31, 32, 33, 64, 65, 100, 127, 128, 129, 200]
    check_attention(dtype, heads, kv_heads, width, page, lengths, [1] * len(lengths), uniform=True)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("counts, heads, kv_heads, width", [([2] * 5, 8, 8, 52), ([4] * 5, 8, 8, 36), ([8] * 5, 8, 2, 64), ([3, 0, 17, 1, 5], 6, 2, 128),
                                                            ([40, 1, 0, 33, 9], 4, 2, 96), ([100, 3, 64, 200, 1], 4, 4, 52), ([70, 0, 130, 5, 1], 3, 1, 256)])
@pytest.mark.parametrize("causal, window", [(True, 0), (False, 0), (True, 1), (True, 37)])
def test_attention_several_rows(dtype, counts, heads, kv_heads, width, causal, window):
    """Beams, drafts and chunks of prompts: every variant of the kernel, masks that leave rows empty (more rows than tokens)."""
    lengths = [5, 64, 150, 203, 1]
    check_attention(dtype, heads, kv_heads, width, 32, lengths, counts, causal, window, seed=5)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("batch, heads, kv_heads, width, n", [(1, 8, 8, 52, 415), (2, 8, 1, 64, 3001), (1, 16, 2, 128, 5000), (3, 4, 2, 256, 1111)])
def test_attention_long_is_split_and_joined(dtype, batch, heads, kv_heads, width, n):
    """Few rows over long caches: the key ranges of several workgroups are joined; one sequence is far shorter than the table."""
    lengths = [n] + [n // 3, 2][:batch - 1]
    check_attention(dtype, heads, kv_heads, width, 64, lengths, [1] * batch, uniform=True, seed=9)
    check_attention(dtype, heads, kv_heads, width, 64, lengths, [3] * batch, window=n // 2, seed=10)


@pytest.mark.parametrize("width", [32, 96, 128, 256])
def test_attention_many_ranges(width):
    """More key ranges than an eighth or a half of a wave, also odd numbers of them: each must find its weight when they are joined."""
    for others in (3, 58):
        check_attention("bf16", 1, 1, width, 64, [18000] + ([300, 0, 7] * 20)[:others], [1] * (others + 1), uniform=True, seed=11)
    check_attention("bf16", 2, 2, width, 64, [7400, 33], [1, 1], uniform=True, seed=12)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("window", [0, 700])
def test_attention_long_chunks(dtype, window):
    """Chunks of prompts behind long beginnings: key ranges are split here too, some of them with nothing that a row sees."""
    check_attention(dtype, 4, 2, 128, 64, [3000, 700, 40, 0], [300, 33, 40, 2], window=window, seed=12)
    check_attention(dtype, 2, 2, 52, 32, [2111], [129], causal=window > 0, window=window, seed=13)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("heads, kv_heads, width, page", [(8, 8, 52, 32), (8, 8, 32, 64), (16, 8, 128, 64), (24, 8, 96, 32), (8, 8, 160, 32), (8, 8, 224, 32), (8, 8, 256, 128)])
@pytest.mark.parametrize("causal, window", [(True, 0), (False, 0), (True, 37)])
def test_attention_batches_of_chunks(dtype, heads, kv_heads, width, page, causal, window):
    """A batch with room for enough prompts that a block is expanded once for four waves: whole and broken tiles, more rows than tokens,
    sequences without rows or tokens."""
    counts, lengths = [70, 0, 128, 1, 0, 129, 65] + [0] * 57 + [30, 90], [300, 64, 150, 203, 1, 0, 33] + [0] * 57 + [97, 64]
    check_attention(dtype, heads, kv_heads, width, page, lengths, counts, causal, window, seed=14)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("window", [0, 5000])
def test_attention_batches_of_long_chunks(dtype, window):
    """The same with key ranges of two workgroups, one sequence far longer than the others."""
    check_attention(dtype, 8, 8, 64, 64, [8200, 100, 0, 33] + [40] * 60, [70, 70, 3, 65] + [7] + [0] * 59, window=window, seed=15)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("width", [52, 96, 128, 224, 256])
@pytest.mark.parametrize("batch", [60, 110, 300])
def test_attention_single_tokens_of_large_batches(dtype, width, batch):
    """Sequences enough that four, two or one wave take a tile, in short tables and longer ones; most have no tokens."""
    lengths = [33, 0, 120, 1, 64] + [0] * (batch - 7) + [95, 32]
    check_attention(dtype, 8, 8, width, 32, lengths, [1] * batch, uniform=True, seed=16)
    lengths[7] = 300
    check_attention(dtype, 16, 8, width, 64, lengths, [1] * batch, seed=17)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("width", [36, 64, 80, 128, 192, 256])
@pytest.mark.parametrize("causal, window", [(True, 0), (False, 0), (True, 37)])
def test_attention_drafts_of_large_batches(dtype, width, causal, window):
    """The same with several rows a sequence: tiles of 32."""
    counts, lengths = [40, 0, 17, 1, 64, 33] + [0] * 60 + [2, 50], [100, 64, 150, 203, 33, 1] + [0] * 60 + [97, 0]
    check_attention(dtype, 8, 8, width, 32, lengths, counts, causal, window, seed=18)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_attention_drafts_over_a_long_cache(dtype):
    """Tiles of 32 and key ranges."""
    check_attention(dtype, 8, 8, 52, 64, [16500, 40, 0, 300] + [1] * 40, [33, 20, 1, 2] + [1] + [0] * 39, seed=19)


def test_attention_chunks_with_pages_that_are_not_there():
    """A page outside the cache counts as absent in every form: its tokens get no weight."""
    batch, rows, n = 64, 70, 160
    k, v = values(gen(3), (batch * 5, 8, 32, 64)), values(gen(4), (batch * 5, 8, 32, 64))
    cache = ops.kv4_cache(batch * 5, 8, 32, 64)
    slots = torch.arange(batch * 160, device="cuda")
    ops.kv4_write(cache, dev(np.ascontiguousarray(k.transpose(0, 2, 1, 3)).reshape(-1, 8, 64)), dev(np.ascontiguousarray(v.transpose(0, 2, 1, 3)).reshape(-1, 8, 64)), slots)
    table = torch.arange(batch * 5, dtype=torch.int32, device="cuda").view(batch, 5).clone()
    q = dev(values(gen(5), (batch * rows, 8, 64)), torch.bfloat16)
    lens = i32([n] * batch)
    bad = table.clone()
    bad[:, 1], bad[:, 3] = -1, batch * 5
    out = ops.kv4_attention(q, cache, bad, lens, max_q=rows, causal=False)
    short = table[:, [0, 2, 4]].contiguous()
    want = ops.kv4_attention(q, cache, short, i32([96] * batch), max_q=rows, causal=False)
    assert torch.equal(out, want)


@pytest.mark.parametrize("batch, rows, n", [(2, 1, 90), (2, 20, 90), (64, 70, 90), (1, 1, 5000)])
def test_attention_into_its_own_queries_and_rows_of_nan(batch, rows, n):
    """out may be q; a NaN query gives NaN (lse too) in its own row and in no other."""
    cache = ops.kv4_cache(80, 8, 64, 64)
    t = torch.arange(80 * 64, device="cuda")
    ops.kv4_write(cache, dev(values(gen(6), (len(t), 8, 64))), dev(values(gen(7), (len(t), 8, 64))), t)
    table = i32([[(b + j) % 80 for j in range(80)] for b in range(batch)])
    q = dev(values(gen(8), (batch * rows, 8, 64)), torch.bfloat16)
    lens = i32([n] * batch)
    want, lse = ops.kv4_attention(q, cache, table, lens, max_q=rows, return_lse=1)
    bad = q.clone()
    bad[0, 3, 5] = float("nan")
    got, got_lse = ops.kv4_attention(bad, cache, table, lens, max_q=rows, return_lse=True, out=bad)
    assert got.data_ptr() == bad.data_ptr() and got[0, 3].isnan().all() and got_lse[0, 3].isnan()
    got[0, 3], got_lse[0, 3] = want[0, 3], lse[0, 3]
    assert torch.equal(got, want) and torch.equal(got_lse, lse)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_attention_sharp_and_flat_rows(dtype):
    """Scores of hundreds (one token takes all; the running maximum moves often) and of nothing."""
    check_attention(dtype, 4, 2, 64, 32, [300, 64, 33], [2, 2, 2], magnitude=60.0, seed=1)
    check_attention(dtype, 4, 2, 64, 32, [300, 64, 33], [2, 2, 2], scale=0.0, seed=2)
    check_attention(dtype, 4, 2, 64, 32, [300, 64, 33], [90, 2, 33], scale=-2.0, seed=3)


@pytest.mark.parametrize("fill", [0x00, 0x7F, 0x80, 0xFF])
def test_attention_never_sees_bytes_behind_the_end(fill):
    """Whatever stands behind the last token (0xFF: scales that mean NaN), in pages that end inside a tile, single tokens and chunks."""
    check_attention("f32", 4, 2, 52, 64, [1, 33, 70], [1, 1, 1], fill=fill, seed=4)
    check_attention("bf16", 4, 2, 128, 32, [40, 70, 95], [40, 33, 70], fill=fill, seed=4)


def test_attention_ascending_scores():
    """Each block's scores pass the earlier maximum: what was summed before is scaled down every time, also in the wide variant."""
    n, width = 260, 32
    k = np.zeros((n, 1, width), np.float32)
    k[:, 0, 0] = np.arange(n) * 0.5
    v = values(gen(2), (n, 1, width))
    cache = ops.kv4_cache(9, 1, 32, width)
    ops.kv4_write(cache, dev(k), dev(v), torch.arange(n, device="cuda"))
    table = i32([list(range(9))])
    for rows in (1, 20, 80):
        q = np.zeros((rows, 1, width), np.float32)
        q[:, 0, 0] = np.linspace(0.5, 4.0, rows)
        want, _, mass, top, spread = ref.attention(q.astype(np.float64), ref.quantise(k), ref.quantise(v), ref.visible(rows, n, False), 1.0)
        out = ops.kv4_attention(dev(q), cache, table, i32([n]), scale=1.0, causal=False)
        assert (np.abs(host(out) - want) <= bound("f32", width, n, want, mass, top, spread)[0]).all()


@pytest.mark.parametrize("rows", [1, 30, 100])
def test_attention_bad_pages_count_as_masked(rows):
    """Page numbers that are not in the cache: their tokens are left out, in every variant; all bad: an empty row."""
    n, width, page = 200, 64, 32
    rng = gen(8)
    k, v = values(rng, (n, 2, width)), values(rng, (n, 2, width))
    cache = ops.kv4_cache(7, 2, page, width)
    ops.kv4_write(cache, dev(k), dev(v), torch.arange(n, device="cuda"))
    table = np.arange(7, dtype=np.int32)[None].copy()
    table[0, [1, 4]] = [-1, 7]
    table[0, 5] = np.iinfo(np.int32).max
    q = values(rng, (rows, 4, width))
    see = ref.visible(rows, n, True)
    see[:, (np.arange(n) // page == 1) | (np.arange(n) // page == 4) | (np.arange(n) // page == 5)] = False
    out, lse = ops.kv4_attention(dev(q), cache, dev(table), i32([n]), return_lse=True)
    want, want_lse, mass, top, spread = ref.attention(q.astype(np.float64), ref.quantise(k), ref.quantise(v), see, width ** -0.5)
    assert (np.abs(host(out) - want) <= bound("f32", width, n, want, mass, top, spread)[0]).all()
    out, lse = ops.kv4_attention(dev(q), cache, torch.full((1, 7), -5, dtype=torch.int32, device="cuda"), i32([n]), return_lse=True)
    assert not out.any() and (lse == -torch.inf).all()


def test_attention_lengths_and_starts_that_do_not_fit_are_cut():
    """Device values the host cannot see: negative and too long lengths, row ranges outside the call."""
    width = 32
    rng = gen(6)
    x = values(rng, (64, 1, width))
    cache = ops.kv4_cache(2, 1, 32, width)
    ops.kv4_write(cache, dev(x), dev(x), torch.arange(64, device="cuda"))
    q = dev(values(rng, (4, 1, width)))
    table = i32([[0, 1], [0, 1], [1, 0], [0, 1]])
    out = ops.kv4_attention(q, cache, table, i32([-3, 10 ** 9, 40, 64]), causal=False)
    same = ops.kv4_attention(q, cache, table, i32([0, 64, 40, 64]), causal=False)
    assert torch.equal(out, same) and not out[0].any()
    keep = torch.full((4, 1, width), 3.0, device="cuda")
    ops.kv4_attention(q, cache, table, i32([64] * 4), q_start=i32([0, 2, 9, 1, -4]), max_q=2, causal=False, out=keep)
    want = ops.kv4_attention(q, cache, table[:2], i32([64, 64]), causal=False)     # of rows 2 .. 8 the first max_q
    assert torch.equal(keep, want)
    keep.fill_(3.0)
    ops.kv4_attention(q, cache, table, i32([64] * 4), q_start=i32([0, 2, 9, 1, -4]), max_q=8, causal=False, out=keep)
    assert torch.equal(keep[:2], want[:2]) and (keep[2:] == 3.0).all()             # rows 2 .. 8 are not in the call


@pytest.mark.parametrize("dtype", list(TYPES))
def test_attention_strided_rows_and_outputs(dtype):
    """q inside a fused projection, out inside a wider buffer, rows at odd element offsets."""
    rng = gen(12)
    n, heads, width = 90, 4, 52
    cache = ops.kv4_cache(3, 2, 32, width)
    x = values(rng, (n, 2, width))
    ops.kv4_write(cache, dev(x), dev(x), torch.arange(n, device="cuda"))
    fused = dev(values(rng, (3, 2, heads, width + 5)), TYPES[dtype])
    q = fused[:, 1, :, 3:3 + width]
    wide = torch.zeros((3, heads, 2 * width + 1), dtype=TYPES[dtype], device="cuda")
    table = i32([[2, 0, 1]] * 3)
    lens = i32([90, 41, 7])
    ops.kv4_attention(q, cache, table, lens, out=wide[:, :, width:2 * width])
    want = ops.kv4_attention(q.contiguous(), cache, table, lens)
    assert torch.equal(wide[:, :, width:2 * width], want) and not wide[:, :, :width].any() and not wide[:, :, 2 * width:].any()


# ------------------------------------------------------------------ plan
@pytest.mark.parametrize("batch, page, longest, n_free", [(1, 32, 40, 99), (3, 32, 200, 99), (5, 64, 500, 7), (300, 32, 300, 10000), (1500, 128, 900, 400),
                                                          (4, 256, 100000, 5000), (2100, 32, 70, 3000)])
def test_plan(batch, page, longest, n_free):
    rng = gen(batch + page)
    held = rng.integers(0, longest + 1, batch)
    new = np.minimum(rng.integers(0, 80, batch), held)
    if batch > 3:
        held[1], new[1] = -5, 3
        new[2] = held[2] + 9
        held[3], new[3] = longest * 3, 10                  # past the table
    width = -(-longest // page) + 1
    table = rng.integers(0, 1 << 20, (batch, width)).astype(np.int32)
    gaps = rng.integers(0, 3, batch)
    cut = np.clip(new, 0, np.clip(held, 0, width * page))
    start = (np.cumsum(cut + gaps) - cut).astype(np.int32)
    rows = int(start[-1] + cut[-1] + 5) if batch else 0
    free = rng.permutation(1 << 20)[:n_free].astype(np.int32)
    want = ref.page_plan(table, held, new, start, rows, free, page)
    got = dev(table)
    slots, used = ops.page_plan(got, i32(held.tolist()), i32(new.tolist()), dev(start), rows, dev(free), page)
    assert int(used) == want[2]
    assert np.array_equal(host(got), want[0])
    assert np.array_equal(host(slots), want[1])


def test_plan_without_rows_or_pages():
    table = torch.full((2, 3), 4, dtype=torch.int32, device="cuda")
    slots, used = ops.page_plan(table, i32([33, 0]), i32([1, 0]), i32([0, 1]), 0, i32([]), 32)
    assert slots.numel() == 0 and int(used) == 1 and host(table).tolist() == [[4, -1, -1], [-1, -1, -1]]


# ------------------------------------------------------------------ selection
def check_select(logits, scores, finished, eos, sure=0.9, **layout):
    got = [host(t) for t in ops.beam_select(logits, dev(scores.astype(np.float32)), dev(finished.astype(np.uint8)), eos)]
    s, p, t, f, order = ref.beam_select(host(logits), scores.astype(np.float32), finished, eos)
    # fp32 exponentials (argument (x - max) * log2 e rounded: 40 * 2^-24, exp2 2^-23), summed in part in 64 bits; a score rounded to fp32
    tol = 2.0 ** -19
    clear = 0
    for b in range(s.shape[0]):
        near = [abs(x - y) <= tol and i != j for (x, i), (y, j) in zip(zip(*order[b]), list(zip(*order[b]))[1:])]
        fin = np.isfinite(s[b])
        assert np.array_equal(np.isfinite(got[0][b]), fin)
        assert (np.abs(got[0][b][fin] - s[b][fin]) <= tol + 2.0 ** -24 * np.abs(s[b][fin])).all()
        if any(near):
            continue                                         # two beams' candidates closer than the sums are exact
        clear += 1
        assert got[1][b].tolist() == p[b].tolist() and got[2][b].tolist() == t[b].tolist() and got[3][b].astype(bool).tolist() == f[b].tolist(), b
    assert clear >= sure * s.shape[0]
    return got


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("batch, beams, vocab", [(1, 1, 1), (2, 3, 2), (1, 4, 512), (3, 2, 33), (5, 16, 17), (4, 5, 1000), (2, 8, 2049), (1, 4, 32768),
                                                 (40, 3, 5003), (2, 16, 30001), (300, 2, 700), (1, 2, 150001), (1, 7, 193001), (2, 11, 90000),
                                                 (1, 16, 70001), (1, 5, 140000), (3, 10, 50)])
def test_select(dtype, batch, beams, vocab):
    rng = gen(batch * 7 + vocab)
    logits = dev((3 * rng.standard_normal((batch, beams, vocab))).astype(np.float32), TYPES[dtype])
    scores = -np.sort(rng.exponential(4.0, (batch, beams)), 1)
    finished = rng.random((batch, beams)) < 0.2
    scores[rng.random((batch, beams)) < 0.1] = -np.inf
    check_select(logits, scores, finished, min(2, vocab - 1))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("beams", [1, 4, 16])
def test_select_ties_go_to_the_lowest(dtype, beams):
    """All logits equal, many equal at the border, equal scores: exact ties, within a row and between rows."""
    for vocab in (40, 3000, 9000):
        x = torch.zeros((2, beams, vocab), dtype=TYPES[dtype], device="cuda")
        x[1, :, vocab // 2:] = 2.0
        scores = np.zeros((2, beams))
        got = check_select(x, scores, np.zeros((2, beams)), -1, sure=0.0)
        assert got[1][0].tolist() == [0] * beams and got[2][0].tolist() == list(range(min(beams, vocab)))
        assert got[2][1].tolist() == list(range(vocab // 2, vocab // 2 + beams))
        x[0, :, 5::3] = 1.5
        got = check_select(x, scores, np.zeros((2, beams)), -1, sure=0.0)
        ids = list(range(5, vocab, 3))                       # of 40 ids, twelve: the next beam's follow
        assert got[2][0].tolist() == [ids[i % len(ids)] for i in range(beams)]
        assert got[1][0].tolist() == [i // len(ids) for i in range(beams)]


@pytest.mark.parametrize("beams", [3, 8, 13])
def test_select_ties_over_long_rows(beams):
    """As many lists and candidates as the second pass can hold, all equal."""
    got = check_select(torch.zeros((2, beams, 140000), device="cuda"), np.zeros((2, beams)), np.zeros((2, beams)), 5, sure=0.0)
    assert got[1].tolist() == [[0] * beams] * 2 and got[2].tolist() == [list(range(beams))] * 2 and got[3][:, 5:6].all()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_select_masked_infinite_and_nan_logits(dtype):
    rng = gen(4)
    x = (2 * rng.standard_normal((6, 3, 4100))).astype(np.float32)
    x[0, 0] = -np.inf                                        # a row with nothing left
    x[1] = -np.inf
    x[1, 1, 4090] = 1.0                                      # one candidate in all
    x[2, :, 100:4000] = -np.inf
    x[3, 0, 77] = np.inf
    x[3, 1, [5, 9]] = np.inf
    x[4, :, ::3] = np.nan
    x[5, :, 1:] = torch.finfo(TYPES[dtype]).min              # masked by the type's lowest value: still candidates
    t = dev(x, TYPES[dtype])
    scores = np.tile([-0.5, -1.0, -1.5], (6, 1))
    got = check_select(t, scores, np.zeros((6, 3)), 2, sure=0.8)
    assert got[2][1].tolist() == [4090, 2, 2] and got[1][1].tolist() == [1, 1, 2] and got[3][1].tolist() == [0, 1, 1]
    assert got[2][5].tolist() == [0, 0, 0]


def test_select_finished_and_dead_beams_do_not_read_their_logits():
    x = torch.full((1, 4, 50), float("nan"), device="cuda")
    x[0, 0] = torch.arange(50, 0, -1, device="cuda") * 0.1
    scores = np.array([[-3.0, -1.0, -np.inf, -np.inf]])
    got = check_select(x, scores, np.array([[0, 1, 0, 1]]), 7)
    assert got[2][0, 0] == 7 and got[1][0, 0] == 1 and got[3][0, 0] == 1 and got[0][0, 0] == -1.0
    got = check_select(x, np.full((1, 4), -np.inf), np.zeros((1, 4)), 7)
    assert got[1][0].tolist() == [0, 1, 2, 3] and (got[2] == 7).all() and got[3].all()
    s, p, t, f = ops.beam_select(x, dev(scores.astype(np.float32)), torch.tensor([[False, True, False, True]], device="cuda"), -1)
    assert f.dtype is torch.bool and int(t[0, 0]) == -1 and bool(f[0, 0]) and not bool(f[0, 1])


@pytest.mark.parametrize("dtype", list(TYPES))
def test_select_rows_inside_a_wider_buffer(dtype):
    rng = gen(14)
    wide = dev(rng.standard_normal((3, 4, 1111)).astype(np.float32), TYPES[dtype])
    x = wide[:, :, 1:1004]                                   # odd addresses, garbage (NaN) before and behind
    wide[:, :, 0] = float("nan")
    wide[:, :, 1004:] = float("nan")
    check_select(x, -rng.random((3, 4)), np.zeros((3, 4)), 2)


# ------------------------------------------------------------------ reordering
@pytest.mark.parametrize("outer, batch, beams, inner, room, row, dtype", [
    (8, 1, 4, 8, 72, 52, torch.bfloat16), (2, 3, 2, 3, 5, 1, torch.uint8), (1, 2, 5, 1, 7, 3, torch.int16), (3, 2, 8, 2, 9, 36, torch.bfloat16),
    (1, 4, 16, 2, 33, 20, torch.float32), (2, 2, 7, 1, 1, 1, torch.int32), (1, 1, 1, 4, 8, 8, torch.float32), (1, 2, 3, 2, 40, 13, torch.uint8)])
@pytest.mark.parametrize("how", ["each", "one", "all"])
def test_reorder(outer, batch, beams, inner, room, row, dtype, how):
    rng = gen(batch * 100 + beams + room)
    x = torch.from_numpy(rng.integers(0, 100, (outer, batch, beams, inner, room, row))).to(dtype).cuda()
    parents = rng.integers(0, beams, (batch, beams))
    parents[0, beams - 1] = [beams, -1, 1 << 30][room % 3]   # no beam
    lengths = {"each": rng.integers(0, room + 3, batch), "one": np.full(batch, room // 2), "all": np.full(batch, room)}[how]
    want = ref.reorder(host(x), parents, lengths)
    given = {"each": i32(lengths.tolist()), "one": i32([room // 2]), "all": None}[how]
    if how == "each":
        given[0] = -2 if batch > 1 else given[0]
        if batch > 1:
            lengths[0] = 0
            want = ref.reorder(host(x), parents, lengths)
    ops.beam_reorder([x], i32(parents.tolist()), given, batch_dims=[1], row_dims=[4])
    assert np.array_equal(host(x), want)


def test_reorder_several_states_at_once():
    """Keys, values, ids and a strided view, one launch; what lies between the rows stays."""
    rng = gen(21)
    batch, beams, room = 3, 4, 19
    k = dev(rng.standard_normal((2, batch, beams, 3, room, 20)).astype(np.float32), torch.bfloat16)
    v = dev(rng.standard_normal((batch, beams, room, 5)).astype(np.float32))
    ids = dev(rng.integers(0, 99, (batch, beams, room)).astype(np.int32))
    wide = dev(rng.integers(0, 99, (batch, beams, 2, room + 6)).astype(np.int16))
    view = wide[:, :, 1, 3:3 + room]
    parents, lengths = rng.integers(0, beams, (batch, beams)), rng.integers(0, room + 1, batch)
    w = [ref.reorder(host(k), parents, lengths), ref.reorder(host(v)[None, :, :, None], parents, lengths)[0, :, :, 0],
         ref.reorder(host(ids)[None, :, :, None], parents, lengths)[0, :, :, 0]]
    wide_want = host(wide).copy()
    wide_want[:, :, 1, 3:3 + room] = ref.reorder(host(view)[None, :, :, None], parents, lengths)[0, :, :, 0]
    ops.beam_reorder([k, v, ids, view], i32(parents.tolist()), i32(lengths.tolist()), batch_dims=[1, 0, 0, 0], row_dims=[4, 2, 2, 2])
    for got, want in zip((k, v, ids, wide), w + [wide_want]):
        assert np.array_equal(host(got), want)


# ------------------------------------------------------------------ refusals of the wrappers, streams, graphs, the whole step
def test_wrappers_refuse():
    z = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
    cache = ops.kv4_cache(2, 2, 32, 40)
    slots, table, lens, scores = z(3, t=torch.int64), z(1, 2, t=torch.int32), z(1, t=torch.int32), z(2, 3, 4)
    bad = [
        lambda: ops.kv4_write(cache, z(3, 2, 40).requires_grad_(), z(3, 2, 40), slots),
        lambda: ops.kv4_write(cache, z(3, 2, 40, t=torch.float64), z(3, 2, 40, t=torch.float64), slots),
        lambda: ops.kv4_write(cache, z(3, 1, 40), z(3, 1, 40), slots),
        lambda: ops.kv4_write(cache, z(3, 2, 65), z(3, 2, 65), slots),
        lambda: ops.kv4_write(cache, z(3, 2, 40), z(3, 2, 40), slots.int()),
        lambda: ops.kv4_write(cache, z(3, 2, 40), z(3, 2, 40), slots[:2]),
        lambda: ops.kv4_write(cache, z(3, 2, 40), z(3, 2, 40), slots.cpu()),
        lambda: ops.kv4_write(cache.transpose(0, 1), z(3, 2, 40), z(3, 2, 40), slots),
        lambda: ops.kv4_read(cache, slots, 40, torch.int32),
        lambda: ops.kv4_attention(z(1, 3, 40), cache, table, lens),
        lambda: ops.kv4_attention(z(3, 2, 40), cache, table.expand(2, 2).contiguous(), lens.expand(2).contiguous()),
        lambda: ops.kv4_attention(z(1, 2, 40), cache, table, lens.long()),
        lambda: ops.kv4_attention(z(1, 2, 40), cache, table, lens, causal=False, window=3),
        lambda: ops.kv4_attention(z(1, 2, 40), cache, table, lens, q_start=z(2, t=torch.int32)),
        lambda: ops.kv4_attention(z(1, 2, 80)[:, :, ::2], cache, table, lens),
        lambda: ops.kv4_attention(z(1, 2, 40), cache, table, lens, out=z(1, 2, 40, t=torch.bfloat16)),
        lambda: ops.kv4_attention(z(1, 2, 40).requires_grad_(), cache, table, lens),
        lambda: ops.kv4_attention(z(1, 2, 40), cache, table, lens, out=z(1, 2, 40).requires_grad_()),
        lambda: ops.kv4_attention(z(1, 2, 40), cache, table, lens, out=z(1, 1, 40).expand(1, 2, 40)),
        lambda: ops.kv4_attention(z(2, 2, 40), cache, table, lens, max_q=2, out=z(160).as_strided((2, 2, 40), (60, 40, 1))),
        lambda: ops.page_plan(table, lens, lens, lens, -1, lens, 32),
        lambda: ops.page_plan(table, lens, lens, lens, 1, lens, 31),
        lambda: ops.page_plan(table.long(), lens, lens, lens, 1, lens, 32),
        lambda: ops.beam_select(z(1, 17, 30), z(1, 17), z(1, 17, t=torch.uint8), 2),
        lambda: ops.beam_select(z(1, 2, 30), z(1, 2), z(1, 2, t=torch.uint8), 30),
        lambda: ops.beam_select(z(1, 2, 30), z(1, 2), z(1, 2, t=torch.int32), 2),
        lambda: ops.beam_select(z(3, 4, 30)[:, :2], z(3, 2), z(3, 2, t=torch.uint8), 2),
        lambda: ops.beam_reorder([z(2, 3, 4).transpose(1, 2)], z(2, 4, t=torch.int32), batch_dims=[0], row_dims=[2]),
        lambda: ops.beam_reorder([z(2, 3, 4)], z(2, 4, t=torch.int32), batch_dims=[0], row_dims=[2]),
        lambda: ops.beam_reorder([z(2, 3, 4)], z(2, 3, t=torch.int32), batch_dims=[0], row_dims=[1]),
        lambda: ops.beam_reorder([z(1, 3, 4).expand(2, 3, 4)], z(2, 3, t=torch.int32), batch_dims=[0], row_dims=[2]),
        lambda: ops.beam_reorder([z(2, 3, 4)], z(2, 3, t=torch.int32), z(3, t=torch.int32), batch_dims=[0], row_dims=[2]),
        lambda: ops.beam_reorder([z(1, 2, 3, 4).expand(5, 2, 3, 4)], z(2, 3, t=torch.int32), batch_dims=[1], row_dims=[3]),
        lambda: ops.beam_reorder([scores, scores], z(2, 3, t=torch.int32), batch_dims=[0, 0], row_dims=[2, 2]),
        lambda: ops.beam_reorder([z(2, 3, 4)] * 5, z(2, 3, t=torch.int32), batch_dims=[0] * 5, row_dims=[2] * 5),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(MshError) as e:
            call()
        assert e.value.code == -3, i
    with torch.no_grad():                                    # no gradient is asked for: fine
        ops.kv4_write(cache, z(3, 2, 40).requires_grad_(), z(3, 2, 40), torch.arange(3, device="cuda"))
    ops.kv4_write(cache, z(0, 2, 40), z(0, 2, 40), slots[:0])
    assert ops.kv4_attention(z(0, 2, 40), cache, table[:0], lens[:0]).shape == (0, 2, 40)
    assert [t.shape for t in ops.beam_select(z(0, 2, 30), z(0, 2), z(0, 2, t=torch.uint8), 2)] == [(0, 2)] * 4


class Step:
    """A decode step of four requests with two beams each as a server would run it: plan, write, attend, select, reorder."""

    def __init__(self, seed, page=32, width=52, heads=4, kv_heads=2, vocab=3001, rows=8):
        rng = gen(seed)
        self.width, self.page = width, page
        self.cache = ops.kv4_cache(40, kv_heads, page, width)
        self.lens0 = np.array([31, 32, 40, 64, 1, 90, 33, 96])
        free = rng.permutation(40).astype(np.int32)
        kept = -(-self.lens0 // page)
        self.table = np.full((rows, 6), -1, np.int32)
        at = 0
        for b in range(rows):
            self.table[b, :kept[b]] = free[at:at + kept[b]]
            at += kept[b]
        self.free = dev(free[at:])
        self.table = dev(self.table)
        self.past = []
        for b in range(rows):
            t = np.arange(self.lens0[b])
            k, v = values(rng, (len(t), kv_heads, width)), values(rng, (len(t), kv_heads, width))
            ops.kv4_write(self.cache, dev(k), dev(v), dev(host(self.table)[b, t // page].astype(np.int64) * page + t % page))
            self.past.append((k, v))
        self.lens = i32((self.lens0 + 1).tolist())
        self.ones, self.start = i32([1] * rows), i32(list(range(rows)))
        self.k, self.v = dev(values(rng, (rows, kv_heads, width))), dev(values(rng, (rows, kv_heads, width)))
        self.q = dev(values(rng, (rows, heads, width)))
        self.head = dev((rng.standard_normal((heads * width, vocab)) / np.sqrt(heads * width)).astype(np.float32))
        self.scores, self.finished = dev(-np.sort(rng.random((4, 2)).astype(np.float32) * 3, 1)), torch.zeros((4, 2), dtype=torch.uint8, device="cuda")
        self.state = dev(rng.standard_normal((4, 2, 5, 6)).astype(np.float32))

    def run(self):
        table, state = self.table.clone(), self.state.clone()
        slots, used = ops.page_plan(table, self.lens, self.ones, self.start, 8, self.free, self.page)
        ops.kv4_write(self.cache, self.k, self.v, slots)
        out = ops.kv4_attention(self.q, self.cache, table, self.lens)
        logits = torch.mm(out.flatten(1), self.head).view(4, 2, -1)
        picked = ops.beam_select(logits, self.scores, self.finished, 2)
        ops.beam_reorder([state], picked[1], batch_dims=[0], row_dims=[2])
        return [out, logits, *picked, state, slots, used, table]


def test_a_decode_step_as_a_whole():
    s = Step(1)
    out, logits, scores, parents, tokens, finished, state, slots, used, table = s.run()
    outs = []
    for b in range(8):
        k, v = (np.concatenate([p, host(n[b:b + 1])]) for p, n in zip(s.past[b], (s.k, s.v)))
        want, _, mass, top, spread = ref.attention(host(s.q[b:b + 1]), ref.quantise(k), ref.quantise(v), ref.visible(1, len(k), True), s.width ** -0.5)
        assert (np.abs(host(out[b:b + 1]) - want) <= bound("f32", s.width, len(k), want, mass, top, spread)[0]).all()
        outs.append(want)
    assert int(used) == int((s.lens0 % s.page == 0).sum())
    w = ref.beam_select(host(logits), host(s.scores).astype(np.float32), np.zeros((4, 2)), 2)
    assert np.array_equal(host(parents), w[1]) and np.array_equal(host(tokens), w[2])
    assert np.array_equal(host(state), ref.reorder(host(s.state)[None, :, :, None], w[1], [5] * 4)[0, :, :, 0])


def test_replayed_graphs_and_other_streams():
    """Two steps captured into graphs, replayed in turn on two streams beside eager calls of others: every replay is the eager result."""
    steps = [Step(2), Step(3, width=128, page=64)]
    want = [s.run() for s in steps]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s, stream in zip(steps, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(s.run())
        graphs.append(g)
    other = Step(4)
    alone = other.run()
    for turn in range(4):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for g, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
        beside = other.run()
        torch.cuda.synchronize()
        for a, b in zip(want[0] + want[1] + alone, outs[0] + outs[1] + beside):
            assert torch.equal(a, b), turn


def test_same_call_same_bits():
    """The order of sums goes by the call alone."""
    s = Step(5)
    first = s.run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, s.run()))


def test_threads_call_at_once():
    import threading

    steps = [Step(6 + i) for i in range(4)]
    want = [s.run() for s in steps]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got = steps[i].run()
            torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, b) for a, b in zip(want[i], got)):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong

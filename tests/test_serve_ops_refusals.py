"""What the serving operators refuse, on the CPU: every refusal comes before anything touches a device, so none of these needs one."""
import ctypes as C
import struct

import numpy as np
import pytest
import torch

import serve_ref
from moonshine_amd import ops
from moonshine_amd.hip_api import MshError, load_library

CACHE = struct.Struct("Pqiiixxxx")                        # msh_kv4_cache
ATTENTION = struct.Struct("PPPqqqqPPPPqiiixxxxqiiiiiiif")   # msh_kv4_attention_args
STATE = struct.Struct("Pqqqqqqq")                         # msh_beam_state
STRIDES = struct.Struct("qqq")
FAKE = 1 << 20   # a 16-byte aligned address that nothing reads


def _attention(**change):
    a = dict(q=FAKE, out=FAKE, lse=0, q_row=64, q_head=64, out_row=64, out_head=64, table=FAKE, lens=FAKE, starts=0, data=FAKE, pages=4,
             kv_heads=1, page=32, width=64, rows=2, dtype=0, heads=1, batch=2, table_width=2, max_q=1, causal=1, window=0, scale=1.0)
    assert set(change) <= set(a)
    a.update(change)
    return ATTENTION.pack(*a.values())


@pytest.mark.parametrize("change, says", [
    (dict(dtype=3), "dtype"), (dict(page=48), "page_size"), (dict(page=16), "page_size"), (dict(page=131072), "page_size"),
    (dict(width=0), "head_dim"), (dict(width=257), "head_dim"), (dict(kv_heads=0), "heads"), (dict(heads=3, kv_heads=2), "multiple"),
    (dict(pages=0), "pages"), (dict(data=FAKE + 8), "aligned"), (dict(data=0), "aligned"), (dict(rows=3), "q_start"), (dict(rows=-1), "rows"),
    (dict(max_q=0), "max_q"), (dict(table_width=0), "table_width"), (dict(table_width=1 << 26), "table_width"),
    (dict(causal=0, window=4), "window needs causal"), (dict(window=-1), "window"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(q=0), "null"), (dict(out=0), "null"), (dict(table=0), "null"), (dict(lens=0), "null"),
    (dict(heads=65537), "heads"), (dict(batch=1 << 21, rows=1 << 21, heads=1024, kv_heads=1024), "too large"), (dict(batch=1 << 20, rows=1 << 20, heads=16, kv_heads=16), "too large"),
    (dict(batch=1 << 30, rows=0, starts=FAKE, heads=1024, kv_heads=1024, max_q=1 << 24), "too large"),
])
def test_attention_refuses(change, says):
    lib = load_library()
    rc = lib.msh_kv4_attention(0, None, _attention(**change), None, 0)
    assert rc == -3 and says in lib.msh_op_last_error().decode()


def test_attention_refuses_a_small_workspace():
    lib = load_library()
    args = _attention(table_width=64)                       # room for 2048 tokens, two sequences: split into ranges
    need = lib.msh_kv4_attention_workspace(args)
    assert need > 0
    for work, size in ((None, 0), (FAKE, need - 1), (FAKE + 4, need)):
        assert lib.msh_kv4_attention(0, None, args, work, size) == -3
        assert "workspace" in lib.msh_op_last_error().decode()


def test_nothing_to_do_is_no_error():
    """Empty calls return before they touch a device."""
    lib = load_library()
    assert lib.msh_kv4_attention(0, None, _attention(rows=0, batch=0, q=0), None, 0) == 0
    cache = CACHE.pack(FAKE, 4, 1, 32, 64)
    assert lib.msh_kv4_write(0, None, cache, None, None, None, None, 0, 0, None) == 0
    assert lib.msh_kv4_read(0, None, cache, None, 0, None, None, 0) == 0
    assert lib.msh_beam_select_workspace(0, 4, 100) == 0
    assert lib.msh_beam_select(0, None, None, 0, 0, 0, 4, 100, None, None, 2, None, None, None, None, None, 0) == 0
    assert lib.msh_beam_reorder(0, None, None, 0, 3, 4, None, None, 0) == 0


def test_plan_write_select_reorder_refuse():
    lib = load_library()
    says = lambda rc: (rc, lib.msh_op_last_error().decode())  # noqa: E731

    def plan(batch=2, width=2, rows=2, n_free=2, page=32, table=FAKE, slots=FAKE):
        return says(lib.msh_page_plan(0, None, table, batch, width, FAKE, FAKE, FAKE, rows, FAKE, n_free, page, slots, FAKE))

    for kw, word in ((dict(page=33), "page_size"), (dict(batch=0), "batch"), (dict(width=0), "table_width"), (dict(rows=-1), "rows"),
                     (dict(n_free=-1), "n_free"), (dict(table=None), "null"), (dict(slots=None), "null"), (dict(width=1 << 26), "table_width")):
        rc, msg = plan(**kw)
        assert rc == -3 and word in msg
    strides = STRIDES.pack(64, 64, 1)

    def write(pages=4, heads=1, page=32, width=64, dtype=0, rows=2, k=FAKE):
        return says(lib.msh_kv4_write(0, None, CACHE.pack(FAKE, pages, heads, page, width), k, strides, FAKE, strides, dtype, rows, FAKE))

    for kw, word in ((dict(pages=0), "pages"), (dict(heads=0), "heads"), (dict(page=40), "page_size"), (dict(width=300), "head_dim"),
                     (dict(dtype=-1), "dtype"), (dict(rows=-1), "rows"), (dict(rows=1 << 40), "rows"), (dict(k=None), "null")):
        rc, msg = write(**kw)
        assert rc == -3 and word in msg

    def select(batch=1, beams=2, vocab=10, dtype=0, row=10, eos=2, logits=FAKE, scores=FAKE, out=FAKE + 64, done=FAKE, done_out=FAKE + 64, work=FAKE, size=1 << 20):
        return says(lib.msh_beam_select(0, None, logits, dtype, row, batch, beams, vocab, scores, done, eos, out, FAKE, FAKE, done_out, work, size))

    for kw, word in ((dict(beams=0), "beams"), (dict(beams=17), "beams"), (dict(vocab=0), "vocab"), (dict(vocab=1 << 25), "vocab"), (dict(batch=-1), "batch"),
                     (dict(eos=10), "eos"), (dict(eos=-2), "eos"), (dict(dtype=5), "dtype"), (dict(logits=None), "null"), (dict(logits=FAKE + 2), "aligned"),
                     (dict(out=FAKE), "inputs"), (dict(done_out=FAKE), "inputs"), (dict(work=None), "workspace"), (dict(size=8), "workspace"), (dict(row=-1), "row_stride")):
        rc, msg = select(**kw)
        assert rc == -3 and word in msg

    def reorder(n=1, batch=1, beams=2, lstride=0, parents=FAKE, data=FAKE, outer=1, outer_stride=0, beam_stride=64, inner=1, inner_stride=0, row_bytes=8, n_rows=8):
        state = STATE.pack(data, outer, outer_stride, beam_stride, inner, inner_stride, row_bytes, n_rows)
        return says(lib.msh_beam_reorder(0, None, state * max(n, 1), n, batch, beams, parents, None, lstride))

    for kw, word in ((dict(n=5), "states"), (dict(n=-1), "states"), (dict(beams=17), "beams"), (dict(beams=0), "beams"), (dict(lstride=2), "length_stride"),
                     (dict(parents=None), "null"), (dict(data=0), "null"), (dict(beam_stride=63), "overlap"), (dict(inner=2, inner_stride=8), "overlap"),
                     (dict(row_bytes=-8), "sizes"), (dict(outer=1 << 20, inner=1 << 20, inner_stride=64), "too large")):
        rc, msg = reorder(**kw)
        assert rc == -3 and word in msg
    for kw, word in ((dict(outer=2, outer_stride=64), "overlap"), (dict(outer=2, outer_stride=0), "overlap"), (dict(batch=2, beams=1, beam_stride=0), "overlap"),
                     (dict(inner=4, inner_stride=-64), "overlap"), (dict(inner=3, inner_stride=64, beam_stride=128), "overlap"), (dict(n=2), "twice"),
                     (dict(n=1, outer=1 << 24, outer_stride=128), "too large")):
        rc, msg = reorder(**kw)
        assert rc == -3 and word in msg, (kw, rc, msg)
    for kw, word in ((dict(batch=1 << 22), "batch"), (dict(batch=(1 << 21) + 1, beams=1), "batch")):
        rc, msg = select(**kw)
        assert rc == -3 and word in msg
    rc, msg = write(rows=1 << 26)
    assert rc == -3 and "rows" in msg
    assert lib.msh_kv4_page_bytes(8, 64, 52) == 8 * 2 * 2176
    assert lib.msh_kv4_page_bytes(8, 64, 0) == -3


def test_messages_belong_to_their_thread():
    import threading

    lib = load_library()
    lib.msh_kv4_page_bytes(1, 33, 52)
    seen = []
    t = threading.Thread(target=lambda: seen.append(lib.msh_op_last_error()))
    t.start()
    t.join()
    assert seen == [b""] and b"page_size" in lib.msh_op_last_error()


def test_tensors_on_the_cpu_are_refused():
    z = torch.zeros
    with pytest.raises(MshError, match="no CPU fallback"):
        ops.kv4_write(z(1, 1, 1, 1088, dtype=torch.uint8), z(1, 1, 8), z(1, 1, 8), z(1, dtype=torch.int64))
    with pytest.raises(MshError, match="no CPU fallback"):
        ops.beam_select(z(1, 2, 8), z(1, 2), z(1, 2, dtype=torch.uint8), 2)
    with pytest.raises(MshError, match="no CPU fallback"):
        ops.beam_reorder([z(1, 2, 4)], z(1, 2, dtype=torch.int32), batch_dims=[0], row_dims=[2])
    with pytest.raises(MshError, match="page_size"):
        ops.kv4_cache(1, 1, 33, 8)


# ---- the oracles themselves (what the GPU tests hold the kernels to) ----
def test_oracle_quantiser_by_hand():
    x = np.array([[7.0, 6.99, 1.0, 0.25, -0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.1] + [0.0] * 20])
    # amax 7 = 1.75 * 4: power 1, unit 2
    want = 2.0 * np.array([4.0, 3.0, 0.5, 0.0, -0.0, 0.5, 0.5, 1.0, 1.0, 2.0, 2.0, -3.0] + [0.0] * 20)
    assert np.array_equal(serve_ref.quantise(x)[0], want)
    assert np.array_equal(serve_ref.quantise(x / 7 * 6.999)[0, :2], [6.0, 6.0])         # power 0: saturates
    ties = np.array([[4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5]])                           # unit 1
    assert np.array_equal(serve_ref.quantise(ties)[0], [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0])
    odd = serve_ref.quantise(np.array([[np.nan, 1.0, -np.inf]]))[0]
    assert odd[0] == 0.0 and odd[1] == 0.0 and odd[2] == -6.0 * 2.0 ** 125
    assert not serve_ref.quantise(np.full((1, 40), 1e-40)).any()


def test_oracle_selection_by_hand():
    logits = np.log(np.array([[[0.5, 0.25, 0.25, 0.0], [0.25, 0.25, 0.25, 0.25]]]) + 1e-300)
    s, p, t, f, _ = serve_ref.beam_select(logits, np.array([[0.0, np.log(0.9)]], np.float32), np.array([[0, 1]]), 3)
    assert p.tolist() == [[1, 0]] and t.tolist() == [[3, 0]] and f.tolist() == [[True, False]]
    assert abs(s[0, 1] - np.log(0.5)) < 1e-12
    s, p, t, f, _ = serve_ref.beam_select(np.zeros((1, 2, 3)), np.array([[0.0, -np.inf]]), np.zeros((1, 2)), 2)
    assert p.tolist() == [[0, 0]] and t.tolist() == [[0, 1]]                             # ties to the lowest id


def test_oracle_plan_by_hand():
    table, slots, used = serve_ref.page_plan(np.array([[5, 9, 9], [9, 9, 9]], np.int32), [33, 64], [2, 64], [0, 2], 67, [7, 1, 3], 32)
    assert table.tolist() == [[5, 7, -1], [1, 3, -1]] and used == 3
    assert slots.tolist()[:3] == [5 * 32 + 31, 7 * 32, 32] and slots[65] == 3 * 32 + 31 and slots[66] == -1


def test_ctypes_structs_match_the_header():
    """The packed argument blocks have the size and the alignment of the C structs."""
    class Cache(C.Structure):
        _fields_ = [("data", C.c_void_p), ("pages", C.c_int64), ("heads", C.c_int32), ("page_size", C.c_int32), ("head_dim", C.c_int32)]

    class Attention(C.Structure):
        _fields_ = [("q", C.c_void_p), ("out", C.c_void_p), ("lse", C.c_void_p), ("s", C.c_int64 * 4), ("t", C.c_void_p * 3), ("cache", Cache),
                    ("rows", C.c_int64), ("i", C.c_int32 * 7), ("scale", C.c_float)]

    assert C.sizeof(Cache) == CACHE.size and C.sizeof(Attention) == ATTENTION.size and STATE.size == 64
    raw = Attention.from_buffer_copy(_attention(scale=0.5, window=7))
    assert raw.scale == 0.5 and raw.i[6] == 7 and raw.cache.head_dim == 64 and raw.rows == 2

"""The largest calls of the serving operators, on the CPU: a launch has fewer than 2^32 threads along an axis, and a call that would need more is refused
before it.  (Only refused calls and calls that launch nothing are made here.)"""
import pytest

from moonshine_amd.hip_api import load_library
from test_serve_ops_refusals import CACHE, FAKE, STRIDES, _attention


@pytest.mark.parametrize("rows", [(1 << 26) - 31, (1 << 26) - 1, 1 << 26, (1 << 63) - 1, -1])
def test_rows_of_a_write_or_read_that_fill_a_grid(rows):
    lib = load_library()
    cache, strides = CACHE.pack(FAKE, 4, 1, 32, 64), STRIDES.pack(64, 64, 1)
    assert lib.msh_kv4_write(0, None, cache, FAKE, strides, FAKE, strides, 0, rows, FAKE) == -3 and b"rows" in lib.msh_op_last_error()
    assert lib.msh_kv4_read(0, None, cache, FAKE, rows, FAKE, FAKE, 0) == -3 and b"rows" in lib.msh_op_last_error()


def test_a_join_that_would_fill_a_grid_is_not_made():
    """Few sequences over long tables are split into ranges that a second launch joins, a wave per (row, head): from 2^26 - 3 of them on there is one range."""
    lib = load_library()

    def workspace(rows):
        return lib.msh_kv4_attention_workspace(_attention(rows=rows, starts=FAKE, table_width=64, batch=2))

    ranges = workspace(1) // (68 * 4)
    assert ranges > 1 and workspace((1 << 26) - 4) == ((1 << 26) - 4) * ranges * 68 * 4
    for rows in ((1 << 26) - 3, (1 << 26) - 1, 1 << 26):
        assert workspace(rows) == 0


@pytest.mark.parametrize("max_q, heads, batch, fits", [((1 << 24) - 1, 16, 1, False), ((1 << 24) - 7, 16, 1, False), ((1 << 24) - 8, 16, 1, True),
                                                       ((1 << 20) - 1, 16, 9, True), ((1 << 20), 16, 16, False)])
def test_chunks_that_would_fill_a_grid(max_q, heads, batch, fits):
    """One (sequence, head) pair has its workgroups, one for 128 rows, on every eighth place of the grid: 16 (2^24 - 8) rows are 2^21 - 1 of them."""
    lib = load_library()
    rc = lib.msh_kv4_attention_workspace(_attention(rows=5, starts=FAKE, max_q=max_q, heads=heads, batch=batch))
    assert rc == 0 if fits else rc == -3 and b"too large" in lib.msh_op_last_error()

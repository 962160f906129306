"""Serving operators on torch tensors: a paged key / value cache held in 4 bits with the attention that reads it, and the
selection and state reordering of a beam search (include/moonshine_hip.h, "serving operators").

Every call runs on the tensors' device and on torch's current stream there, enqueues and returns: no synchronisation, no state
between calls, results independent of what else runs; all of it may be captured into a graph.  Outputs and workspaces come from
torch's allocator.  There is no backward pass: inputs that require a gradient are refused.  A refused argument raises
``MshError`` (code -3) before anything is launched.

A decode step over a paged cache::

    cache = ops.kv4_cache(n_pages, kv_heads, page_size, head_dim)                 # once
    slots, used = ops.page_plan(table, kv_lens, new_lens, row_start, rows, free_pages, page_size)
    ops.kv4_write(cache, k, v, slots)                                             # k, v [rows, kv_heads, head_dim]
    out = ops.kv4_attention(q, cache, table, kv_lens, causal=True)                # q [rows, heads, head_dim]

and one of a beam search::

    scores, parents, tokens, finished = ops.beam_select(logits, scores, finished, eos)
    ops.beam_reorder([keys, values], parents, lengths, batch_dims=[1, 1], row_dims=[4, 4])
"""
from __future__ import annotations

import struct

import torch

from .hip_api import MshError, load_library

_INVALID = -3
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_CACHE = struct.Struct("Pqiiixxxx")                      # msh_kv4_cache
_ATTENTION = struct.Struct("PPPqqqqPPPPqiiixxxxqiiiiiiif")   # msh_kv4_attention_args
_STATE = struct.Struct("Pqqqqqqq")                       # msh_beam_state
_STRIDES = struct.Struct("qqq")

_lib = None


def _library():
    global _lib
    if _lib is None:
        _lib = load_library()
    return _lib


def _refuse(what: str):
    raise MshError(_INVALID, what)


def _check(rc: int) -> int:
    if rc < 0:
        raise MshError(rc, _library().msh_op_last_error().decode())
    return rc


def _place(first: torch.Tensor, *others: torch.Tensor | None):
    """The device index all tensors share, and torch's current stream there."""
    device = first.device
    if device.type != "cuda":
        _refuse(f"tensors must be on the GPU, not on {device}: there is no CPU fallback")
    for t in others:
        if t is not None and t.device != device:
            _refuse(f"tensors on {device} and {t.device}: one call, one device")
    return device.index, torch._C._cuda_getCurrentRawStream(device.index)


def _no_grad(*tensors: torch.Tensor):
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                _refuse("an input requires a gradient: this operator has no backward pass (call it under torch.no_grad())")


def _array(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple) -> int:
    """Address of a contiguous tensor of this type and shape."""
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        _refuse(f"{name}: a contiguous {dtype} tensor of shape {tuple(shape)} is wanted, not {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _cache_fields(cache: torch.Tensor, head_dim: int) -> tuple:
    if cache.dtype is not torch.uint8 or cache.dim() != 4 or not cache.is_contiguous():
        _refuse("cache: the contiguous uint8 tensor [pages, heads, page_size / 32, bytes] of kv4_cache() is wanted")
    pages, heads, blocks, size = cache.shape
    if size != 1088 * ((head_dim + 31) // 32):
        _refuse(f"cache: its blocks of {size} bytes are not those of head_dim {head_dim}")
    return cache.data_ptr(), pages, heads, blocks * 32, head_dim


def kv4_cache(pages: int, heads: int, page_size: int, head_dim: int, device="cuda") -> torch.Tensor:
    """A cache of ``pages`` pages (uint8 [pages, heads, page_size / 32, bytes], zeroed): token t of a page is slot
    ``page * page_size + t``.  4.25 bits an element, in groups of 32 of a head's width."""
    size = _check(_library().msh_kv4_page_bytes(heads, page_size, head_dim))
    if pages < 1:
        _refuse("pages: at least 1")
    return torch.zeros((pages, heads, page_size // 32, size // heads // (page_size // 32)), dtype=torch.uint8, device=device)


def page_plan(block_table: torch.Tensor, kv_lens: torch.Tensor, new_lens: torch.Tensor, row_start: torch.Tensor, rows: int,
              free_pages: torch.Tensor, page_size: int):
    """Extend ``block_table`` (int32 [batch, width], in place) to ``kv_lens`` tokens per request with pages from ``free_pages``,
    and map the step's packed rows to slots.  ``new_lens[b]`` of the tokens are new and stand in rows ``row_start[b]``...
    Returns (slots int64 [rows], -1 for rows of no request; used int32 [1]: pages taken from ``free_pages``, which were too few
    if it exceeds their number -- the entries and slots that found no page are then -1)."""
    index, stream = _place(block_table, kv_lens, new_lens, row_start, free_pages)
    if block_table.dim() != 2 or free_pages.dim() != 1:
        _refuse("block_table: [batch, width]; free_pages: [n]")
    batch, width = block_table.shape
    n_free = free_pages.shape[0]
    if rows < 0:
        _refuse("rows: not negative")
    args = (_array(block_table, "block_table", torch.int32, (batch, width)), batch, width, _array(kv_lens, "kv_lens", torch.int32, (batch,)),
            _array(new_lens, "new_lens", torch.int32, (batch,)), _array(row_start, "row_start", torch.int32, (batch,)), rows,
            _array(free_pages, "free_pages", torch.int32, (n_free,)), n_free, page_size)
    slots = torch.empty((rows,), dtype=torch.int64, device=block_table.device)
    used = torch.empty((1,), dtype=torch.int32, device=block_table.device)
    _check(_library().msh_page_plan(index, stream, *args, slots.data_ptr(), used.data_ptr()))
    return slots, used


def _slots(slots: torch.Tensor, rows: int) -> int:
    return _array(slots, "slots", torch.int64, (rows,))


def kv4_write(cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Store rows of keys and values [rows, heads, head_dim] (fp32, bf16 or fp16, any strides) in their slots; a slot outside the
    cache (-1: padding) is skipped.  The slots of a call must differ.  NaN is stored as 0, infinities as the largest finite."""
    index, stream = _place(cache, k, v, slots)
    _no_grad(k, v)
    if k.dim() != 3 or k.shape != v.shape or k.dtype is not v.dtype or k.dtype not in _DTYPES:
        _refuse("k and v: [rows, heads, head_dim], both fp32, bf16 or fp16")
    rows, heads, head_dim = k.shape
    fields = _cache_fields(cache, head_dim)
    if heads != fields[2]:
        _refuse(f"k and v have {heads} heads, the cache {fields[2]}")
    _check(_library().msh_kv4_write(index, stream, _CACHE.pack(*fields), k.data_ptr(), _STRIDES.pack(*k.stride()), v.data_ptr(),
                                    _STRIDES.pack(*v.stride()), _DTYPES[k.dtype], rows, _slots(slots, rows)))


def kv4_read(cache: torch.Tensor, slots: torch.Tensor, head_dim: int, dtype: torch.dtype = torch.bfloat16):
    """The keys and values that slots hold, [rows, heads, head_dim]; zeros for a slot outside the cache.  Exact in fp32 and bf16."""
    index, stream = _place(cache, slots)
    if dtype not in _DTYPES or slots.dim() != 1:
        _refuse("dtype: fp32, bf16 or fp16; slots: [rows]")
    rows = slots.shape[0]
    fields = _cache_fields(cache, head_dim)
    k = torch.empty((rows, fields[2], head_dim), dtype=dtype, device=cache.device)
    v = torch.empty_like(k)
    _check(_library().msh_kv4_read(index, stream, _CACHE.pack(*fields), _slots(slots, rows), rows, k.data_ptr(), v.data_ptr(), _DTYPES[dtype]))
    return k, v


def kv4_attention(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, *,
                  q_start: torch.Tensor | None = None, max_q: int | None = None, scale: float | None = None, causal: bool = True,
                  window: int = 0, return_lse: bool = False, out: torch.Tensor | None = None):
    """Attention of packed query rows ``q`` [rows, heads, head_dim] over the cached tokens of their sequences.

    Sequence b has the rows ``q_start[b]`` to ``q_start[b + 1] - 1``, at most ``max_q`` of them (``q_start`` None: rows / batch
    each), and ``kv_lens[b]`` tokens in the pages ``block_table[b]``.  ``causal``: its rows are its last tokens, each sees what
    stands up to itself, of that the last ``window`` tokens if window > 0; otherwise every row sees all tokens (a clip's
    encoder frames).  heads must be a multiple of the cache's: neighbouring query heads share one.  ``scale`` defaults to
    head_dim ** -0.5.  A row that sees nothing gives zeros and lse -inf; rows of no sequence are left as they are (in ``out``,
    [rows, heads, head_dim] with a contiguous last dimension; uninitialised if none is given).
    Returns out, or (out, lse fp32 [rows, heads])."""
    index, stream = _place(q, cache, block_table, kv_lens, q_start, out)
    _no_grad(q)
    if q.dim() != 3 or q.dtype not in _DTYPES or (q.stride(2) != 1 and q.shape[2] > 1):
        _refuse("q: [rows, heads, head_dim] in fp32, bf16 or fp16 with a contiguous last dimension")
    if block_table.dim() != 2:
        _refuse("block_table: [batch, width]")
    rows, heads, head_dim = q.shape
    batch, width = block_table.shape
    fields = _cache_fields(cache, head_dim)
    if q_start is None:
        if max_q is None:
            max_q = rows // batch if batch > 0 else 1
        if rows != batch * max_q:
            _refuse(f"{rows} rows are not {max_q} for each of {batch} sequences: give q_start")
        if rows == 0:
            max_q = max(max_q, 1)
            batch = 0
    elif max_q is None:
        _refuse("max_q: the most rows of a sequence (q_start is on the device)")
    if out is None:
        out = torch.empty((rows, heads, head_dim), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype is not q.dtype or (out.stride(2) != 1 and head_dim > 1):
        _refuse("out: q's shape and type, with a contiguous last dimension")
    lse = torch.empty((rows, heads), dtype=torch.float32, device=q.device) if return_lse else None
    table = _array(block_table, "block_table", torch.int32, block_table.shape)
    lens = _array(kv_lens, "kv_lens", torch.int32, (block_table.shape[0],))
    starts = _array(q_start, "q_start", torch.int32, (batch + 1,)) if q_start is not None else 0
    qs, os_ = q.stride(), out.stride()
    args = _ATTENTION.pack(q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0, qs[0], qs[1], os_[0], os_[1], table, lens,
                           starts, *fields, rows, _DTYPES[q.dtype], heads, batch, width, max_q, causal, window,
                           head_dim ** -0.5 if scale is None else scale)
    lib = _library()
    size = _check(lib.msh_kv4_attention_workspace(args))
    work = torch.empty((size,), dtype=torch.uint8, device=q.device) if size > 0 else None
    _check(lib.msh_kv4_attention(index, stream, args, work.data_ptr() if size > 0 else None, size))
    return (out, lse) if return_lse else out


def beam_select(logits: torch.Tensor, scores: torch.Tensor, finished: torch.Tensor, eos: int):
    """One selection of a beam search over ``logits`` [batch, beams, vocab] (fp32, bf16 or fp16, rows evenly spaced) with the
    beams' accumulated log probabilities ``scores`` (fp32 [batch, beams], -inf: not in use) and ``finished`` flags (uint8 or bool).
    Returns (scores, parents int32, tokens int32, finished) [batch, beams]: the best of score + log_softmax(logits), ties to the
    lowest beam * vocab + id; a finished beam stays as it is with the token ``eos`` (-1: no id ends a beam).  1 to 16 beams."""
    index, stream = _place(logits, scores, finished)
    _no_grad(logits, scores)
    if logits.dim() != 3 or logits.dtype not in _DTYPES or (logits.stride(2) != 1 and logits.shape[2] > 1):
        _refuse("logits: [batch, beams, vocab] in fp32, bf16 or fp16 with a contiguous last dimension")
    batch, beams, vocab = logits.shape
    row = logits.stride(1)
    if beams == 1:
        row = logits.stride(0)
    elif batch > 1 and logits.stride(0) != beams * row:
        _refuse("logits: the rows of all beams must be evenly spaced")
    if finished.dtype is not torch.uint8 and finished.dtype is not torch.bool:
        _refuse("finished: uint8 or bool")
    shape = (batch, beams)
    inputs = _array(scores, "scores", torch.float32, shape), _array(finished, "finished", finished.dtype, shape)
    next_scores = torch.empty(shape, dtype=torch.float32, device=logits.device)
    parents = torch.empty(shape, dtype=torch.int32, device=logits.device)
    tokens = torch.empty(shape, dtype=torch.int32, device=logits.device)
    next_finished = torch.empty(shape, dtype=finished.dtype, device=logits.device)
    lib = _library()
    size = _check(lib.msh_beam_select_workspace(batch, beams, vocab))
    work = torch.empty((size,), dtype=torch.uint8, device=logits.device)
    _check(lib.msh_beam_select(index, stream, logits.data_ptr(), _DTYPES[logits.dtype], row, batch, beams, vocab, *inputs, eos,
                               next_scores.data_ptr(), parents.data_ptr(), tokens.data_ptr(), next_finished.data_ptr(), work.data_ptr(), size))
    return next_scores, parents, tokens, next_finished


def _merge(sizes, strides, what: str):
    """(count, stride in elements) of several dimensions walked as one."""
    n, step = 1, 0
    for size, stride in zip(reversed(sizes), reversed(strides)):
        if size == 1:
            continue
        if n == 1:
            step = stride
        elif stride != n * step:
            _refuse(f"state: its {what} dimensions cannot be walked as one")
        n *= size
    return n, step


def beam_reorder(states, parents: torch.Tensor, lengths: torch.Tensor | None = None, *, batch_dims, row_dims) -> None:
    """In place, all at once: the first ``lengths`` rows of beam k of entry b become those of beam ``parents[b, k]`` (int32 [batch,
    beams]; a number that is no beam leaves its child as it is).  Up to four states of any type; state i has the entries in
    dimension ``batch_dims[i]``, the beams in the next one and the rows (decode steps) in ``row_dims[i]``, with what follows it
    contiguous.  ``lengths``: int32 [batch] or [1] on the GPU, None: all rows.  The states must not overlap."""
    states = list(states)
    index, stream = _place(parents, lengths, *states)
    if parents.dim() != 2 or not 0 < len(states) <= 4 or not len(states) == len(batch_dims) == len(row_dims):
        _refuse("parents: [batch, beams]; one to four states, each with a batch and a row dimension")
    batch, beams = parents.shape
    par = _array(parents, "parents", torch.int32, (batch, beams))
    packed = b""
    for t, b, r in zip(states, batch_dims, row_dims):
        _no_grad(t)
        shape, strides, size = t.shape, t.stride(), t.element_size()
        if not 0 <= b < b + 1 < r < len(shape) or shape[b] != batch or shape[b + 1] != beams:
            _refuse(f"state: dimensions {b}, {b + 1} of {tuple(shape)} are not the {batch} entries and {beams} beams, or {r} does not follow them")
        outer, outer_step = _merge(shape[:b], strides[:b], "outer")
        inner, inner_step = _merge(shape[b + 2:r], strides[b + 2:r], "inner")
        row, row_step = _merge(shape[r + 1:], strides[r + 1:], "last")
        if row > 1 and row_step != 1:
            _refuse("state: what follows the row dimension must be contiguous")
        if shape[r] > 1 and strides[r] != row:
            _refuse("state: its rows must be contiguous")
        beam = strides[b + 1] if beams > 1 else strides[b]
        if batch > 1 and strides[b] != beams * beam:
            _refuse("state: its beams must be evenly spaced over all entries")
        packed += _STATE.pack(t.data_ptr(), outer, outer_step * size, beam * size, inner, inner_step * size, row * size, shape[r])
    if lengths is not None and (lengths.dtype is not torch.int32 or lengths.dim() != 1 or lengths.shape[0] not in (1, batch) or not lengths.is_contiguous()):
        _refuse("lengths: a contiguous int32 tensor [batch] or [1]")
    per_entry = int(lengths is not None and lengths.shape[0] == batch)
    _check(_library().msh_beam_reorder(index, stream, packed, len(states), batch, beams, par, lengths.data_ptr() if lengths is not None else None,
                                       per_entry))

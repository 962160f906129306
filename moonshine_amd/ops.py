"""Serving operators on torch tensors: a paged key / value cache held in 4 bits with the attention that reads it, and the
selection and state reordering of a beam search (include/moonshine_hip.h, "serving operators").

Every call runs on the tensors' device and on torch's current stream there, enqueues and returns: no synchronisation, no state
between calls, results independent of what else runs; all of it may be captured into a graph.  Outputs and workspaces come from
torch's allocator.  There is no backward pass: inputs that require a gradient, or have a tangent of forward differentiation, are refused;
what a call writes in place counts as changed to autograd.  A refused argument raises ``MshError`` (code -3) before anything is launched.

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

import importlib.util
import os

import torch

from .hip_api import MshError, load_library

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _load():
    """The module that checks tensors, allocates outputs and calls the library (csrc/torch_ops.cpp)."""
    load_library()
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "msh_torch_ops.so")
    if not os.path.exists(path):
        raise FileNotFoundError(f"{path} not found: run `python -m moonshine_amd.build`")
    spec = importlib.util.spec_from_file_location("msh_torch_ops", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    if module.torch_version != torch.__version__:
        raise ImportError(f"{path} was built for torch {module.torch_version}, this is {torch.__version__}: run `python -m moonshine_amd.build`")
    module.set_up(MshError)
    return module


_ops = _load()


def kv4_cache(pages: int, heads: int, page_size: int, head_dim: int, device="cuda") -> torch.Tensor:
    """A cache of ``pages`` pages (uint8 [pages, heads, page_size / 32, bytes], zeroed): token t of a page is slot
    ``page * page_size + t``.  4.25 bits an element, in groups of 32 of a head's width."""
    lib = load_library()
    size = lib.msh_kv4_page_bytes(heads, page_size, head_dim)
    if size < 0:
        raise MshError(size, lib.msh_op_last_error().decode())
    if pages < 1:
        raise MshError(-3, "pages: at least 1")
    return torch.zeros((pages, heads, page_size // 32, size // heads // (page_size // 32)), dtype=torch.uint8, device=device)


def page_plan(block_table: torch.Tensor, kv_lens: torch.Tensor, new_lens: torch.Tensor, row_start: torch.Tensor, rows: int,
              free_pages: torch.Tensor, page_size: int):
    """Extend ``block_table`` (int32 [batch, width], in place) to ``kv_lens`` tokens per request with pages from ``free_pages``,
    and map the step's packed rows to slots.  ``new_lens[b]`` of the tokens are new and stand in rows ``row_start[b]``... (not decreasing).
    Returns (slots int64 [rows], -1 for rows of no request; used int32 [1]: pages taken from ``free_pages``, which were too few
    if it exceeds their number -- the entries and slots that found no page are then -1)."""
    return _ops.page_plan(block_table, kv_lens, new_lens, row_start, rows, free_pages, page_size)


def kv4_write(cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Store rows of keys and values [rows, heads, head_dim] (fp32, bf16 or fp16, any strides) in their slots; a slot outside the
    cache (-1: padding) is skipped.  The slots of a call must differ.  NaN is stored as 0, infinities as the largest finite."""
    _ops.kv4_write(cache, k, v, slots)


def kv4_read(cache: torch.Tensor, slots: torch.Tensor, head_dim: int, dtype: torch.dtype = torch.bfloat16):
    """The keys and values that slots hold, [rows, heads, head_dim]; zeros for a slot outside the cache.  Exact in fp32 and bf16."""
    if dtype not in _DTYPES:
        raise MshError(-3, "dtype: fp32, bf16 or fp16")
    return _ops.kv4_read(cache, slots, head_dim, _DTYPES[dtype])


def kv4_attention(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, *,
                  q_start: torch.Tensor | None = None, max_q: int | None = None, scale: float | None = None, causal: bool = True,
                  window: int = 0, return_lse: bool = False, out: torch.Tensor | None = None):
    """Attention of packed query rows ``q`` [rows, heads, head_dim] over the cached tokens of their sequences.

    Sequence b has the rows ``q_start[b]`` to ``q_start[b + 1] - 1``, at most ``max_q`` of them (``q_start``, not decreasing, int32 on
    the GPU; None: rows / batch each), and ``kv_lens[b]`` tokens in the pages ``block_table[b]``.  ``causal``: its rows are its last tokens, each sees what
    stands up to itself, of that the last ``window`` tokens if window > 0; otherwise every row sees all tokens (a clip's
    encoder frames).  heads must be a multiple of the cache's: neighbouring query heads share one.  ``scale`` defaults to
    head_dim ** -0.5.  A row that sees nothing gives zeros and lse -inf; rows of no sequence are left as they are (in ``out``,
    [rows, heads, head_dim] with a contiguous last dimension; uninitialised if none is given; it may be q itself).
    Returns out, or (out, lse fp32 [rows, heads])."""
    return _ops.kv4_attention(q, cache, block_table, kv_lens, q_start, max_q, scale, causal, window, return_lse, out)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, finished: torch.Tensor, eos: int):
    """One selection of a beam search over ``logits`` [batch, beams, vocab] (fp32, bf16 or fp16, rows evenly spaced) with the
    beams' accumulated log probabilities ``scores`` (fp32 [batch, beams], -inf: not in use) and ``finished`` flags (uint8 or bool).
    Returns (scores, parents int32, tokens int32, finished) [batch, beams]: the best of score + log_softmax(logits), ties to the
    lowest beam * vocab + id; a finished beam stays as it is with the token ``eos`` (-1: no id ends a beam).  1 to 16 beams."""
    return _ops.beam_select(logits, scores, finished, eos)


def beam_reorder(states, parents: torch.Tensor, lengths: torch.Tensor | None = None, *, batch_dims, row_dims) -> None:
    """In place, all at once: the first ``lengths`` rows of beam k of entry b become those of beam ``parents[b, k]`` (int32 [batch,
    beams]; a number that is no beam leaves its child as it is).  Up to four states of any type; state i has the entries in
    dimension ``batch_dims[i]``, the beams in the next one and the rows (decode steps) in ``row_dims[i]``, with what follows it
    contiguous.  ``lengths``: int32 [batch] or [1] on the GPU, None: all rows.  The states must not overlap."""
    _ops.beam_reorder(list(states), parents, lengths, list(batch_dims), list(row_dims))

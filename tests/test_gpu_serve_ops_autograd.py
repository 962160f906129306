"""The serving operators beside torch's own bookkeeping: what they write in place counts as changed (a backward pass that saved it says so instead of
using the new values), and inputs whose derivative or pending sign they would drop are refused."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from moonshine_amd import ops
from moonshine_amd.hip_api import MshError

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Setting:
    def __init__(self):
        g = torch.Generator(device="cuda").manual_seed(1)
        self.cache = ops.kv4_cache(4, 2, 32, 40)
        self.k, self.v, self.q = (torch.randn((6, 2, 40), generator=g, device="cuda") for _ in range(3))
        self.slots = torch.arange(6, device="cuda")
        ops.kv4_write(self.cache, self.k, self.v, self.slots)
        self.table, self.lens = i32([[0]] * 6), i32([6] * 6)
        self.states = [torch.randn((2, 3, 4), generator=g, device="cuda") for _ in range(2)]
        self.parents = i32([[1, 0, 2], [2, 2, 2]])
        self.logits, self.scores = torch.randn((2, 3, 50), generator=g, device="cuda"), -torch.rand((2, 3), generator=g, device="cuda")
        self.finished = torch.zeros((2, 3), dtype=torch.uint8, device="cuda")


def writes():
    s = Setting()
    out = torch.zeros_like(s.q)
    plan = i32([[0, -1]])
    return {"cache": (s.cache, lambda: ops.kv4_write(s.cache, s.k, s.v, s.slots)),
            "out": (out, lambda: ops.kv4_attention(s.q, s.cache, s.table, s.lens, out=out)),
            "its own queries": (s.q, lambda: ops.kv4_attention(s.q, s.cache, s.table, s.lens, out=s.q)),
            "block_table": (plan, lambda: ops.page_plan(plan, i32([33]), i32([1]), i32([0]), 1, i32([3]), 32)),
            "states": (s.states[1], lambda: ops.beam_reorder(s.states, s.parents, batch_dims=[0, 0], row_dims=[2, 2]))}


@pytest.mark.parametrize("what", ["cache", "out", "its own queries", "block_table", "states"])
def test_what_is_written_in_place_counts_as_changed(what):
    t, call = writes()[what]
    view, before = t[:1], t._version
    call()
    assert t._version == before + 1 and view._version == t._version


def test_a_backward_pass_over_a_state_that_was_reordered_says_so():
    s = Setting()
    w = torch.ones((2, 3, 4), device="cuda", requires_grad=True)
    loss = (w * s.states[0]).sum()
    ops.beam_reorder(s.states, s.parents, batch_dims=[0, 0], row_dims=[2, 2])
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()


def test_tensors_made_under_inference_mode():
    with torch.inference_mode():
        s = Setting()
        for t, call in writes().values():
            call()
    ops.beam_reorder(s.states, s.parents, batch_dims=[0, 0], row_dims=[2, 2])     # they have no version to count
    ops.kv4_write(s.cache, s.k, s.v, s.slots)
    assert s.states[0].is_inference()


def inputs():
    """name -> (a call that takes the tensor, the tensor)"""
    s = Setting()
    return {"k": (lambda x: ops.kv4_write(s.cache, x, s.v, s.slots), s.k), "v": (lambda x: ops.kv4_write(s.cache, s.k, x, s.slots), s.v),
            "q": (lambda x: ops.kv4_attention(x, s.cache, s.table, s.lens), s.q),
            "out": (lambda x: ops.kv4_attention(s.q, s.cache, s.table, s.lens, out=x), torch.zeros_like(s.q)),
            "logits": (lambda x: ops.beam_select(x, s.scores, s.finished, 2), s.logits), "scores": (lambda x: ops.beam_select(s.logits, x, s.finished, 2), s.scores),
            "state": (lambda x: ops.beam_reorder([x], s.parents, batch_dims=[0], row_dims=[2]), s.states[0])}


NAMES = ["k", "v", "q", "out", "logits", "scores", "state"]


@pytest.mark.parametrize("name", NAMES)
def test_a_forward_derivative_is_not_dropped(name):
    call, x = inputs()[name]
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        with pytest.raises(MshError, match="forward") as e:
            call(dual)
        assert e.value.code == -3
    call(x)


@pytest.mark.parametrize("name", NAMES)
def test_a_pending_sign_is_not_dropped(name):
    """The imaginary part of a conjugate is a view whose sign torch has not applied yet: its memory holds the other sign."""
    call, x = inputs()[name]
    z = torch.complex(torch.zeros_like(x), -x).conj().imag
    assert z.is_neg() and torch.equal(z, x)
    with pytest.raises(MshError, match="sign") as e:
        call(z)
    assert e.value.code == -3
    call(z.resolve_neg().contiguous())

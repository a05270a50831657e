"""What the drafts' operators do ahead of a launch, without a GPU: the calls that are refused, and what a refused call leaves."""
import numpy as np
import pytest
import torch

from fllm_amd.kernels import KernelError, Ops, load_library


@pytest.fixture
def ops(monkeypatch):
    """Operators of a process that has launched nothing yet; tensors on the CPU are refused behind the other checks."""
    monkeypatch.setattr(Ops, "_streams", {})
    monkeypatch.setattr(Ops, "_current_stream", staticmethod(lambda: (0, 0x1234)))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    made = Ops.__new__(Ops)
    made.lib = load_library()
    return made


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def calls():
    k, v = torch.zeros((1, 3, 2, 4, 16, 8)), torch.zeros((1, 3, 2, 32, 16))
    yield "tree_attention", lambda ops: ops.tree_attention(torch.zeros(4, 128), k[0], v[0], i32(2, 3), i32(4), i32(3), i32(2), torch.zeros((4, 1), dtype=torch.int64), torch.zeros(4, 128),
                                                          4, 2, 32, 16, 0.2, 40)
    yield "follow_tree", lambda ops: ops.follow_tree(i32(4), i32(4), i32(3), i32(4), i32(2, 3), i32(2), i32(2))
    yield "move_tokens", lambda ops: ops.move_tokens(k, v, i32(2, 3), i32(2), i32(2, 3), i32(2))
    yield "copy_pages", lambda ops: ops.copy_pages((k, v), [0], [1])
    yield "rope_kv_store", lambda ops: ops.rope_kv_store(torch.zeros(4, 256), i32(4), i32(4), i32(2, 3), torch.zeros(40, 16), torch.zeros(40, 16), k[0], v[0], 4, 2, 32, 32, 1, 16,
                                                         row_slot=i32(4))


@pytest.mark.parametrize("name,call", list(calls()), ids=[name for name, _ in calls()])
def test_a_refused_call_does_not_choose_the_stream(ops, name, call):
    """The first launch makes its stream the device's; a call that launches nothing does not."""
    with pytest.raises(KernelError):
        call(ops)
    assert Ops._streams == {}


def test_copying_nothing_does_not_choose_the_stream(ops, monkeypatch):
    monkeypatch.setattr("fllm_amd.kernels._held", lambda t, *_: t.data_ptr())
    ops.copy_pages((torch.zeros((1, 3, 8)),), [], [])
    assert Ops._streams == {}


@pytest.mark.parametrize("kind", [list, tuple, torch.tensor, np.array, lambda v: [torch.tensor(p) for p in v]], ids=["list", "tuple", "tensor", "array", "tensors"])
def test_pages_that_meet_are_refused_in_whatever_they_are_given(ops, kind):
    """Two pairs that write one page, or one that reads what another writes, run at the same time: which is first is anyone's guess."""
    store = (torch.zeros((1, 9, 8)),)
    for source, target, message in (([0, 1], [2, 2], "copied to twice"), ([0, 1], [1, 2], "copied from and to"), ([0, 1], [2, 9], "has 9 pages"), ([0, -1], [2, 3], "has 9 pages")):
        with pytest.raises(KernelError, match=message if "has" not in message else "must be on the GPU|has 9 pages"):
            ops.copy_pages(store, kind(source), kind(target))


def test_page_numbers_are_whole(ops):
    for wrong in ([0.0], [0.5], ["0"], [None]):
        with pytest.raises((KernelError, TypeError)):
            ops.copy_pages((torch.zeros((1, 9, 8)),), wrong, [1])
        with pytest.raises((KernelError, TypeError)):
            ops.copy_pages((torch.zeros((1, 9, 8)),), [1], wrong)


@pytest.mark.parametrize("kind", [list, torch.tensor, np.array], ids=["list", "tensor", "array"])
def test_pages_that_do_not_meet_are_copied(ops, monkeypatch, kind):
    seen = []

    class Library:
        def fllm_copy_pages(self, stores, layers, pages, sizes, count, source, target, pairs, stream):
            seen.append((list(layers), list(pages), list(sizes), count, list(source), list(target), pairs, stream))
            return 0
    ops.lib = Library()
    monkeypatch.setattr("fllm_amd.kernels._held", lambda t, *_: t.data_ptr())
    ops.copy_pages((torch.zeros((2, 9, 8)), torch.zeros((3, 10, 4), dtype=torch.bfloat16)), kind([0, 0, 5]), kind([1, 8, 2]))
    assert seen == [([2, 3], [9, 10], [32, 8], 2, [0, 0, 5], [1, 8, 2], 3, 0x1234)]

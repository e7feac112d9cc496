"""Selections used on several streams, with no ordering by the caller: the
stream that sets the ids is held up by queued work, so a plan that did not wait
for it would be sorted from what the memory held before."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def _held_up(stream, fn):
    """fn() on `stream`, behind about ten milliseconds of queued copies."""
    a = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        b = torch.empty_like(a)
        for _ in range(100):
            b.copy_(a, non_blocking=True)
        return fn()


def _operands(batch, seq):
    g = torch.Generator(device="cuda").manual_seed(batch)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    m = batch * seq
    return rn(m, 64), rn(m, 64), rn(3, 8, 64), rn(3, 8, 64), torch.ones(3, device="cuda")


def test_a_plan_waits_for_its_ids():
    from diffuser_b200 import modules, ops
    batch, seq = 4, 5
    operands = _operands(batch, seq)
    ids = torch.tensor([2, -1, 0, 1], dtype=torch.int32, device="cuda")
    other = torch.tensor([0, 1, 1, -1], dtype=torch.int32, device="cuda")
    offsets = torch.arange(batch + 1, dtype=torch.int32, device="cuda") * seq
    want = [ops.adapter_add(*operands, ops.adapter_plan(i, offsets, batch * seq, 3)) for i in (ids, other)]
    torch.cuda.synchronize()
    a, b, c = (torch.cuda.Stream() for _ in range(3))
    # made on a, its plan built on b
    sel = _held_up(a, lambda: modules.AdapterSelection(ids, 3))
    with torch.cuda.stream(b):
        got = ops.adapter_add(*operands, sel.plan(batch * seq))
    # updated on a (behind b's use, as the caller has to), read on c and, for a new token count, on b
    a.wait_stream(b)
    _held_up(a, lambda: sel.update_(other))
    with torch.cuda.stream(c):
        again = ops.adapter_add(*operands, sel.plan(batch * seq))
    with torch.cuda.stream(b):
        fresh = sel.plan(2 * batch * seq)
        half = torch.cat([torch.arange(i * 2 * seq, i * 2 * seq + seq, device="cuda") for i in range(batch)])
        wide = [torch.zeros(2 * batch * seq, 64, dtype=torch.bfloat16, device="cuda").index_copy_(0, half, t)
                for t in operands[:2]]
        longer = ops.adapter_add(*wide, *operands[2:], fresh)[half]
    # a copy made on another stream
    a.wait_stream(b)
    a.wait_stream(c)
    _held_up(a, lambda: sel.update_(ids))
    with torch.cuda.stream(c):
        twin = copy.deepcopy(sel)
        copied = ops.adapter_add(*operands, twin.plan(batch * seq))
    torch.cuda.synchronize()
    assert torch.equal(got, want[0])
    assert torch.equal(again, want[1]) and torch.equal(longer, want[1])
    assert torch.equal(copied, want[0]) and twin.ids.tolist() == ids.tolist()
    assert ops.device_error() == 0


def test_a_dropped_selection_leaves_its_ids_to_the_build():
    # the build of one plan is queued on b when the selection goes; a's next
    # tensors may not take the ids' block before it has run
    from diffuser_b200 import modules, ops
    batch, seq = 4, 3
    operands = _operands(batch, seq)
    ids = torch.tensor([1, 2, -1, 0], dtype=torch.int32, device="cuda")
    offsets = torch.arange(batch + 1, dtype=torch.int32, device="cuda") * seq
    want = ops.adapter_add(*operands, ops.adapter_plan(ids, offsets, batch * seq, 3))
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(a):
        sel = modules.AdapterSelection(ids, 3)
    plan = _held_up(b, lambda: sel.plan(batch * seq))
    del sel
    with torch.cuda.stream(a):
        taken = [torch.zeros(batch, dtype=torch.int32, device="cuda") for _ in range(64)]
    with torch.cuda.stream(b):
        got = ops.adapter_add(*operands, plan)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and not any(t.any() for t in taken)


def test_no_selection_is_made_inside_a_capture():
    from diffuser_b200 import modules
    ids = torch.zeros(2, dtype=torch.int32, device="cuda")
    out = torch.zeros(1, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out.add_(1)
        with pytest.raises(RuntimeError, match="capture"):
            modules.AdapterSelection(ids, 2)
    graph.replay()
    assert out.item() == 1


def test_plans_of_many_lengths_are_not_all_kept():
    """Prompts of ever other lengths: the plans used last are kept, with those a
    capture took and those in use, and every one alive follows an update."""
    import gc
    import weakref
    from diffuser_b200 import modules, ops
    ids = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    sel = modules.AdapterSelection(ids, 3)
    operands = _operands(2, 3)
    sel.plan(6)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.adapter_add(*operands, sel.plan(6))
    mine = sel.plan(10)
    seen = [weakref.ref(sel.plan(2 * n)) for n in range(10, 60)]
    gc.collect()
    alive = [r for r in seen if r() is not None]
    assert len(alive) == sel.KEPT and alive == seen[-sel.KEPT:]
    assert sel.plan(10) is mine  # held here
    sel.update_(torch.tensor([2, -1], dtype=torch.int32, device="cuda"))
    graph.replay()
    offsets = torch.tensor([0, 3, 6], dtype=torch.int32, device="cuda")
    assert torch.equal(out, ops.adapter_add(*operands, ops.adapter_plan(sel.ids, offsets, 6, 3)))
    fresh = ops.adapter_plan(sel.ids, torch.tensor([0, 5, 10], dtype=torch.int32, device="cuda"), 10, 3)
    wide = [torch.cat([t, t])[:10] for t in operands[:2]]
    assert torch.equal(ops.adapter_add(*wide, *operands[2:], mine), ops.adapter_add(*wide, *operands[2:], fresh))


@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy])
def test_a_copy_has_ids_of_its_own(how):
    from diffuser_b200 import modules, ops
    sel = modules.AdapterSelection(torch.tensor([1, 0], dtype=torch.int32, device="cuda"), 3)
    operands = _operands(2, 3)
    twin = how(sel)
    want = ops.adapter_add(*operands, twin.plan(6))
    sel.update_(torch.tensor([2, 2], dtype=torch.int32, device="cuda"))
    assert twin.ids.tolist() == [1, 0] and sel.ids.tolist() == [2, 2]
    assert torch.equal(ops.adapter_add(*operands, how(twin).plan(6)), want)
    assert not torch.equal(ops.adapter_add(*operands, sel.plan(6)), want)

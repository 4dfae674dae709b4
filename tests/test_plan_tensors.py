"""Tensors that lose their memory after a plan over them was made (geeps_amd.clipping.GradPlan)."""
import pytest
import torch

from geeps_amd import clipping, native


def halve(t):
    t.data = t.data.half()


def swap(t):
    t.data = torch.zeros_like(t)


def point_elsewhere(t):
    t.set_(torch.zeros_like(t))


def shorten(t):
    t.data = t.data[:-1]


def grow(t):
    t.resize_(1 << 16)


def let_go(t):
    t.untyped_storage().resize_(0)


def retype(t):
    t.data = t.data.view(torch.int32)


def turn(t):
    t.data = t.data.view(8, 8).t()


def exchange(t):
    torch.utils.swap_tensors(t, torch.zeros_like(t))


CHANGES = [halve, swap, point_elsewhere, shorten, grow, let_go, retype, turn, exchange]


@pytest.mark.parametrize("change", CHANGES)
@pytest.mark.parametrize("which", [0, 2])
def test_a_change_is_seen(change, which):
    facts = native.tensor_facts()
    tensors = (torch.zeros(64), torch.zeros(0), torch.zeros(64), torch.zeros(5, dtype=torch.bfloat16))
    was = facts.facts(tensors)
    tensors[0].add_(1)
    assert facts.moved(tensors, was) == -1
    change(tensors[which])
    assert facts.moved(tensors, was) == which


def test_facts_refuse_what_is_no_list_of_tensors():
    facts = native.tensor_facts()
    one = (torch.zeros(3),)
    for call in (lambda: facts.facts([torch.zeros(3)]), lambda: facts.facts((3,)), lambda: facts.moved(one, b""),
                 lambda: facts.moved(one), lambda: facts.moved((3,), facts.facts(one)),
                 lambda: facts.moved(one * 2, facts.facts(one)), lambda: facts.moved(list(one), facts.facts(one))):
        with pytest.raises(TypeError):
            call()
    assert facts.moved((), facts.facts(())) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("change", CHANGES)
@pytest.mark.parametrize("which", ["grads", "outs", "in place"])
def test_a_plan_refuses_moved_tensors(dev, change, which):
    grads = [torch.full((n,), 2.0, device=dev) for n in (64, 300)]
    outs = None if which == "in place" else [torch.zeros_like(g) for g in grads]
    plan = clipping.GradPlan(grads, outs)
    plan.clip(1.0)
    other = clipping.GradPlan([torch.ones(7, device=dev)])
    moved = (outs if which == "outs" else grads)[0]
    change(moved)
    watched = [t for t in (*grads, *(outs or ())) if t is not moved]
    before = [t.clone() for t in watched]
    name = "outs" if which == "outs" else "grads"
    for call in (lambda: plan.clip(1.0), plan.sum_squares, plan.norm,
                 lambda: plan.clip(1.0, stream=torch.cuda.Stream())):
        with pytest.raises(ValueError, match=rf"{name}\[0\] is not where it was"):
            call()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, watched))
    other.clip(1.0)  # another plan goes on
    plan.close()
    with pytest.raises(ValueError, match="closed"):
        plan.clip(1.0)


@pytest.mark.gpu
def test_a_plan_keeps_the_memory_that_it_points_at(dev):
    """A graph replayed after a tensor was given other memory writes to nothing that another tensor got."""
    grad = torch.full((1 << 20,), 2.0, device=dev)
    plan = clipping.GradPlan([grad])
    plan.clip(1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.clip(1.0)
    at = grad.data_ptr()
    grad.data = torch.zeros_like(grad)
    others = [torch.full((1 << 20,), 3.0, device=dev) for _ in range(20)]
    assert at not in [t.data_ptr() for t in others]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(bool((t == 3.0).all()) for t in others) and not bool(grad.any())
    plan.close()


@pytest.mark.gpu
def test_a_plan_of_copy_on_write_clones(dev):
    """Asking for a clone's address gives it memory of its own: that is the plan's, and no move."""
    base = torch.full((5000,), 2.0, device=dev)
    grads, outs = [torch._lazy_clone(base)], [torch._lazy_clone(base)]
    plan = clipping.GradPlan(grads, outs)
    for _ in range(2):
        plan.clip(1.0)
    f = 1.0 / (4.0 * 5000) ** 0.5
    assert bool((base == 2.0).all()) and bool((grads[0] == 2.0).all())
    assert bool(((outs[0].double() - 2.0 * f).abs() <= 3 * 2.0 ** -24 * 2.0 * f).all())

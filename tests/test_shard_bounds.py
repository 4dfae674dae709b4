"""What ShardedReducer takes beside a bound on its update (CPU, one rank)."""
import pytest
import torch

from geeps_amd.shard import ShardedReducer


def add(master, buckets):
    for b in buckets:
        master += b


def squares(updates, scratch):
    return sum(updates).double().square().sum()


def clipped(master, updates, max_norm, scratch, total):
    u = sum(updates)
    norm = u.double().square().sum().sqrt()
    master += (u.double() * min(1.0, max_norm / float(norm))).float()
    return norm.float()


def test_no_stand_in_is_dropped():
    """apply_fn was left unused where max_norm was given, and clip_fns where it was not."""
    with pytest.raises(ValueError, match="apply_fn"):
        ShardedReducer(4, 3, 2, "cpu", max_norm=1.0, apply_fn=add)
    with pytest.raises(ValueError, match="apply_fn"):
        ShardedReducer(4, 3, 2, "cpu", max_norm=1.0, apply_fn=add, clip_fns=(squares, clipped))
    with pytest.raises(ValueError, match="clip_fns"):
        ShardedReducer(4, 3, 2, "cpu", clip_fns=(squares, clipped))


def test_each_stand_in_where_it_belongs():
    deltas = [torch.full((12,), 1.0), torch.full((12,), 2.0)]
    plain = ShardedReducer(4, 3, 2, "cpu", apply_fn=add)
    assert torch.equal(plain.step(deltas)[:12], torch.full((12,), 3.0)) and plain.norm is None
    bound = ShardedReducer(4, 3, 2, "cpu", max_norm=0.0, clip_fns=(squares, clipped))
    assert torch.equal(bound.step(deltas)[:12], torch.zeros(12))
    assert abs(float(bound.norm) - 108 ** 0.5) <= 2.0 ** -24 * 11

"""The work lists of attention over shared prefixes: every (token, key) pair is covered once, and what is refused."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from rapid_llm_b200.ops import kernels
from rapid_llm_b200.parts.attention import SharedItems
from rapid_llm_b200.parts.base import StepShape


def shape_of(lengths, starts, groups, shared, page=16):
    return StepShape(lengths=np.asarray(lengths, dtype=np.int32), starts=np.asarray(starts, dtype=np.int32), decode_only=max(lengths) == 1,
                     page_size=page, prefix_group=np.asarray(groups, dtype=np.int32), prefix_tokens=np.asarray(shared, dtype=np.int32))


def random_shape(seed, page=16):
    rng = np.random.RandomState(seed)
    n = rng.randint(1, 70)
    prefix = rng.randint(0, 3000, size=5)
    groups = rng.randint(-1, 5, size=n)
    shared = np.where(groups >= 0, prefix[groups], 0)
    return shape_of(rng.choice([1, 1, 1, 2, 5], n), shared + rng.randint(0, 400, n), groups, shared, page)


@pytest.mark.parametrize("dtype,dim,group", [(torch.float32, 64, 4), (torch.bfloat16, 64, 4), (torch.bfloat16, 128, 4), (torch.bfloat16, 128, 5),
                                             (torch.bfloat16, 128, 40), (torch.float32, 128, 33)])
@pytest.mark.parametrize("seed", range(6))
def test_every_key_of_every_row_is_covered_once(dtype, dim, group, seed):
    shape = random_shape(seed)
    planner = SharedItems(group, 2, dim, dtype=dtype)
    plan = planner.plan(shape)
    lengths, starts = np.asarray(shape.lengths), np.asarray(shape.starts)
    entry_of = np.repeat(np.arange(len(lengths)), lengths)
    positions = np.concatenate([np.arange(s, s + n) for s, n in zip(starts, lengths)])
    seen = [np.zeros((group, p + 1), dtype=int) for p in positions]
    parts = [set() for _ in positions]
    most = 0
    for bucket, height in (("tile_items", plan["tile_rows"]), ("row_items", 16)):
        for entry, first, end, member, row0, rows, part, fresh in plan[bucket]:
            assert 0 < rows <= height and first < end
            if bucket == "row_items":
                most = max(most, rows)
            for p in range(row0, row0 + rows):
                token = plan["members"][member + p // group]
                mine = entry_of[token]
                if mine != entry:          # a shared range: the entry named is one of the token's group
                    assert shape.prefix_group[mine] == shape.prefix_group[entry] >= 0 and end <= shape.prefix_tokens[mine]
                assert fresh <= starts[mine] if mine == entry and end > shape.prefix_tokens[mine] else fresh >= end
                seen[token][p % group, first : min(end, positions[token] + 1)] += 1
                parts[token].add((part, p % group))
    assert all((s == 1).all() for s in seen)
    counts = np.diff(plan["part_first"])
    for token, its in enumerate(parts):
        assert its == {(part, head) for part in range(counts[token]) for head in range(group)}
    assert plan["parts"] == counts.sum() and planner.part_rows(plan) == plan["parts"] * group * 2
    assert most == plan["most_rows"]
    for bucket in ("tile_items", "row_items"):
        spans = plan[bucket][:, 2] - plan[bucket][:, 1]
        assert (np.diff(spans) <= 0).all()


def test_nothing_shared_needs_no_arrays():
    plan = SharedItems(4, 2, 128).plan(StepShape(lengths=np.array([1, 3]), starts=np.array([9, 0]), decode_only=False, page_size=16))
    assert plan["entries"] == 2 and plan["tokens"] == 4 and len(plan["tile_items"]) == 0


@pytest.mark.parametrize("shape", [
    shape_of([1, 1], [5, 9], [0, 0], [6, 6]),             # shares a position that is new
    shape_of([1, 1], [9, 9], [0, 0], [4, 6]),             # one group, two lengths
    shape_of([1, 1], [9, 9], [0, 0], [-1, -1]),
    shape_of([1, 0], [9, 9], [0, 0], [4, 4]),
    StepShape(lengths=np.array([1, 1]), starts=np.array([9, 9]), decode_only=True, page_size=16, prefix_group=np.array([0]), prefix_tokens=np.array([4])),
], ids=["new", "lengths", "negative", "empty", "shapes"])
def test_refused(shape):
    with pytest.raises(ValueError):
        SharedItems(4, 2, 128).plan(shape)


def test_there_is_no_cpu_path():
    with pytest.raises(kernels.KernelError):
        kernels.attention_shared(torch.zeros((1, 64)), torch.zeros((2, 2, 1, 16, 64)), torch.zeros((1, 64)), plan={}, part_out=None, part_lse=None,
                                 positions=torch.zeros(1, dtype=torch.int32), cu_seqlens=None, entry_start=None, entry_slot=None,
                                 block_table=None, num_heads=1, num_kv_heads=1, head_dim=64, scale=1.0, fault=None)


def test_the_rule_of_a_decode_step():
    """Shared where that saves enough for groups of enough members; lists filled up to powers of two; never in steps with portions."""
    from rapid_llm_b200.parts import attention

    items = SharedItems(4, 8, 128)
    def shape(members, prefix, own=5, lengths=None):
        return shape_of(lengths or [1] * members, [prefix + own] * members, [3] * members, [prefix] * members)

    per_position = 2 * 8 * 128 * 2
    assert items.saved_bytes(shape(8, 1000)) == 7 * 1000 * per_position and items.saved_bytes(shape(4, 1000)) == 0
    edge = -(-attention.WORTH_SHARING // (7 * per_position))
    assert items.step_plan(shape(8, edge)) is not None and items.step_plan(shape(8, edge - 1)) is None
    assert items.step_plan(shape(4, 100_000)) is None and items.step_plan(shape(8, 5000, lengths=[1] * 7 + [2])) is None
    wide = SharedItems(4, 8, 128, dtype=torch.float32)
    assert wide.step_plan(shape(2, 16)) is not None and wide.step_plan(shape(1, 16)) is None and wide.step_plan(shape(2, 0)) is None
    plan = items.step_plan(shape(11, 5000, 300))
    assert plan["shared"] is True
    for name in ("tile_items", "row_items"):
        count = len(plan[name])
        assert count & (count - 1) == 0 and (plan[name][plan[name][:, 5] == 0] == 0).all()
    assert plan["parts"] & (plan["parts"] - 1) == 0 and plan["parts"] >= plan["part_first"][-1]
    counts = {tuple((k, len(v) if isinstance(v, np.ndarray) else v) for k, v in items.step_plan(shape(11, 5000, own)).items()) for own in range(1, 400)}
    assert len(counts) <= 6                  # what a captured step has baked in, over 400 steps


def test_the_lists_fit_what_the_planner_asks_for():
    for members in (5, 33, 64):
        for prefix in (200, 5000, 200_000):
            items = SharedItems(4, 1, 128)
            plan = items.step_plan(shape_of([1] * members, [prefix + 9000] * members, [0] * members, [prefix] * members))
            if plan is not None:
                size = sum(v.size + 3 for v in plan.values() if isinstance(v, np.ndarray))
                assert size <= items.capacity(members, members)

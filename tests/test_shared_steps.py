"""What a captured decode step over shared prefixes has baked in, while the requests of a family come to their ends."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from rapid_llm_b200.engine.runner import decode_bucket
from rapid_llm_b200.parts.attention import SharedItems
from rapid_llm_b200.parts.base import StepShape


def step_shape(bucket, live, shared, own, others=0):
    """``live`` members of one family, ``others`` requests of their own, padding rows behind them."""
    pad = bucket - live - others
    return StepShape(
        lengths=np.ones(bucket, dtype=np.int32), starts=np.asarray([shared + own] * live + [own] * others + [0] * pad, dtype=np.int32),
        decode_only=True, page_size=16, padding=pad, prefix_group=np.asarray([3] * live + [-1] * (others + pad), dtype=np.int32),
        prefix_tokens=np.asarray([shared] * live + [0] * (others + pad), dtype=np.int32))


def baked_in(plan):
    return tuple((name, value.shape if isinstance(value, np.ndarray) else value) for name, value in sorted(plan.items()))


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 128)])
def test_members_that_end_one_by_one_leave_few_kinds_of_step(dtype, dim):
    """64 members end one by one, a token later each: the buckets of the batch and the powers of two of the lists, not a
    kind for every count of members."""
    items = SharedItems(4, 8, dim, dtype=dtype)
    kinds, shared_steps = set(), 0
    for gone, live in enumerate(range(64, 4, -1)):
        bucket = decode_bucket(live, 64, 64)
        plan = items.step_plan(step_shape(bucket, live, 8192, 40 + gone))
        if plan is not None:
            shared_steps += 1
            kinds.add((bucket, baked_in(plan)))
    assert shared_steps > 40 and len(kinds) <= 16, (shared_steps, len(kinds))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_same_batch_with_fewer_members(dtype):
    """In a batch of one size, requests of their own in the members' places: the list of members has one size."""
    items = SharedItems(4, 8, 128, dtype=dtype)
    sizes, offsets = set(), set()
    for live in range(5, 33):
        plan = items.step_plan(step_shape(32, live, 20000, 30, others=32 - live))
        sizes.add(plan["members"].shape)
        offsets.add(plan["part_first"].shape)
        # every member an item names lies inside what the list holds
        for bucket in ("tile_items", "row_items"):
            for _, _, _, first, row0, rows, _, _ in plan[bucket]:
                if rows > 0:
                    assert first + (row0 + rows - 1) // 4 < 32 + live
        assert sorted(plan["members"][32 : 32 + live]) == list(range(live))
    assert len(sizes) == 1 and len(offsets) == 1


@pytest.mark.parametrize("members,prefix,shares", [
    (8, 4096, False), (16, 2048, False), (32, 1328, False), (20, 2160, False), (16, 2752, False), (64, 512, False), (4, 100_000, False),
    (8, 6144, True), (12, 4096, True), (16, 4096, True), (32, 2048, True), (64, 8192, True), (5, 16384, True)])
def test_a_step_shares_where_that_pays_for_its_plan(members, prefix, shares):
    """8 key heads of 128 in groups of 4: shared where a step that the host waits for was no slower than the ordinary one."""
    bucket = decode_bucket(members, 64, 64)
    assert (SharedItems(4, 8, 128).step_plan(step_shape(bucket, members, prefix, 20)) is not None) == shares

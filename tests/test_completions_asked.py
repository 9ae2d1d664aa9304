"""How many completions a request asks for, in whatever number type, and what a refused request leaves behind."""

from __future__ import annotations

import numpy as np
import pytest
from test_scheduler_completions import scheduler_of, several

from rapid_llm_b200.sampling import SamplingParams


@pytest.mark.parametrize("n", [2, 2.0, np.int64(2), np.float32(2)])
def test_whole_numbers_of_any_type(n):
    params = several(n, 3, top_k=5.0)
    assert type(params.n) is int and type(params.top_k) is int and (params.n, params.top_k) == (2, 5)
    scheduler, executor = scheduler_of()
    request = scheduler.add_request(list(range(20)), params, "a")
    scheduler.run_to_completion()
    assert [len(r.output_token_ids) for r in request.completions] == [3, 3]
    assert executor.cache.num_free_slots == 4


def test_a_request_that_fails_leaves_nothing_in_the_queue():
    params = SamplingParams(temperature=0.0, repetition_penalty=1.0, max_gen_len=3)
    params.n = 2.5                                    # changed after it was checked
    scheduler, _ = scheduler_of()
    with pytest.raises(TypeError):
        scheduler.add_request(list(range(20)), params, "a")
    assert not scheduler.waiting and not scheduler.has_unfinished()


@pytest.mark.parametrize("steps", [0, 1, 2])
@pytest.mark.parametrize("gone", [1, 2, 3])
def test_the_prompt_is_computed_once_for_those_that_are_left(steps, gone):
    """The completion that computes the prompt is aborted before the others are forked from it, and the next one, and the next."""
    scheduler, executor = scheduler_of(max_num_seqs=8)
    request = scheduler.add_request(list(range(90)), several(6, 3), "a")       # 90 tokens in portions of 32
    for _ in range(steps):
        scheduler.step()
    for each in request.completions[:gone]:
        scheduler.abort(each)
    before = len(executor.steps)
    scheduler.run_to_completion()
    left = [r.request_id for r in request.completions[gone:]]
    assert executor.forked == [(left[0], left[1:])]
    assert [r.finish_reason for r in request.completions] == ["abort"] * gone + ["length"] * len(left)
    assert all(len(r.output_token_ids) == 3 for r in request.completions[gone:])
    assert sum(count for step in executor.steps[before:] for _, start, count, _ in step if start < 89) == 89
    assert executor.cache.num_free_slots == 8 and not scheduler.has_unfinished()

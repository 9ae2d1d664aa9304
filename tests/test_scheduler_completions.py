"""Several completions of one prompt through the scheduler, with a scripted executor (no GPU)."""

from __future__ import annotations

import pytest
from test_scheduler import ScriptedExecutor, greedy, make

from rapid_llm_b200.config import EngineConfig
from rapid_llm_b200.engine.scheduler import Scheduler
from rapid_llm_b200.sampling import SamplingParams


class Forking(ScriptedExecutor):
    forks: list

    def fork(self, parent, children):
        copies = self.cache.fork(parent, children)
        self.cache.check()
        if copies is None:
            return False
        self.__dict__.setdefault("forked", []).append((parent, list(children)))
        return True


def scheduler_of(pages=64, **overrides):
    values = dict(max_seq_len=256, page_size=16, max_num_seqs=4, max_num_batched_tokens=64, max_chunk_size=32)
    values.update(overrides)
    config = EngineConfig(**values)
    executor = Forking(config, pages)
    return Scheduler(executor, config, stop_token_ids=[7]), executor


def several(n, tokens, **more):
    return SamplingParams(temperature=0.0, top_p=1.0, repetition_penalty=1.0, max_gen_len=tokens, n=n, **more)


def test_the_prompt_is_computed_once():
    scheduler, executor = scheduler_of()
    request = scheduler.add_request(list(range(70)), several(3, 4), "a")
    scheduler.run_to_completion()
    assert executor.forked == [("a", [("a", 1), ("a", 2)])]
    assert [r.output_token_ids for r in request.completions] == [[1000, 1001, 1002, 1003]] * 3
    assert all(r.finish_reason == "length" for r in request.completions) and len({r.seed for r in request.completions}) == 3
    prompt_tokens = sum(count for step in executor.steps for _, start, count, _ in step if start < 69)
    assert prompt_tokens == 69                                        # once, but for the last token of each
    fork_step = next(step for step in executor.steps if len(step) == 3)
    assert [(start, count, samples) for _, start, count, samples in fork_step] == [(69, 1, True)] * 3
    assert executor.cache.num_free_slots == 4 and executor.cache.num_free_pages() == 64


@pytest.mark.parametrize("length", [1, 2, 16, 17, 32, 33])
def test_prompts_of_any_length(length):
    scheduler, executor = scheduler_of()
    request = scheduler.add_request(list(range(length)), several(2, 3), "a")
    other = scheduler.add_request(list(range(5)), greedy(2), "b")
    scheduler.run_to_completion()
    assert [len(r.output_token_ids) for r in request.completions] == [3, 3] and len(other.output_token_ids) == 2
    assert bool(getattr(executor, "forked", [])) == (length > 1)
    assert executor.cache.num_free_slots == 4


def test_those_that_find_no_place_compute_the_prompt_themselves():
    scheduler, executor = scheduler_of(max_num_seqs=3)
    request = scheduler.add_request(list(range(40)), several(6, 3), "a")
    later = scheduler.add_request(list(range(9)), greedy(2), "b")
    scheduler.run_to_completion()
    assert [len(r.output_token_ids) for r in request.completions] == [3] * 6 and later.finished
    assert executor.forked == [("a", [("a", 1), ("a", 2)])]
    scheduler, executor = scheduler_of(pages=4, max_num_seqs=4)        # the prompt takes three pages, a fork one more
    request = scheduler.add_request(list(range(40)), several(3, 3), "a")
    scheduler.run_to_completion()
    assert [len(r.output_token_ids) for r in request.completions] == [3] * 3 and executor.forked == [("a", [("a", 1)])]
    assert executor.cache.num_free_pages() == 4


def test_eviction_of_some_of_them():
    scheduler, executor = scheduler_of(pages=7, max_num_seqs=4, max_seq_len=100)
    request = scheduler.add_request(list(range(36)), several(3, 40), "a")
    scheduler.run_to_completion()
    assert [len(r.output_token_ids) for r in request.completions] == [40] * 3 and scheduler.num_preemptions > 0
    assert executor.cache.num_free_pages() == 7


def test_aborts_at_any_time():
    for when in range(6):
        for whom in range(3):
            scheduler, executor = scheduler_of()
            request = scheduler.add_request(list(range(50)), several(3, 6), "a")
            for _ in range(when):
                scheduler.step()
            scheduler.abort(request.completions[whom])
            scheduler.run_to_completion()
            reasons = [r.finish_reason for r in request.completions]
            assert reasons[whom] == "abort" and [r for i, r in enumerate(reasons) if i != whom] == ["length"] * 2
            assert executor.cache.num_free_slots == 4 and not scheduler.has_unfinished()
    scheduler, executor = scheduler_of()
    request = scheduler.add_request(list(range(50)), several(3, 6), "a")
    scheduler.abort(("a", 2))                                          # by its id, before the fork
    scheduler.run_to_completion()
    assert [r.finish_reason for r in request.completions] == ["length", "length", "abort"]


def test_an_executor_that_cannot_fork():
    scheduler, executor = make()
    request = scheduler.add_request(list(range(20)), several(2, 3), "a")
    scheduler.run_to_completion()
    assert [len(r.output_token_ids) for r in request.completions] == [3, 3]


def test_seeds():
    scheduler, _ = scheduler_of()
    request = scheduler.add_request([1, 2, 3], several(4, 2, seed=2**63 - 5), "a")
    assert request.seed == 2**63 - 5 and all(0 <= r.seed < 2**63 for r in request.completions) and len({r.seed for r in request.completions}) == 4


@pytest.mark.parametrize("wrong", [{"top_k": -1}, {"top_k": 1.5}, {"min_p": -0.1}, {"min_p": 1.1}, {"n": 0}, {"n": 2.5},
                                   {"top_k": float("inf")}, {"n": float("inf")}, {"top_k": float("nan")}])
def test_refused_parameters(wrong):
    with pytest.raises(ValueError):
        SamplingParams(**wrong)

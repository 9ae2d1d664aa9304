"""Requests forked from one another through the step function and the entry point: pages shared, states copied, shared prefixes
read once, several completions of one prompt."""

from __future__ import annotations

import importlib

import pytest
import torch
from tiny_configs import PAGE_SIZES
from tolerances import assert_rows_close, assert_rows_close_by_size, for_dtype

pytestmark = pytest.mark.gpu
DTYPES = ["float32", "bfloat16"]


def tokens_of(vocab: int, count: int, seed: int) -> list[int]:
    return torch.randint(0, vocab, (count,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.fixture(params=[False, True], ids=["ordinary", "shared"])
def sharing(request, monkeypatch):
    """Both ways a decode step can read shared pages, whatever its size."""
    from rapid_llm_b200.parts import attention

    for name in ("WORTH_SHARING", "WORTH_SHARING_F32"):
        monkeypatch.setattr(attention, name, 0 if request.param else 1 << 62)
    monkeypatch.setattr(attention, "MEMBERS_WORTH_SHARING", 2)
    return request.param


def step_of(request_id, tokens):
    from rapid_llm_b200.engine.runner import StepEntry

    return StepEntry(request_id, tokens, [len(tokens) - 1])


def shared_plans(runner) -> int:
    """How many of the captured graphs hold attention over shared prefixes."""
    return sum(any(name == "shared" for _, name, _ in constants) for _, constants in runner._graphs)


def make_runner(folder, dtype: str, page_size: int):
    from rapid_llm_b200.config import EngineConfig
    from rapid_llm_b200.engine.runner import ModelRunner

    return ModelRunner.from_folder(folder, EngineConfig(dtype=getattr(torch, dtype), max_seq_len=128, page_size=page_size, num_pages=80,
                                                        max_num_seqs=8, max_num_batched_tokens=64))


def run_family(runner, vocab, prompt_len, count, steps, graph=True, compact_at=None, drop_at=None):
    """A prompt, ``count`` requests forked from it, each fed tokens of its own one by one; logits by (request, step)."""
    prompt = tokens_of(vocab, prompt_len, 1)
    names = ["p"] + [f"c{i}" for i in range(1, count)]
    fed = {name: tokens_of(vocab, steps, 10 + i) for i, name in enumerate(names)}
    assert runner.admit("p")
    at = 0
    while at < prompt_len:                         # in two portions
        size = min(prompt_len - at, max(1, prompt_len // 2 + 1))
        runner.step([step_of("p", prompt[at : at + size])])
        at += size
    assert runner.fork("p", names[1:])
    rows = {}
    for step in range(steps):
        live = [name for name in names if drop_at is None or step < drop_at or name != names[1]]
        if drop_at == step:
            runner.release(names[1])
        if compact_at == step:
            runner.compact()
        order = live[step % len(live) :] + live[: step % len(live)]         # another order every step
        entries = [step_of(name, [fed[name][step]]) for name in order]
        logits = runner.step_decode(entries) if graph else runner.step(entries)
        for name, row in zip(order, logits.float().cpu().clone()):
            rows[name, step] = row
        runner.check_fault()
        runner.cache.check()
    for name in names:
        if runner.cache.has(name):
            runner.release(name)
    runner.cache.check()
    return prompt, fed, rows


@pytest.mark.parametrize("graph", [True, False], ids=["graph", "eager"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_a_fork_goes_on_as_a_request_of_its_own(name, dtype, graph, sharing, tiny_dirs, tiny_dirs_bf16, tiny_plain, tiny_plain_bf16):
    from plain_qwen3 import forward_logits

    dirs, plains = (tiny_dirs, tiny_plain) if dtype == "float32" else (tiny_dirs_bf16, tiny_plain_bf16)
    config, weights = plains[name]
    runner = make_runner(dirs[name], dtype, PAGE_SIZES[name])
    for prompt_len, count in ((PAGE_SIZES[name] * 3, 3), (PAGE_SIZES[name] * 2 + 5, 7), (3, 2)):
        prompt, fed, rows = run_family(runner, config["vocab_size"], prompt_len, count, 12, graph=graph)
        for request, tokens in fed.items():
            plain = forward_logits(config, weights, prompt + tokens)
            for step in range(12):
                torch.testing.assert_close(rows[request, step], plain[prompt_len + step], **for_dtype(dtype))
    if graph:
        assert (shared_plans(runner) > 0) == sharing


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_member_leaves_and_pages_move(dtype, sharing, tiny_dirs, tiny_dirs_bf16, tiny_plain, tiny_plain_bf16):
    from plain_qwen3 import forward_logits

    dirs, plains = (tiny_dirs, tiny_plain) if dtype == "float32" else (tiny_dirs_bf16, tiny_plain_bf16)
    config, weights = plains["B"]
    runner = make_runner(dirs["B"], dtype, 8)
    runner.admit("old")
    runner.step([step_of("old", tokens_of(config["vocab_size"], 40, 3))])
    runner.admit("p0")                             # holds pages between
    runner.step([step_of("p0", [1, 2, 3])])
    runner.release("old")
    prompt, fed, rows = run_family(runner, config["vocab_size"], 37, 4, 14, compact_at=6, drop_at=9)
    for (request, step), row in rows.items():
        plain = forward_logits(config, weights, prompt + fed[request])
        torch.testing.assert_close(row, plain[37 + step], **for_dtype(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("family", ["kopatar", "mezadra", "basitar", "zupupel", "bidetar", "danalorn"])
def test_every_architecture_forks(family, dtype, sharing):
    """A fork's logits are those of a request that was given the same tokens from the start: states, windows, chunks, cached
    latents and shared caches included."""
    from rapid_llm_b200.config import EngineConfig
    from rapid_llm_b200.config.registry import resolve_architecture
    from rapid_llm_b200.engine.runner import ModelRunner

    draw = importlib.import_module(f"test_{family}_random_gpu").draw_config
    for seed in range(3):
        raw = draw(seed)
        config = resolve_architecture(raw).from_dict(raw)
        runner = ModelRunner.from_random(config, seed, EngineConfig(
            dtype=getattr(torch, dtype), max_seq_len=64, page_size=8, num_pages=60, max_num_seqs=6, max_num_batched_tokens=64), std=0.08)
        vocab = runner.model.spec.vocab_size
        prompt, fed, rows = run_family(runner, vocab, 21, 3, 8)
        for request, tokens in fed.items():
            runner.admit("alone")
            runner.step([step_of("alone", prompt[:11])])
            runner.step([step_of("alone", prompt[11:])])
            for step, token in enumerate(tokens):
                want = runner.step_decode([step_of("alone", [token])])[0].float().cpu()
                close = assert_rows_close if dtype == "float32" else assert_rows_close_by_size
                close(rows[request, step][None], want[None], dtype)
            runner.release("alone")


@pytest.mark.parametrize("dtype", DTYPES)
def test_wide_heads_share_long_prefixes_without_being_asked(dtype):
    """Heads of 128, a prompt of some thousand tokens: the step is large enough that sharing is chosen, and equals the ordinary step."""
    from rapid_llm_b200.config import EngineConfig, Qwen3Config
    from rapid_llm_b200.engine.runner import ModelRunner
    from rapid_llm_b200.parts import attention
    from tiny_configs import TINY_A

    config = Qwen3Config.from_dict({**TINY_A, "head_dim": 128, "num_attention_heads": 32, "num_key_value_heads": 8, "max_position_embeddings": 8192})
    runner = ModelRunner.from_random(config, 5, EngineConfig(
        dtype=getattr(torch, dtype), max_seq_len=4200, page_size=16, num_pages=700, max_num_seqs=12, max_num_batched_tokens=4096), std=0.05)
    _, _, rows = run_family(runner, 256, 4001, 12, 5)
    assert shared_plans(runner) == 1                # five lengths, one graph
    before = attention.WORTH_SHARING, attention.WORTH_SHARING_F32
    attention.WORTH_SHARING = attention.WORTH_SHARING_F32 = 1 << 62
    try:
        _, _, ordinary = run_family(runner, 256, 4001, 12, 5)
    finally:
        attention.WORTH_SHARING, attention.WORTH_SHARING_F32 = before
    for key, row in rows.items():
        assert_rows_close(row[None], ordinary[key][None], dtype)


def make_llm(folder, **overrides):
    from rapid_llm_b200 import LLM

    return LLM(folder, **{**dict(dtype="float32", max_seq_len=128, max_gpu_num_blocks=64, page_size=16, max_num_seqs=6, max_chunk_size=13,
                                 max_num_batched_tokens=64), **overrides})


@pytest.mark.parametrize("run_ahead", [True, False], ids=["ahead", "lockstep"])
@pytest.mark.parametrize("penalty", [1.0, 1.2])
def test_completions_are_those_of_requests_of_their_own(run_ahead, penalty, sharing, tiny_dirs):
    from rapid_llm_b200 import SamplingParams
    from rapid_llm_b200.engine.scheduler import SEED_STRIDE

    llm = make_llm(tiny_dirs["A"], run_ahead=run_ahead)
    prompts = [tokens_of(256, n, 40 + n) for n in (37, 1, 16, 50)]
    kind = dict(temperature=0.9, top_p=0.9, repetition_penalty=penalty, max_gen_len=14, top_k=60, min_p=0.01)
    several = llm.generate(prompts, [SamplingParams(n=n, seed=70 + i, **kind) for i, n in enumerate((4, 3, 1, 8))])
    assert [len(o.outputs) for o in several] == [4, 3, 1, 8]
    for i, (prompt, output) in enumerate(zip(prompts, several)):
        for index, completion in enumerate(output.outputs):
            alone = llm.generate([prompt], SamplingParams(seed=(70 + i + index * SEED_STRIDE) % 2**63, **kind))[0]
            assert completion.token_ids == alone.token_ids and completion.index == index
    greedy = llm.generate([prompts[0]], SamplingParams(temperature=0.0, top_p=1.0, repetition_penalty=1.0, max_gen_len=9, n=3))[0]
    assert len({tuple(c.token_ids) for c in greedy.outputs}) == 1 and len(greedy.token_ids) == 9
    llm.runner.cache.check()
    assert llm.runner.cache.num_free_slots == 6 and not llm.scheduler.has_unfinished()
    with pytest.raises(ValueError):
        next(llm.stream(prompts, SamplingParams(n=2)))


def test_filters_of_one_request_leave_the_others_alone(tiny_dirs):
    from rapid_llm_b200 import SamplingParams

    llm = make_llm(tiny_dirs["A"])
    prompts = [tokens_of(256, n, n) for n in (9, 30, 12)]
    params = [SamplingParams(temperature=0.8, top_p=0.9, repetition_penalty=1.0, max_gen_len=12, seed=i, **more)
              for i, more in enumerate(({}, {"top_k": 1}, {"min_p": 0.2, "top_k": 20}))]
    together = llm.generate(prompts, params)
    alone = [llm.generate([p], [sp])[0] for p, sp in zip(prompts, params)]
    assert [o.token_ids for o in together] == [o.token_ids for o in alone]
    greedy = llm.generate([prompts[1]], SamplingParams.greedy(max_gen_len=12))[0]
    assert together[1].token_ids == greedy.token_ids


def test_the_command_line_prints_every_completion(tiny_dirs, tmp_path):
    import subprocess
    import sys
    from pathlib import Path

    ids = tmp_path / "prompts.txt"
    ids.write_text("5 6 7 8 9\n11 12\n")
    done = subprocess.run(
        [sys.executable, "-m", "rapid_llm_b200.cli", "batch", "--model-dir", str(tiny_dirs["A"]), "--dtype", "float32", "--prompt-ids-file", str(ids),
         "--temperature", "0.8", "--top-k", "30", "--min-p", "0.01", "--n", "3", "--seed", "4", "--max-gen-len", "6", "--max-seq-len", "64",
         "--max-gpu-num-blocks", "40"], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stderr[-2000:]
    assert [line.split()[1] for line in done.stdout.splitlines() if line.startswith("---")] == ["[0.0]", "[0.1]", "[0.2]", "[1.0]", "[1.1]", "[1.2]"]

"""A family whose members end one by one, its decode steps replayed from captured graphs that read the shared pages once."""

from __future__ import annotations

import pytest
import torch
from test_fork_gpu import make_runner, shared_plans, step_of, tokens_of
from tolerances import for_dtype

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_members_end_one_by_one(dtype, monkeypatch, tiny_dirs, tiny_dirs_bf16, tiny_plain, tiny_plain_bf16):
    from plain_qwen3 import forward_logits
    from rapid_llm_b200.parts import attention

    for name in ("WORTH_SHARING", "WORTH_SHARING_F32"):
        monkeypatch.setattr(attention, name, 0)
    monkeypatch.setattr(attention, "MEMBERS_WORTH_SHARING", 2)
    dirs, plains = (tiny_dirs, tiny_plain) if dtype == "float32" else (tiny_dirs_bf16, tiny_plain_bf16)
    config, weights = plains["B"]
    runner = make_runner(dirs["B"], dtype, 8)
    vocab, prompt = config["vocab_size"], tokens_of(config["vocab_size"], 32, 1)
    names = ["p"] + [f"c{i}" for i in range(1, 8)]
    assert runner.admit("p")
    runner.step([step_of("p", prompt)])
    assert runner.fork("p", names[1:])
    fed = {name: tokens_of(vocab, 6, 20 + i) for i, name in enumerate(names)}
    rows, live = {}, list(names)
    for step in range(6):                        # 8, 7, 6, 5, 5, 5 members, all in the batch of eight
        if step in (1, 2, 3):
            runner.release(live.pop(step))       # one from the middle
        logits = runner.step_decode([step_of(name, [fed[name][step]]) for name in live])
        for name, row in zip(live, logits.float().cpu().clone()):
            rows[name, step] = row
        runner.check_fault()
    assert shared_plans(runner) == len(runner._graphs) == 1
    for (name, step), row in rows.items():
        plain = forward_logits(config, weights, prompt + fed[name][: step + 1])
        torch.testing.assert_close(row, plain[32 + step], **for_dtype(dtype))

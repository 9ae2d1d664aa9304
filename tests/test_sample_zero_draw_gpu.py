"""A draw of exactly zero: the first index that the cuts leave, however little it weighs."""

from __future__ import annotations

import numpy as np
import pytest
import torch
from test_sample_filters_gpu import DEV, choose, logits_of, run_case

from rapid_llm_b200.ops import kernels

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("vocab", [3, 700, 20011, 151936])
@pytest.mark.parametrize("temperature", [1e-30, 0.003, 0.05, 0.1, 0.2, 0.3, 1.0])
def test_top_k_holds_where_fewer_tokens_weigh_anything(dtype, vocab, temperature):
    """Low temperatures leave fewer tokens of any weight in 43 bits than top-k keeps; those it does not keep are never drawn."""
    x = logits_of(4, vocab, dtype, seed=vocab)
    x[2, : vocab // 2] = x[2, vocab // 2]            # many equal ones: of these the lowest indices stay
    x[3, ::3] = -float("inf")
    for top_k in (1, 2, 5, 50, 300, 3000):
        run_case(x, temperature, top_k, 1.0, 0.0, torch.zeros(4))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_three_tokens_far_apart(dtype):
    x = torch.tensor([[-100.0, -90.0, 0.0], [-90.0, -100.0, 0.0], [0.0, -100.0, -90.0]], device=DEV).to(dtype)
    assert run_case(x, 1.0, 2, 1.0, 0.0, torch.zeros(3)) == [1, 0, 0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_rows_with_and_without_a_draw_of_zero(dtype):
    rows = 40
    u = torch.rand((rows,), generator=torch.Generator().manual_seed(9))
    u[::2] = 0.0
    rng = np.random.RandomState(4)
    run_case(logits_of(rows, 50021, dtype, seed=7), torch.from_numpy(rng.choice([0.02, 0.1, 0.25, 0.9], rows)),
             torch.from_numpy(rng.choice([0, 2, 40, 700, 9000], rows)), 1.0, 0.0, u)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("vocab", [6, 3000, 151936])
@pytest.mark.parametrize("top_k", [0, 5, 400])
def test_min_p_far_below_the_smallest_weight(dtype, vocab, top_k):
    """A share of 1e-20 lies between e^-47 and e^-46: with a draw of zero the first token within 46 temperatures is taken.  (No token
    is nearer to the border than a tenth of an octave, so nothing here depends on how an exponential is rounded.)"""
    x = torch.full((3, vocab), -200.0, device=DEV)
    for row, values in enumerate(([-60.0, -50.0, -40.0, 0.0, -44.0], [-47.0, -48.0, -45.0, -45.0, 0.0], [-47.0, -70.0, 0.0, -10.0, -1.0])):
        x[row, :5] = torch.tensor(values, device=DEV)
    of = lambda value, kind=torch.float32: torch.full((3,), value, dtype=kind, device=DEV)
    out = of(-7, torch.int32)
    kernels.sample(x.to(dtype), out, temperature=of(1.0), top_k=of(top_k, torch.int32), min_p=of(1e-20), uniforms=of(0.0))
    assert out.tolist() == [2, 2, 2]
    for row in range(3):
        assert choose(x[row].double().cpu().numpy(), 1.0, top_k, 1.0, float(np.float32(1e-20)), 0.0)[0] == 2

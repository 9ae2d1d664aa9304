"""The choice of a token with top-k, top-p and min-p from given random numbers, against the definition in 64 bits."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from rapid_llm_b200.ops import kernels

DEV = "cuda:0"


def choose(x, temperature, top_k, top_p, min_p, u):
    """The definition over one row of float64 logits; also the distance of the draw and of the cuts from the next border, as
    a share of the mass: below 1e-9 a row says nothing about a kernel whose masses are exact to 1e-13 a token."""
    x = np.where(np.isnan(x), -np.inf, x)
    if not (x > -np.inf).any():
        return 0, 1.0
    top = int(np.argmax(x))
    if not temperature > 0:
        return top, 1.0
    if x[top] == np.inf:
        x = np.where(x == np.inf, 0.0, -np.inf)
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp((x - x.max()) / temperature)
    order = np.lexsort((np.arange(len(x)), -x))
    chosen = order[:top_k] if 0 < top_k else order
    margin = 1.0
    kept = chosen
    if top_p < 1:
        z = math.fsum(w[chosen])
        xs = x[chosen]
        upto = np.cumsum(w[chosen])
        starts = np.flatnonzero(np.concatenate(([True], xs[1:] != xs[:-1])))
        run = np.cumsum(np.concatenate(([True], xs[1:] != xs[:-1]))) - 1
        above = (upto - w[chosen])[starts][run]
        near = np.abs(above[(w[chosen] > 0) & (above > 0)] / z - top_p)          # nothing above is exactly nothing
        margin = min(margin, float(near.min())) if len(near) else margin
        kept = chosen[above <= max(top_p, 0.0) * z]
    if min_p > 0:
        margin = min(margin, float(np.abs(w[kept] - min(min_p, 1.0)).min()) if min_p < 1 else 1.0)
    kept = np.sort(kept[w[kept] >= min(min_p, 1.0)])
    running = np.cumsum(w[kept])
    target = u * running[-1]
    margin = min(margin, float(np.abs(running[w[kept] > 0] - target).min() / running[-1])) if u > 0 else margin
    return int(kept[np.searchsorted(running, target, side="right")]), margin


def run_case(logits, temperature, top_k, top_p, min_p, u, **more):
    rows = logits.shape[0]
    spread = lambda v, dtype: (v if isinstance(v, torch.Tensor) else torch.full((rows,), v)).to(dtype).to(DEV)
    out = torch.full((rows,), -7, dtype=torch.int32, device=DEV)
    params = {"temperature": spread(temperature, torch.float32), "top_k": spread(top_k, torch.int32),
              "top_p": spread(top_p, torch.float32), "min_p": spread(min_p, torch.float32), "uniforms": spread(u, torch.float32)}
    kernels.sample(logits, out, **params, **more)
    got = out.tolist()
    host = {k: v.double().cpu().numpy() for k, v in params.items()}
    x = logits.double().cpu().numpy()
    told = 0
    for row in range(rows):
        want, margin = choose(x[row], host["temperature"][row], int(host["top_k"][row]), host["top_p"][row], host["min_p"][row],
                              host["uniforms"][row])
        if margin > 1e-9:
            told += 1
            assert got[row] == want, (row, got[row], want, margin, {k: v[row] for k, v in host.items()})
    assert told >= rows // 2
    return got


def logits_of(rows, vocab, dtype, spread=2.5, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn((rows, vocab), generator=gen, device=DEV) * spread
    x[:, torch.randint(0, vocab, (min(3, vocab),), generator=gen, device=DEV)] += 2 * spread
    return x.to(dtype)


def draws(rows, seed=1):
    u = torch.rand((rows,), generator=torch.Generator().manual_seed(seed))
    u[0] = 0.0
    if rows > 1:
        u[1] = 1.0 - 2.0**-24
    return u


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 400, 4099, 32003, 151936])
@pytest.mark.parametrize("cut", [(0, 1.0, 0.0), (1, 1.0, 0.0), (5, 0.8, 0.0), (50, 0.9, 0.02), (0, 0.9, 0.0), (0, 1.0, 0.05), (300, 1.0, 0.0),
                                 (300, 0.7, 0.001), (3000, 0.98, 0.0), (0, 0.999, 0.0), (20, 0.0, 0.0), (0, 0.0, 0.0), (0, 0.5, 1.0), (40000, 1.0, 0.0)], ids=str)
def test_cuts_and_draws(vocab, dtype, cut):
    top_k, top_p, min_p = cut
    run_case(logits_of(9, vocab, dtype, seed=vocab), 0.9, top_k, top_p, min_p, draws(9))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_rows_that_disagree(dtype):
    rng = np.random.RandomState(5)
    rows = 70
    pick = lambda values: torch.tensor(rng.choice(values, rows))
    run_case(logits_of(rows, 50021, dtype, seed=3), pick([0.0, 0.3, 0.7, 1.0, 1.5, 30.0]), pick([0, 0, 1, 40, 700, 60000]),
             pick([1.0, 0.95, 0.5, 0.999]), pick([0.0, 0.0, 0.01, 0.3]), draws(rows))


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [10, 777, 20000])
def test_equal_logits(vocab):
    """All equal, and equal in a few levels: the cut of top-k goes by the index, the others take equal ones together."""
    for x in (torch.zeros((6, vocab), device=DEV), torch.full((6, vocab), torch.finfo(torch.float32).min, device=DEV),
              (torch.arange(6 * vocab, device=DEV) % 5).float().view(6, vocab)):
        for top_k in (0, 1, vocab // 3, vocab - 1, vocab):
            for top_p in (1.0, 0.63):
                run_case(x, 1.0, top_k, top_p, 0.0, draws(6, seed=vocab))


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [300, 5000, 60000])
def test_zeros_of_both_signs_are_equal(vocab):
    x = torch.zeros((5, vocab), device=DEV)
    x[:, torch.rand((vocab,), generator=torch.Generator(device=DEV).manual_seed(vocab), device=DEV) < 0.5] = -0.0
    x[3, 7] = 1.0
    for dtype in (torch.float32, torch.bfloat16):
        for top_k, top_p in ((0, 0.5), (1, 1.0), (40, 0.5), (vocab // 2, 1.0), (vocab - 3, 0.9)):
            run_case(x.to(dtype), 0.7, top_k, top_p, 0.0, draws(5))
        run_case(x.to(dtype), 0.0, 0, 1.0, 0.0, draws(5))


@pytest.mark.gpu
def test_values_nearer_than_the_codes():
    """Thousands of different values within a tiny part of the row's range."""
    x = torch.full((4, 9000), -9.0, device=DEV)
    x[:, :8000] = -8.0 + torch.rand((4, 8000), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV) * 2e-6
    x[:, 17] = 9.0
    for top_k, top_p in ((0, 1.0), (4000, 1.0), (0, 0.9999998), (5000, 0.9999997), (300, 1.0)):
        run_case(x, 2.0, top_k, top_p, 0.0, torch.tensor([0.1, 0.9999999, 0.99999994, 0.99999]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_infinities_nan_and_lowest_values(dtype):
    lowest = torch.finfo(dtype).min
    x = logits_of(8, 5003, dtype, seed=8)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, 7:] = -math.inf
    x[3, ::2] = lowest
    x[4, 40] = x[4, 4000] = math.inf
    x[5, ::3] = math.nan
    x[6] = lowest
    x[7, :5000] = -math.inf
    for top_k, top_p, min_p in ((0, 1.0, 0.0), (3, 1.0, 0.0), (50, 0.9, 0.1), (0, 0.9, 0.0)):
        got = run_case(x, 1.0, top_k, top_p, min_p, draws(8))
        assert got[0] == 0 and got[1] == 0 and got[4] in (40, 4000) and got[5] % 3 != 0
        run_case(x, 0.0, top_k, top_p, min_p, draws(8))


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [1e-30, 1e-6, 0.05, 20.0, 1e6])
def test_temperatures(temperature):
    for top_k, top_p in ((0, 1.0), (30, 0.9), (0, 0.9), (2000, 0.9)):
        run_case(logits_of(6, 20011, torch.float32, seed=2), temperature, top_k, top_p, 0.0, draws(6))


@pytest.mark.gpu
def test_strided_rows_and_rows_off_the_vector_boundary():
    wide = logits_of(7, 3001, torch.bfloat16, seed=4)
    for begin, end in ((0, 2999), (1, 3000), (8, 1500)):
        run_case(wide[:, begin:end], 0.8, 20, 0.9, 0.0, draws(7))
        run_case(wide[::2, begin:end], 0.8, 0, 0.9, 0.0, draws(4))


@pytest.mark.gpu
def test_penalty_and_seeds_as_the_plain_call():
    """Without a cut that only this form has, seeded draws are those of the call without one; a penalty meets each token once."""
    x = logits_of(12, 4000, torch.float32, seed=6)
    seeds = torch.arange(12, dtype=torch.int64, device=DEV) * 977 + 5
    counters = torch.arange(12, dtype=torch.int32, device=DEV)
    seen = torch.tensor([3, 9, 3, 3999, 70000, -4] * 12, dtype=torch.int32, device=DEV)
    offsets = torch.arange(13, dtype=torch.int32, device=DEV) * 6
    args = {"temperature": torch.full((12,), 0.7, device=DEV), "top_p": torch.full((12,), 0.9, device=DEV),
            "penalty": torch.full((12,), 1.3, device=DEV), "seeds": seeds, "counters": counters, "seen_tokens": seen, "seen_offsets": offsets}
    plain, here = (torch.empty((12,), dtype=torch.int32, device=DEV) for _ in range(2))
    kernels.sample(x, plain, **args)
    kernels.sample(x, here, top_k=torch.zeros((12,), dtype=torch.int32, device=DEV), **args)
    assert torch.equal(plain, here)
    penalised = x.clone()
    for id in (3, 9, 3999):
        column = penalised[:, id]
        penalised[:, id] = torch.where(column < 0, column * 1.3, column / 1.3)
    u = draws(12)
    out = torch.empty((12,), dtype=torch.int32, device=DEV)
    kernels.sample(x, out, temperature=args["temperature"], top_p=args["top_p"], penalty=args["penalty"], seen_tokens=seen,
                   seen_offsets=offsets, uniforms=u.to(DEV))
    assert out.tolist() == run_case(penalised, 0.7, 0, 0.9, 0.0, u)


@pytest.mark.gpu
def test_replayed_and_on_another_stream():
    x = logits_of(5, 30011, torch.bfloat16, seed=11)
    u = draws(5).to(DEV)
    t, k = torch.full((5,), 0.8, device=DEV), torch.full((5,), 30, dtype=torch.int32, device=DEV)
    want = torch.empty((5,), dtype=torch.int32, device=DEV)
    kernels.sample(x, want, temperature=t, top_k=k, uniforms=u)
    out = torch.empty_like(want)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        kernels.sample(x, out, temperature=t, top_k=k, uniforms=u)
    for _ in range(3):
        out.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def _arguments():
    x = torch.randn((3, 50), device=DEV)
    return {"logits": x, "out": torch.zeros((3,), dtype=torch.int32, device=DEV), "temperature": torch.ones((3,), device=DEV),
            "top_k": torch.full((3,), 5, dtype=torch.int32, device=DEV), "uniforms": torch.rand((3,), device=DEV)}


@pytest.mark.gpu
@pytest.mark.parametrize("name,value", [
    ("top_k", lambda: torch.full((3,), 5, device=DEV)), ("top_k", lambda: torch.full((2,), 5, dtype=torch.int32, device=DEV)),
    ("uniforms", lambda: torch.rand((3,), dtype=torch.float64, device=DEV)), ("uniforms", lambda: torch.rand((6,), device=DEV)[::2]),
    ("min_p", lambda: torch.rand((4,), device=DEV)), ("uniforms", lambda: None), ("logits", lambda: torch.randn((50, 3), device=DEV).T),
    ("logits", lambda: torch.randn((3, 50), device=DEV).half()), ("logits", lambda: torch.randn((3, 400000), device=DEV)),
    ("out", lambda: torch.zeros((3,), dtype=torch.int64, device=DEV)), ("seen_tokens", lambda: torch.zeros((3,), dtype=torch.int32, device=DEV)),
    ("temperature", lambda: torch.ones((3,))),
])
def test_refused(name, value):
    arguments = _arguments()
    arguments[name] = value()
    with pytest.raises(kernels.KernelError):
        kernels.sample(arguments.pop("logits"), arguments.pop("out"), **arguments)


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [1e-44, 3e-39, 3e38, float("inf")])
def test_temperatures_at_the_ends_of_the_type(temperature):
    for top_k, top_p, min_p in ((0, 1.0, 0.0), (30, 0.9, 0.0), (0, 0.7, 0.5), (2000, 0.9, 0.0)):
        run_case(logits_of(6, 20011, torch.float32, seed=2), temperature, top_k, top_p, min_p, draws(6))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_the_largest_vocabulary(dtype):
    largest = kernels.core().rl_sample_filtered_max_vocab()
    for top_k, top_p in ((0, 0.9), (40, 0.9), (largest - 1, 0.99)):
        run_case(logits_of(3, largest, dtype, seed=top_k), 1.0, top_k, top_p, 0.0, draws(3))
    with pytest.raises(kernels.KernelError):
        run_case(logits_of(3, largest + 1, dtype), 1.0, 40, 0.9, 0.0, draws(3))


@pytest.mark.gpu
def test_calls_side_by_side():
    calls = []
    for seed, (rows, vocab) in enumerate(((70, 32003), (9, 151936))):
        x = logits_of(rows, vocab, torch.bfloat16, seed=seed)
        of = lambda v, dtype=torch.float32: torch.full((rows,), v, dtype=dtype, device=DEV)
        arguments = dict(temperature=of(0.9), top_k=of(0, torch.int32), top_p=of(0.95), uniforms=draws(rows, seed=seed).float().to(DEV))
        calls.append((x, arguments, torch.cuda.Stream(), of(-7, torch.int32), kernels.sample(x, of(-7, torch.int32), **arguments)))
    torch.cuda.synchronize()
    for _ in range(20):
        for x, arguments, stream, out, _ in calls:
            with torch.cuda.stream(stream):
                out.fill_(-7)
                kernels.sample(x, out, **arguments)
    torch.cuda.synchronize()
    for _, _, _, out, want in calls:
        assert torch.equal(out, want)

"""Attention over shared prefixes against every request's own attention in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from rapid_llm_b200.ops import kernels
from rapid_llm_b200.parts.attention import SharedItems
from rapid_llm_b200.parts.base import StepShape

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Step:
    """A step over a random cache: ``requests`` are (group or -1, own positions, new tokens), ``prefix`` the groups' positions."""

    def __init__(self, prefix, requests, *, heads, kv_heads, dim, page, dtype, seed=0, spread=2.0):
        self.prefix, self.requests = prefix, requests
        self.heads, self.kv_heads, self.dim, self.page, self.dtype = heads, kv_heads, dim, page, dtype
        rng = np.random.RandomState(seed)
        shared = [prefix[g] if g >= 0 else 0 for g, _, _ in requests]
        lengths = [s + own for s, (_, own, _) in zip(shared, requests)]
        # a group's whole pages are shared; where its positions end inside a page every member has a page of its own with the same rows
        needed = sum(-(-length // page) for length in lengths) + sum(-(-p // page) for p in prefix) + 1
        ids = list(rng.permutation(needed) + 1)
        gen = torch.Generator(device=DEV).manual_seed(seed)
        self.cache = torch.randn((needed + 2, 2, kv_heads, page, dim), generator=gen, device=DEV).to(dtype)
        group_pages = [[ids.pop() for _ in range(-(-p // page))] for p in prefix]
        self.table = np.zeros((len(requests) + 2, max(-(-length // page) for length in lengths) + 1), dtype=np.int32)
        self.slots = rng.permutation(len(requests)) + 1              # slots in another order than the entries
        for slot, (g, _, _), s, length in zip(self.slots, requests, shared, lengths):
            whole = s // page
            pages = (group_pages[g][:whole] if g >= 0 else []) + [ids.pop() for _ in range(-(-length // page) - whole)]
            self.table[slot, : len(pages)] = pages
            if s % page:
                self.cache[pages[whole], :, :, : s % page] = self.cache[group_pages[g][whole], :, :, : s % page]
        self.starts = [length - new for length, (_, _, new) in zip(lengths, requests)]
        self.new = [new for _, _, new in requests]
        self.positions = np.concatenate([np.arange(s, s + n) for s, n in zip(self.starts, self.new)])
        self.entry_of = np.repeat(np.arange(len(requests)), self.new)
        tokens = len(self.positions)
        self.q = (torch.randn((tokens, heads * dim), generator=gen, device=DEV) * spread).to(dtype)
        self.scale = dim**-0.5
        self.planner = SharedItems(heads // kv_heads, kv_heads, dim, dtype=dtype)
        self.shape = StepShape(lengths=np.asarray(self.new), starts=np.asarray(self.starts), decode_only=max(self.new) == 1,
                               page_size=page, prefix_group=np.asarray([g for g, _, _ in requests]), prefix_tokens=np.asarray(shared))
        self.fault = torch.zeros(1, dtype=torch.int32, device=DEV)

    def device_plan(self):
        plan = self.planner.plan(self.shape)
        return {k: torch.from_numpy(v).to(DEV) if isinstance(v, np.ndarray) else v for k, v in plan.items()}

    def run(self, out=None, plan=None, **options):
        plan = plan or self.device_plan()
        rows = self.planner.part_rows(plan)
        to = lambda values: torch.from_numpy(np.ascontiguousarray(np.asarray(values, dtype=np.int32))).to(DEV)
        # scratch with the worst that may lie there
        part_out = torch.full((max(rows, 1), self.dim), float("nan"), device=DEV)
        part_lse = torch.full((max(rows, 1),), float("nan"), device=DEV)
        out = torch.full_like(self.q, float("nan")) if out is None else out
        kernels.attention_shared(
            self.q, self.cache, out, plan=plan, part_out=part_out, part_lse=part_lse, positions=to(self.positions),
            cu_seqlens=to(np.concatenate(([0], np.cumsum(self.new)))), entry_start=to(self.starts), entry_slot=to(self.slots),
            block_table=to(self.table), num_heads=self.heads, num_kv_heads=self.kv_heads, head_dim=self.dim, scale=self.scale,
            fault=self.fault, **options)
        torch.cuda.synchronize()
        assert int(self.fault.item()) == 0
        return out

    def want(self, sink=None, gate=None, slopes=None):
        """The result, the same sums over |v| (what a weight's rounding acts on), and the largest score, in 64 bits."""
        group = self.heads // self.kv_heads
        q = self.q.double().view(-1, self.heads, self.dim)
        out, size, largest = torch.empty_like(q), torch.empty_like(q), 0.0
        for t, position in enumerate(self.positions):
            used = torch.from_numpy(self.table[self.slots[self.entry_of[t]], : position // self.page + 1].astype(np.int64)).to(DEV)
            k = self.cache[used, 0].double().permute(1, 0, 2, 3).flatten(1, 2)[:, : position + 1]
            v = self.cache[used, 1].double().permute(1, 0, 2, 3).flatten(1, 2)[:, : position + 1]
            s = torch.einsum("kgd,kjd->kgj", q[t].view(self.kv_heads, group, self.dim), k) * self.scale
            largest = max(largest, float(s.abs().max()))
            if slopes is not None:
                away = int(position) - torch.arange(int(position) + 1, device=DEV)
                s = s - slopes.double().view(self.kv_heads, group, 1) * away
            if sink is not None:
                s = torch.cat([s, sink.double().view(self.kv_heads, group, 1)], -1)
            w = torch.softmax(s, -1)[..., : int(position) + 1]
            out[t] = torch.einsum("kgj,kjd->kgd", w, v).reshape(self.heads, self.dim)
            size[t] = torch.einsum("kgj,kjd->kgd", w, v.abs()).reshape(self.heads, self.dim)
        if gate is not None:
            out, size = (x * torch.sigmoid(gate.double())[..., None] for x in (out, size))
        return out.view(self.q.shape), size.view(self.q.shape), largest


def check(got, reference, dtype, dim):
    """A weight that is off by a relative e moves the result by at most e times the sum over |v|.  Both types: a score is a sum of
    d products, whose roundings walk like sqrt(d) of 2^-24 of its size; four standard deviations of that, on a weight and on the
    sum of weights, and sixteen roundings for the exponential, the sums and the join.  bfloat16: also the weight's rounding
    (half a step, 2^-8 of it) and the result's (2^-8 of it)."""
    want, size, largest = reference
    allowed = size * 2.0**-24 * (8 * dim**0.5 * max(largest, 1.0) + 16)
    if dtype == torch.bfloat16:
        allowed = allowed + 2.0**-8 * (size + want.abs())
    excess = ((got.double() - want).abs() - allowed).max()
    assert bool(torch.isfinite(got).all()) and float(excess) <= 0.0, float(excess)


SHAPES = [
    dict(heads=8, kv_heads=2, dim=64, page=16),
    dict(heads=6, kv_heads=2, dim=128, page=16),
    dict(heads=5, kv_heads=1, dim=128, page=20),
    dict(heads=32, kv_heads=8, dim=128, page=64),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s['heads']}_{s['kv_heads']}_{s['dim']}_{s['page']}")
@pytest.mark.parametrize("layout", ["two", "one_key", "ragged", "odd_prefix", "many", "none", "single_member"])
def test_equals_each_requests_own_attention(shape, dtype, layout):
    page = shape["page"]
    prefix, requests = {
        "two": ([4 * page], [(0, 3, 1), (0, 40, 1)]),
        "one_key": ([page], [(0, 1, 1), (-1, 1, 1), (0, 1, 1)]),                # a request whose only key is its own
        "ragged": ([11 * page, 3 * page, 25 * page], [(0, 5, 1), (2, 130, 3), (-1, 77, 2), (0, 1, 1), (1, 200, 1), (2, 9, 5), (0, 64, 1)]),
        "odd_prefix": ([3 * page + 5, 129], [(0, 4, 1), (1, 70, 1), (0, 12, 2), (1, 1, 1)]),
        "many": ([700 // page * page], [(0, 1 + 7 * i % 50, 1) for i in range(40)]),
        "none": ([], [(-1, 300, 1), (-1, 1, 1), (-1, 65, 4)]),
        "single_member": ([600 // page * page], [(0, 17, 1)]),
    }[layout]
    step = Step(prefix, requests, dtype=dtype, seed=len(requests), **shape)
    check(step.run(), step.want(), dtype, shape["dim"])


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256, 24])
@pytest.mark.parametrize("members,group", [(5, 4), (30, 4), (33, 4), (64, 4), (52, 5), (70, 8), (7, 16)])
def test_tiles_of_every_height_and_page(page, members, group):
    """128 wide heads: one tile, two tiles, several items of two; prefixes that end inside a block of 128 keys, and one beyond."""
    for prefix in (page * 3, max(page, 1100 // page * page)):
        step = Step([prefix], [(0, 1 + 13 * i % 150, 1) for i in range(members)], heads=2 * group, kv_heads=2, dim=128, page=page,
                    dtype=torch.bfloat16, seed=members + page)
        check(step.run(), step.want(), torch.bfloat16, 128)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_what_lies_behind_a_request_is_not_seen(dtype, dim):
    """NaN in every place of the cache that no request holds, the places behind a request's last key in its own page among them."""
    for members in (3, 40):
        step = Step([176, 32], [(0, 1 + 7 * i % 40, 1) for i in range(members)] + [(1, 3, 2), (-1, 130, 1)], heads=8, kv_heads=2, dim=dim,
                    page=16, dtype=dtype, seed=3)
        held = torch.zeros(step.cache.shape[0], step.page, dtype=torch.bool, device=DEV)
        for e, (start, new) in enumerate(zip(step.starts, step.new)):
            at = np.arange(start + new)
            held[torch.from_numpy(step.table[step.slots[e], at // step.page].astype(np.int64)).to(DEV), torch.from_numpy(at % step.page).to(DEV)] = True
        step.cache.permute(0, 3, 1, 2, 4)[~held] = float("nan")
        check(step.run(), step.want(), dtype, dim)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("members", [2, 12, 40])
def test_sink_gate_slopes_and_wider_rows(dtype, members, dim):
    step = Step([320], [(0, 1 + 11 * i % 90, 1 + i % 2) for i in range(members)] + [(-1, 40, 1)], heads=12, kv_heads=3, dim=dim, page=16,
                dtype=dtype, seed=members)
    gen = torch.Generator(device=DEV).manual_seed(5)
    tokens = len(step.positions)
    sink = torch.randn((12,), generator=gen, device=DEV) * 3
    sink[1] = -float("inf")
    slopes = torch.rand((12,), generator=gen, device=DEV) * 0.2
    slopes[0] = 0.0
    wide_gate = torch.randn((tokens, 40), generator=gen, device=DEV).to(dtype)
    gate = wide_gate[:, 16:28]
    wide_out = torch.full((tokens, 12 * dim + 32), 7.0, dtype=dtype, device=DEV)
    out = wide_out[:, 16 : 16 + 12 * dim]
    for options in ({"sink": sink}, {"slopes": slopes}, {"gate": gate}, {"sink": sink, "slopes": slopes, "gate": gate}):
        got = step.run(out=out, **options)
        want, size, largest = step.want(**options)
        check(got, (want, size, largest + float(slopes.max()) * 420), dtype, dim)
    assert bool((wide_out[:, :16] == 7.0).all()) and bool((wide_out[:, 16 + 12 * dim :] == 7.0).all())


def test_the_largest_head_and_wide_groups():
    for dtype, dim, heads, kv in ((torch.float32, 256, 4, 2), (torch.float32, 16, 40, 1), (torch.bfloat16, 128, 20, 1), (torch.bfloat16, 128, 150, 1)):
        step = Step([400], [(0, 1 + 3 * i, 1) for i in range(9)], heads=heads, kv_heads=kv, dim=dim, page=16, dtype=dtype, seed=heads)
        check(step.run(), step.want(), dtype, dim)


def test_equals_the_unshared_kernel_on_a_captured_step():
    """The captured call on another stream, replayed with the scratch and the result spoiled in between, new queries each time."""
    step = Step([1024], [(0, 1 + 9 * i, 1) for i in range(20)], heads=16, kv_heads=4, dim=128, page=16, dtype=torch.bfloat16)
    plan = step.device_plan()
    rows = step.planner.part_rows(plan)
    part_out, part_lse = torch.empty((rows, 128), device=DEV), torch.empty((rows,), device=DEV)
    to = lambda values: torch.from_numpy(np.ascontiguousarray(np.asarray(values, dtype=np.int32))).to(DEV)
    out = torch.empty_like(step.q)
    fixed = dict(plan=plan, part_out=part_out, part_lse=part_lse, positions=to(step.positions), cu_seqlens=to(np.arange(21)),
                 entry_start=to(step.starts), entry_slot=to(step.slots), block_table=to(step.table), num_heads=16, num_kv_heads=4,
                 head_dim=128, scale=step.scale, fault=step.fault)
    kernels.attention_shared(step.q, step.cache, out, **fixed)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    previous, kernels.PDL = kernels.PDL, True
    try:
        with torch.cuda.graph(graph, stream=stream):
            for _ in range(3):                     # layers one after the other on the same scratch
                kernels.attention_shared(step.q, step.cache, out, **fixed)
    finally:
        kernels.PDL = previous
    for seed in range(3):
        step.q.copy_(torch.randn(step.q.shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV))
        part_out.fill_(float("nan")), part_lse.fill_(float("nan")), out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        check(out, step.want(), torch.bfloat16, 128)
    assert int(step.fault.item()) == 0


def test_the_same_bits_every_time():
    for dtype, dim in ((torch.float32, 80), (torch.bfloat16, 64), (torch.bfloat16, 128)):
        step = Step([900 // 16 * 16], [(0, 1 + 9 * i, 1) for i in range(40)], heads=16, kv_heads=4, dim=dim, page=16, dtype=dtype)
        first = step.run()
        for _ in range(5):
            assert torch.equal(step.run(), first)


def test_a_page_or_slot_outside_the_pool_is_reported():
    """Indices that the kernels look at before they use them (no access is made through a bad one)."""
    for dtype, dim in ((torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 128)):
        for spoil, word in ((lambda s: s.table.__setitem__((s.slots[0], 2), 10_000), 2), (lambda s: s.table.__setitem__((s.slots[1], 12), -3), 2),
                            (lambda s: s.slots.__setitem__(1, 77), 8)):
            step = Step([160], [(0, 40, 1) for _ in range(8)], heads=8, kv_heads=2, dim=dim, page=16, dtype=dtype)
            step.slots = step.slots.copy()
            spoil(step)
            with pytest.raises(AssertionError):
                step.run()
            assert int(step.fault.item()) & word


def _call(step, **changed):
    plan = step.device_plan()
    rows = step.planner.part_rows(plan)
    to = lambda values: torch.from_numpy(np.ascontiguousarray(np.asarray(values, dtype=np.int32))).to(DEV)
    arguments = dict(q=step.q, cache=step.cache, out=torch.empty_like(step.q), plan=plan, part_out=torch.empty((rows, step.dim), device=DEV),
                     part_lse=torch.empty((rows,), device=DEV), positions=to(step.positions), cu_seqlens=to(np.arange(len(step.new) + 1)),
                     entry_start=to(step.starts), entry_slot=to(step.slots), block_table=to(step.table), num_heads=step.heads,
                     num_kv_heads=step.kv_heads, head_dim=step.dim, scale=step.scale, fault=step.fault)
    arguments.update({k: v(arguments) for k, v in changed.items()})
    return kernels.attention_shared(arguments.pop("q"), arguments.pop("cache"), arguments.pop("out"), **arguments)


REFUSED = [
    dict(q=lambda a: a["q"][:1]), dict(q=lambda a: a["q"].float()), dict(q=lambda a: a["q"].half()), dict(cache=lambda a: a["cache"][:, :1]), dict(cache=lambda a: a["cache"].float()),
    dict(part_out=lambda a: a["part_out"][1:]), dict(part_lse=lambda a: None), dict(part_out=lambda a: a["part_out"].bfloat16()),
    dict(positions=lambda a: a["positions"].long()), dict(positions=lambda a: a["positions"][:2]), dict(entry_slot=lambda a: a["entry_slot"][:2]),
    dict(scale=lambda a: 0.0), dict(scale=lambda a: float("nan")), dict(num_heads=lambda a: 7), dict(head_dim=lambda a: 32),
    dict(out=lambda a: a["out"].float()), dict(sink=lambda a: torch.zeros(3, device=DEV)), dict(gate=lambda a: torch.zeros((3, 2), device=DEV)),
    dict(fault=lambda a: a["fault"].cpu()), dict(plan=lambda a: {**a["plan"], "dtype": 0}), dict(plan=lambda a: {**a["plan"], "tokens": 9}),
    dict(plan=lambda a: {**a["plan"], "members": a["plan"]["members"].cpu()}), dict(block_table=lambda a: a["block_table"].T),
]


@pytest.mark.parametrize("changed", REFUSED, ids=lambda c: next(iter(c)))
def test_refused(changed):
    step = Step([64], [(0, 3, 1), (0, 5, 1), (0, 1, 1)], heads=8, kv_heads=2, dim=64, page=16, dtype=torch.bfloat16)
    with pytest.raises(kernels.KernelError):
        _call(step, **changed)


@pytest.mark.parametrize("own", [129, 500, 1024, 1500])
def test_long_keys_of_their_own_walked_by_one_item(own):
    """Many requests behind a long prefix: an item walks all of a request's own keys, in several blocks, with the ring of one
    tile a multiprocessor shares; and values behind the last key that are NaN."""
    step = Step([16000], [(0, max(1, own - 17 * i % own), 1) for i in range(64)], heads=20, kv_heads=4, dim=128, page=16, dtype=torch.bfloat16, seed=own)
    held = torch.zeros(step.cache.shape[0], step.page, dtype=torch.bool, device=DEV)
    for e, (start, new) in enumerate(zip(step.starts, step.new)):
        at = np.arange(start + new)
        held[torch.from_numpy(step.table[step.slots[e], at // step.page].astype(np.int64)).to(DEV), torch.from_numpy(at % step.page).to(DEV)] = True
    step.cache.permute(0, 3, 1, 2, 4)[~held] = float("nan")
    want = step.want()
    for _ in range(4):
        check(step.run(), want, torch.bfloat16, 128)


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 128)])
def test_a_nan_that_is_seen_stays_one(dtype, dim):
    """In a request's own key: its rows; in a shared one: every row of the group; nowhere else."""
    for members in (3, 40):
        step = Step([160, 48], [(0, 1 + 7 * i % 40, 1) for i in range(members)] + [(1, 3, 1), (-1, 130, 1)], heads=4, kv_heads=2, dim=dim,
                    page=16, dtype=dtype, seed=3)
        clean = step.run()
        own_page = int(step.table[step.slots[1], step.positions[1] // 16])
        step.cache[own_page, 0, 0, step.positions[1] % 16] = float("nan")
        got = step.run().view(-1, 4, dim)
        assert bool(got[1, :2].isnan().all()) and not bool(got[1, 2:].isnan().any())
        got[1] = clean.view(-1, 4, dim)[1]
        assert torch.equal(got.view(clean.shape), clean)
        step.cache[int(step.table[step.slots[0], 4]), 0, 1, 5] = float("nan")
        got = step.run().view(-1, 4, dim)
        assert bool(got[:members, 2:].isnan().all()) and torch.equal(got[members:], clean.view(-1, 4, dim)[members:])


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 128), (torch.bfloat16, 128), (torch.bfloat16, 64)])
def test_pages_beyond_32_bits(dtype, dim):
    """The same rows in pages whose first number lies behind 2^31 numbers and more: the same bits."""
    step = Step([160, 37], [(0, 5 + 30 * i, 1) for i in range(9)] + [(1, 70, 2), (1, 3, 1)], heads=16, kv_heads=8, dim=dim, page=16, dtype=dtype)
    near = step.run()
    held = step.cache.shape[0]
    first = 2**31 // step.cache[0].numel() + 5
    cache = torch.zeros((first + held, *step.cache.shape[1:]), dtype=dtype, device=DEV)
    cache[first:] = step.cache
    step.cache, step.table = cache, np.where(step.table > 0, step.table + first, 0).astype(np.int32)
    assert torch.equal(step.run(), near)


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.bfloat16, 128), (torch.bfloat16, 64)])
def test_calls_side_by_side(dtype, dim):
    """Two steps on two streams, each with scratch and a result of its own."""
    steps = [Step([2048], [(0, 1 + 40 * i, 1) for i in range(n)], heads=16, kv_heads=4, dim=dim, page=16, dtype=dtype, seed=n) for n in (12, 30)]
    want = [step.run() for step in steps]
    to = lambda values: torch.from_numpy(np.ascontiguousarray(np.asarray(values, dtype=np.int32))).to(DEV)
    calls = []
    for step in steps:
        plan = step.device_plan()
        rows = step.planner.part_rows(plan)
        calls.append((step, torch.cuda.Stream(), torch.zeros_like(step.q), dict(
            plan=plan, part_out=torch.empty((rows, dim), device=DEV), part_lse=torch.empty((rows,), device=DEV), positions=to(step.positions),
            cu_seqlens=to(np.arange(len(step.new) + 1)), entry_start=to(step.starts), entry_slot=to(step.slots), block_table=to(step.table),
            num_heads=16, num_kv_heads=4, head_dim=dim, scale=step.scale, fault=step.fault)))
    torch.cuda.synchronize()
    for _ in range(20):
        for step, stream, out, arguments in calls:
            with torch.cuda.stream(stream):
                out.fill_(float("nan"))
                kernels.attention_shared(step.q, step.cache, out, **arguments)
    torch.cuda.synchronize()
    for (step, _, out, _), expected in zip(calls, want):
        assert torch.equal(out, expected) and int(step.fault.item()) == 0


@pytest.mark.parametrize("page", [16, 20])
@pytest.mark.parametrize("dim", [16, 32, 80, 144, 256])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_every_head_size(dtype, dim, page):
    step = Step([400, 90], [(0, 1 + 37 * i, 1) for i in range(7)] + [(1, 250, 2), (1, 3, 1), (-1, 130, 3)], heads=6, kv_heads=2, dim=dim,
                page=page, dtype=dtype, seed=dim)
    check(step.run(), step.want(), dtype, dim)

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

"""Several continuations of one prompt: attention that reads a shared prefix once, copies of cache pages, the choice of tokens.

The calls are those of :mod:`rapid_llm_b200.ops.kernels` (``attention_shared``, ``copy_pages``, ``sample`` with ``top_k``,
``min_p`` and given random numbers), with a step's lists cut by ``SharedItems`` as the engine's planner cuts them.  Beside
each stands its plain form in elementary torch operations and, in :func:`exact`, its definition in 64 bits.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False       # False: the plain forms; True: the framework's kernels

DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}

# -- the cases --------------------------------------------------------------------------------------------------------------
# attention: `groups` groups of `members` requests share `prefix` positions each; every request has up to `own` positions of its
# own, its `tokens` new ones among them.  `ragged` (not 0): lengths, group sizes and the requests' order vary, by that number.
HEADS_8B = {"heads": 32, "kv_heads": 8, "dim": 128}
HEADS_14B = {"heads": 40, "kv_heads": 8, "dim": 128}
VOCAB = 151936


def listed() -> list[dict]:
    return [
        # two continuations of a short prompt have just begun: the smallest step
        {"name": "shared_2x256", "kind": "attention", "dtype": "bf16", **HEADS_8B, "page": 16, "groups": 1, "members": 2,
         "prefix": 256, "own": 9, "tokens": 1, "ragged": 1},
        # eight samples of one prompt of the benchmark's length and more, some hundred tokens in
        {"name": "shared_8x4096", "kind": "attention", "dtype": "bf16", **HEADS_8B, "page": 16, "groups": 1, "members": 8,
         "prefix": 4096, "own": 300, "tokens": 1, "ragged": 2},
        # a full serving batch behind one system prompt, each with a question and an answer under way
        {"name": "shared_64x8192", "kind": "attention", "dtype": "bf16", **HEADS_8B, "page": 16, "groups": 1, "members": 64,
         "prefix": 8192, "own": 512, "tokens": 1, "ragged": 3},
        # several prompts with uneven numbers of samples, lengths that end inside tiles, heads of 64, two new tokens a request
        {"name": "shared_groups", "kind": "attention", "dtype": "bf16", "heads": 24, "kv_heads": 4, "dim": 64, "page": 32,
         "groups": 5, "members": 7, "prefix": 2500, "own": 333, "tokens": 2, "ragged": 4},
        # the 32-bit path: eight samples
        {"name": "shared_32_bit", "kind": "attention", "dtype": "f32", **HEADS_8B, "page": 16, "groups": 1, "members": 8,
         "prefix": 2048, "own": 100, "tokens": 1, "ragged": 5},
        # a document of 32,000 tokens behind which a full batch asks, five heads a key head
        {"name": "shared_64x32000", "kind": "attention", "dtype": "bf16", **HEADS_14B, "page": 16, "groups": 1, "members": 64,
         "prefix": 32000, "own": 1024, "tokens": 1, "ragged": 6},
        # a fork into eight: the ragged last page of a prompt, in every layer of the 8B model
        {"name": "fork_8", "kind": "pages", "dtype": "bf16", "layers": 36, "kv_heads": 8, "dim": 128, "page": 16, "pages": 700,
         "moved": 7},
        # compaction of a cache after a burst of requests has ended
        {"name": "compact_600", "kind": "pages", "dtype": "bf16", "layers": 36, "kv_heads": 8, "dim": 128, "page": 16,
         "pages": 1500, "moved": 600},
        # one request's next token
        {"name": "sample_1", "kind": "sample", "dtype": "bf16", "rows": 1, "vocab": VOCAB, "top_k": 50, "top_p": 0.9, "min_p": 0.0,
         "temperature": 0.6, "spread": 2.5, "mixed": 0},
        # a full batch whose requests disagree about everything, greedy ones and unfiltered ones among them
        {"name": "sample_64_mixed", "kind": "sample", "dtype": "bf16", "rows": 64, "vocab": VOCAB, "top_k": 200, "top_p": 0.95,
         "min_p": 0.02, "temperature": 0.9, "spread": 2.5, "mixed": 7},
        # the 32-bit path, a hot and flat distribution: nearly the whole vocabulary stays in
        {"name": "sample_32_flat", "kind": "sample", "dtype": "f32", "rows": 32, "vocab": VOCAB, "top_k": 0, "top_p": 0.98,
         "min_p": 0.0, "temperature": 1.3, "spread": 1.0, "mixed": 0},
        # many rows of a small vocabulary
        {"name": "sample_256_small", "kind": "sample", "dtype": "bf16", "rows": 256, "vocab": 32003, "top_k": 40, "top_p": 1.0,
         "min_p": 0.05, "temperature": 0.8, "spread": 2.0, "mixed": 0},
    ]


def _spread(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    kind = rng.choice(("attention", "attention", "attention", "pages", "sample", "sample"))
    if kind == "attention":
        dtype = rng.choice(("bf16", "bf16", "bf16", "f32"))
        kv_heads = rng.choice((1, 2, 4, 8))
        case = {"kind": kind, "dtype": dtype, "heads": kv_heads * rng.randint(1, 8), "kv_heads": kv_heads,
                "dim": rng.choice((64, 128, 128)) if dtype == "bf16" else rng.choice((16, 64, 80, 128, 256)),
                "page": rng.choice((8, 16, 16, 32, 64, 20)), "groups": rng.choice((1, 1, 1, 2, 3, rng.randint(4, 9))),
                "members": _spread(rng, 1, 64), "prefix": _spread(rng, 1, 32000), "own": _spread(rng, 4, 1024),
                "tokens": rng.choice((1, 1, 1, rng.randint(2, 4))), "ragged": rng.randint(1, 1 << 20)}
        while case["groups"] * case["members"] > 64:
            case["members"] = max(1, case["members"] // 2)
        while dtype == "f32" and case["prefix"] * case["members"] * case["groups"] > 1 << 16:
            case["prefix"] = max(1, case["prefix"] // 2)
        return case
    if kind == "pages":
        pages = _spread(rng, 16, 1500)
        return {"kind": kind, "dtype": rng.choice(("bf16", "f32")), "layers": _spread(rng, 1, 36), "kv_heads": rng.choice((1, 2, 8)),
                "dim": rng.choice((64, 80, 128)), "page": rng.choice((8, 16, 16, 20)), "pages": pages, "moved": _spread(rng, 1, max(1, pages // 3))}
    vocab = _spread(rng, 50, VOCAB)
    return {"kind": kind, "dtype": rng.choice(("bf16", "bf16", "f32")), "rows": _spread(rng, 1, 64), "vocab": vocab,
            "top_k": rng.choice((0, 1, _spread(rng, 1, vocab))), "top_p": rng.choice((1.0, round(rng.uniform(0.05, 0.999), 3))),
            "min_p": rng.choice((0.0, round(math.exp(rng.uniform(math.log(1e-4), math.log(0.5))), 5))),
            "temperature": round(math.exp(rng.uniform(math.log(0.2), math.log(2.0))), 3), "spread": round(rng.uniform(0.5, 4.0), 2),
            "mixed": rng.choice((0, rng.randint(1, 1 << 20)))}


def _layout(case):
    """Per group its shared positions; per request (in the step's order) its group and its own positions."""
    rng = random.Random(case["ragged"])
    groups, requests = [], []
    for index in range(case["groups"]):
        whole = max(1, case["prefix"] // case["page"])
        pages = whole if index == 0 or not case["ragged"] else max(1, int(whole * rng.uniform(0.3, 1.0)))
        groups.append(pages * case["page"])
        members = case["members"] if index == 0 or not case["ragged"] else rng.randint(1, case["members"])
        longest = max(case["own"], case["tokens"])
        for member in range(members):
            ragged = case["ragged"] and (index or member)
            requests.append((index, rng.randint(case["tokens"], longest) if ragged else longest))
    if case["ragged"]:
        rng.shuffle(requests)
    return groups, requests


def _generator(seed: int, salt: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed * 1000 + salt)


def _on_device(values) -> torch.Tensor:
    return torch.as_tensor(np.asarray(values, dtype=np.int32)).to(DEV)


# -- inputs -----------------------------------------------------------------------------------------------------------------
def _prepare_attention(case, seed):
    groups, requests = _layout(case)
    page, tokens, dtype = case["page"], case["tokens"], TYPES[case["dtype"]]
    needed = sum(g // page for g in groups) + sum(-(-length // page) for _, length in requests)
    ids = np.random.RandomState(seed % (1 << 32)).permutation(needed) + 1          # pages lie anywhere; 0 is the null page
    at, group_pages = 0, []
    for length in groups:
        group_pages.append(ids[at : at + length // page])
        at += length // page
    lengths = [groups[g] + length for g, length in requests]
    table = np.zeros((len(requests) + 1, -(-max(lengths) // page)), dtype=np.int32)
    own_pages = np.zeros((len(requests), -(-max(length for _, length in requests) // page)), dtype=np.int64)
    for slot, (g, length) in enumerate(requests):
        count = -(-length // page)
        mine = ids[at : at + count]
        at += count
        table[slot, : len(group_pages[g])] = group_pages[g]
        table[slot, len(group_pages[g]) : len(group_pages[g]) + count] = mine
        own_pages[slot, :count] = mine
    starts = [length - tokens for length in lengths]
    positions = np.concatenate([np.arange(s, s + tokens) for s in starts])
    gen = _generator(seed, 1)
    # queries and keys of size one as behind a norm; scores have a spread of two
    q = torch.randn((len(positions), case["heads"] * case["dim"]), generator=gen, device=DEV).mul_(2.0).to(dtype)
    cache = torch.empty((needed + 1, 2, case["kv_heads"], page, case["dim"]), dtype=dtype, device=DEV)
    for first in range(0, needed + 1, 4096):          # in slices: the 32-bit numbers of a long cache are not all held at once
        part = cache[first : first + 4096]
        part.copy_(torch.randn(part.shape, generator=gen, device=DEV))
    state = {"case": case, "q": q, "cache": cache, "out": torch.empty_like(q), "positions": _on_device(positions),
             "scale": case["dim"] ** -0.5, "table": _on_device(table), "slots": _on_device(range(len(requests))),
             "starts": _on_device(starts), "fault": torch.zeros(1, dtype=torch.int32, device=DEV)}
    # for the plain form: the groups' pages and their tokens as padded matrices
    prefix_pages = np.zeros((len(groups), max(len(p) for p in group_pages)), dtype=np.int64)
    for g, pages in enumerate(group_pages):
        prefix_pages[g, : len(pages)] = pages
    group_of = np.repeat([g for g, _ in requests], tokens)
    place, seen = np.zeros(len(group_of), dtype=np.int64), {}
    for t, g in enumerate(group_of):
        place[t] = seen.setdefault(int(g), 0)
        seen[int(g)] += 1
    members = np.zeros((len(groups), max(seen.values())), dtype=np.int64)
    members[group_of, place] = np.arange(len(group_of))
    state["plain"] = {name: torch.as_tensor(np.asarray(value, dtype=np.int64)).to(DEV) for name, value in (
        ("prefix_pages", prefix_pages), ("own_pages", own_pages), ("group_of", group_of), ("place", place), ("members", members),
        ("prefix", groups), ("entry_of", np.repeat(np.arange(len(requests)), tokens)))}
    if own:
        from rapid_llm_b200.parts.attention import SharedItems
        from rapid_llm_b200.parts.base import StepShape

        # the step's lists, cut on the host and uploaded with its metadata, once for all layers
        planner = SharedItems(case["heads"] // case["kv_heads"], case["kv_heads"], case["dim"], dtype=dtype)
        plan = planner.plan(StepShape(
            lengths=np.full(len(requests), tokens, dtype=np.int32), starts=np.asarray(starts, dtype=np.int32),
            decode_only=tokens == 1, page_size=page, prefix_group=np.asarray([g for g, _ in requests], dtype=np.int32),
            prefix_tokens=np.asarray([groups[g] for g, _ in requests], dtype=np.int32)))
        state["plan"] = {name: _on_device(value) if isinstance(value, np.ndarray) else value for name, value in plan.items()}
        state["cu_seqlens"] = _on_device(np.arange(len(requests) + 1) * tokens)
        rows = planner.part_rows(plan)
        state["part_out"] = torch.empty((rows, case["dim"]), dtype=torch.float32, device=DEV)
        state["part_lse"] = torch.empty((rows,), dtype=torch.float32, device=DEV)
    return state


def _prepare_pages(case, seed):
    dtype = TYPES[case["dtype"]]
    gen = _generator(seed, 2)
    pages = torch.empty((case["layers"], case["pages"] + 1, 2, case["kv_heads"], case["page"], case["dim"]), dtype=dtype, device=DEV)
    for layer in range(case["layers"]):
        pages[layer].copy_(torch.randn(pages.shape[1:], generator=gen, device=DEV))
    ids = np.random.RandomState(seed % (1 << 32)).permutation(case["pages"]) + 1
    moved = min(case["moved"], case["pages"] // 2)
    pairs = np.stack([ids[:moved], ids[moved : 2 * moved]], axis=1).astype(np.int32)
    if case["moved"] <= 8:
        pairs[:, 0] = pairs[0, 0]        # a fork: every new request gets a copy of the same page
    return {"case": case, "pages": pages, "pairs": pairs, "source": torch.as_tensor(pairs[:, 0].astype(np.int64)).to(DEV),
            "target": torch.as_tensor(pairs[:, 1].astype(np.int64)).to(DEV)}


def _prepare_sample(case, seed):
    rows, vocab = case["rows"], case["vocab"]
    gen = _generator(seed, 3)
    logits = torch.randn((rows, vocab), generator=gen, device=DEV).mul_(case["spread"])
    logits[:, torch.randint(0, vocab, (3,), generator=gen, device=DEV)] += 3.0 * case["spread"]      # what the model is sure of
    logits[:, vocab - vocab // 500 :] = -math.inf                                                    # entries no token has
    logits = logits.to(TYPES[case["dtype"]])
    params = {"temperature": [case["temperature"]] * rows, "top_k": [case["top_k"]] * rows, "top_p": [case["top_p"]] * rows,
              "min_p": [case["min_p"]] * rows}
    if case["mixed"]:
        rng = random.Random(case["mixed"])
        for row in range(rows):
            params["temperature"][row] = rng.choice((0.0, case["temperature"], case["temperature"], 1.0))
            params["top_k"][row] = rng.choice((0, case["top_k"], 1 + case["top_k"] // 7))
            params["top_p"][row] = rng.choice((1.0, case["top_p"], 0.5))
            params["min_p"][row] = rng.choice((0.0, 0.0, case["min_p"]))
    state = {name: torch.tensor(value, dtype=torch.int32 if name == "top_k" else torch.float32, device=DEV)
             for name, value in params.items()}
    uniforms = torch.rand((rows,), generator=gen, device=DEV)
    return {"case": case, "logits": logits, "uniforms": uniforms, "out": torch.empty((rows,), dtype=torch.int32, device=DEV), **state}


def prepare(case: dict, seed: int):
    return {"attention": _prepare_attention, "pages": _prepare_pages, "sample": _prepare_sample}[case["kind"]](case, seed)


# -- one pass ---------------------------------------------------------------------------------------------------------------
def _plain_attention(s):
    case, plain = s["case"], s["plain"]
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    group_of, place, entry_of = plain["group_of"], plain["place"], plain["entry_of"]
    q = s["q"].float().view(-1, kv_heads, heads // kv_heads, dim) * s["scale"]

    def rows(pages, plane):               # [n, pages, kv heads, page, dim] -> [n, kv heads, keys, dim]
        return s["cache"][pages, plane].float().permute(0, 2, 1, 3, 4).flatten(2, 3)

    prefix_len = plain["prefix"][group_of]
    keys = torch.arange(plain["prefix_pages"].shape[1] * page, device=DEV)
    prefix_scores = torch.einsum("gmkhd,gkjd->gmkhj", q[plain["members"]], rows(plain["prefix_pages"], 0))[group_of, place]
    prefix_scores = prefix_scores.masked_fill((keys >= prefix_len[:, None])[:, None, None], -math.inf)
    own_keys = torch.arange(plain["own_pages"].shape[1] * page, device=DEV)
    own_scores = torch.einsum("tkhd,tkjd->tkhj", q, rows(plain["own_pages"], 0)[entry_of])
    hidden = prefix_len[:, None] + own_keys > s["positions"][:, None]
    own_scores = own_scores.masked_fill(hidden[:, None, None], -math.inf)
    weights = torch.cat([prefix_scores, own_scores], -1)
    weights = torch.exp(weights - weights.amax(-1, keepdim=True))
    weights = weights / weights.sum(-1, keepdim=True)
    by_group = torch.zeros((*plain["members"].shape, *weights.shape[1:3], len(keys)), device=DEV)
    by_group[group_of, place] = weights[..., : len(keys)]
    out = torch.einsum("gmkhj,gkjd->gmkhd", by_group, rows(plain["prefix_pages"], 1))[group_of, place]
    out = out + torch.einsum("tkhj,tkjd->tkhd", weights[..., len(keys) :], rows(plain["own_pages"], 1)[entry_of])
    return out.reshape(out.shape[0], -1).to(s["q"].dtype)


def _plain_sample(s):
    x = s["logits"].double()
    vocab = x.shape[1]
    places = torch.arange(vocab, device=DEV)
    top = x.amax(-1, keepdim=True)
    greedy = torch.where(x == top, places, vocab).amin(-1)
    temperature = s["temperature"].double()[:, None]
    ranked, order = torch.sort(x, dim=-1, descending=True, stable=True)
    weight = torch.exp((ranked - top) / torch.where(temperature > 0, temperature, 1.0))
    top_k = torch.where(s["top_k"] > 0, s["top_k"], vocab)[:, None]
    weight = torch.where(places < top_k, weight, 0.0)
    running = torch.cumsum(weight, -1)
    begins = torch.ones_like(ranked, dtype=torch.bool)
    begins[:, 1:] = ranked[:, 1:] != ranked[:, :-1]
    first_equal = torch.cummax(torch.where(begins, places, 0), -1).values
    above = (running - weight).gather(-1, first_equal)          # the mass that lies strictly above
    kept = (above <= s["top_p"].double()[:, None] * running[:, -1:]) | (s["top_p"][:, None] >= 1)
    kept = kept & (weight >= s["min_p"].double()[:, None].clamp(max=1.0))
    by_place = torch.zeros_like(weight).scatter_(-1, order, torch.where(kept, weight, 0.0))
    running = torch.cumsum(by_place, -1)
    target = s["uniforms"].double()[:, None] * running[:, -1:]
    drawn = (running <= target).sum(-1).clamp(max=vocab - 1)
    return torch.where(s["temperature"] > 0, drawn, greedy).to(torch.int32)


def run(state):
    kind = state["case"]["kind"]
    if own:
        from rapid_llm_b200.ops import kernels

        if kind == "attention":
            case = state["case"]
            return kernels.attention_shared(
                state["q"], state["cache"], state["out"], plan=state["plan"], part_out=state["part_out"], part_lse=state["part_lse"],
                positions=state["positions"], cu_seqlens=state["cu_seqlens"], entry_start=state["starts"], entry_slot=state["slots"],
                block_table=state["table"], num_heads=case["heads"], num_kv_heads=case["kv_heads"], head_dim=case["dim"],
                scale=state["scale"], fault=state["fault"])
        if kind == "pages":
            return kernels.copy_pages(state["pages"], state["pairs"])
        return kernels.sample(state["logits"], state["out"], temperature=state["temperature"], top_k=state["top_k"],
                              top_p=state["top_p"], min_p=state["min_p"], uniforms=state["uniforms"])
    if kind == "attention":
        return _plain_attention(state)
    if kind == "pages":
        state["pages"][:, state["target"]] = state["pages"][:, state["source"]]
        return state["pages"]
    return _plain_sample(state)


def work(case: dict) -> dict:
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "attention":
        groups, requests = _layout(case)
        cached = sum(groups) + sum(length for _, length in requests)
        rows = len(requests) * case["tokens"] * case["heads"]
        keys = sum(case["tokens"] * (groups[g] + length) - case["tokens"] * (case["tokens"] - 1) // 2 for g, length in requests)
        return {"bytes": size * case["dim"] * (2 * cached * case["kv_heads"] + 2 * rows), "flops": 4 * case["dim"] * case["heads"] * keys}
    if case["kind"] == "pages":
        one = 2 * case["kv_heads"] * case["page"] * case["dim"] * size
        moved = min(case["moved"], case["pages"] // 2)
        return {"bytes": case["layers"] * one * ((1 if case["moved"] <= 8 else moved) + moved), "flops": 0}
    return {"bytes": case["rows"] * (case["vocab"] * size + 24), "flops": 4 * case["rows"] * case["vocab"]}


# -- the definitions in 64 bits ---------------------------------------------------------------------------------------------
def _exact_attention(s):
    """Request by request over its own block table, as if nothing were shared."""
    case = s["case"]
    group, dim, page, tokens = case["heads"] // case["kv_heads"], case["dim"], case["page"], case["tokens"]
    out = torch.empty((s["q"].shape[0], case["heads"], dim), dtype=torch.float64, device=DEV)
    q = s["q"].double().view(-1, case["heads"], dim)
    positions, table = s["positions"].tolist(), s["table"].long()
    for t, position in enumerate(positions):
        used = table[t // tokens, : position // page + 1]
        for head in range(case["kv_heads"]):
            k = s["cache"][used, 0, head].reshape(-1, dim)[: position + 1].double()
            v = s["cache"][used, 1, head].reshape(-1, dim)[: position + 1].double()
            mine = slice(head * group, (head + 1) * group)
            out[t, mine] = torch.softmax(q[t, mine] @ k.T * s["scale"], -1) @ v
    return out.view(s["q"].shape)


def _exact_sample(s):
    """Row by row: the definition over a sorted list, in numpy."""
    ids = []
    rows = s["logits"].double().cpu().numpy()
    params = {name: s[name].cpu().numpy() for name in ("temperature", "top_k", "top_p", "min_p", "uniforms")}
    for row, x in enumerate(rows):
        top = int(np.argmax(x))                                   # the first of equal ones
        if params["temperature"][row] <= 0:
            ids.append(top)
            continue
        weight = np.exp((x - x[top]) / float(params["temperature"][row]))
        order = np.lexsort((np.arange(len(x)), -x))
        count = int(params["top_k"][row])
        chosen = order[: count] if count > 0 else order
        mass, kept, above = math.fsum(weight[chosen]), [], 0.0
        runs = np.split(chosen, np.flatnonzero(np.diff(x[chosen])) + 1)
        for equal in runs:
            if params["top_p"][row] < 1 and above > float(params["top_p"][row]) * mass:
                break
            if weight[equal[0]] < min(float(params["min_p"][row]), 1.0):
                break
            kept.append(equal)
            above += float(weight[equal[0]]) * len(equal)
        kept = np.sort(np.concatenate(kept))
        running = np.cumsum(weight[kept])
        ids.append(int(kept[min(np.searchsorted(running, float(params["uniforms"][row]) * running[-1], side="right"), len(kept) - 1)]))
    return torch.tensor(ids, dtype=torch.int32)


def exact(case: dict, seed: int):
    if case["kind"] == "attention":
        return _exact_attention(prepare(case, seed))
    if case["kind"] == "sample":
        return _exact_sample(prepare(case, seed))
    return None                       # copies have no rounding

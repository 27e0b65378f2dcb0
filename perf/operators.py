"""Cases that say how fast the operators of beam search are: attention of tokens whose requests
share a long prefix (the beams of a prompt, requests behind one system prompt), the choice of the
next beams over beams and vocabulary, and the beams' caches put in their new order.

``listed`` are the cases by name, ``draw`` gives another one of the same ranges.  ``prepare`` makes
what a program has in hand before the call, ``run`` is one call: in plain torch operations, or,
where ``own`` is true, of this framework's operators.  Head layouts are those of the benchmark's
Llama shapes (TinyLlama-1.1B, Llama-2-7B, Llama-3-8B).
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
# query heads, key/value heads, head size
HEADS = {"tinyllama": (32, 4, 64), "llama2_7b": (32, 32, 128), "llama3_8b": (32, 8, 128)}
# the rows that a beam search moves, as [layers, rows, width]: a layer's row of one request
ROWS = {"delta": (6, 16 * 128 * 128, "f32"),           # states of gated delta rule layers
        "recurrence": (8, 2048, "f32"),                # states of a gated linear recurrence
        "conv": (6, 3 * 6144 + 1, "f32"),              # rows behind a convolution, of odd width
        "pages_7b": (32, 32 * 16 * 128, "bf16"),       # a page of keys, Llama-2-7B shape
        "pages_tiny": (22, 4 * 16 * 64, "bf16")}       # the same, TinyLlama-1.1B shape


def listed() -> list[dict]:
    return [
        # the smallest: four beams of one prompt decode a token each
        {"name": "shared_four_beams", "kind": "shared", "dtype": "bf16", "shape": "tinyllama",
         "groups": 1, "members": 4, "tokens": 1, "prefix": 512, "tail": 20, "page": 16},
        # sixteen prompts of uneven lengths, four beams each, every query head with keys of its own
        {"name": "shared_many_prompts", "kind": "shared", "dtype": "bf16", "shape": "llama2_7b",
         "groups": 16, "members": 4, "tokens": 1, "prefix": 1003, "tail": 70, "page": 16},
        # sixty-four requests behind one long system prompt, each with a conversation of its own
        {"name": "shared_system_prompt", "kind": "shared", "dtype": "bf16", "shape": "llama3_8b",
         "groups": 1, "members": 64, "tokens": 1, "prefix": 8192, "tail": 500, "page": 16},
        # the largest: 128 answers drawn to one very long document
        {"name": "shared_long_document", "kind": "shared", "dtype": "bf16", "shape": "llama3_8b",
         "groups": 1, "members": 128, "tokens": 1, "prefix": 65003, "tail": 300, "page": 64},
        # questions of a few tokens each, put to one document
        {"name": "shared_questions", "kind": "shared", "dtype": "bf16", "shape": "tinyllama",
         "groups": 2, "members": 9, "tokens": 21, "prefix": 4100, "tail": 0, "page": 32},
        # eight beams in the 32-bit mode
        {"name": "shared_eight_beams_f32", "kind": "shared", "dtype": "f32",
         "shape": "tinyllama", "groups": 1, "members": 8, "tokens": 1, "prefix": 2001,
         "tail": 40, "page": 16},
        # the next four beams of one prompt, with as many again for beams that end
        {"name": "select_four_beams", "kind": "select", "groups": 1, "beams": 4,
         "vocabulary": 32000, "take": 8, "allowed": 1.0, "first": False},
        # five beams of each of seven prompts, an odd vocabulary of which a grammar allows a part
        {"name": "select_masked", "kind": "select", "groups": 7, "beams": 5,
         "vocabulary": 50021, "take": 10, "allowed": 0.3, "first": False},
        # the largest: eight beams of 64 prompts over a large vocabulary
        {"name": "select_large", "kind": "select", "groups": 64, "beams": 8,
         "vocabulary": 128256, "take": 16, "allowed": 1.0, "first": False},
        # four beams' small recurrent states: latency
        {"name": "reorder_small_states", "kind": "reorder", "rows": "recurrence", "groups": 1,
         "beams": 4, "pool": 64},
        # the last pages of four beams of each of sixteen prompts
        {"name": "reorder_pages", "kind": "reorder", "rows": "pages_7b", "groups": 16, "beams": 4,
         "pool": 200},
        # eight beams' states of 64 requests, a megabyte a layer each
        {"name": "reorder_large_states", "kind": "reorder", "rows": "delta", "groups": 8,
         "beams": 8, "pool": 96},
    ]


def _log(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["shared", "shared", "shared", "select", "reorder"])
    if kind == "select":
        beams, groups = _log(rng, 1, 16), _log(rng, 1, 64)
        while groups * beams > 512:
            groups = max(1, groups // 2)
        return {"kind": kind, "groups": groups, "beams": beams,
                "vocabulary": _log(rng, 1000, 128256), "take": beams * rng.choice([1, 2]),
                "allowed": rng.choice([1.0, 1.0, 0.1]), "first": rng.random() < 0.2}
    if kind == "reorder":
        rows = rng.choice(sorted(ROWS))
        groups, beams = _log(rng, 1, 16), _log(rng, 2, 16)
        while groups * beams > 64:
            groups = max(1, groups // 2)
        return {"kind": kind, "rows": rows, "groups": groups, "beams": beams,
                "pool": groups * beams + rng.randint(0, 32)}
    dtype = rng.choice(["bf16", "bf16", "f32"])
    wide = dtype == "f32"
    groups, members = _log(rng, 1, 16), _log(rng, 2, 16 if wide else 128)
    while groups * members > (32 if wide else 128):
        groups = max(1, groups // 2)
    tokens = rng.choice([1, 1, 1, _log(rng, 2, 24)])
    if groups * members * tokens > 256:
        tokens = 1
    prefix = _log(rng, 100, (8000 if wide else 32000) // groups)
    return {"kind": kind, "dtype": dtype, "shape": rng.choice(sorted(HEADS)), "groups": groups,
            "members": members, "tokens": tokens, "prefix": prefix,
            "tail": rng.choice([0, _log(rng, 1, 400)]), "page": rng.choice([16, 16, 32, 64])}


# ----------------------------------------------------------------------------- inputs
def _generator(seed: int) -> torch.Generator:
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(1000003 * int(seed) + 29)
    return gen


def _lengths(case) -> "tuple[list[int], list[int]]":
    """Keys that the members of each group share, and keys that each member has of its own before
    this step's tokens; ragged."""
    prefix = [case["prefix"] - (g * 37) % (case["prefix"] // 4 + 1) for g in range(case["groups"])]
    tail = [case["tail"] - (s * 29) % (case["tail"] // 2 + 1)
            for s in range(case["groups"] * case["members"])]
    return prefix, tail


def _shared_inputs(case, seed):
    """q [tokens, heads * d] in rows that also hold k and v, the pages, and every request's pages
    in order (a group's first pages are the same ones; where the shared keys end inside a page,
    each request has that page for itself, with the shared keys in it)."""
    heads, kv_heads, dim = HEADS[case["shape"]]
    dtype, page, members, new = DTYPES[case["dtype"]], case["page"], case["members"], case["tokens"]
    prefix, tail = _lengths(case)
    gen = _generator(seed)
    width = (heads + 2 * kv_heads) * dim
    qkv = torch.randn(len(tail) * new, width, generator=gen, device=DEVICE).to(dtype)
    tables, used = [], 0
    for g, p in enumerate(prefix):
        common = list(range(used, used + p // page))
        used += len(common)
        for s in range(g * members, (g + 1) * members):
            more = -(-(p + tail[s] + new) // page) - len(common)
            tables.append(common + list(range(used, used + more)))
            used += more
    order = torch.randperm(used, generator=gen, device=DEVICE)
    longest = max(len(t) for t in tables)
    table = torch.tensor([t + [-1] * (longest - len(t)) for t in tables], device=DEVICE)
    table = torch.where(table < 0, table, order[table.clamp_min(0)])
    k, v = (torch.randn(used, kv_heads, page, dim, generator=gen, device=DEVICE).to(dtype)
            for _ in range(2))
    ragged = [g for g, p in enumerate(prefix) if p % page]
    if ragged:                      # the page in which the shared keys end: the same keys in each
        first = torch.tensor([g * members for g in ragged], device=DEVICE)
        at = torch.tensor([prefix[g] // page for g in ragged], device=DEVICE)
        keep = torch.tensor([prefix[g] % page for g in ragged], device=DEVICE)
        mask = (torch.arange(page, device=DEVICE)[None] < keep[:, None])[:, None, :, None]
        source = table[first, at]
        for m in range(1, members):
            copy = table[first + m, at]
            for pages in (k, v):
                pages[copy] = torch.where(mask, pages[source], pages[copy])
    return qkv, k, v, table, prefix, tail


def _select_inputs(case, seed):
    gen = _generator(seed)
    groups, beams, vocabulary = case["groups"], case["beams"], case["vocabulary"]
    logits = torch.randn(groups * beams, vocabulary, generator=gen, device=DEVICE) * 2.5
    if case["allowed"] < 1.0:
        drop = torch.rand(groups * beams, vocabulary, generator=gen, device=DEVICE)
        logits.masked_fill_(drop >= case["allowed"], -math.inf)
    scores = -12.0 + torch.randn(groups, beams, generator=gen, device=DEVICE)
    scores = scores.sort(dim=1, descending=True).values.contiguous()
    if case["first"]:                       # behind the prompt only one beam counts
        scores[:, 1:] = -math.inf
        scores[:, 0] = 0.0
    return logits, scores


def _moves(case) -> "tuple[list[list[int]], list[list[int]]]":
    """Row of every beam in the pool, and the beam of its group whose row it takes: a few beams
    have the most children, as after a choice over all of them."""
    rng = random.Random(case["groups"] * 1009 + case["beams"] * 31 + case["pool"])
    rows = rng.sample(range(case["pool"]), case["groups"] * case["beams"])
    beams = case["beams"]
    parents = [[min(beams - 1, int(beams * rng.random() ** 1.7)) for _ in range(beams)]
               for _ in range(case["groups"])]
    return [rows[g * beams: (g + 1) * beams] for g in range(case["groups"])], parents


def _reorder_inputs(case, seed):
    layers, width, dtype = ROWS[case["rows"]]
    state = torch.randn(layers, case["pool"], width, generator=_generator(seed),
                        device=DEVICE).to(DTYPES[dtype])
    slots, parents = _moves(case)
    return state, torch.tensor(slots, dtype=torch.int32, device=DEVICE), torch.tensor(
        parents, dtype=torch.int32, device=DEVICE)


def prepare(case, seed) -> dict:
    state = {"case": case}
    if case["kind"] == "select":
        state["logits"], state["scores"] = _select_inputs(case, seed)
        return state
    if case["kind"] == "reorder":
        state["rows"], state["slots"], state["parents"] = _reorder_inputs(case, seed)
        return state
    heads, kv_heads, dim = HEADS[case["shape"]]
    qkv, state["k"], state["v"], table, prefix, tail = _shared_inputs(case, seed)
    groups, members, new = case["groups"], case["members"], case["tokens"]
    before = [prefix[s // members] + tail[s] for s in range(groups * members)]
    state.update(
        q=qkv[:, : heads * dim], scale=dim ** -0.5, table=table.int(),
        slots=torch.arange(len(tail), dtype=torch.int32, device=DEVICE),
        positions=torch.tensor(before, dtype=torch.int32, device=DEVICE),
        prefix=torch.tensor(prefix, device=DEVICE), tail=torch.tensor(tail, device=DEVICE),
        most_shared=max(prefix), most_own=max(tail) + new)
    if own:
        from distengine_b200.kernels.shared_prefix import SharedPrefixAttention
        layer = SharedPrefixAttention(DTYPES[case["dtype"]], heads, kv_heads, dim, dim ** -0.5,
                                      torch.device(DEVICE))
        state["layer"] = layer
        # which tokens belong together: kept from step to step, until a request ends
        state["plan"] = layer.plan([new] * len(tail), [members] * groups, prefix,
                                   tail=max(tail) + new)
    return state


# ----------------------------------------------------------------------------- one pass
def _gathered(pages, table, at, mask):
    """Keys or values at the positions ``at`` [rows, n] of the requests with the page tables
    ``table`` [rows, pages], as float32 [rows, n, kv heads, d]; zero where ``mask`` is false."""
    page = pages.shape[2]
    ids = table.gather(1, (at // page).clamp_max(table.shape[1] - 1)).clamp_min(0).long()
    rows = pages.transpose(1, 2)[ids, at % page]
    return rows.float().masked_fill_(~mask[:, :, None, None], 0.0)


def _shared_plain(s):
    case = s["case"]
    heads, kv_heads, dim = HEADS[case["shape"]]
    G, M, T = case["groups"], case["members"], case["tokens"]
    q = s["q"].float().view(G, M, T, kv_heads, heads // kv_heads, dim)
    table = s["table"].long()
    # the shared keys, once a group
    at = torch.arange(s["most_shared"], device=DEVICE).expand(G, -1)
    seen = at < s["prefix"][:, None]
    first = table[:: M]
    k, v = (_gathered(s[n], first, at, seen) for n in "kv")
    score = torch.einsum("gmthrd,gphd->gmthrp", q, k) * s["scale"]
    score.masked_fill_(~seen[:, None, None, None, None, :], -math.inf)
    # every request's own keys, up to the token's own
    own_at = torch.arange(s["most_own"], device=DEVICE)
    start = s["prefix"].repeat_interleave(M)
    mask = own_at[None] < (s["tail"] + T)[:, None]
    k_own, v_own = (_gathered(s[n], table, start[:, None] + own_at[None], mask) for n in "kv")
    q_own = q.view(G * M, T, kv_heads, heads // kv_heads, dim)
    score_own = torch.einsum("sthrd,sphd->sthrp", q_own, k_own) * s["scale"]
    last = s["tail"][:, None] + torch.arange(T, device=DEVICE)[None]
    hidden = own_at[None, None] > last[:, :, None]
    score_own.masked_fill_(hidden[:, :, None, None, :], -math.inf)
    score_own = score_own.view(G, M, T, kv_heads, heads // kv_heads, -1)
    top = torch.maximum(score.amax(-1, keepdim=True), score_own.amax(-1, keepdim=True))
    weight = score.sub_(top).exp_()
    weight_own = score_own.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True) + weight_own.sum(-1, keepdim=True)
    out = torch.einsum("gmthrp,gphd->gmthrd", weight, v)
    weight_own = weight_own.view(G * M, T, kv_heads, heads // kv_heads, -1)
    out = out + torch.einsum("sthrp,sphd->sthrd", weight_own, v_own).reshape(out.shape)
    return (out / total).reshape(G * M * T, heads * dim).to(s["q"].dtype)


def _select_plain(s):
    """[scores, beams, tokens] of the best candidates of each group, best first; of equal ones the
    lower beam, then the lower token; where fewer are left, -1 and a score of minus infinity."""
    G, B, V = s["case"]["groups"], s["case"]["beams"], s["case"]["vocabulary"]
    # in 64 bits: which of two nearly equal candidates comes first is part of the answer
    x = s["logits"].double()
    top = x.amax(1, keepdim=True)
    total = s["scores"].double().view(-1, 1) + (x - (top + (x - top).exp().sum(1, keepdim=True).log()))
    total = torch.where(total.isnan(), -math.inf, total).view(G, B * V)
    best, index = total.sort(dim=1, descending=True, stable=True)
    best, index = best[:, : s["case"]["take"]], index[:, : s["case"]["take"]]
    there = best > -math.inf
    return [best.float(), torch.where(there, index // V, -1).int(),
            torch.where(there, index % V, -1).int()]


def _reorder_plain(s):
    from_rows = s["slots"].gather(1, s["parents"].long()).view(-1).long()
    s["rows"][:, s["slots"].view(-1).long()] = s["rows"][:, from_rows]
    return s["rows"]


def run(s):
    case = s["case"]
    if not own:
        return {"shared": _shared_plain, "select": _select_plain,
                "reorder": _reorder_plain}[case["kind"]](s)
    from distengine_b200.kernels import ops
    if case["kind"] == "reorder":
        ops.beam_reorder(s["rows"], s["slots"], s["parents"])
        return s["rows"]
    if case["kind"] == "select":
        shape = (case["groups"], case["take"])
        best = torch.empty(shape, device=DEVICE)
        beam, token = (torch.empty(shape, dtype=torch.int32, device=DEVICE) for _ in range(2))
        ops.beam_select(s["logits"], s["scores"], best, beam, token)
        return [best, beam, token]
    out = torch.empty(s["q"].shape, dtype=s["q"].dtype, device=DEVICE)
    s["layer"].run(s["q"], out, s["k"], s["v"], s["table"], s["slots"], s["positions"], s["plan"])
    return out


def work(case) -> dict:
    if case["kind"] == "select":
        n = case["groups"] * case["beams"] * case["vocabulary"]
        # a logit is read once, and enters a maximum, an exponential and a sum
        return {"bytes": 4 * n + 12 * case["groups"] * case["take"], "flops": 4 * n}
    if case["kind"] == "reorder":
        layers, width, dtype = ROWS[case["rows"]]
        size = width * (4 if dtype == "f32" else 2) * layers
        _, parents = _moves(case)
        moved = [[p for b, p in enumerate(ps) if p != b] for ps in parents]
        return {"bytes": size * sum(len(set(ps)) + len(ps) for ps in moved), "flops": 0}
    heads, kv_heads, dim = HEADS[case["shape"]]
    size = 2 if case["dtype"] == "bf16" else 4
    prefix, tail = _lengths(case)
    new, members = case["tokens"], case["members"]
    keys = sum(prefix) + sum(tail) + new * len(tail)
    pairs = sum(new * (prefix[s // members] + t) + new * (new + 1) // 2
                for s, t in enumerate(tail))
    return {"bytes": size * dim * (2 * kv_heads * keys + 2 * heads * new * len(tail)),
            "flops": 4 * heads * dim * pairs}


# ----------------------------------------------------------------------------- 64-bit results
def _exact_shared(case, seed):
    """Token by token from the definition: a request's keys are one sequence, whoever shares them."""
    heads, kv_heads, dim = HEADS[case["shape"]]
    qkv, k, v, table, prefix, tail = _shared_inputs(case, seed)
    new, members, page = case["tokens"], case["members"], case["page"]
    out = torch.empty(qkv.shape[0], heads, dim, dtype=torch.float64, device=DEVICE)
    repeat = heads // kv_heads
    for s in range(len(tail)):
        before = prefix[s // members] + tail[s]
        ids = table[s, : -(-(before + new) // page)]
        keys, values = (x[ids].permute(1, 0, 2, 3).reshape(kv_heads, -1, dim)[:, : before + new]
                        .double() for x in (k, v))
        q = qkv[s * new: (s + 1) * new, : heads * dim].double().view(new, heads, dim)
        # query head h reads key/value head h // repeat
        q = q.permute(1, 0, 2).reshape(kv_heads, repeat * new, dim)
        score = torch.bmm(q, keys.transpose(1, 2)) * dim ** -0.5
        for t in range(new - 1):
            score.view(kv_heads, repeat, new, -1)[:, :, t, before + t + 1:] = -math.inf
        mixed = torch.bmm(torch.softmax(score, 2), values)
        out[s * new: (s + 1) * new] = mixed.view(heads, new, dim).permute(1, 0, 2)
    return out.view(-1, heads * dim)


def _exact_select(case, seed):
    """One candidate after the other: the largest of all that are left, the first of equal ones."""
    logits, scores = _select_inputs(case, seed)
    G, B, V, K = case["groups"], case["beams"], case["vocabulary"], case["take"]
    best = torch.full((G, K), -math.inf, dtype=torch.float64, device=DEVICE)
    beam, token = (torch.full((G, K), -1, dtype=torch.int32, device=DEVICE) for _ in range(2))
    for g in range(G):
        left = torch.log_softmax(logits[g * B: (g + 1) * B].double(), 1) + scores[g].double()[:, None]
        left = left.view(-1)
        for i in range(K):
            top = left.max()
            if not bool(top > -math.inf):
                break
            at = int((left == top).nonzero()[0])
            best[g, i], beam[g, i], token[g, i] = top, at // V, at % V
            left[at] = -math.inf
    return [best, beam, token]


def exact(case, seed):
    if case["kind"] == "select":
        return _exact_select(case, seed)
    if case["kind"] == "shared":
        return _exact_shared(case, seed)
    state, _, _ = _reorder_inputs(case, seed)
    moved = state.clone()
    for rows, parents in zip(*_moves(case)):
        for row, parent in zip(rows, parents):
            moved[:, row] = state[:, rows[parent]]
    return moved.double()

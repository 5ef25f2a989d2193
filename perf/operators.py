"""What requests of one batch have in common, computed once: the work that these two operators are measured on.

``prefix``    attention of a step whose requests begin with the same keys (a system prompt, a document, several answers to one prompt):
              the shared pages are named by every request's block table, groups of neighbouring requests share their first keys, and
              behind them each request has keys of its own (``ops.prefix_attention``).
``adapters``  a projection with weights for all and a low-rank adapter for most requests of the step, another one for each or the
              same for several (``ops.adapter_linear``).

Head layouts and widths are those of ``tempura_amd.config.PRESETS`` and of ``bench.py``.  The plain forms are elementary torch
operations in 32 bits; ``exact`` computes the same from the definitions, request by request, in 64 bits.
"""
import math

import torch

own = False
DEVICE = "cuda:0"
PAGE = 16
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ---- the cases --------------------------------------------------------------------------------------------------------------
def _prefix(name, groups, own_keys, tokens=1, heads=32, kv_heads=8, dim=128, dtype="bfloat16", cap=0.0, sink=False):
    """``groups``: "requests x shared keys" of each group; ``own_keys``, ``tokens``: the most that a request has."""
    return {"name": name, "kind": "prefix", "groups": groups, "own_keys": own_keys, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "cap": cap, "sink": sink}


def _adapters(name, singles, portions, k, n, slices=1, rank=16, slots=8, dtype="bfloat16"):
    """``singles`` requests of one token, then ``portions`` (lengths in a text); ``slices`` projections stacked into n columns."""
    return {"name": name, "kind": "adapters", "singles": singles, "portions": portions, "k": k, "n": n, "slices": slices, "rank": rank,
            "slots": slots, "dtype": dtype}


def listed():
    return [
        # four answers to one short prompt, just begun: the least a call can be
        _prefix("prefix_4_answers", "4x1008", 24),
        # the headline batch of bench.py behind a system prompt
        _prefix("prefix_decode_8", "8x2048", 400),
        # a busy server: one long system prompt with examples, contexts of every length behind it
        _prefix("prefix_decode_64", "64x8192", 1200),
        # three services on one machine, and requests that share nothing; pages that end inside a tile; the 3B shape's heads
        _prefix("prefix_groups", "24x4112,13x1600,7x528,4x0", 700, heads=24),
        # short questions to one document, in one step: a few tokens a request
        _prefix("prefix_questions", "16x6000", 60, tokens=24),
        # narrow heads with capped scores and a sink
        _prefix("prefix_capped_64", "48x4096", 500, heads=32, kv_heads=8, dim=64, cap=30.0, sink=True),
        # one very long document read by many: the largest
        _prefix("prefix_document", "32x65536", 900),
        # the float32 path
        _prefix("prefix_float32", "16x2000", 300, heads=24, dtype="float32"),
        # one user's token with an adapter on q, k and v
        _adapters("adapters_1", 1, "", 4096, 6144, slices=3, slots=4),
        # a serving step: 48 users, adapters of 16 customers, some without
        _adapters("adapters_48", 48, "", 4096, 6144, slices=3, slots=16),
        # portions of two prompts beside running requests, down projection of bench.py's width 2,048
        _adapters("adapters_mixed_700", 31, "512,188", 8192, 2048, rank=32),
        # whole prompts of several customers in one long step
        _adapters("adapters_prompts", 0, "1500,700,1030,866", 4096, 4096, rank=64),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        heads, kv_heads, dim = rng.choice(((32, 8, 128), (24, 8, 128), (32, 8, 64), (16, 4, 64), (8, 8, 128), (64, 8, 128)))
        dtype = "float32" if rng.random() < 0.2 else "bfloat16"
        tokens = rng.choice((1, 1, 1, log(2, 30)))
        groups, left = [], log(2, 24 if tokens > 1 or dtype == "float32" else 90)
        while left > 0 and len(groups) < 4:
            n = min(left, log(1, 64))
            groups.append("%dx%d" % (n, 16 * log(2, 1000 if dtype == "bfloat16" else 250) if rng.random() < 0.85 else 0))
            left -= n
        return _prefix("", ",".join(groups), log(tokens, 900), tokens, heads, kv_heads, dim, dtype,
                       30.0 if rng.random() < 0.2 else 0.0, rng.random() < 0.2)
    dtype = "float32" if rng.random() < 0.2 else "bfloat16"
    widths = (512, 1024, 1100, 2048, 4096, 8192)
    k, slices = rng.choice(widths), rng.choice((1, 1, 2, 3))
    n = slices * 8 * log(20, 700)
    portions = [str(log(2, 1200 if dtype == "bfloat16" else 300)) for _ in range(rng.choice((0, 0, 1, 3)))]
    return _adapters("", log(1, 128), ",".join(portions), k, n, slices, rng.choice((4, 8, 12, 16, 16, 32, 64)), log(1, 32), dtype)


# ---- sizes that a case stands for (whatever the seed) ------------------------------------------------------------------------
def _part(i, most):
    """A number from 1 to ``most`` for the i-th of a row of things, spread over the range."""
    return 1 + int((i * 0.6180339887498949 + 0.35) % 1.0 * most)


def _requests(case):
    """(requests, shared keys) of each group, and of each request (shared keys, own keys, new tokens)."""
    groups = [tuple(int(v) for v in g.split("x")) for g in case["groups"].split(",")]
    each = []
    for count, shared in groups:
        for _ in range(count):
            t = _part(len(each), case["tokens"])
            each.append((shared, max(t, _part(3 * len(each) + 1, case["own_keys"])), t))
    return groups, each


def _rows(case):
    """Tokens of each request, and its adapter (-1: none; a quarter of many requests)."""
    runs = [1] * case["singles"] + [int(t) for t in case["portions"].split(",") if t]
    return runs, [-1 if len(runs) > 3 and i % 4 == 3 else (i * 7 + 1) % case["slots"] for i in range(len(runs))]


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32) * std).to(dtype)
    if case["kind"] == "prefix":
        return _prepare_prefix(case, gen, normal)
    runs, slot = _rows(case)
    k, n, rank, slices = case["k"], case["n"], case["rank"], case["slices"]
    s = {"case": case, "x": normal(sum(runs), k), "w": normal(n, k, std=k ** -0.5),
         "a": normal(case["slots"], slices * rank, k, std=k ** -0.5), "b": normal(case["slots"], n, rank, std=0.05),
         "scales": 0.5 + torch.rand(case["slots"], generator=gen, device=DEVICE),
         "ids": torch.tensor([v for t, v in zip(runs, slot) for _ in range(t)], dtype=torch.int32, device=DEVICE),
         "ends": [n // slices * (i + 1) for i in range(slices)], "max_run": max(runs)}
    if own:
        from tempura_amd.kernels import ops
        s["weight"], s["adapters"] = ops.tile_weight(s["w"]), ops.Adapters(s["a"], s["b"], s["scales"], s["ends"])
    return s


def _prepare_prefix(case, gen, normal):
    groups, each = _requests(case)
    heads, kvh, dim = case["heads"], case["kv_heads"], case["dim"]
    pages_of = lambda keys: -(-keys // PAGE)  # noqa: E731
    # a group's whole pages are its requests' first ones; the page that its keys end in, if they do not end with one, too
    total = sum(pages_of(p) for _, p in groups) + sum(pages_of(p + o) - pages_of(p) for p, o, _ in each) + 2
    names = torch.randperm(total, generator=gen, device=DEVICE).to(torch.int32).cpu()
    width = max(pages_of(p + o) for p, o, _ in each)
    tables, at, r = torch.full((len(each), width), -1, dtype=torch.int32), 0, 0
    for count, shared in groups:
        first = names[at: at + pages_of(shared)]
        at += len(first)
        for _ in range(count):
            more = pages_of(sum(each[r][:2])) - len(first)
            tables[r, :len(first)] = first
            tables[r, len(first): len(first) + more] = names[at: at + more]
            at, r = at + more, r + 1
    new = [t for _, _, t in each]
    starts = torch.tensor([0] + new).cumsum(0)
    ints = lambda v: torch.as_tensor(v).to(torch.int32).to(DEVICE)  # noqa: E731
    ctx = [p + o for p, o, _ in each]
    s = {"case": case, "q": normal(sum(new), heads, dim), "k": normal(total, kvh, PAGE, dim), "v": normal(total, kvh, dim, PAGE),
         "tables": ints(tables), "starts": ints(starts), "ctx": ints(ctx),
         "token_req": ints([i for i, t in enumerate(new) for _ in range(t)]), "place": ints([j for t in new for j in range(t)]),
         "scale": dim ** -0.5, "max_new": max(new), "max_ctx": max(ctx), "max_own": max(o for _, o, _ in each),
         "single": sum(t == 1 for t in new),
         "sink": torch.randn(heads, generator=gen, device=DEVICE, dtype=torch.float32) if case["sink"] else None}
    if own:
        from tempura_amd.kernels import ops
        s["shared"] = ops.SharedKeys([c for c, _ in groups], [p for _, p in groups], DEVICE)
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        from tempura_amd.kernels import ops
        if state["case"]["kind"] == "prefix":
            return ops.prefix_attention(state["q"], state["k"], state["v"], state["tables"], state["starts"], state["ctx"], state["token_req"],
                                        state["scale"], state["shared"], state["max_new"], state["max_ctx"], max_own_len=state["max_own"],
                                        num_single=state["single"], sink=state["sink"], softcap=state["case"]["cap"])
        return ops.adapter_linear(state["x"], state["weight"], state["adapters"], state["ids"], max_run=state["max_run"])
    return _plain_prefix(state) if state["case"]["kind"] == "prefix" else _plain_adapters(state)


def _plain_prefix(s):
    """Every request's keys gathered by its table, padded to the longest; one product, a masked softmax, one product."""
    q, kvh, dim, r = s["q"].float(), s["k"].shape[1], s["k"].shape[3], s["tables"].shape[0]
    heads, group, t = q.shape[1], q.shape[1] // kvh, s["max_new"]
    pages = s["tables"].long().clamp(min=0)
    k = s["k"][pages].float().permute(0, 2, 1, 3, 4).reshape(r, kvh, -1, dim)
    v = s["v"][pages].float().permute(0, 2, 3, 1, 4).reshape(r, kvh, dim, -1)
    req, place = s["token_req"].long(), s["place"].long()
    rows = torch.zeros((r, t, heads, dim), device=q.device)
    rows[req, place] = q
    rows = rows.view(r, t, kvh, group, dim).permute(0, 2, 1, 3, 4).reshape(r, kvh, t * group, dim)
    score = rows @ k.transpose(2, 3).contiguous() * s["scale"]
    if s["case"]["cap"]:
        score = s["case"]["cap"] * torch.tanh(score / s["case"]["cap"])
    new = s["starts"][1:] - s["starts"][:-1]
    pos = (s["ctx"] - new)[:, None] + torch.arange(t, device=q.device)[None]
    seen = torch.arange(k.shape[2], device=q.device)[None, None] <= pos[:, :, None]
    score = score.view(r, kvh, t, group, -1).masked_fill(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    if s["sink"] is not None:
        sink = s["sink"].view(1, kvh, 1, group, 1)
        top = torch.maximum(top, sink)
    weight = torch.exp(score - top)
    total = weight.sum(-1, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(sink - top)
    exists = torch.arange(k.shape[2], device=q.device)[None] < s["ctx"][:, None]
    v = v.masked_fill(~exists[:, None, None], 0.0)
    o = (weight / total).view(r, kvh, t * group, -1) @ v.transpose(2, 3).contiguous()
    o = o.view(r, kvh, t, group, dim).permute(0, 2, 1, 3, 4).reshape(r, t, heads * dim)
    return o[req, place].to(s["q"].dtype)


def _plain_adapters(s):
    """All adapters' low-rank rows in one product, those of other adapters than a row's own cleared, all adapters' columns in one more."""
    x, slots, rank = s["x"].float(), s["a"].shape[0], s["b"].shape[2]
    n, slices, ids = s["b"].shape[1], s["case"]["slices"], s["ids"].long()
    y = x @ s["w"].float().t()
    low = (x @ s["a"].float().reshape(-1, x.shape[1]).t()).view(-1, slots, slices, rank)
    own_slot = torch.arange(slots, device=x.device)[None] == ids[:, None]
    low = low * (own_slot * s["scales"])[:, :, None, None]
    up = s["b"].float().view(slots, slices, n // slices, rank).permute(1, 0, 3, 2).reshape(slices, slots * rank, n // slices)
    more = low.permute(2, 0, 1, 3).reshape(slices, -1, slots * rank) @ up
    return y + more.permute(1, 0, 2).reshape(-1, n)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "prefix":
        groups, each = _requests(case)
        keys = sum(p for _, p in groups) + sum(o for _, o, _ in each)
        seen = sum(t * (p + o) - t * (t - 1) // 2 for p, o, t in each)
        return {"bytes": size * case["dim"] * (2 * case["kv_heads"] * keys + 2 * case["heads"] * sum(t for _, _, t in each)),
                "flops": 4 * case["dim"] * case["heads"] * seen}
    runs, slot = _rows(case)
    m, k, n, rank = sum(runs), case["k"], case["n"], case["rank"]
    used, with_one = len({v for v in slot if v >= 0}), sum(t for t, v in zip(runs, slot) if v >= 0)
    return {"bytes": size * (n * k + m * k + used * rank * (case["slices"] * k + n)) + 4 * m * n,
            "flops": 2 * m * n * k + 2 * with_one * rank * (case["slices"] * k + n)}


# ---- the same in 64 bits ----------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_prefix(s) if case["kind"] == "prefix" else _exact_adapters(s)


def _exact_prefix(s):
    out, heads, kvh = [], s["q"].shape[1], s["k"].shape[1]
    starts, ctx = s["starts"].tolist(), s["ctx"].tolist()
    for i, length in enumerate(ctx):
        page = s["tables"][i, : -(-length // PAGE)].long()
        k = s["k"].index_select(0, page).double().transpose(1, 2).flatten(0, 1)[:length]                      # [keys, kv heads, dim]
        v = s["v"].index_select(0, page).double().permute(0, 3, 1, 2).flatten(0, 1)[:length]
        q = s["q"][starts[i]: starts[i + 1]].double()
        rows = []
        for h in range(heads):
            score = s["scale"] * torch.mm(q[:, h], k[:, h * kvh // heads].t())
            if s["case"]["cap"]:
                score = torch.tanh(score / s["case"]["cap"]) * s["case"]["cap"]
            for j in range(score.shape[0]):
                score[j, length - score.shape[0] + j + 1:] = -math.inf
            if s["sink"] is not None:
                score = torch.cat([score, s["sink"][h].double().expand(score.shape[0], 1)], 1)
            p = torch.softmax(score, 1)[:, :length]
            rows.append(torch.mm(p, v[:, h * kvh // heads]))
        out.append(torch.cat(rows, 1))
    return torch.cat(out)


def _exact_adapters(s):
    x = s["x"].double()
    y = torch.mm(x, s["w"].double().t())
    rank, first = s["b"].shape[2], 0
    for i, end in enumerate(s["ends"]):
        for slot in sorted(set(s["ids"].tolist()) - {-1}):
            rows = (s["ids"] == slot).nonzero().flatten()
            low = torch.mm(x[rows], s["a"][slot, i * rank: (i + 1) * rank].double().t())
            y[rows, first: end] += s["scales"][slot].double() * torch.mm(low, s["b"][slot, first: end].double().t())
        first = end
    return y

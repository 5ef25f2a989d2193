"""Steps whose requests begin with the same keys, and their attention in 64 bits."""
import torch


def step(runs, own, new, heads, kv, dim, page, dtype, seed, cut=0, poison=True, spare=2):
    """``runs``: (requests, shared keys) of each run; ``own[i]``, ``new[i]``: request i's keys behind the shared ones, its new tokens among them, and how many
    those are.  Shared keys that end inside a page (``cut`` of them) share that page's keys, copied into a page of each request's own.
    ``poison``: what lies behind a request's last key is not finite.  Everything on the CPU."""
    g = torch.Generator().manual_seed(seed)
    ctx, each = [], []
    for c, shared in runs:
        each += [shared + (cut if shared else 0)] * c
    ctx = [p + o for p, o in zip(each, own)]
    r, width = len(ctx), -(-max(ctx) // page) + spare
    total = r * width + sum(-(-p // page) for _, p in runs) + 3
    names = torch.randperm(total, generator=g).tolist()
    k = torch.randn(total, kv, page, dim, generator=g).to(dtype)
    v = torch.randn(total, kv, dim, page, generator=g).to(dtype)
    tables = torch.full((r, width), -1, dtype=torch.int32)
    i = 0
    for c, shared in runs:
        whole = shared // page
        first = [names.pop() for _ in range(whole)]
        part = shared + (cut if shared else 0) - whole * page
        source = None
        for _ in range(c):
            n = -(-ctx[i] // page)
            rest = [names.pop() for _ in range(n - whole)]
            tables[i, :n] = torch.tensor(first + rest, dtype=torch.int32)
            if part and rest:       # (the keys of the page that the shared ones end in are the same for all)
                if source is None:
                    source = rest[0]
                k[rest[0], :, :part], v[rest[0], :, :, :part] = k[source, :, :part].clone(), v[source, :, :, :part].clone()
            i += 1
    if poison:
        used = torch.zeros(total, page, dtype=torch.bool)
        for j, c in enumerate(ctx):
            for p in range(-(-c // page)):
                used[tables[j, p], : min(page, c - p * page)] = True
        bad = ~used
        k.masked_fill_(bad[:, None, :, None], float("nan"))
        v.masked_fill_(bad[:, None, None, :], float("inf"))
    n = sum(new)
    starts = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    return {"q": torch.randn(n, heads, dim, generator=g).to(dtype), "k": k, "v": v, "tables": tables, "starts": starts,
            "ctx": torch.tensor(ctx, dtype=torch.int32), "req": torch.tensor([j for j, t in enumerate(new) for _ in range(t)], dtype=torch.int32),
            "each": each, "new": new, "scale": dim ** -0.5, "counts": [c for c, _ in runs], "lens": [p + (cut if p else 0) for _, p in runs],
            "own": max(own)}


def exact(s, sink=None, cap=0.0):
    """(outputs in 64 bits, the weights' sum over |values|, the largest sum of |q k| behind a score) of every token and head."""
    out, size, reach = [], [], []
    heads, kv = s["q"].shape[1], s["k"].shape[1]
    for i, c in enumerate(s["ctx"].tolist()):
        page = s["tables"][i, : -(-c // s["k"].shape[2])].long()
        k = s["k"][page].double().transpose(1, 2).flatten(0, 1)[:c]
        v = s["v"][page].double().permute(0, 3, 1, 2).flatten(0, 1)[:c]
        t0, t1 = int(s["starts"][i]), int(s["starts"][i + 1])
        for t in range(t0, t1):
            last = c - (t1 - t0) + (t - t0)
            row, a, b = [], [], []
            for h in range(heads):
                kk, vv = k[: last + 1, h * kv // heads], v[: last + 1, h * kv // heads]
                q = s["q"][t, h].double()
                score = kk @ q * s["scale"]
                if cap:
                    score = cap * torch.tanh(score / cap)
                if sink is not None:
                    score = torch.cat([score, sink[h].double().reshape(1)])
                w = torch.softmax(score, 0)[: last + 1]
                row.append(w @ vv)
                a.append(w @ vv.abs())
                b.append(float((kk.abs() @ q.abs()).max()) * s["scale"])
            out.append(torch.cat(row))
            size.append(torch.cat(a))
            reach.append(max(b))
    return torch.stack(out), torch.stack(size), torch.tensor(reach, dtype=torch.float64)


def tolerance(s, want, size, reach):
    """How far a result may be off, element by element.  A float32 score is a sum of dim products, off by dim half steps of the
    sum of their magnitudes (``reach``), and passes a handful of further roundings; an error e of every score moves a weighted mean of
    values by at most 2 e of their weighted magnitudes (``size``).  The sums over the keys add a half step a key and part.  bfloat16: the
    weights are rounded in front of the second product (2^-8 of each, so 2^-8 of ``size``), the result once more.  A result below the
    smallest normal number of either type, 2^-126 (a head whose sink takes all but e^-200 of the weight), may come as zero: it is off by
    itself, less than 2^-126."""
    half, keys = 2.0 ** -24, int(s["ctx"].max())
    score = 2 * (s["q"].shape[2] + 16) * half * (reach[:, None] + 1)
    tol = size * (score + (keys + 64) * half) + 2.0 ** -126
    if s["q"].dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * size + 2.0 ** -8 * want.abs()
    else:
        tol = tol + half * want.abs()
    return tol

"""Every form of the attention of shared keys against its definition in 64 bits, whatever the rule on sizes would take: blocks of 16, 64 and 128 rows for shared
and for own keys, parts of few steps, joins in one pass and in several."""
import ctypes

import pytest
import torch

import prefix_cases as P

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32
FORMS = [(16, 16), (64, 16), (128, 16), (64, 64), (128, 64), (128, 128)]


def run(monkeypatch, s, form, shared_steps, own_steps, sink=None, cap=0.0):
    """The step laid out in blocks of ``form`` rows and parts of so many steps; the launch is asserted to be that one."""
    from tempura_amd.kernels import ops
    rows, own_rows = form
    heads, kv = s["q"].shape[1], s["k"].shape[1]
    shared = ops.SharedKeys(s["counts"], s["lens"], DEV, requests=len(s["new"]))
    tokens, blocks, i = s["new"], 0, 0
    for c, v in zip(s["counts"], s["lens"]):
        blocks += -(-sum(tokens[i: i + c]) * (heads // kv) // rows) if v else 0
        i += c
    steps, own = -(-shared.max_keys // 32), (s["own"] + 15 + 31) // 32
    plan = (rows, own_rows, blocks, shared_steps, -(-steps // shared_steps), own_steps, -(-own // own_steps))
    assert plan[4] + plan[6] <= 128
    monkeypatch.setattr(ops, "prefix_least_keys", (0, 0, 0))
    monkeypatch.setattr(ops, "_prefix_plan", lambda *a: plan)
    launched, real = [], ops._call

    def call(name, *a, **kw):
        launched.append((name, [list(x) for x in a if isinstance(x, ctypes.Array)]))
        return real(name, *a, **kw)
    monkeypatch.setattr(ops, "_call", call)
    to = lambda name: s[name].to(DEV)  # noqa: E731
    out = ops.prefix_attention(to("q"), to("k"), to("v"), to("tables"), to("starts"), to("ctx"), to("req"), s["scale"], shared, max(s["new"]),
                               int(s["ctx"].max()), max_own_len=s["own"], sink=None if sink is None else sink.to(DEV), softcap=cap)
    assert [n for n, _ in launched] == ["tp_prefix_attention"] and tuple(launched[0][1][0][10:]) == plan
    return out.cpu().double()


def check(monkeypatch, s, *args, sink=None, cap=0.0):
    want, size, reach = P.exact(s, sink, cap)
    got = run(monkeypatch, s, *args, sink=sink, cap=cap)
    over = (got - want).abs() - P.tolerance(s, want, size, reach)
    assert got.shape == want.shape and bool(torch.isfinite(got).all()) and float(over.max()) <= 0, float(over.max())


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (6, 2, 64), (5, 1, 32)])
def test_portions(monkeypatch, form, dtype, heads, kv, dim):
    """Portions beside single tokens, rows that fill blocks and that leave waves without any, a request that shares nothing; shared keys that end inside a page; what lies
    behind the last key is not finite."""
    new, own = [1, 5, 17, 1, 33, 2, 3], [60, 5, 40, 1, 33, 70, 9]
    check(monkeypatch, P.step([(4, 208), (2, 96), (1, 0)], own, new, heads, kv, dim, 16, dtype, seed=dim + heads, cut=7), form, 2, 1)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim,cap", [(128, 0.0), (128, 20.0), (64, 20.0), (32, 0.0)])
def test_single_tokens_with_sinks(monkeypatch, form, dtype, dim, cap):
    """Single tokens of two runs, with sinks, with and without a cap; parts of unequal length."""
    n = 40
    s = P.step([(n - 5, 592), (5, 64)], [1 + (37 * i) % 130 for i in range(n)], [1] * n, 8, 2, dim, 32, dtype, seed=dim, cut=3)
    check(monkeypatch, s, form, 5, 2, sink=torch.tensor([0.0, 3.0, -50.0, 9.0, float("-inf"), 1.0, 20.0, -1.0]), cap=cap)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,dim,parts", [(32, 128, 11), (32, 64, 20), (32, 32, 37), (2, 128, 37), (2, 64, 75), (4, 32, 110)])
def test_joins(monkeypatch, dtype, heads, dim, parts):
    """Rows of many parts, by one wave (more than 4,096 rows) and by four, in more than one pass; requests of fewer parts than the longest."""
    requests = 4128 // 32 if heads == 32 else 6
    runs = [(requests - 3, 32 * (parts - 2) - 16), (2, 64), (1, 0)]
    s = P.step(runs, [1 + (11 * i) % 40 for i in range(requests)], [1] * requests, heads, 1, dim, 16, dtype, seed=parts)
    check(monkeypatch, s, (128, 16) if heads == 32 else (16, 16), 1, 2)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("cap", [50.0, 1000.0, 30000.0])
def test_caps_far_above_the_scores(monkeypatch, form, cap):
    """float32 scores small beside their cap are as exact as scores without one: cap * tanh(score / cap) is a product of a few roundings, each relative to the score."""
    s = P.step([(5, 560), (1, 0)], [3, 40, 64, 100, 1, 7], [1, 1, 2, 1, 1, 1], 8, 2, 64, 16, F32, seed=int(cap))
    check(monkeypatch, s, form, 4, 2, cap=cap)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [128, 32])
def test_what_is_not_finite_behind_a_token(monkeypatch, form, dtype, dim):
    """Keys and values of a request's later tokens that are infinite or no numbers leave the tokens in front of them as they are, and give those that see them what the
    definition gives: an element whose values hold one infinity is infinite, with two of opposite signs or with what is no number it is none."""
    new, own, inf = [1, 9, 40, 40], [20, 30, 61, 75], float("inf")
    s = P.step([(4, 80)], own, new, 8, 2, dim, 16, dtype, seed=dim, cut=5)
    last = dict(enumerate(s["ctx"].tolist()))

    def put(request, behind, name, values):      # (into the key or value `behind` places in front of the request's last)
        at = last[request] - 1 - behind
        page = int(s["tables"][request, at // 16])
        row = s[name][page, :, at % 16] if name == "k" else s[name][page, :, :, at % 16]
        for element, x in values.items():
            row[:, element] = x
    put(1, 3, "v", {0: inf, 5: -inf, 17: float("nan")})
    put(1, 0, "v", {0: -inf, 5: -inf})
    put(2, 20, "v", {3: inf, 31: inf})
    put(2, 11, "v", {3: inf, 4: -inf, dim - 1: float("nan")})
    put(3, 0, "v", {i: inf for i in range(dim)})
    put(3, 18, "k", {2: float("nan")})
    want, size, reach = P.exact(s)
    got = run(monkeypatch, s, form, 2, 1)
    finite = torch.isfinite(want)
    assert bool((~finite).any()) and bool(finite[: 1 + 5].all())
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[want.abs() == inf], want[want.abs() == inf])
    tol = P.tolerance(s, want, torch.where(finite, size, torch.zeros_like(size)), torch.where(torch.isfinite(reach), reach, torch.zeros_like(reach)))
    assert float(((got - want).abs() - tol)[finite].max()) <= 0


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_same_call_gives_the_same_bits(monkeypatch, form, dtype):
    s = P.step([(9, 640)], [1 + (61 * i) % 200 for i in range(9)], [1, 4, 1, 9, 1, 1, 30, 1, 2], 8, 2, 128, 16, dtype, seed=2)
    first = run(monkeypatch, s, form, 3, 2)
    assert all(torch.equal(run(monkeypatch, s, form, 3, 2), first) for _ in range(3))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_queries_at_odd_places(monkeypatch, dtype):
    """q may lie anywhere that an element may: the same bits as from an aligned place."""
    from tempura_amd.kernels import ops
    monkeypatch.setattr(ops, "prefix_least_keys", (0, 0, 0))
    s = P.step([(5, 320)], [1, 40, 64, 100, 7], [1, 3, 1, 1, 2], 8, 2, 64, 16, dtype, seed=4)
    t = {name: s[name].to(DEV) for name in ("q", "k", "v", "tables", "starts", "ctx", "req")}
    shared = ops.SharedKeys(s["counts"], s["lens"], DEV)
    call = lambda q: ops.prefix_attention(q, t["k"], t["v"], t["tables"], t["starts"], t["ctx"], t["req"], s["scale"], shared, 3,  # noqa: E731
                                          int(s["ctx"].max()), max_own_len=s["own"])
    odd = torch.empty(t["q"].numel() + 1, dtype=dtype, device=DEV)[1:].view(t["q"].shape)
    odd.copy_(t["q"])
    assert odd.data_ptr() % 16 and torch.equal(call(odd), call(t["q"]))

"""Attention of requests that begin with the same keys against its definition in 64 bits, and against the attention that reads
every request's pages for itself."""
import pytest
import torch

import prefix_cases as P

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def few_keys_too(monkeypatch):
    """Shared keys are read once for all however few they are (``test_few_shared_keys`` apart)."""
    from tempura_amd.kernels import ops
    monkeypatch.setattr(ops, "prefix_least_keys", (0, 0, 0))


def _run(s, sink=None, cap=0.0, own=True, dev=DEV):
    from tempura_amd.kernels import ops
    shared = ops.SharedKeys(s["counts"], s["lens"], dev, requests=len(s["new"]))
    to = lambda name: s[name].to(dev)  # noqa: E731
    return ops.prefix_attention(to("q"), to("k"), to("v"), to("tables"), to("starts"), to("ctx"), to("req"), s["scale"], shared, max(s["new"]),
                                int(s["ctx"].max()), max_own_len=s["own"] if own else None, sink=None if sink is None else sink.to(dev), softcap=cap)


def _check(s, sink=None, cap=0.0, **more):
    want, size, reach = P.exact(s, sink, cap)
    got = _run(s, sink, cap, **more).cpu().double()
    assert got.shape == want.shape
    over = (got - want).abs() - P.tolerance(s, want, size, reach)
    assert bool(torch.isfinite(got).all()) and float(over.max()) <= 0, float(over.max())
    return got


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv,dim,page", [(8, 2, 128, 16), (4, 4, 64, 32), (10, 1, 64, 16), (6, 2, 32, 64), (34, 2, 32, 16), (2, 1, 128, 128)])
@pytest.mark.parametrize("shared", [128, 384, 1152])
def test_single_tokens(dtype, heads, kv, dim, page, shared):
    """Groups of one, some and many rows; own keys of one, at the edges of steps and pages; what lies behind the last key is not finite."""
    own = [1, 2, 31, 32, 33, 15, 16, 17, 100, 257]
    _check(P.step([(len(own), shared)], own, [1] * len(own), heads, kv, dim, page, dtype, seed=shared + dim))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("runs", [[(3, 48), (1, 16), (5, 640)], [(2, 0), (6, 256), (2, 0)], [(1, 2048)], [(4, 32), (3, 0)], [(1, 16)] * 70])
def test_runs(dtype, runs):
    """Several runs of requests, requests that share nothing among them, runs of one request, more runs than lanes."""
    n = sum(c for c, _ in runs)
    own = [1 + (37 * i) % 90 for i in range(n)]
    _check(P.step(runs, own, [1] * n, 8, 2, 64, 16, dtype, seed=n))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cut", [1, 8, 15])
def test_shared_keys_that_end_inside_a_page(dtype, cut):
    _check(P.step([(3, 160), (2, 16)], [40, 7, 19, 16, 90], [1] * 5, 8, 2, 128, 16, dtype, seed=cut, cut=cut))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv", [(8, 2), (4, 4), (6, 1)])
def test_several_tokens_a_request(dtype, heads, kv):
    """Portions beside single tokens: a token sees the request's own keys up to itself."""
    new = [1, 5, 17, 1, 33, 2]
    own = [60, 5, 40, 1, 33, 70]
    _check(P.step([(4, 208), (2, 96)], own, new, heads, kv, 64, 16, dtype, seed=heads))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cap,with_sink", [(0.0, True), (5.0, False), (30.0, True)])
def test_cap_and_sink(dtype, cap, with_sink):
    s = P.step([(4, 96), (2, 0), (3, 304)], [1 + 13 * i for i in range(9)], [1] * 8 + [4], 8, 2, 64, 16, dtype, seed=int(cap) + 1)
    sink = torch.tensor([0.0, 3.0, -50.0, 9.0, float("-inf"), 1.0, 200.0, -1.0]) if with_sink else None
    _check(s, sink, cap)


def test_many_requests_and_parts():
    """Keys in many parts, blocks beyond the chip; bounds that are not tight."""
    n = 40
    s = P.step([(n, 4096)], [1 + (61 * i) % 600 for i in range(n)], [1] * n, 4, 1, 128, 16, BF16, seed=5, poison=False)
    _check(s)
    _check(s, own=False)


def test_other_sizes_run_the_attention_of_each_request():
    """Head sizes and pages that the kernel is not built for, and steps without shared keys: the same bits as without sharing."""
    from tempura_amd.kernels import ops
    for dim, page, runs in ((96, 16, [(3, 64)]), (64, 8, [(3, 64)]), (64, 16, [(3, 0)]), (40, 16, [(3, 32)])):
        s = P.step(runs, [9, 30, 41], [1, 1, 1], 4, 2, dim, page, BF16, seed=dim)
        _check(s)
        to = {name: s[name].to(DEV) for name in ("q", "k", "v", "tables", "starts", "ctx", "req")}
        plain = ops.paged_attention(to["q"], to["k"], to["v"], to["tables"], to["starts"], to["ctx"], to["req"], s["scale"], 0, 1, int(s["ctx"].max()))
        assert torch.equal(_run(s), plain)


def test_few_shared_keys(monkeypatch):
    """By the rule on how many keys are shared: the same bits as without sharing where they are few, the result as defined on both sides."""
    from tempura_amd.kernels import ops
    monkeypatch.undo()
    for dtype, new, below, above in ((BF16, 1, 752, 768), (F32, 1, 496, 512), (BF16, 3, 176, 192), (BF16, 20, 304, 320)):
        for shared in (below, above):
            s = P.step([(3, shared)], [20, 30, 41], [new] * 3, 4, 2, 64, 16, dtype, seed=shared)
            _check(s)
            to = {name: s[name].to(DEV) for name in ("q", "k", "v", "tables", "starts", "ctx", "req")}
            plain = ops.paged_attention(to["q"], to["k"], to["v"], to["tables"], to["starts"], to["ctx"], to["req"], s["scale"], 0, new, int(s["ctx"].max()))
            if shared == below:
                assert torch.equal(_run(s), plain)


def test_large_scores_and_equal_keys():
    """Scores far apart and all alike: the running maximum moves late, or never."""
    for dtype in (BF16, F32):
        s = P.step([(5, 320)], [3, 40, 64, 100, 1], [1] * 5, 8, 2, 64, 16, dtype, seed=3, poison=False)
        s["q"] = (s["q"].float() * 8).to(dtype)
        _check(s)
        s["q"] = torch.zeros_like(s["q"])
        _check(s)


def test_the_same_call_gives_the_same_bits_on_any_stream_and_in_a_graph():
    from tempura_amd.kernels import ops
    s = P.step([(6, 512), (3, 128)], [1 + 29 * i for i in range(9)], [1] * 9, 8, 2, 128, 16, BF16, seed=11, poison=False)
    shared = ops.SharedKeys(s["counts"], s["lens"], DEV)
    t = {name: s[name].to(DEV) for name in ("q", "k", "v", "tables", "starts", "ctx", "req")}
    call = lambda: ops.prefix_attention(t["q"], t["k"], t["v"], t["tables"], t["starts"], t["ctx"], t["req"], s["scale"], shared, 1,  # noqa: E731
                                        int(s["ctx"].max()) + 9, max_own_len=250)
    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(call(), first)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):      # (contexts and queries move between replays)
        t["q"].copy_(torch.randn(t["q"].shape, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        t["ctx"].sub_((t["ctx"] > 600).to(torch.int32) * 7)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_runs_of_a_captured_step_move_between_replays(dtype):
    """Launches laid out for bounds: other runs, lengths and tables with every replay, each against the definition."""
    import numpy as np
    from tempura_amd.kernels import ops
    n, groups, bound, own_bound = 12, 17, 1024, 512
    steps = [P.step(runs, [1 + (53 * i + 7 * k) % 500 for i in range(n)], [1] * n, 8, 2, 64, 16, dtype, seed=20 + k, spare=(1536 - bound) // 16)
             for k, runs in enumerate([[(12, 1008)], [(1, 0), (5, 512), (6, 0)], [(2, 16 * j) for j in (1, 9, 30, 64, 2, 5)], [(12, 0)], [(3, 128), (9, 976)]])]
    width, pages = 96, max(s["k"].shape[0] for s in steps)
    t = {"q": steps[0]["q"].to(DEV), "k": torch.zeros((pages,) + steps[0]["k"].shape[1:], dtype=dtype, device=DEV), "ctx": torch.ones(n, dtype=torch.int32, device=DEV),
         "v": torch.zeros((pages,) + steps[0]["v"].shape[1:], dtype=dtype, device=DEV), "tables": torch.zeros((n, width), dtype=torch.int32, device=DEV),
         "starts": steps[0]["starts"].to(DEV), "req": steps[0]["req"].to(DEV)}
    data = torch.zeros(2 * groups + 1 + n, dtype=torch.int32, device=DEV)
    host = np.zeros(2 * groups + 1 + n, dtype=np.int32)
    ops.SharedKeys.pack([], n, groups, host)
    data.copy_(torch.from_numpy(host))
    shared = ops.SharedKeys.captured(data, n, groups, bound)
    call = lambda: ops.prefix_attention(t["q"], t["k"], t["v"], t["tables"], t["starts"], t["ctx"], t["req"], steps[0]["scale"], shared, 1, width * 16,  # noqa: E731
                                        max_own_len=own_bound)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for s in steps + steps[::-1]:
        for name in ("q", "k", "v", "ctx"):
            t[name][: s[name].shape[0]].copy_(s[name])
        t["tables"].fill_(-1)
        wide = min(width, s["tables"].shape[1])
        t["tables"][:, :wide].copy_(s["tables"][:, :wide])
        ops.SharedKeys.pack(list(zip(s["counts"], s["lens"])), n, groups, host)
        data.copy_(torch.from_numpy(host))
        graph.replay()
        torch.cuda.synchronize()
        want, size, reach = P.exact(s)
        over = (out.cpu().double() - want).abs() - P.tolerance(s, want, size, reach)
        assert bool(torch.isfinite(out).all()) and float(over.max()) <= 0, float(over.max())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_pages_beyond_two_to_the_31_elements(dtype):
    """The same step at the far end of a pool of more than 2^31 elements (and 2^32 bytes): the same bits."""
    s = P.step([(6, 512), (2, 0)], [1 + 41 * i for i in range(8)], [1] * 7 + [5], 8, 2, 128, 16, dtype, seed=9, poison=False)
    near = _run(s)
    pages, first = s["k"].shape[0], 2 ** 31 // (2 * 16 * 128) + 7
    assert (first + pages) * 2 * 16 * 128 > 2 ** 31
    from tempura_amd.kernels import ops
    k = torch.empty((first + pages,) + s["k"].shape[1:], dtype=dtype, device=DEV)
    v = torch.empty((first + pages,) + s["v"].shape[1:], dtype=dtype, device=DEV)
    k[first:], v[first:] = s["k"].to(DEV), s["v"].to(DEV)
    t = {name: s[name].to(DEV) for name in ("q", "tables", "starts", "ctx", "req")}
    tables = torch.where(t["tables"] >= 0, t["tables"] + first, t["tables"])
    shared = ops.SharedKeys(s["counts"], s["lens"], DEV)
    far = ops.prefix_attention(t["q"], k, v, tables, t["starts"], t["ctx"], t["req"], s["scale"], shared, 5, int(s["ctx"].max()), max_own_len=s["own"])
    assert torch.equal(near, far)


def test_tokens_that_are_not_there_are_not_written():
    """No requests: an empty result.  A step's outputs are its own: the scratch of one call does not reach the next."""
    from tempura_amd.kernels import ops
    none = lambda *shape: torch.empty(shape, dtype=torch.int32, device=DEV)  # noqa: E731
    cache = torch.zeros(3, 2, 16, 64, dtype=BF16, device=DEV)
    out = ops.prefix_attention(torch.empty(0, 4, 64, dtype=BF16, device=DEV), cache, cache.transpose(2, 3).contiguous(), none(0, 1), none(1).zero_(), none(0), none(0), 0.125,
                               ops.SharedKeys([], [], DEV), 1, 1)
    assert out.shape == (0, 256)
    s = P.step([(3, 64)], [5, 6, 7], [1, 1, 1], 4, 2, 64, 16, BF16, seed=1)
    a, b = _run(s), _run(s)
    assert a.data_ptr() != b.data_ptr() and torch.equal(a, b)


def test_refusals():
    from tempura_amd.kernels import ops
    from tempura_amd.kernels.ops import KernelError
    s = P.step([(3, 64)], [5, 6, 7], [1, 1, 1], 4, 2, 64, 16, BF16, seed=1)
    t = {name: s[name].to(DEV) for name in ("q", "k", "v", "tables", "starts", "ctx", "req")}
    good = ops.SharedKeys([3], [64], DEV)

    def call(shared=good, max_ctx=71, **other):
        o = {**t, **other}
        return ops.prefix_attention(o["q"], o["k"], o["v"], o["tables"], o["starts"], o["ctx"], o["req"], 0.125, shared, 1, max_ctx,
                                    max_own_len=o.get("own"), sink=o.get("sink"), softcap=o.get("cap", 0.0))
    call()
    for bad in (dict(shared=ops.SharedKeys([2], [64], DEV)), dict(shared=ops.SharedKeys([3], [80], DEV)), dict(max_ctx=10 ** 6),
                dict(q=t["q"].float()), dict(q=t["q"].transpose(0, 1)), dict(k=t["k"][:, :1].contiguous()), dict(q=t["q"].cpu()),
                dict(own=0), dict(own=72), dict(sink=torch.zeros(3, device=DEV)), dict(cap=-1.0), dict(ctx=t["ctx"].long())):
        with pytest.raises(KernelError):
            call(**bad)
    for counts, lens in (([1], [1, 2]), ([-1], [3]), ([1], [-3])):
        with pytest.raises(KernelError):
            ops.SharedKeys(counts, lens, DEV)

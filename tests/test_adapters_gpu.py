"""A projection with low-rank adapters of many requests against its definition in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def _case(ids, k, n, rank, slots, ends=None, dtype=BF16, seed=0, interleaved=False):
    g = torch.Generator().manual_seed(seed)
    slices = 2 if interleaved else len(ends or [n])
    s = {"x": torch.randn(len(ids), k, generator=g).to(dtype), "w": (torch.randn(n, k, generator=g) * k ** -0.5).to(dtype),
         "a": (torch.randn(slots, slices * rank, k, generator=g) * k ** -0.5).to(dtype), "b": torch.randn(slots, n, rank, generator=g).mul(0.3).to(dtype),
         "scales": torch.rand(slots, generator=g) + 0.5, "ids": torch.tensor(ids, dtype=torch.int32)}
    return s, ends, interleaved


def _exact(s, ends, interleaved, residual=None):
    """(the result in 64 bits, how far a float32 result may be off).  A float32 sum of k products, in whatever order, is off by at most k half
    steps of the sum of their magnitudes (the products of bfloat16 operands are exact in float32, those of float32 operands off by a half
    step each); the low-rank sums carry theirs through the second sum of rank terms, and each sum is rounded a few more times on its way."""
    x, w = s["x"].double(), s["w"].double()
    m, n = x.shape[0], w.shape[0]
    k, rank = x.shape[1], s["b"].shape[2]
    half = 2.0 ** -24
    y, tol = x @ w.t(), (k + 8) * half * (x.abs() @ w.abs().t())
    col = torch.arange(n)
    ends = ends or [n]
    slice_of = (col // 8) % 2 if interleaved else sum((col >= e).long() for e in ends[:-1]) + torch.zeros(n, dtype=torch.long)
    for t, i in enumerate(s["ids"].tolist()):
        if not 0 <= i < s["b"].shape[0]:
            continue
        a, b = s["a"][i].double().view(-1, rank, k), s["b"][i].double()
        v, va = a @ x[t], a.abs() @ x[t].abs()
        y[t] += s["scales"][i].double() * (b * v[slice_of]).sum(1)
        tol[t] += s["scales"][i].double() * (k + rank + 24) * half * (b.abs() * va[slice_of]).sum(1)
    if residual is not None:
        y = y + residual.double()
    return y, tol + 4 * half * y.abs() + (0 if residual is None else 4 * half * residual.double().abs())


def _run(case, residual=None, tiled=True, max_run=0):
    from tempura_amd.kernels import ops
    s, ends, interleaved = case
    t = {name: v.to(DEV) for name, v in s.items()}
    ad = ops.Adapters(t["a"], t["b"], t["scales"], ends, interleaved)
    return ops.adapter_linear(t["x"], ops.tile_weight(t["w"]) if tiled else t["w"], ad, t["ids"], residual=residual, max_run=max_run)


def _check(case, residual=None, **more):
    want, tol = _exact(*case, residual=residual)
    res = None if residual is None else residual.to(DEV)
    got = _run(case, residual=res, **more)
    assert got.dtype == F32 and (res is None or got.data_ptr() == res.data_ptr())
    over = (got.cpu().double() - want).abs() - tol
    assert float(over.max()) <= 0, float(over.max())
    return got


@pytest.fixture(params=["rule", "one launch", "two launches", "together"])
def way(request, monkeypatch):
    """Rows one by one in a launch or in two, and together by adapter, whatever the rule on sizes would take."""
    from tempura_amd.kernels import ops
    if request.param != "rule":
        monkeypatch.setattr(ops, "adapter_row_limits", (0, 0) if request.param == "together" else (1 << 16, 1 << 16))
        monkeypatch.setattr(ops, "adapter_row_weights", {BF16: 1 << 40, F32: 1 << 40})
        monkeypatch.setattr(ops, "adapter_block_bytes", 0 if request.param == "two launches" else 1 << 40)
        monkeypatch.setattr(ops, "adapter_blocks_bytes", 1 << 40)
    return request.param


MANY = [i % 5 - 1 for i in range(70)]
PORTIONS = [3] * 40 + [-1] * 30 + [0] * 17 + [2] + [3] + [1] * 90


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("ids", [[2], [-1], [0, 0, 3, -1, 2, 1, 1], MANY, PORTIONS], ids=["one", "none", "seven", "singles", "portions"])
@pytest.mark.parametrize("k,n,rank", [(512, 320, 16), (264, 1000, 8), (100, 37, 3), (1024, 48, 40), (129, 256, 12)])
def test_rows(dtype, ids, k, n, rank, way):
    """One row to many, rows without an adapter, adapters that several requests share; widths and ranks of every alignment."""
    case = _case(ids, k, n, rank, 4, dtype=dtype, seed=k + len(ids))
    _check(case)
    _check(case, max_run=1)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("ids", [[1, 0, 2], MANY, PORTIONS], ids=["three", "singles", "portions"])
@pytest.mark.parametrize("ends,interleaved", [([64, 80, 96], False), ([100, 101, 400], False), ([17, 300], False), ([320], True), ([1, 2, 3, 4, 5, 6, 7, 333], False)])
def test_slices(dtype, ids, ends, interleaved, way):
    """Stacked projections: slices that end inside a tile, narrow ones, and two that alternate by eights."""
    for rank in (16, 72):
        _check(_case(ids, 256, ends[-1], rank, 4, None if interleaved else ends, dtype, seed=len(ends), interleaved=interleaved))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("ids", [[1, -1, 2], PORTIONS], ids=["three", "portions"])
def test_residual(dtype, ids, way):
    case = _case(ids, 512, 272, 16, 4, dtype=dtype)
    _check(case, residual=torch.randn(len(ids), 272, generator=torch.Generator().manual_seed(4)))


def test_a_row_does_not_hang_on_the_rows_beside_it(way):
    """Rows of other requests move nothing, whatever they hold; ids outside the slots are rows without an adapter."""
    case = _case(PORTIONS, 512, 320, 16, 4)
    first = _run(case)
    other = ({**case[0], "x": case[0]["x"].clone(), "ids": case[0]["ids"].clone()},) + case[1:]
    other[0]["x"][::2] = float("nan")
    other[0]["ids"][::2] = 17
    got = _run(other)
    assert torch.equal(got[1::2], first[1::2]) and bool(torch.isnan(got[::2]).all())


@pytest.mark.parametrize("ids", [[1, -1, 2], PORTIONS], ids=["three", "portions"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("ends,interleaved", [([320], True), ([100, 320], False)])
def test_a_slice_that_is_not_finite_leaves_the_others(ids, dtype, ends, interleaved, way):
    """Low-rank values of one slice that are infinite or no numbers: the other slice's columns, beside or between its own, are as without it."""
    from tempura_amd.kernels import ops
    case = _case(ids, 256, 320, 16, 4, None if interleaved else ends, dtype, seed=3, interleaved=interleaved)
    want, tol = _exact(*case)
    col = torch.arange(320)
    other = (col // 8) % 2 == 1 if interleaved else col >= 100
    case[0]["a"][:, :16] = float("inf")
    got = _run(case).cpu().double()
    assert float(((got - want).abs() - tol)[:, other].max()) <= 0
    some = case[0]["ids"] >= 0
    assert not bool(torch.isfinite(got[some][:, ~other]).any()) and bool(torch.isfinite(got[~some]).all())


def test_no_rows():
    case = _case([], 64, 48, 8, 2)
    assert _run(case).shape == (0, 48) and _run(case, residual=torch.empty(0, 48, device=DEV), max_run=1).shape == (0, 48)


def test_streams_and_graphs(way):
    from tempura_amd.kernels import ops
    for ids in ([0, 3, -1, 2], PORTIONS):
        s, ends, _ = _case(ids, 512, 320, 16, 4, [128, 320])
        t = {name: v.to(DEV) for name, v in s.items()}
        ad, w = ops.Adapters(t["a"], t["b"], t["scales"], ends), ops.tile_weight(t["w"])
        call = lambda: ops.adapter_linear(t["x"], w, ad, t["ids"])  # noqa: E731
        first = call()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            assert torch.equal(call(), first)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        for i in range(4):      # (rows, and who has which adapter, change between replays)
            t["x"].copy_(torch.randn(t["x"].shape, generator=torch.Generator().manual_seed(i)))
            t["ids"].copy_(torch.roll(s["ids"], i))
            graph.replay()
            want = call()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_refusals():
    from tempura_amd.kernels import ops
    from tempura_amd.kernels.ops import KernelError
    s, _, _ = _case([0, 1], 64, 48, 8, 3)
    t = {name: v.to(DEV) for name, v in s.items()}
    ad = ops.Adapters(t["a"], t["b"], t["scales"])
    ops.adapter_linear(t["x"], t["w"], ad, t["ids"])
    for bad in (dict(x=t["x"].float()), dict(x=t["x"][:, :32].contiguous()), dict(ids=t["ids"].long()), dict(ids=t["ids"][:1]), dict(w=t["w"][:32].contiguous()),
                dict(x=t["x"].t()), dict(ids=t["ids"].cpu()), dict(residual=torch.zeros(2, 47, device=DEV))):
        o = {"residual": None, **t, **bad}
        with pytest.raises(KernelError):
            ops.adapter_linear(o["x"], o["w"], ad, o["ids"], residual=o["residual"])
    for a, b, sc, ends, inter in ((t["a"], t["b"], t["scales"], [20, 20, 48], False), (t["a"], t["b"], t["scales"], [24, 40], False),
                                  (t["a"], t["b"].float(), t["scales"], None, False), (t["a"], t["b"], t["scales"][:2], None, False),
                                  (t["a"][:, :6].contiguous(), t["b"], t["scales"], None, False), (t["a"], t["b"], t["scales"], None, True),
                                  (t["a"].cpu(), t["b"], t["scales"], None, False)):
        with pytest.raises(KernelError):
            ops.Adapters(a, b, sc, ends, inter)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_adapters_and_long_rows(dtype, way):
    """More adapters than one pass of the plan takes, most of them with one row; one adapter with rows all over the batch; K in several parts."""
    _check(_case([(i * 37) % 1300 - 1 for i in range(400)], 64, 48, 8, 1299, dtype=dtype))
    _check(_case([0 if i % 3 else (i // 3) % 4 for i in range(700)], 4104, 80, 16, 4, dtype=dtype))

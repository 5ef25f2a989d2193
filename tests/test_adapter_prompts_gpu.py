"""A projection with low-rank adapters for so many rows that its second product takes 128 columns a wave, against its definition in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32
ROWS = 4100


def _ids(kind, slots):
    if kind == "singles":          # (more adapters in a window of 64 rows than blocks that share it out)
        return torch.tensor([(i * 37) % (slots + 1) - 1 for i in range(ROWS)], dtype=torch.int32)
    out, i = torch.full((ROWS,), -1, dtype=torch.int32), 0
    for length, slot in ((1000, 2), (37, -1), (700, 0), (1, 3), (900, 1), (64, 17), (1200, 3)):
        out[i: i + length] = slot
        i += length
    return out


def _exact(t, slice_of, residual):
    """(the result in 64 bits, how far a float32 result may be off).  A float32 sum of k products, in whatever order, is off by at most k half steps of the sum of
    their magnitudes (products of bfloat16 operands are exact in float32, those of float32 operands off by a half step each); the low-rank sums carry theirs
    through the second sum of rank terms, and each sum is rounded a few more times on its way."""
    half, (n, k), rank = 2.0 ** -24, t["w"].shape, t["b"].shape[2]
    x, w = t["x"].double(), t["w"].double()
    y, tol = x @ w.t(), (k + 8) * half * (x.abs() @ w.abs().t())
    for i in range(t["b"].shape[0]):
        rows = (t["ids"] == i).nonzero()[:, 0]
        if rows.numel() == 0:
            continue
        a, b, s = t["a"][i].double(), t["b"][i].double(), t["scales"][i].double()
        for j in range(int(slice_of.max()) + 1):
            cols = (slice_of == j).nonzero()[:, 0]
            aj, bj = a[j * rank: (j + 1) * rank], b[cols]
            y[rows[:, None], cols] += s * (x[rows] @ aj.t()) @ bj.t()
            tol[rows[:, None], cols] += s * (k + rank + 24) * half * ((x[rows].abs() @ aj.abs().t()) @ bj.abs().t())
    if residual is not None:
        y, tol = y + residual.double(), tol + 4 * half * residual.double().abs()
    return y, tol + 4 * half * y.abs()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind,n,ends,rank", [("portions", 2048, None, 16), ("portions", 2048, [1000, 1030, 2048], 72), ("portions", 2048, "alternate", 16),
                                              ("portions", 1538, [700, 1538], 16), ("singles", 2048, [300, 2048], 24), ("singles", 1600, "alternate", 8)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_prompts(dtype, kind, n, ends, rank, with_residual):
    """Slices that end inside a wave's columns, that alternate by eights, columns that are no multiple of four, ranks beyond one pass; rows without an adapter."""
    from tempura_amd.kernels import ops
    k, slots, g = 256, 9 if kind == "singles" else 4, torch.Generator().manual_seed(n + rank)
    alternate = ends == "alternate"
    slices = 2 if alternate else len(ends or [n])
    t = {"x": torch.randn(ROWS, k, generator=g).to(dtype), "w": (torch.randn(n, k, generator=g) * k ** -0.5).to(dtype),
         "a": (torch.randn(slots, slices * rank, k, generator=g) * k ** -0.5).to(dtype), "b": torch.randn(slots, n, rank, generator=g).mul(0.3).to(dtype),
         "scales": torch.rand(slots, generator=g) + 0.5, "ids": _ids(kind, slots)}
    residual = torch.randn(ROWS, n, generator=g) if with_residual else None
    col = torch.arange(n)
    slice_of = (col // 8) % 2 if alternate else sum((col >= e).long() for e in (ends or [n])[:-1]) + torch.zeros(n, dtype=torch.long)
    assert -(-ROWS // 64) * -(-n // 512) >= 192          # (what the wide form is taken from on)
    want, tol = _exact(t, slice_of, residual)
    d = {name: v.to(DEV) for name, v in t.items()}
    ad = ops.Adapters(d["a"], d["b"], d["scales"], None if alternate else ends, alternate)
    run = lambda: ops.adapter_linear(d["x"], ops.tile_weight(d["w"]), ad, d["ids"], residual=None if residual is None else residual.to(DEV))  # noqa: E731
    got = run()
    over = (got.cpu().double() - want).abs() - tol
    assert got.dtype == F32 and float(over.max()) <= 0, float(over.max())
    assert torch.equal(run(), got)

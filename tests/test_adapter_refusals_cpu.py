"""Operands of adapters that lie on different devices are refused, on the host."""
import pytest
import torch


class Elsewhere(torch.Tensor):
    """A host tensor that names another device as its own than the current one."""

    def get_device(self):
        return 3


@pytest.fixture
def launched(monkeypatch):
    from tempura_amd.kernels import ops
    made = []
    monkeypatch.setattr(ops, "_dev_ok", lambda *ts: None)
    monkeypatch.setattr(ops, "_call", lambda name, *args, tag=None: made.append(name))
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "linear", lambda x, w, dt, residual=None, **kw: made.append("linear") or torch.zeros(x.shape[0], w.shape[0]))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)      # (what host tensors name as theirs)
    return made


def test_operands_of_several_devices(launched):
    from tempura_amd.kernels import ops
    a, b, scales = torch.zeros(3, 8, 64), torch.zeros(3, 48, 8), torch.zeros(3)
    for where in ((a.to("meta"), b, scales), (a, b.to("meta"), scales), (a, b, scales.to("meta"))):
        with pytest.raises(ops.KernelError, match="one device"):
            ops.Adapters(*where)
    good = dict(x=torch.zeros(2, 64), w=torch.zeros(48, 64), ids=torch.zeros(2, dtype=torch.int32), residual=torch.zeros(2, 48))
    ad = ops.Adapters(a, b, scales)
    for name in good:
        o = {**good, name: good[name].as_subclass(Elsewhere)}
        with pytest.raises(ops.KernelError, match="current device"):
            ops.adapter_linear(o["x"], o["w"], ad, o["ids"], residual=o["residual"])
    with pytest.raises(ops.KernelError, match="current device"):
        ops.adapter_linear(good["x"], ops.TiledWeight(torch.zeros(3, 2, 64, 8).as_subclass(Elsewhere), 48, 64), ad, good["ids"])
    with pytest.raises(ops.KernelError, match="current device"):
        ops.adapter_linear(good["x"], good["w"], ops.Adapters(a.as_subclass(Elsewhere), b, scales), good["ids"])
    assert not launched
    ops.adapter_linear(good["x"], good["w"], ad, good["ids"])
    assert launched == ["linear", "tp_adapter_add"]


def test_tensors_are_kept_or_copied_as_documented(launched):
    """Kept where the kernels can read them as they are; with ranks that are no multiple of 8, or a b at an odd place, both are copied once."""
    from tempura_amd.kernels import ops
    a, b, scales = torch.randn(3, 8, 64), torch.randn(3, 48, 8), torch.ones(3)
    ad = ops.Adapters(a, b, scales)
    assert ad.a.data_ptr() == a.data_ptr() and ad.b.data_ptr() == b.data_ptr() and ad.scales is scales
    odd = torch.randn(3 * 48 * 8 + 1)[1:].view(3, 48, 8)
    assert odd.data_ptr() % 16 != 0
    ad = ops.Adapters(a, odd, scales)
    assert ad.b.data_ptr() % 16 == 0 and torch.equal(ad.b, odd) and torch.equal(ad.a, a) and ad.a.data_ptr() != a.data_ptr()
    ad = ops.Adapters(a[:, :5].contiguous(), b[..., :5].contiguous(), scales)
    assert ad.rank == 8 and torch.equal(ad.a[:, :5], a[:, :5]) and torch.equal(ad.b[..., :5], b[..., :5]) and not ad.a[:, 5:].any() and not ad.b[..., 5:].any()

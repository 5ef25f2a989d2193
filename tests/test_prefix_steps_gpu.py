"""Which kernels an engine's steps run behind a held prefix, and what the steps that read shared keys once compute."""
import pytest
import torch

import helpers
import plain

pytestmark = pytest.mark.gpu


@pytest.fixture
def launches(monkeypatch):
    """The library's calls, and the steps whose attention takes the projection's rows, by name."""
    from tempura_amd.kernels import ops
    made, call, rows = [], ops._call, ops.attention_rows
    monkeypatch.setattr(ops, "_call", lambda name, *a, **kw: (made.append(name), call(name, *a, **kw))[1])
    monkeypatch.setattr(ops, "attention_rows", lambda *a, **kw: (made.append("attention_rows"), rows(*a, **kw))[1])
    return made


def _generate(tiny_dirs, dtype, prefix, tails, n, **kw):
    from tempura_amd.engine import Engine
    from tempura_amd.sampling import SamplingParams
    eng = Engine(tiny_dirs.path("D", dtype), dtype=dtype, page_size=16, kv_pages=128, max_batch_size=6, max_num_batched_tokens=96, prefill_chunk_size=40, max_prefixes=1, **kw)
    return eng.generate(tails, SamplingParams(temperature=0.0, max_new_tokens=n), prefix=eng.hold_prefix(prefix))


@pytest.mark.parametrize("kw", [dict(use_graph=False), dict(), dict(chain_steps=False)], ids=["eager", "captured and chained", "captured"])
def test_steps_that_read_shared_keys_once(tiny_dirs, monkeypatch, launches, kw):
    """Eager, captured and chained steps all launch the kernel, single tokens and portions, and give the plain model's tokens."""
    from tempura_amd.kernels import ops
    monkeypatch.setattr(ops, "shared_keys_pay_bytes", 0)
    monkeypatch.setattr(ops, "prefix_least_keys", (0, 0, 0))
    cfg, W = tiny_dirs.plain_model("D")
    prefix, tails = helpers.random_tokens(cfg["vocab_size"], 70, seed=3), [helpers.random_tokens(cfg["vocab_size"], n, seed=n) for n in (5, 33, 1, 60, 12)]
    got = _generate(tiny_dirs, "float32", prefix, tails, 9, **kw)
    assert got == [plain.greedy_generate(cfg, W, prefix + t, 9) for t in tails]
    # (two layers; eager: every step that several requests share)
    assert launches.count("tp_prefix_attention") >= (2 * 9 if kw.get("use_graph") is False else 2 * 2)

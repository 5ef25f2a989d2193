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


@pytest.mark.parametrize("kind", ["rows", "plain"])
def test_steps_that_do_not_are_as_without(launches, kind):
    """Where each request reads its keys for itself, because they are few, a step keeps the kernels that it has without runs of requests: the one that takes the
    projection's rows (of an attention with a norm per head), or the attention with the order of its requests; the same bits."""
    from tempura_amd.cache import LayerCache
    from tempura_amd.config.spec import PartSpec
    from tempura_amd.kernels import ops
    from tempura_amd.parts import build_part
    heads, kv, dim, width, page, dev = 8, 2, 64, 128, 16, "cuda:0"
    g = torch.Generator().manual_seed(1)
    shapes = {"q": (heads * dim, width), "k": (kv * dim, width), "v": (kv * dim, width), "o": (width, heads * dim), "qn": (dim,), "kn": (dim,)}
    weights = {n: torch.randn(*s, generator=g) * 0.1 for n, s in shapes.items()}
    more = {"qk_norm": {"eps": 1e-6}} if kind == "rows" else {}
    part = build_part("mixer", PartSpec("attention", {"num_heads": heads, "num_kv_heads": kv, "head_dim": dim, "scale": 0.125, **more,
                                                      "position": PartSpec("rope", {"head_dim": dim, "rotary_dim": dim, "theta": 1e4})},
                                        {"q": "q", "k": "k", "v": "v", "o": "o", "q_norm": "qn", "k_norm": "kn"}), width, torch.bfloat16, dev)
    part.load_weights(lambda n: weights[n])
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    r, lens = 5, [50, 61, 49, 80, 70]

    class Ctx:
        positions, token_req, cu_seqlens, context_lens = i32(*[n - 1 for n in lens]), i32(*range(r)), i32(*range(r + 1)), i32(*lens)
        block_tables = [i32(*[[0, 1, 2] + [3 + 3 * i + j for j in range(3)] for i in range(r)])]
        slot_mapping = [i32(*[(3 + 3 * i + (n - 1 - 48) // page) * page + (n - 1) % page for i, n in enumerate(lens)])]
        max_q_len, max_context_len, num_single, num_tokens, num_requests, max_own_len = 1, 80, r, r, r, 32
        shared_keys = None
    pools = [torch.randn(20, kv, page, dim, generator=g).to(torch.bfloat16).to(dev), torch.randn(20, kv, dim, page, generator=g).to(torch.bfloat16).to(dev)]
    x = torch.randn(r, width, generator=g).to(torch.bfloat16).to(dev)

    def step(shared_keys):
        del launches[:]
        Ctx.shared_keys, Ctx.shared = shared_keys, {}
        return part.forward(x, Ctx, LayerCache(0, {"k": pools[0].clone(), "v": pools[1].clone()}, True, page, None), torch.zeros(r, width, device=dev)), list(launches), dict(Ctx.shared)
    residual, real = [], part.forward
    part.forward = lambda x, ctx, cache, h: (real(x, ctx, cache, h), residual.append(h))[0]
    _, made, kept = step(None)
    _, again, kept_again = step(ops.SharedKeys([r], [48], dev))
    assert made == again and ("attention_rows" in made) == (kind == "rows") and kept.keys() == kept_again.keys()
    assert torch.equal(residual[0], residual[1]) and float(residual[0].abs().max()) > 0

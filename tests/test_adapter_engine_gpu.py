"""Requests with adapters through the engine on the GPU: mixed steps, captured and chained decode steps, both element types."""
import pytest
import torch

import adapter_cases
import helpers
import plain

pytestmark = pytest.mark.gpu


def _engine(tiny_dirs, name, dtype, **kw):
    from tempura_amd.engine import Engine
    args = dict(dtype=dtype, page_size=helpers.PAGE_SIZE[name], kv_pages=128, max_batch_size=6, max_num_batched_tokens=96, prefill_chunk_size=40,
                max_adapters=3, max_adapter_rank=8)
    args.update(kw)
    return Engine(tiny_dirs.path(name, dtype), **args)


@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
@pytest.mark.parametrize("graph", [True, False])
def test_greedy_generation_matches_plain(tiny_dirs, name, graph):
    """float32: the tokens of the plain model with each request's adapter merged in; requests without one beside them."""
    from tempura_amd.sampling import SamplingParams
    cfg, W = tiny_dirs.plain_model(name)
    sets = {"one": (adapter_cases.make(W, 1), 1.5), "two": (adapter_cases.make(W, 2, rank=8, targets=("q_proj", "v_proj", "down_proj")), 0.5)}
    eng = _engine(tiny_dirs, name, "float32", use_graph=graph)
    for key, (pairs, scale) in sets.items():
        eng.load_adapter(key, pairs, scale=scale)
    prompts = [helpers.random_tokens(cfg["vocab_size"], n, seed=n) for n in (9, 70, 33, 5, 1)]
    names = ["one", None, "two", "one", "two"]
    got = eng.generate(prompts, SamplingParams(temperature=0.0, max_new_tokens=12), adapters=names)
    for p, a, o in zip(prompts, names, got):
        assert o == plain.greedy_generate(cfg, W if a is None else adapter_cases.merged(W, *sets[a]), p, 12)
    assert (eng.stats()["graph_steps"] > 0) == graph
    # nobody with an adapter: the tokens of an engine without room for any
    alone = _engine(tiny_dirs, name, "float32", max_adapters=0).generate(prompts, SamplingParams(temperature=0.0, max_new_tokens=12))
    assert eng.generate(prompts, SamplingParams(temperature=0.0, max_new_tokens=12)) == alone


@pytest.mark.parametrize("name", ["C", "D"])
def test_bfloat16_logits_against_plain(tiny_dirs, name):
    """Prompts and single tokens in bfloat16 against the plain model on merged weights, within the bound that every bfloat16 engine test here is held to: a
    small multiple of what rounding the stored rows of the same request to bfloat16 moves (the adapters' share is added to float32 sums and rounds no further row)."""
    from tempura_amd.engine import StepEntry
    cfg, W = tiny_dirs.plain_model(name, "bfloat16")
    pairs = adapter_cases.make(W, 4, rank=8, dtype=torch.bfloat16)
    eng = _engine(tiny_dirs, name, "bfloat16")
    eng.load_adapter("a", pairs, scale=1.0)
    toks = [helpers.random_tokens(cfg["vocab_size"], n, seed=n) for n in (50, 17)]
    r = eng.runner
    for rid, adapted in (("x", True), ("y", False)):
        r.add_request(rid)
        if adapted:
            r.adapter_of[rid] = eng._adapters["a"]
    got = {"x": [], "y": []}
    cuts = [((0, 40), (0, 9)), ((40, 9), (9, 7)), ((49, 1), (16, 1))]
    for (sx, cx), (sy, cy) in cuts:
        logits = r.step([StepEntry("x", toks[0][sx: sx + cx], [cx - 1]), StepEntry("y", toks[1][sy: sy + cy], [cy - 1])]).double().cpu()
        got["x"].append((sx + cx - 1, logits[0]))
        got["y"].append((sy + cy - 1, logits[1]))
    for rid, t, weights in (("x", toks[0], adapter_cases.merged(W, pairs, 1.0)), ("y", toks[1], W)):
        ref, bound = helpers.plain_reference(cfg, weights, t, "bfloat16")
        places = [place for place, _ in got[rid]]
        assert float((torch.stack([row for _, row in got[rid]]) - ref[places]).abs().max() / ref.abs().max()) <= bound
    for rid in got:
        r.end_request(rid)


def test_captured_and_eager_steps_agree(tiny_dirs):
    from tempura_amd.sampling import SamplingParams
    cfg, W = tiny_dirs.plain_model("D", "bfloat16")
    pairs = adapter_cases.make(W, 6, rank=8, dtype=torch.bfloat16)
    prompts = [helpers.random_tokens(cfg["vocab_size"], n, seed=80 + n) for n in (3, 30, 21)]
    out = []
    for kw in (dict(), dict(use_graph=False), dict(chain_steps=False)):
        eng = _engine(tiny_dirs, "D", "bfloat16", **kw)
        eng.load_adapter("a", pairs, scale=1.0)
        out.append(eng.generate(prompts, SamplingParams(temperature=0.0, max_new_tokens=16), adapters=["a", None, "a"]))
    assert out[0] == out[1] == out[2]


def test_an_adapter_that_takes_anothers_place(tiny_dirs):
    """Unloaded and replaced between requests: captured steps read the new tensors."""
    from tempura_amd.sampling import SamplingParams
    cfg, W = tiny_dirs.plain_model("A")
    eng = _engine(tiny_dirs, "A", "float32", max_adapters=1)
    p = helpers.random_tokens(cfg["vocab_size"], 20, seed=9)
    for seed in (1, 2):
        pairs = adapter_cases.make(W, seed)
        eng.load_adapter("a", pairs, scale=1.0)
        assert eng.generate([p], SamplingParams(temperature=0.0, max_new_tokens=10), adapters="a") == [plain.greedy_generate(cfg, adapter_cases.merged(W, pairs, 1.0), p, 10)]
        eng.unload_adapter("a")
    with pytest.raises(ValueError):
        eng.add_request(p, adapter="a")

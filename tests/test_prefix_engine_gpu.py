"""Requests that begin with the pages of a held prefix, on the GPU: tokens of the plain model on whole prompts in eager, captured and chained steps."""
import pytest
import torch

import adapter_cases
import helpers
import plain

pytestmark = pytest.mark.gpu


@pytest.fixture
def always(monkeypatch):
    """Shared keys are read once however little that saves; counts the calls."""
    from tempura_amd.kernels import ops
    monkeypatch.setattr(ops, "shared_keys_pay_bytes", 0)
    calls, real = [], ops.prefix_attention

    def counted(*a, **kw):
        calls.append(a[9])
        return real(*a, **kw)
    monkeypatch.setattr(ops, "prefix_attention", counted)
    return calls


def _engine(tiny_dirs, name, dtype, **kw):
    from tempura_amd.engine import Engine
    args = dict(dtype=dtype, page_size=helpers.PAGE_SIZE[name], kv_pages=128, max_batch_size=6, max_num_batched_tokens=96, prefill_chunk_size=40, max_prefixes=3)
    args.update(kw)
    return Engine(tiny_dirs.path(name, dtype), **args)


@pytest.mark.parametrize("name", ["A", "B", "D", "E"])
@pytest.mark.parametrize("kw", [dict(), dict(use_graph=False), dict(chain_steps=False)])
def test_tokens_are_those_of_whole_prompts(tiny_dirs, always, name, kw):
    """float32; two prefixes at a time, requests without one, requests that join and end at different steps, one prefix released on the way."""
    from tempura_amd.sampling import SamplingParams
    cfg, W = tiny_dirs.plain_model(name)
    vocab, ps = cfg["vocab_size"], helpers.PAGE_SIZE[name]
    eng = _engine(tiny_dirs, name, "float32", **kw)
    one, two = helpers.random_tokens(vocab, 3 * ps + 5, seed=1), helpers.random_tokens(vocab, 2 * ps, seed=2)
    a, b = eng.hold_prefix(one), eng.hold_prefix(two)
    tails = [helpers.random_tokens(vocab, n, seed=n) for n in (7, 1, 41, 3, 11, 2, 5, 9)]
    which = [(a, one), (b, two), (a, one), (None, []), (b, two), (a, one), (a, one), (None, [])]
    lengths = [6, 14, 9, 12, 14, 14, 3, 8]
    rids = [eng.add_request(t, SamplingParams(temperature=0.0, max_new_tokens=n), prefix=p) for t, (p, _), n in zip(tails[:6], which, lengths)]
    for _ in range(4):
        eng.step()
    eng.release_prefix(b)
    late = eng.hold_prefix(two + one)      # (between steps of others, one of them queued ahead)
    eng.step()
    tails.append(tails[0])
    which.append((late, two + one))
    lengths.append(5)
    rids += [eng.add_request(t, SamplingParams(temperature=0.0, max_new_tokens=n), prefix=p) for t, (p, _), n in zip(tails[6:], which[6:], lengths[6:])]
    while eng.has_unfinished():
        eng.step()
    for rid, t, (_, tokens), n in zip(rids, tails, which, lengths):
        assert eng.request(rid).output == plain.greedy_generate(cfg, W, tokens + t, n)
    assert always and (eng.stats()["graph_steps"] > 0) == kw.get("use_graph", True)
    eng.release_prefix(a)
    eng.release_prefix(late)
    assert eng.runner.cache.free_pages() == [128]


def test_bfloat16_logits_against_plain(tiny_dirs, always):
    """Portions and single tokens of two requests behind a prefix, captured and eager, within the bound of every bfloat16 engine test here."""
    from tempura_amd.engine import StepEntry
    cfg, W = tiny_dirs.plain_model("D", "bfloat16")
    ps, vocab = helpers.PAGE_SIZE["D"], cfg["vocab_size"]
    eng = _engine(tiny_dirs, "D", "bfloat16")
    prefix = helpers.random_tokens(vocab, 4 * ps, seed=1)
    eng.hold_prefix(prefix)
    donor, r = next(iter(eng._prefixes.values()))[0], eng.runner
    tails = {"x": helpers.random_tokens(vocab, 30, seed=2), "y": helpers.random_tokens(vocab, 19, seed=3)}
    got = {rid: [] for rid in tails}
    for rid in tails:
        r.add_request(rid)
        r.cache.share(rid, donor, 4 * ps)
    at = {rid: 0 for rid in tails}
    for cx, cy in ((27, 16), (1, 1), (1, 1), (1, 1)):
        entries = []
        for rid, c in (("x", cx), ("y", cy)):
            entries.append(StepEntry(rid, tails[rid][at[rid]: at[rid] + c], [c - 1]))
            at[rid] += c
        logits = r.step(entries).double().cpu()
        for rid, row in zip(tails, logits):
            got[rid].append((4 * ps + at[rid] - 1, row))
    for rid, tail in tails.items():
        ref, bound = helpers.plain_reference(cfg, W, prefix + tail, "bfloat16")
        places = [place for place, _ in got[rid]]
        assert float((torch.stack([row for _, row in got[rid]]) - ref[places]).abs().max() / ref.abs().max()) <= bound
        r.end_request(rid)
    assert len(always) > 0


def test_prefixes_and_adapters_together(tiny_dirs, always):
    from tempura_amd.sampling import SamplingParams
    cfg, W = tiny_dirs.plain_model("D")
    ps, vocab = helpers.PAGE_SIZE["D"], cfg["vocab_size"]
    pairs = adapter_cases.make(W, 6, rank=8)
    tokens, tails = helpers.random_tokens(vocab, 2 * ps + 3, seed=1), [helpers.random_tokens(vocab, n, seed=n) for n in (4, 12, 1, 30)]
    eng = _engine(tiny_dirs, "D", "float32", max_adapters=2, max_adapter_rank=8)
    eng.load_adapter("a", pairs, scale=1.0)
    p, q = eng.hold_prefix(tokens, adapter="a"), eng.hold_prefix(tokens)
    greedy = SamplingParams(temperature=0.0, max_new_tokens=10)
    rids = [eng.add_request(t, greedy, prefix=(p, q)[i % 2], adapter=("a", None)[i % 2]) for i, t in enumerate(tails)]
    while eng.has_unfinished():
        eng.step()
    for i, (rid, t) in enumerate(zip(rids, tails)):
        assert eng.request(rid).output == plain.greedy_generate(cfg, (adapter_cases.merged(W, pairs, 1.0), W)[i % 2], tokens + t, 10)
    assert always

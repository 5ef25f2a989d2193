"""Requests that begin with the pages of a held prefix, on the host: bookkeeping, tokens against the plain implementation, refusals."""
import pytest
import torch

import adapter_cases
import helpers
import plain


@pytest.fixture
def emu(monkeypatch):
    from tempura_amd.kernels import ops

    class Emu(adapter_cases.Emu):
        seen = []

        def prefix_attention(self, q, k_cache, v_cache, block_tables, cu_seqlens, context_lens, token_req, scale, shared, max_q_len, max_context_len,
                             max_own_len=None, *rest):
            # what the runs say is so: their requests' tables begin alike, and no bound is exceeded
            page = k_cache.shape[2]
            for g in range(shared.groups):
                lo, hi, keys = int(shared.starts[g]), int(shared.starts[g + 1]), int(shared.keys[g])
                assert shared.each[lo:hi].tolist() == [keys] * (hi - lo) and keys % page == 0 and keys <= shared.max_keys
                assert bool((block_tables[lo:hi, : keys // page] == block_tables[lo:lo + 1, : keys // page]).all())
            new = cu_seqlens[1:] - cu_seqlens[:-1]
            assert bool((context_lens - new >= shared.each).all()) and int((context_lens - shared.each).max()) <= max_own_len
            Emu.seen.append((shared.max_keys, max_q_len))
            return super().prefix_attention(q, k_cache, v_cache, block_tables, cu_seqlens, context_lens, token_req, scale, shared, max_q_len, max_context_len,
                                            max_own_len, *rest)
    Emu.seen.clear()
    ops.set_backend(Emu())
    monkeypatch.setattr(ops, "shared_keys_pay_bytes", 0)
    yield Emu
    ops.set_backend(None)


class _Greedy:
    def sample(self, logits, params, *a, **kw):
        return logits.argmax(1).tolist()


def _engine(tiny_dirs, name="A", **kw):
    from tempura_amd.engine import Engine
    args = dict(dtype="float32", device="cpu", page_size=helpers.PAGE_SIZE[name], kv_pages=64, max_batch_size=4, max_num_batched_tokens=48,
                prefill_chunk_size=16, max_prefixes=2)
    args.update(kw)
    eng = Engine(tiny_dirs.path(name, "float32"), **args)
    eng.sampler = _Greedy()
    return eng


def _greedy(n):
    from tempura_amd.sampling import SamplingParams
    return SamplingParams(temperature=0.0, max_new_tokens=n)


@pytest.mark.parametrize("name", ["A", "B", "D", "E"])
def test_tokens_are_those_of_whole_prompts(tiny_dirs, emu, name):
    """Prefixes that end inside a page and at its end, requests with and without one, two prefixes at a time; every page comes back."""
    cfg, W = tiny_dirs.plain_model(name)
    vocab, ps = cfg["vocab_size"], helpers.PAGE_SIZE[name]
    eng = _engine(tiny_dirs, name)
    one, two = helpers.random_tokens(vocab, 3 * ps + 5, seed=1), helpers.random_tokens(vocab, 2 * ps, seed=2)
    a, b = eng.hold_prefix(one), eng.hold_prefix(two)
    tails = [helpers.random_tokens(vocab, n, seed=n) for n in (7, 1, 20, 3, 11)]
    which = [(a, one), (b, two), (a, one), (None, []), (b, two)]
    rids = [eng.add_request(t, _greedy(6), prefix=p) for t, (p, _) in zip(tails, which)]
    while eng.has_unfinished():
        eng.step()
        assert eng.runner.cache._lib.cc_check(eng.runner.cache._h) == 0
    for rid, t, (_, tokens) in zip(rids, tails, which):
        assert eng.request(rid).output == plain.greedy_generate(cfg, W, tokens + t, 6)
    assert any(keys == 3 * ps for keys, _ in emu.seen)
    eng.release_prefix(a)
    eng.release_prefix(b)
    assert eng.runner.cache.free_pages() == [64] and not eng.runner.cache.live_requests() and eng.scheduler.pages_kept == 0


def test_a_prefix_that_is_released_while_requests_have_it(tiny_dirs, emu):
    cfg, W = tiny_dirs.plain_model("A")
    eng = _engine(tiny_dirs)
    tokens = helpers.random_tokens(cfg["vocab_size"], 40, seed=3)
    p = eng.hold_prefix(tokens)
    tails = [helpers.random_tokens(cfg["vocab_size"], n, seed=n) for n in (4, 9)]
    rids = [eng.add_request(t, _greedy(8), prefix=p) for t in tails]
    eng.step()
    eng.release_prefix(p)
    late = eng.add_request(tails[0], _greedy(3))
    while eng.has_unfinished():
        eng.step()
        assert eng.runner.cache._lib.cc_check(eng.runner.cache._h) == 0
    for rid, t in zip(rids, tails):
        assert eng.request(rid).output == plain.greedy_generate(cfg, W, tokens + t, 8)
    assert eng.request(late).output == plain.greedy_generate(cfg, W, tails[0], 3)
    assert eng.runner.cache.free_pages() == [64]


def test_preempted_requests_begin_with_the_prefix_again(tiny_dirs, emu):
    cfg, W = tiny_dirs.plain_model("A")
    tokens = helpers.random_tokens(cfg["vocab_size"], 32, seed=4)
    tails = [helpers.random_tokens(cfg["vocab_size"], 14, seed=70 + i) for i in range(2)]
    for release in (False, True):
        eng = _engine(tiny_dirs, kv_pages=2 + 4, admit_headroom=None)
        p = eng.hold_prefix(tokens)
        rids = [eng.add_request(t, _greedy(40), prefix=p) for t in tails]
        for _ in range(3):
            eng.step()
        if release:
            eng.release_prefix(p)
        while eng.has_unfinished():
            eng.step()
        assert eng.scheduler.num_preemptions > 0
        assert [eng.request(r).output for r in rids] == [plain.greedy_generate(cfg, W, tokens + t, 40) for t in tails]


def test_prefixes_with_adapters(tiny_dirs, emu):
    cfg, W = tiny_dirs.plain_model("A")
    pairs = adapter_cases.make(W, 8)
    eng = _engine(tiny_dirs, max_adapters=1)
    eng.load_adapter("a", pairs, scale=1.0)
    tokens, tail = helpers.random_tokens(cfg["vocab_size"], 35, seed=5), helpers.random_tokens(cfg["vocab_size"], 6, seed=6)
    p, q = eng.hold_prefix(tokens, adapter="a"), eng.hold_prefix(tokens)
    with pytest.raises(ValueError):
        eng.add_request(tail, prefix=p)
    with pytest.raises(ValueError):
        eng.add_request(tail, prefix=q, adapter="a")
    with pytest.raises(ValueError):
        eng.unload_adapter("a")
    rids = [eng.add_request(tail, _greedy(5), prefix=p, adapter="a"), eng.add_request(tail, _greedy(5), prefix=q), eng.add_request(tail, _greedy(5), prefix=p, adapter="a")]
    while eng.has_unfinished():
        eng.step()
    assert eng.generate([tail, tail[:2]], _greedy(4), adapters="a", prefix=p) == \
        [plain.greedy_generate(cfg, adapter_cases.merged(W, pairs, 1.0), tokens + t, 4) for t in (tail, tail[:2])]
    for wrong in (dict(prefix=p), dict(prefix=q, adapters=[None, "a"]), dict(prefix=77)):
        with pytest.raises(ValueError):
            eng.generate([tail, tail], _greedy(2), **wrong)
    assert not eng.has_unfinished()
    with_one = plain.greedy_generate(cfg, adapter_cases.merged(W, pairs, 1.0), tokens + tail, 5)
    assert [eng.request(r).output for r in rids] == [with_one, plain.greedy_generate(cfg, W, tokens + tail, 5), with_one]
    eng.release_prefix(p)
    eng.unload_adapter("a")


def test_refusals(tiny_dirs, emu):
    eng = _engine(tiny_dirs, kv_pages=8, max_seq_len=200)
    vocab = eng.model.spec.vocab_size
    for tokens in ([1] * 15, [], [vocab] * 32, [-1] * 32, [1] * 199):
        with pytest.raises(ValueError):
            eng.hold_prefix(tokens)
    for call in (lambda: eng.add_request([1], prefix=9), lambda: eng.hold_prefix([1] * 32, adapter="x")):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(KeyError):
        eng.release_prefix(3)
    p = eng.hold_prefix([1] * 40)
    with pytest.raises(ValueError):
        eng.add_request([], prefix=p)
    with pytest.raises(ValueError):      # 8 pages, two of them held
        eng.add_request([1] * 90, _greedy(20))
    eng.add_request([1] * 60, _greedy(20), prefix=p)      # (116 tokens and more, two pages of them shared)
    with pytest.raises(ValueError):
        eng.hold_prefix([2] * 32)
    while eng.has_unfinished():
        eng.step()
    eng.hold_prefix([2] * 32)
    with pytest.raises(ValueError):
        eng.hold_prefix([3] * 32)      # (two are held)
    with pytest.raises(ValueError):
        _engine(tiny_dirs, "C")        # (layers with a window give pages back)
    with pytest.raises(ValueError):
        _engine(tiny_dirs, max_prefixes=0).hold_prefix([1] * 32)


def test_the_cache_shares_whole_pages():
    from tempura_amd.cache.manager import CacheManager
    from tempura_amd.parts.base import CacheSpec
    spec = CacheSpec("full", 1, 8)
    c = CacheManager([spec], 4, 10, 5)
    for r in "abc":
        c.add(r)
    c.reserve("a", 11)
    c.commit("a", 11)
    for bad in (lambda: c.share("b", "a", 0), lambda: c.share("b", "a", 6), lambda: c.share("b", "a", 12), lambda: c.share("a", "a", 4), lambda: c.share("a", "b", 4)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(KeyError):
        c.share("z", "a", 4)
    c.share("b", "a", 8)
    c.share("c", "b", 4)
    assert c.num_tokens("b") == 8 and c.table("b", 0) == c.table("a", 0)[:2] and c.table("c", 0) == c.table("a", 0)[:1] and c.free_pages() == [7]
    assert c.shared("b")[1] == 8 and c.shared("c") != c.shared("b") and c.shared("a") is None
    c.reserve("b", 5)
    c.commit("b", 5)
    assert c.free_pages() == [5] and len(set(c.table("a", 0) + c.table("b", 0))) == 5 and c._lib.cc_check(c._h) == 0
    with pytest.raises(ValueError):      # (the next token would be written into a page that others read)
        c.truncate("b", 6)
    with pytest.raises(ValueError):
        c.truncate("a", 3)
    assert c.waste_ratio() == pytest.approx(1 - (4 + 4 + 3 + 4 + 1) / 20)      # (a's, of which the first two pages are b's too and the first is c's; b's own)
    c.truncate("a", 8)
    c.truncate("b", 4)
    assert c.shared("b") is None and c._lib.cc_check(c._h) == 0
    c.release("a")
    assert c.waste_ratio() == 0.0      # (one page, full, that b and c have)
    assert c.free_pages() == [9] and c._lib.cc_check(c._h) == 0
    c.release("c")
    c.release("b")
    assert c.free_pages() == [10] and c._lib.cc_check(c._h) == 0
    w = CacheManager([spec, CacheSpec("window", 1, 8, 8)], 4, 10, 5)
    w.add("a"), w.add("b")
    w.reserve("a", 8), w.commit("a", 8)
    with pytest.raises(ValueError):
        w.share("b", "a", 4)
    assert w._lib.cc_share(w._h, w.state_slot("b"), w.state_slot("a"), 4) != 0


def test_runs_of_a_captured_step():
    import numpy as np
    from tempura_amd.kernels import ops
    out = np.empty(2 * 5 + 1 + 9, dtype=np.int32)
    ops.SharedKeys.pack([(2, 32), (1, 0), (3, 16)], 9, 5, out)
    s = ops.SharedKeys.captured(torch.from_numpy(out), 9, 5, 64)
    assert s.starts.tolist() == [0, 2, 3, 6, 9, 9] and s.keys.tolist() == [32, 0, 16, 0, 0] and s.each.tolist() == [32, 32, 0, 16, 16, 16, 0, 0, 0]
    with pytest.raises(ops.KernelError):      # (three that share, room for two)
        ops.SharedKeys.pack([(2, 32), (1, 0), (2, 16), (1, 0), (2, 64)], 9, 5, out)
    with pytest.raises(ops.KernelError):
        ops.SharedKeys.pack([(2, 32), (8, 0)], 9, 5, out)
    import random
    rng = random.Random(2)
    for _ in range(500):
        runs, left = [], ops.SharedKeys.runs_in(17)
        for _ in range(rng.randint(1, 40)):
            v = 16 * rng.choice((0, 0, 1, 5, 9)) if left else 0
            runs.append((rng.randint(1, 4), v))
            left -= v > 0
        n = sum(c for c, _ in runs) + rng.randint(0, 5)
        out = np.empty(2 * 17 + 1 + n, dtype=np.int32)
        ops.SharedKeys.pack(runs, n, 17, out)
        s = ops.SharedKeys.captured(torch.from_numpy(out), n, 17, 256)
        assert s.each.tolist() == [v for c, v in runs for _ in range(c)] + [0] * (n - sum(c for c, _ in runs))
        assert s.starts.tolist() == sorted(s.starts.tolist()) and int(s.starts[-1]) == n
        for g in range(17):
            assert s.each[s.starts[g]: s.starts[g + 1]].tolist() == [int(s.keys[g])] * int(s.starts[g + 1] - s.starts[g])


def test_a_captured_step_keeps_the_runs_that_save_most(tiny_dirs, emu):
    eng = _engine(tiny_dirs, kv_pages=64, max_batch_size=32)
    cache, runner = eng.runner.cache, eng.runner
    cache.add("d")
    cache.reserve("d", 10 * 16), cache.commit("d", 10 * 16)
    rids = []
    for g in range(10):
        for i in range(2):
            rids.append((g, i))
            cache.add((g, i))
            cache.share((g, i), "d", 16 * (g + 1))
    assert runner._shared_runs(rids) == [(2, 16 * (g + 1)) for g in range(10)]
    kept = runner._shared_runs(rids, 8)
    assert kept == [(2, 16 * (g + 1) if g >= 2 else 0) for g in range(10)]
    assert runner._shared_bounds(rids) == (256, 256, 8)      # (keys for themselves: 17 to 33)
    assert runner._shared_bounds(rids[:6]) == (256, 256, 4) and runner._shared_bounds(rids[:2]) == (256, 256, 1)


def test_when_shared_keys_pay():
    """By what reading them once saves a layer: less for short portions, more for long ones."""
    from tempura_amd.kernels import ops
    mib = 1 << 20
    for longest, least in ((1, 96), (2, 8), (64, 8), (65, 96), (128, 96), (512, 384), (2048, 1536)):
        assert ops.shared_keys_pay(least * mib, longest) and not ops.shared_keys_pay(least * mib - 1, longest)

"""When shared keys are read once for all, and how such a launch is laid out, on the host."""
import random

import pytest
import torch


@pytest.fixture
def launched(monkeypatch):
    """What the entry point hands to the library: its name for steps that read shared keys once, "paged" for the others."""
    from tempura_amd.kernels import ops
    made = []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)      # (what host tensors name as theirs)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_call", lambda name, *args, tag=None: made.append((name, args)))
    monkeypatch.setattr(ops, "paged_attention", lambda *a, **kw: made.append(("paged", kw)))
    return made


def attend(launched, singles, portion, shared, own, portion_own, heads=32, kv=8, dim=128, dtype=torch.bfloat16, page=16, **kw):
    """The kind of launch of a step of one portion and single tokens behind the same keys."""
    from tempura_amd.kernels import ops
    new = ([portion] if portion else []) + [1] * singles
    ctx = ([shared + portion_own] if portion else []) + [shared + own] * singles
    r, n, longest = len(new), sum(new), max(ctx)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    del launched[:]
    ops.prefix_attention(torch.empty(n, heads, dim, dtype=dtype), torch.empty(2, kv, page, dim, dtype=dtype), torch.empty(2, kv, dim, page, dtype=dtype),
                         torch.zeros(r, -(-longest // page), dtype=torch.int32), torch.tensor([0] + new).cumsum(0).int(), i32(ctx),
                         i32([i for i, t in enumerate(new) for _ in range(t)]), 0.1, ops.SharedKeys([r], [shared], "cpu"), max(new), longest,
                         max_own_len=max(own, portion_own if portion else 0), num_single=singles, **kw)
    return "paged" if launched[0][0] == "paged" else "once"


def test_portions_beside_requests_with_many_keys_of_their_own(launched):
    """A part of own keys is walked by one block: not beside a portion, where that would take longer than reading the shared keys for each request."""
    go = lambda *a, **kw: attend(launched, *a, **kw)  # noqa: E731
    assert go(32, 512, 8192, 32768, 512) == "paged" and go(32, 512, 8192, 8192, 512) == "paged" and go(32, 128, 2048, 4000, 128) == "paged"
    assert go(8, 128, 2048, 100, 20000) == "paged"
    assert go(32, 512, 8192, 1000, 512) == "once" and go(8, 128, 2048, 1000, 128) == "once" and go(32, 64, 2048, 1000, 64) == "once"
    assert go(32, 2, 2048, 16000, 2) == "once"         # (blocks of 16 rows are cut over their waves and parts)
    assert go(33, 0, 8192, 32768, 0) == "once"         # (and single tokens alone)
    for dtype in (torch.bfloat16, torch.float32):
        for portion in (30, 100, 500):
            kinds = [go(16, portion, 8192, own, portion, dtype=dtype) for own in (100, 1000, 4000, 16000, 64000, 256000)]
            assert kinds == sorted(kinds, key=lambda k: k == "paged") and kinds[0] == "once" and kinds[-1] == "paged"


def test_blocks_hold_the_rows_of_every_step():
    """As many blocks of rows as the runs can have at most, however their tokens are spread over the requests, and for every replay of a captured step."""
    from tempura_amd.kernels import ops
    rng = random.Random(9)
    for _ in range(2000):
        counts = [rng.choice((1, 2, 7, 40)) for _ in range(rng.choice((1, 2, 9)))]
        lengths = [16 * rng.choice((0, 1, 30, 4000)) for _ in counts]
        shared = ops.SharedKeys(counts, lengths, "cpu")
        if not shared.max_keys:
            continue
        r, kvh, group, longest = sum(counts), rng.choice((1, 2, 8)), rng.choice((1, 3, 4, 8, 34)), rng.choice((1, 2, 30, 400))
        new = [rng.choice((1, longest, rng.randint(1, longest))) for _ in range(r)]
        plan = ops._prefix_plan(shared, r, sum(new), group, kvh, longest, rng.choice((256, 4096)), rng.choice((32, 64, 128)), rng.choice((torch.bfloat16, torch.float32)))
        at, need = 0, 0
        for c, v in zip(counts, lengths):
            need += -(-sum(new[at: at + c]) * group // plan[0]) if v else 0
            at += c
        assert plan[2] >= need


def test_blocks_hold_the_rows_of_every_replay():
    from tempura_amd.kernels import ops
    rng = random.Random(10)
    for _ in range(2000):
        groups, r, group = rng.choice((3, 5, 9, 17)), rng.choice((2, 8, 64, 200)), rng.choice((1, 3, 4, 8, 34))
        data = torch.zeros(2 * groups + 1 + r, dtype=torch.int32)
        shared = ops.SharedKeys.captured(data, r, groups, 16 * rng.choice((16, 64, 512)))
        plan = ops._prefix_plan(shared, r, r, group, rng.choice((1, 2, 8)), 1, 512, 128, torch.bfloat16)
        runs, left = [], r
        for _ in range(rng.randint(1, ops.SharedKeys.runs_in(groups))):
            if left:
                runs.append((rng.randint(1, left), 16 * rng.randint(1, shared.max_keys // 16)))
                left -= runs[-1][0]
        out = data.numpy()
        ops.SharedKeys.pack(runs, r, groups, out)
        assert plan[2] >= sum(-(-(int(shared.starts[g + 1]) - int(shared.starts[g])) * group // plan[0]) for g in range(groups) if int(shared.keys[g]))
        assert plan[3] * plan[4] * 32 >= shared.max_keys


def test_the_engine_and_the_operator_ask_the_same(launched, tiny_dirs):
    """Keys that the operator would read for each request are no shared keys of a step, however many bytes that would save; nor are those of a model whose heads or
    pages the kernel is not built for."""
    from tempura_amd.kernels import ops
    from tempura_amd.engine import Engine
    for requests, keys, once in ((98, 256, False), (40, 640, False), (50, 512, False), (64, 768, True), (193, 256, True), (2, 800, True)):
        assert ops.prefix_keys_pay([(requests, keys)], torch.bfloat16, 1) == once
        assert attend(launched, requests, 0, keys, 100, 0) == ("once" if once else "paged")
    for name, page, sizes in (("D", 16, True), ("D", 8, False), ("A", 16, False), ("E", 16, False)):
        runner = Engine(tiny_dirs.path(name, "float32"), dtype="float32", device="cpu", page_size=page, kv_pages=256, max_batch_size=8, max_prefixes=1).runner
        runner._key_bytes = 1 << 30
        cache = runner.cache
        cache.add("d"), cache.reserve("d", 640), cache.commit("d", 640)
        for keys in (512, 496, 640):
            for i in range(3):
                cache.add((keys, i)), cache.share((keys, i), "d", keys)
        assert runner._reads_once == sizes
        for keys, enough in ((512, True), (496, False), (640, True)):       # (float32: from 512 on)
            rids = [(keys, i) for i in range(3)]
            assert runner._shared_runs(rids) == ([(3, keys)] if sizes and enough else None)
            assert (runner._shared_bounds(rids) is not None) == (sizes and enough)


def test_runs_of_eager_steps_travel_like_their_other_inputs(tiny_dirs, monkeypatch):
    """New runs of requests go to the device through the runner's ring of pinned buffers: the host does not wait for the steps in flight."""
    from tempura_amd.engine import Engine
    from tempura_amd.kernels import ops
    monkeypatch.setattr(ops, "shared_keys_pay_bytes", 0)
    runner = Engine(tiny_dirs.path("A", "float32"), dtype="float32", device="cpu", page_size=16, kv_pages=256, max_batch_size=8, max_prefixes=1).runner
    cache, sent, real = runner.cache, [], runner._runs_staging.send
    cache.add("d"), cache.reserve("d", 64), cache.commit("d", 64)
    for i in range(4):
        cache.add(i), cache.share(i, "d", 64)
    runner._runs_staging.send = lambda n: (sent.append(n), real(n))[1]
    monkeypatch.setattr(ops.torch, "tensor", lambda *a, **kw: pytest.fail("a copy that waits"))
    from tempura_amd.engine.runner import StepEntry
    for rids in ([0, 1], [0, 1, 2], [0, 1]):
        _, ctx = runner._pack_step([StepEntry(i, [5], [0]) for i in rids])
        n = len(rids)
        assert ctx.shared_keys.starts.tolist() == [0, n] and ctx.shared_keys.keys.tolist() == [64] and ctx.shared_keys.each.tolist() == [64] * n
    assert sent == [2 + 1 + 2, 2 + 1 + 3]       # (the third step's runs are the first's, which are there)


def test_caches_at_odd_places_are_refused(launched):
    """Keys and values go to LDS in pieces of 16 bytes from where they lie."""
    from tempura_amd.kernels import ops
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    shared, q = ops.SharedKeys([3], [1024], "cpu"), torch.empty(3, 4, 64, dtype=torch.bfloat16)

    def call(offset_k, offset_v, q=q):
        k, v = (torch.empty(2 * 2 * 16 * 64 + 8, dtype=torch.bfloat16)[o: o + 2 * 2 * 16 * 64] for o in (offset_k, offset_v))
        return ops.prefix_attention(q, k.view(2, 2, 16, 64), v.view(2, 2, 64, 16), torch.zeros(3, 70, dtype=torch.int32), i32(0, 1, 2, 3), i32(1030, 1031, 1032),
                                    i32(0, 1, 2), 0.125, shared, 1, 1032, max_own_len=8)
    for k, v in ((1, 0), (0, 4), (4, 4), (2, 6)):
        with pytest.raises(ops.KernelError, match="16 bytes"):
            call(k, v)
    assert not launched
    call(8, 0)
    call(0, 0, torch.empty(3 * 4 * 64 + 1, dtype=torch.bfloat16)[1:].view(3, 4, 64))       # (q is read with ordinary loads, from anywhere)
    assert [name for name, _ in launched] == ["tp_prefix_attention"] * 2

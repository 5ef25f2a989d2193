"""Adapters on the host: what the engine does with them over plain stand-ins, folders and their faults, and every refusal of the operations."""
import os

import pytest
import torch

import adapter_cases
import helpers
import plain


@pytest.fixture
def emu():
    from tempura_amd.kernels import ops
    ops.set_backend(adapter_cases.Emu())
    yield
    ops.set_backend(None)


def _engine(tiny_dirs, name, **kw):
    from tempura_amd.engine import Engine
    args = dict(dtype="float32", device="cpu", page_size=helpers.PAGE_SIZE[name], kv_pages=64, max_batch_size=4, max_num_batched_tokens=48,
                prefill_chunk_size=16, max_adapters=2, max_adapter_rank=6)
    args.update(kw)
    return Engine(tiny_dirs.path(name, "float32"), **args)


class _Greedy:
    def sample(self, logits, params, *a, **kw):
        return logits.argmax(1).tolist()


@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_requests_with_adapters_beside_requests_without(tiny_dirs, emu, name, tmp_path):
    """Every request's tokens are those of the plain model with its adapter merged in; rows of other requests move nothing."""
    from tempura_amd.sampling import SamplingParams
    cfg, W = tiny_dirs.plain_model(name)
    one, two = adapter_cases.make(W, 1), adapter_cases.make(W, 2, rank=6, targets=("q_proj", "down_proj"))
    eng = _engine(tiny_dirs, name)
    eng.sampler = _Greedy()
    eng.load_adapter("one", one, scale=1.5)
    eng.load_adapter("two", adapter_cases.write(str(tmp_path / "two"), two, 6, 3))
    prompts = [helpers.random_tokens(cfg["vocab_size"], n, seed=n) for n in (9, 33, 17, 5)]
    names = ["one", None, "two", "one"]
    got = eng.generate(prompts, SamplingParams(temperature=0.0, max_new_tokens=6), adapters=names)
    weights = {"one": adapter_cases.merged(W, one, 1.5), "two": adapter_cases.merged(W, two, 0.5), None: W}
    for p, a, o in zip(prompts, names, got):
        assert o == plain.greedy_generate(cfg, weights[a], p, 6)
    base = [plain.greedy_generate(cfg, W, p, 6) for p in prompts]
    assert any(a != b for a, b in zip(got, base))      # (the adapters are large enough to show)


def test_load_unload_and_refusals(tiny_dirs, emu):
    from tempura_amd.sampling import SamplingParams
    cfg, W = tiny_dirs.plain_model("A")
    pairs = adapter_cases.make(W, 3)
    eng = _engine(tiny_dirs, "A")
    eng.sampler = _Greedy()
    some = sorted(pairs)[0]
    a, b = pairs[some]
    for bad, scale in (({}, 1.0), ({"model.norm.weight": (a, b)}, 1.0), ({some: (a[:, 1:], b)}, 1.0), ({some: (a, b[1:])}, 1.0), ({some: (a[:2], b)}, 1.0),
                       ({some: (torch.zeros(7, a.shape[1]), torch.zeros(b.shape[0], 7 + 2))}, 1.0), ({some: (a, b)}, None),
                       ({some: (torch.zeros(9, a.shape[1]), torch.zeros(b.shape[0], 9))}, 1.0)):
        with pytest.raises(ValueError):
            eng.load_adapter("bad", bad, scale=scale)
    assert len(eng._free_adapters) == 2
    eng.load_adapter("x", pairs, scale=1.0)
    eng.load_adapter("y", pairs, scale=-1.0)
    for call in (lambda: eng.load_adapter("x", pairs, scale=1.0), lambda: eng.load_adapter("z", pairs, scale=1.0),
                 lambda: eng.add_request([1, 2], adapter="z"), lambda: eng.generate([[1]], adapters=["x", "x"]), lambda: eng.generate([[1], [2]], adapters="nobody")):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(KeyError):
        eng.unload_adapter("z")
    rid = eng.add_request([1, 2, 3], SamplingParams(temperature=0.0, max_new_tokens=3), adapter="x")
    with pytest.raises(ValueError):
        eng.unload_adapter("x")
    while eng.has_unfinished():
        eng.step()
    assert rid not in eng.runner.adapter_of
    eng.unload_adapter("x")
    # a slot that another adapter had holds nothing of it
    few = {some: pairs[some]}
    eng.load_adapter("few", few, scale=2.0)
    p = helpers.random_tokens(cfg["vocab_size"], 12, seed=4)
    assert eng.generate([p], SamplingParams(temperature=0.0, max_new_tokens=5), adapters="few") == [plain.greedy_generate(cfg, adapter_cases.merged(W, few, 2.0), p, 5)]
    rid = eng.add_request([1, 2, 3], adapter="few")
    eng.abort(rid)
    eng.unload_adapter("few")
    with pytest.raises(ValueError):
        _engine(tiny_dirs, "A", max_adapters=0).load_adapter("x", pairs, scale=1.0)


def test_preempted_requests_keep_their_adapter(tiny_dirs, emu):
    from tempura_amd.sampling import SamplingParams
    cfg, W = tiny_dirs.plain_model("A")
    pairs = adapter_cases.make(W, 5)
    ps = helpers.PAGE_SIZE["A"]
    eng = _engine(tiny_dirs, "A", kv_pages=52 // ps, admit_headroom=None)
    eng.sampler = _Greedy()
    eng.load_adapter("a", pairs, scale=1.0)
    prompts = [helpers.random_tokens(cfg["vocab_size"], 18, seed=60 + i) for i in range(2)]
    got = eng.generate(prompts, SamplingParams(temperature=0.0, max_new_tokens=20), adapters=["a", None])
    assert eng.scheduler.num_preemptions > 0
    assert got == [plain.greedy_generate(cfg, adapter_cases.merged(W, pairs, 1.0), prompts[0], 20), plain.greedy_generate(cfg, W, prompts[1], 20)]


def test_folders_and_their_faults(tiny_dirs, tmp_path):
    from tempura_amd.weights.adapters import read_adapter
    from tempura_amd.weights.loader import WeightsError
    from tempura_amd.weights.safetensors_io import write_safetensors
    _, W = tiny_dirs.plain_model("A")
    pairs = adapter_cases.make(W, 7)
    got, scale = read_adapter(adapter_cases.write(str(tmp_path / "a"), pairs, 4, 8))
    assert scale == 2.0 and sorted(got) == sorted(pairs) and all(torch.equal(got[n][i], pairs[n][i]) for n in pairs for i in (0, 1))
    assert read_adapter(adapter_cases.write(str(tmp_path / "b"), pairs, 4, 8, use_rslora=True))[1] == 4.0
    for i, more in enumerate((dict(use_dora=True), dict(bias="all"), dict(modules_to_save=["lm_head"]), dict(r=0), dict(rank_pattern={"q_proj": 3}))):
        with pytest.raises(WeightsError):
            read_adapter(adapter_cases.write(str(tmp_path / f"c{i}"), pairs, 4, 8, **more))
    folder = adapter_cases.write(str(tmp_path / "d"), pairs, 4, 8)
    path = os.path.join(folder, "adapter_model.safetensors")
    one = sorted(pairs)[0][: -len(".weight")]
    for tensors in ([("base_model.model." + one + ".lora_A.weight", torch.zeros(4, 4))], [("lm_head.weight", torch.zeros(4, 4))], []):
        write_safetensors(path, tensors)
        with pytest.raises(WeightsError):
            read_adapter(folder)
    os.remove(path)
    with pytest.raises(WeightsError):
        read_adapter(folder)


def test_models_of_other_blocks_take_none(emu, tmp_path):
    from tempura_amd.engine import Engine
    import mifutar_cases
    folder = mifutar_cases.write_model("mix", str(tmp_path / "m"))
    with pytest.raises(ValueError, match="takes adapters"):
        Engine(folder, dtype="float32", device="cpu", kv_pages=8, max_batch_size=2, max_adapters=1)


# ---- the operations' refusals, and what they hand to the library ----------------------------------------------------------
@pytest.fixture
def calls(monkeypatch):
    from tempura_amd.kernels import ops
    made = []
    monkeypatch.setattr(ops, "_dev_ok", lambda *ts: [ops._need(t is None or t.is_contiguous(), "operand is not contiguous") for t in ts])
    monkeypatch.setattr(ops, "_call", lambda name, *args, tag=None: made.append((name, args)))
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)      # (what host tensors name as theirs)
    monkeypatch.setattr(ops, "linear", lambda x, w, dt, residual=None, **kw: residual if residual is not None else torch.zeros(x.shape[0], w.shape[0]))
    return made


def test_adapter_refusals(calls):
    from tempura_amd.kernels import ops
    from tempura_amd.kernels.ops import KernelError
    a, b, sc = torch.zeros(3, 8, 64), torch.zeros(3, 48, 8), torch.zeros(3)
    for args in ((a, b, sc, [20, 20, 48]), (a, b, sc, [24, 40]), (a, b.bfloat16(), sc), (a, b, sc[:2]), (a[:, :6].contiguous(), b, sc), (a, b, sc, None, True),
                 (a, b, sc.double()), (a.half(), b.half(), sc), (a, b[..., :0], sc), (a, b, sc, [8 * i for i in range(1, 10)]), (a, b.transpose(1, 2), sc)):
        with pytest.raises(KernelError):
            ops.Adapters(*args)
    ad = ops.Adapters(a, b, sc)
    x, w, ids = torch.zeros(2, 64), torch.zeros(48, 64), torch.zeros(2, dtype=torch.int32)
    for kw in (dict(x=x.bfloat16()), dict(x=torch.zeros(2, 32)), dict(ids=ids.long()), dict(ids=ids[:1]), dict(w=w[:32]), dict(x=torch.zeros(64, 2).t()), dict(ids=ids[None]),
               dict(residual=torch.zeros(2, 47)), dict(residual=torch.zeros(2, 48).double())):
        o = {"x": x, "w": w, "ids": ids, "residual": None, **kw}
        with pytest.raises(KernelError):
            ops.adapter_linear(o["x"], o["w"], ad, o["ids"], residual=o["residual"])
    assert not calls
    ops.adapter_linear(x, w, ad, ids)
    ops.adapter_linear(torch.zeros(0, 64), w, ad, ids[:0])
    assert [c[0] for c in calls] == ["tp_adapter_add"]
    with pytest.MonkeyPatch.context() as mp:
        mp.setattr(torch.cuda, "current_device", lambda: 1)
        with pytest.raises(KernelError, match="current device"):
            ops.adapter_linear(x, w, ad, ids)
    wide = ops.Adapters(torch.zeros(2, 6, 64), torch.zeros(2, 48, 3), sc[:2], [10, 48])      # (ranks padded once)
    assert wide.rank == 8 and tuple(wide.a.shape) == (2, 16, 64) and tuple(wide.b.shape) == (2, 48, 8)


def test_shared_keys_refusals(calls, monkeypatch):
    from tempura_amd.kernels import ops
    monkeypatch.setattr(ops, "prefix_least_keys", (0, 0, 0))
    from tempura_amd.kernels.ops import KernelError
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    good = dict(q=torch.zeros(3, 4, 64), k=torch.zeros(9, 2, 16, 64), v=torch.zeros(9, 2, 64, 16), t=torch.zeros(3, 6, dtype=torch.int32), cu=i32(0, 1, 2, 3),
                ctx=i32(70, 71, 72), req=i32(0, 1, 2), shared=ops.SharedKeys([3], [64], "cpu"), max_ctx=72, own=8, sink=None, cap=0.0, q_len=1)

    def call(scale=0.125, **kw):
        o = {**good, **kw}
        return ops.prefix_attention(o["q"], o["k"], o["v"], o["t"], o["cu"], o["ctx"], o["req"], scale, o["shared"], o["q_len"], o["max_ctx"], max_own_len=o["own"],
                                    sink=o["sink"], softcap=o["cap"])
    for kw in (dict(shared=ops.SharedKeys([2], [64], "cpu")), dict(shared=ops.SharedKeys([3], [80], "cpu")), dict(max_ctx=97), dict(q=good["q"].bfloat16()),
               dict(q=torch.zeros(4, 3, 64).transpose(0, 1)), dict(k=torch.zeros(9, 3, 16, 64)), dict(v=torch.zeros(9, 2, 16, 64)), dict(own=0), dict(own=73),
               dict(sink=torch.zeros(3)), dict(cap=-1.0), dict(ctx=good["ctx"].long()), dict(cu=i32(0, 1, 2)), dict(req=i32(0, 1)), dict(t=good["t"][0]),
               dict(q=torch.zeros(2, 4, 64)), dict(q_len=0), dict(t=good["t"].long()), dict(scale=0.0),
               dict(scale=-1.0), dict(max_ctx=64)):
        with pytest.raises(KernelError):
            call(**kw)
    assert not calls
    call()
    call(own=None)
    assert [c[0] for c in calls] == ["tp_prefix_attention"] * 2
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    with pytest.raises(KernelError, match="current device"):
        call()
    for counts, lens in (([1], [1, 2]), ([-1], [3]), ([1], [-3]), ([1], [2 ** 31])):
        with pytest.raises(KernelError):
            ops.SharedKeys(counts, lens, "cpu")
    with pytest.raises(KernelError):
        ops.SharedKeys([2, 2], [16, 0], "cpu", requests=3)
    s = ops.SharedKeys([2, 0, 1], [32, 7, 0], "cpu", requests=5)
    assert s.starts.tolist() == [0, 2, 3, 5] and s.keys.tolist() == [32, 0, 0] and s.each.tolist() == [32, 32, 0, 0, 0] and (s.max_keys, s.max_requests, s.sharing) == (32, 2, 1)


def test_parts_fit_every_size():
    """The parts that a launch is laid out in: within the kernel's limits, and enough for the longest keys, whatever the sizes."""
    import random
    from tempura_amd.kernels import ops
    rng = random.Random(3)
    for _ in range(3000):
        counts = [rng.choice((1, 2, 7, 64)) for _ in range(rng.choice((1, 2, 40)))]
        shared = ops.SharedKeys(counts, [rng.choice((0, 1, 16, 500, 70000, 10 ** 6)) for _ in counts], "cpu")
        if not shared.max_keys:
            continue
        kvh, group, q = rng.choice((1, 2, 8, 32)), rng.choice((1, 3, 4, 8, 34)), rng.choice((1, 1, 2, 30, 400))
        r = sum(counts)
        n, own = rng.randint(r, r * q), rng.choice((1, 256, 4096, 10 ** 6))
        rows, own_rows, blocks, steps, parts, own_steps, own_parts = ops._prefix_plan(shared, r, n, group, kvh, q, own, rng.choice((32, 64, 128)),
                                                                                     rng.choice((torch.bfloat16, torch.float32)))
        assert (rows, own_rows) in ((16, 16), (64, 16), (128, 16), (64, 64), (128, 64), (128, 128))
        assert parts >= 1 and own_parts >= 1 and parts + own_parts <= 128
        assert steps * parts * 32 >= shared.max_keys and own_steps * own_parts * 32 >= own + 15
        assert own_rows >= min(128, q * group) or own_rows == 128
        # (at least as many blocks of rows as the runs can have, however their tokens are spread)
        assert blocks >= sum(-(-c * group // rows) for c, _ in shared._runs if q == 1 and n == r)

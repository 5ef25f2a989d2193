"""Holding a prefix beside live requests whose pages it would need, on the host."""
import pytest

import adapter_cases
import helpers
import plain


def test_a_prefix_takes_no_pages_from_running_requests(tiny_dirs):
    """Refused as a whole where too few pages are free, before a token of it is computed; requests go on, and it is held once they have ended."""
    from tempura_amd.cache import PagesExhausted
    from tempura_amd.engine import Engine
    from tempura_amd.kernels import ops
    from tempura_amd.sampling import SamplingParams
    ops.set_backend(adapter_cases.Emu())
    try:
        cfg, W = tiny_dirs.plain_model("A")
        eng = Engine(tiny_dirs.path("A", "float32"), dtype="float32", device="cpu", page_size=16, kv_pages=8, max_batch_size=4, max_num_batched_tokens=32,
                     prefill_chunk_size=16, max_prefixes=1, admit_headroom=None)
        eng.sampler = type("Greedy", (), {"sample": lambda self, logits, *a, **kw: logits.argmax(1).tolist()})()
        prompts = [helpers.random_tokens(cfg["vocab_size"], 40, seed=i) for i in (1, 2)]
        greedy = SamplingParams(temperature=0.0, max_new_tokens=6)
        rids = [eng.add_request(p, greedy) for p in prompts]
        for _ in range(4):
            eng.step()
        free, steps = eng.runner.cache.free_pages(), eng.runner.steps_run
        assert free == [2]
        prefix = helpers.random_tokens(cfg["vocab_size"], 64, seed=3)
        with pytest.raises(PagesExhausted):
            eng.hold_prefix(prefix)
        assert eng.runner.steps_run == steps and eng.runner.cache.free_pages() == free and eng.scheduler.pages_kept == 0
        while eng.has_unfinished():
            eng.step()
        assert [eng.request(r).output for r in rids] == [plain.greedy_generate(cfg, W, p, 6) for p in prompts]
        held = eng.hold_prefix(prefix)
        assert eng.runner.cache.free_pages() == [4]
        assert eng.generate([[7, 8]], greedy, prefix=held) == [plain.greedy_generate(cfg, W, prefix + [7, 8], 6)]
    finally:
        ops.set_backend(None)

"""What the attention part hands to the attention of shared keys, on the host."""
import pytest
import torch

import adapter_cases


@pytest.mark.parametrize("more", [{}, {"softcap": 3.0}, {"sink": True}, {"sink": 1.5, "softcap": 2.0}, {"qk_norm": {"eps": 1e-6}}], ids=str)
def test_sinks_caps_and_scales_are_handed_over(more):
    """A part with each of its options gives the same rows whether the step's requests are named as runs that share keys or not."""
    from tempura_amd.cache import LayerCache
    from tempura_amd.config.spec import PartSpec
    from tempura_amd.kernels import ops
    from tempura_amd.parts import build_part
    heads, kv, dim, width, page, seen = 4, 2, 16, 32, 16, []

    class Emu(adapter_cases.Emu):
        def prefix_attention(self, q, k_cache, v_cache, block_tables, cu_seqlens, context_lens, token_req, scale, shared, max_q_len, max_context_len,
                             max_own_len=None, num_single=None, sink=None, softcap=0.0):
            seen.append((shared.max_keys, max_own_len, num_single))
            options = {**({"sink": sink} if sink is not None else {}), **({"softcap": softcap} if softcap else {})}
            return self.paged_attention(q, k_cache, v_cache, block_tables, cu_seqlens, context_lens, token_req, scale, 0, max_q_len, max_context_len, **options)
    g = torch.Generator().manual_seed(1)
    shapes = {"q": (heads * dim, width), "k": (kv * dim, width), "v": (kv * dim, width), "o": (width, heads * dim), "s": (heads,), "qn": (dim,), "kn": (dim,)}
    weights = {n: torch.randn(*s, generator=g) for n, s in shapes.items()}
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731

    class Ctx:
        positions, token_req, cu_seqlens, context_lens = i32(19, 20, 17), i32(0, 0, 1), i32(0, 2, 3), i32(21, 18)
        block_tables, slot_mapping, shared = [i32(0, 1, 0, 2).view(2, 2)], [i32(16 + 3, 16 + 4, 32 + 1)], {}
        max_q_len, max_context_len, num_single, num_tokens, num_requests, max_own_len, shared_keys = 2, 21, 1, 3, 2, 5, None
    pools = [torch.randn(4, kv, page, dim, generator=g), torch.randn(4, kv, dim, page, generator=g)]
    x = torch.randn(3, width, generator=g)
    ops.set_backend(Emu())
    try:
        part = build_part("mixer", PartSpec("attention", {"num_heads": heads, "num_kv_heads": kv, "head_dim": dim, "scale": 0.3, **more,
                                                          "position": PartSpec("rope", {"head_dim": dim, "rotary_dim": dim, "theta": 1e4})},
                                            {"q": "q", "k": "k", "v": "v", "o": "o", "sink": "s", "q_norm": "qn", "k_norm": "kn"}), width, torch.float32, "cpu")
        part.load_weights(lambda n: weights[n])
        out = []
        for Ctx.shared_keys in (None, ops.SharedKeys([2], [16], "cpu")):
            h = torch.zeros(3, width)
            y = part.forward(x, Ctx, LayerCache(0, {"k": pools[0].clone(), "v": pools[1].clone()}, True, page, None), h)
            out.append(h if y is None else h + y if y.data_ptr() != h.data_ptr() else y)
    finally:
        ops.set_backend(None)
    assert seen == [(16, 5, 1)] and float(out[0].abs().max()) > 0
    assert torch.equal(out[0], out[1])

"""Adapters for the tiny models, and what a model with one computes: the plain implementation on merged weights."""
import json
import os

import torch

from emu_ops import EmuOps
from tempura_amd.weights.safetensors_io import write_safetensors

TARGETS = ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj")


def make(W, seed, rank=4, targets=TARGETS, dtype=torch.float32, scale=0.25):
    """base tensor name -> (A, B) beside every matrix whose name holds one of ``targets``."""
    g = torch.Generator().manual_seed(seed)
    out = {}
    for name, w in sorted(W.items()):
        if any(t in name for t in targets):
            out[name] = ((torch.randn(rank, w.shape[1], generator=g) * w.shape[1] ** -0.5).to(dtype), (torch.randn(w.shape[0], rank, generator=g) * scale).to(dtype))
    return out


def merged(W, pairs, scale):
    return {name: w + scale * pairs[name][1].double() @ pairs[name][0].double() if name in pairs else w for name, w in W.items()}


def write(folder, pairs, rank, alpha, **more):
    os.makedirs(folder, exist_ok=True)
    with open(os.path.join(folder, "adapter_config.json"), "w") as f:
        json.dump({"r": rank, "lora_alpha": alpha, "bias": "none", **more}, f)
    write_safetensors(os.path.join(folder, "adapter_model.safetensors"),
                      [("base_model.model." + n[: -len(".weight")] + f".lora_{h}.weight", t) for n, p in pairs.items() for h, t in zip("AB", p)])
    return folder


class Emu(EmuOps):
    """The host stand-ins with the operations of adapters and of shared keys."""

    def adapter_linear(self, x, w, adapters, ids, residual=None):
        y = x.double() @ w.double().t()
        rank, col = adapters.rank, torch.arange(adapters.n)
        which = (col // 8) % 2 if adapters.interleaved else sum((col >= e).long() for e in list(adapters.ends)[:-1]) + torch.zeros(adapters.n, dtype=torch.long)
        for t, i in enumerate(ids.tolist()):
            if 0 <= i < adapters.slots:
                v = adapters.a[i].double().view(-1, rank, x.shape[1]) @ x[t].double()
                y[t] += adapters.scales[i].double() * (adapters.b[i].double() * v[which]).sum(1)
        if residual is not None:
            residual.copy_((residual.double() + y).float())
            return residual
        return y.float()

    def prefix_attention(self, q, k_cache, v_cache, block_tables, cu_seqlens, context_lens, token_req, scale, shared, max_q_len, max_context_len,
                         max_own_len=None, num_single=None, sink=None, softcap=0.0):
        return self.paged_attention(q, k_cache, v_cache, block_tables, cu_seqlens, context_lens, token_req, scale, 0, max_q_len, max_context_len)

"""Low-rank adapters from a folder as adapter libraries publish them: ``adapter_config.json`` (``r``, ``lora_alpha``, ``use_rslora``) and
``adapter_model.safetensors`` with ``base_model.model.<matrix>.lora_A.weight`` [rank, inputs] and ``.lora_B.weight`` [outputs, rank],
<matrix>.weight being the name of the tensor of the base checkpoint that they stand beside.  All faults are reported in one error."""
from __future__ import annotations

import json
import math
import os
from typing import Dict, Tuple

import torch

from .loader import WeightsError
from .safetensors_io import SafetensorsError, SafetensorsFile

PREFIX, HALVES = "base_model.model.", (".lora_A.weight", ".lora_B.weight")
#: keys of the configuration that ask for something else than W x + scale B A x when they are set
REFUSED = ("use_dora", "modules_to_save", "fan_in_fan_out", "rank_pattern", "alpha_pattern", "layer_replication", "trainable_token_indices")


def read_adapter(folder: str) -> Tuple[Dict[str, Tuple[torch.Tensor, torch.Tensor]], float]:
    """(base tensor name -> (A, B), scale)."""
    try:
        with open(os.path.join(folder, "adapter_config.json"), encoding="utf-8") as f:
            config = json.load(f)
    except (OSError, ValueError) as e:
        raise WeightsError(f"{folder}: adapter_config.json: {e}") from e
    faults = [f"{key} = {config[key]!r}" for key in REFUSED if config.get(key)]
    if config.get("bias", "none") != "none":
        faults.append(f"bias = {config['bias']!r}")
    rank, alpha = config.get("r"), config.get("lora_alpha")
    if not (isinstance(rank, int) and rank > 0 and isinstance(alpha, (int, float))):
        faults.append(f"r = {rank!r}, lora_alpha = {alpha!r}")
    if faults:
        raise WeightsError(f"{folder}: adapter_config.json asks for what is not supported: " + "; ".join(faults))
    path = os.path.join(folder, "adapter_model.safetensors")
    try:
        file = SafetensorsFile(path)
    except (OSError, SafetensorsError) as e:
        raise WeightsError(f"{path}: {e}") from e
    halves: Dict[str, dict] = {}
    unexpected, wrong = [], {}
    try:
        for name in file.names():
            half = next((h for h in HALVES if name.endswith(h)), None)
            if half is None or not name.startswith(PREFIX):
                unexpected.append(name)
                continue
            if file.dtype_tag(name) not in ("F32", "BF16", "F16"):
                wrong[name] = (("F32", "BF16", "F16"), file.dtype_tag(name))
                continue
            halves.setdefault(name[len(PREFIX): -len(half)] + ".weight", {})[half] = file.tensor(name).to(torch.float32)
    finally:
        file.close()
    missing = [PREFIX + base[: -len(".weight")] + h for base, got in halves.items() for h in HALVES if h not in got and PREFIX + base[: -len(".weight")] + h not in wrong]
    if unexpected or wrong or missing or not halves:
        raise WeightsError(f"{path}: " + "; ".join(
            [f"unexpected {n}" for n in unexpected] + [f"{n} stored as {t[1]}" for n, t in wrong.items()] + [f"missing {n}" for n in missing]
            + ([] if halves else ["no adapter tensors"])), missing, unexpected, wrong_dtype=wrong)
    scale = alpha / (math.sqrt(rank) if config.get("use_rslora") else rank)
    return {base: (got[HALVES[0]], got[HALVES[1]]) for base, got in halves.items()}, float(scale)

"""Architecture registry of the token-id language models: config.json's "architecture" -> class.
`load_language_model(dir)` is what `vila_b200.load`, the CLI and the trace runner use."""
from __future__ import annotations

import json
from pathlib import Path
from typing import Dict, Optional

import torch

from .bivizen import BivizenForCausalLM
from .ludazen import LudazenForCausalLM
from .lufatar import LufatarForCausalLM
from .moronex import MoronexForCausalLM
from .nibelix import NibelixForCausalLM
from .nusovik import NusovikForCausalLM

LANGUAGE_MODELS: Dict[str, type] = {"Moronex": MoronexForCausalLM, "Lufatar": LufatarForCausalLM,
                                    "Nusovik": NusovikForCausalLM, "Ludazen": LudazenForCausalLM,
                                    "Bivizen": BivizenForCausalLM, "Nibelix": NibelixForCausalLM}

_DTYPES = {"bfloat16": torch.bfloat16, "bf16": torch.bfloat16, "float32": torch.float32, "fp32": torch.float32}


def language_model_architecture(model_dir) -> Optional[str]:
    """The registered architecture named by <model_dir>/config.json, or None (e.g. a VILA checkpoint)."""
    f = Path(model_dir) / "config.json"
    if not f.exists():
        return None
    arch = json.loads(f.read_text()).get("architecture")
    return arch if arch in LANGUAGE_MODELS else None


# The layers' weights that linear_any alone reads, by class: these may be held in 4 bits.  Projections that a recurrence's step size or
# decay comes from stay as they are (an error in them compounds over the state), as do embeddings, routers, experts, norms and the output
# head.  Where such rows end a fused weight, the layer's `exact_from` says from which row on.
MX4_WEIGHTS: Dict[str, tuple] = {
    "Lufatar": ("qkv", "o", "side_gate", "side_proj"),
    "Nusovik": ("qkg", "attn_o", "ssd_in", "ssd_o", "sel_in", "sel_o", "up", "down"),
    "Ludazen": ("qkv", "in_w", "o", "up", "down", "shared_gu", "shared_down"),
    "Bivizen": ("in_w", "o", "gu", "down"),
    "Nibelix": ("in_w", "o", "gu", "down", "shared_up", "shared_down"),
}


def quantize_weights(model):
    """Hold a bf16 language model's layer weights as microscaled 4-bit rows (ops.Mx4: 17 bytes per 32 of them instead of 64), each
    rounded to the nearest number of its block; rows that step sizes and decays come from, and activations, stay bf16.  In place; -> model.
    state_dict and save_pretrained still give the weights that were loaded, which the model keeps where they were: on the host after from_pretrained.  A model
    made from tensors on the GPU keeps those there, too, and then takes more of its memory, not less.  A TokenEngine that runs the
    model captures its decode steps anew at its next step; what it cached for its sequences stays as the former weights made it.
    Not while another thread runs a step of the model."""
    from .. import ops
    arch = next((a for a, c in LANGUAGE_MODELS.items() if type(model) is c), None)
    names = MX4_WEIGHTS.get(arch)
    if names is None:
        raise ValueError(f"{type(model).__name__} does not hold weights in 4 bits (those that do: {sorted(MX4_WEIGHTS)})")
    if model.dtype != torch.bfloat16:
        raise ValueError(f"4-bit weights go with bfloat16 activations, not {model.dtype}")
    if torch.device(model.device).type == "cuda":
        torch.cuda.synchronize(model.device)      # no step that reads the replaced weights is under way, on whichever stream
    model.weights_version = getattr(model, "weights_version", 0) + 1
    for layer in model.layers:
        for name in names:
            w = getattr(layer, name, None)
            if isinstance(w, torch.Tensor) and w.dim() == 2:      # experts' weights are one tensor of three dimensions
                first = getattr(layer, "exact_from", {}).get(name, w.shape[0])
                first = first // 8 * 8 if first < w.shape[0] else first      # the kept rows' results start on a 16-byte boundary
                if first > 0:
                    setattr(layer, name, ops.mx4_quantize(w, keep=w.shape[0] - first))
    return model


def load_language_model(model_dir, device="cuda", dtype="bfloat16", weights: Optional[str] = None):
    """weights: None (as dtype says) or "mx4" (quantize_weights)"""
    if weights not in (None, "mx4"):
        raise ValueError(f"weights={weights!r}: None or 'mx4'")
    arch = language_model_architecture(model_dir)
    if arch is None:
        raise ValueError(f"{model_dir}: config.json names no registered architecture "
                         f"(known: {sorted(LANGUAGE_MODELS)})")
    dt = _DTYPES[dtype] if isinstance(dtype, str) else dtype
    if weights is not None and (arch not in MX4_WEIGHTS or dt != torch.bfloat16):      # before anything is loaded
        raise ValueError(f"{arch} in {dt}: 4-bit weights are for {sorted(MX4_WEIGHTS)} in bfloat16")
    model = LANGUAGE_MODELS[arch].from_pretrained(model_dir, device=device, dtype=dt)
    return model if weights is None else quantize_weights(model)

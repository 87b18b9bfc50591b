"""Compute dtypes and cache formats by name."""
from __future__ import annotations

import torch


def parse_dtype(name) -> torch.dtype:
    if isinstance(name, torch.dtype):
        if name in (torch.float32, torch.bfloat16):
            return name
        raise ValueError(f"compute dtype must be float32 or bfloat16, not {name}")
    table = {"float32": torch.float32, "fp32": torch.float32, "f32": torch.float32,
             "bfloat16": torch.bfloat16, "bf16": torch.bfloat16}
    try:
        return table[str(name).lower()]
    except KeyError:
        raise ValueError(f"unknown dtype {name!r}; use bfloat16 or float32") from None


def parse_kv_quant(name) -> int:
    """Bits of a cached key or value element: 0 stands for the compute dtype."""
    table = {None: 0, "none": 0, "int8": 8, "int4": 4}
    try:
        return table[name]
    except (KeyError, TypeError):
        raise ValueError(f"unknown kv_quant {name!r}; use int8, int4 or none") from None

"""Where and in which precision a model runs."""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Any, Dict, Optional

import torch

_DTYPE_NAMES = {
    "float32": torch.float32, "f32": torch.float32, "fp32": torch.float32,
    "bfloat16": torch.bfloat16, "bf16": torch.bfloat16,
}


def parse_dtype(name) -> torch.dtype:
    """``bfloat16``/``bf16`` or ``float32``/``f32`` (the reference's ``--dtype`` spellings, inferrs/src/main.rs:101-103;
    float16 is not offered here)."""
    if isinstance(name, torch.dtype):
        if name in (torch.float32, torch.bfloat16):
            return name
        raise ValueError(f"dtype must be float32 or bfloat16, got {name}")
    try:
        return _DTYPE_NAMES[str(name).lower()]
    except KeyError:
        raise ValueError(f"dtype must be one of {sorted(_DTYPE_NAMES)}, got {name!r}") from None


@dataclass
class Runtime:
    """``dtype`` is the element type of activations and of the cache.  The residual stream,
    norms, softmax, rotation and logits are float32 in both cases; with float32 every matrix
    product is true 32-bit as well.

    ``weight_bits`` 4: the projections inside the layers keep their weights in 4 bits with a power of two per 32 of them
    (embedding, head, norms and biases stay as they are); ``cache_bits`` 8: keys and values are cached in 8 bits with a
    scale per vector.  Parts that have no such form refuse."""

    device: torch.device
    dtype: torch.dtype
    shared: Dict[Any, Any] = field(default_factory=dict)  # tables shared by parts with equal descriptions
    weight_bits: Optional[int] = None
    cache_bits: Optional[int] = None

    def __post_init__(self):
        if self.weight_bits not in (None, 4):
            raise ValueError(f"weights are kept in their own type or in 4 bits, got {self.weight_bits} bits")
        if self.cache_bits not in (None, 8):
            raise ValueError(f"keys and values are kept in the activations' type or in 8 bits, got {self.cache_bits} bits")

    @classmethod
    def cuda(cls, dtype, weight_bits: Optional[int] = None, cache_bits: Optional[int] = None) -> "Runtime":
        if not torch.cuda.is_available():
            raise RuntimeError("inferrs_b200 needs a CUDA device (built for sm_100a); there is no CPU path")
        return cls(device=torch.device("cuda", torch.cuda.current_device()), dtype=parse_dtype(dtype),
                   weight_bits=weight_bits, cache_bits=cache_bits)

"""Storage of a quantised KV cache, and the frequencies of rotary positions.

``QuantizedKVCache`` holds the K and V rows of B sequences and Hkv heads in
``[B, Hkv, C, ...]`` arrays, one row per (sequence, head, slot):

* ``"fp8"``: E4M3 codes ``[B, Hkv, C, D]`` and one float32 scale per row,
  ``value = code * row_scale`` (1.03 bytes per element at D = 128);
* ``"nvfp4"``: each row is one ``[1, D]`` matrix of the weight format of
  ``nvfp4_tensor``: packed E2M1 ``[B, Hkv, C, D/2]``, UE4M3 block-16 scales
  ``[B, Hkv, C, D/16]`` and one float32 scale per row (0.59 bytes per element).

Rows are quantised from their own values as they are written, so a cache needs
no calibration and rows of any size keep their relative precision.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

KV_FORMATS = ("fp8", "nvfp4")
CAPACITY_MULTIPLE = 64
MAX_HEAD_DIM = 256


@dataclass(frozen=True)
class QuantizedKVCache:
    """A quantised KV cache (see the module's text for the layout).

    ``allocate`` makes an empty one; the constructor checks given arrays.  The
    operators read only the fields, so any object that has them will do.
    """

    format: str
    head_dim: int
    k_codes: torch.Tensor
    v_codes: torch.Tensor
    k_row_scales: torch.Tensor
    v_row_scales: torch.Tensor
    k_block_scales: torch.Tensor | None = None
    v_block_scales: torch.Tensor | None = None

    def __post_init__(self) -> None:
        if self.format not in KV_FORMATS:
            raise ValueError(f"format must be one of {KV_FORMATS}, got {self.format!r}")
        if isinstance(self.head_dim, bool) or not isinstance(self.head_dim, int):
            raise TypeError("head_dim must be an integer")
        if not 16 <= self.head_dim <= MAX_HEAD_DIM or self.head_dim % 16:
            raise ValueError(f"head_dim must be a multiple of 16 and at most {MAX_HEAD_DIM}, got {self.head_dim}")
        if not isinstance(self.k_codes, torch.Tensor) or self.k_codes.ndim != 4:
            raise TypeError("k_codes must be a rank-4 torch.Tensor")
        lead = tuple(self.k_codes.shape[:3])
        if min(lead) < 1:
            raise ValueError("cache dimensions must all be positive")
        if lead[2] % CAPACITY_MULTIPLE:
            raise ValueError(f"the capacity must be a multiple of {CAPACITY_MULTIPLE}, got {lead[2]}")
        width = self.head_dim if self.format == "fp8" else self.head_dim // 2
        wanted = {"codes": (torch.uint8, (*lead, width)), "row_scales": (torch.float32, lead)}
        if self.format == "nvfp4":
            wanted["block_scales"] = (torch.uint8, (*lead, self.head_dim // 16))
        elif self.k_block_scales is not None or self.v_block_scales is not None:
            raise ValueError("an fp8 cache has no block scales")
        for side in "kv":
            for field, (dtype, shape) in wanted.items():
                name, t = f"{side}_{field}", getattr(self, f"{side}_{field}")
                if not isinstance(t, torch.Tensor):
                    raise TypeError(f"{name} must be a torch.Tensor")
                if t.dtype != dtype:
                    raise TypeError(f"{name} must have dtype {dtype}, got {t.dtype}")
                if tuple(t.shape) != shape:
                    raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
                if not t.is_contiguous():
                    raise ValueError(f"{name} must be contiguous")
                if t.device != self.k_codes.device:
                    raise ValueError(f"{name} must be on device {self.k_codes.device}, got {t.device}")

    @classmethod
    def allocate(cls, batch: int, kv_heads: int, capacity: int, head_dim: int, format: str = "fp8",
                 device="cuda") -> "QuantizedKVCache":
        """An empty cache of at least ``capacity`` slots (rounded up to a multiple of 64)."""
        for name, v in (("batch", batch), ("kv_heads", kv_heads), ("capacity", capacity), ("head_dim", head_dim)):
            if isinstance(v, bool) or not isinstance(v, int):
                raise TypeError(f"{name} must be an integer")
            if v < 1:
                raise ValueError(f"{name} must be positive, got {v}")
        if format not in KV_FORMATS:
            raise ValueError(f"format must be one of {KV_FORMATS}, got {format!r}")
        lead = (batch, kv_heads, -(-capacity // CAPACITY_MULTIPLE) * CAPACITY_MULTIPLE)
        fields = {}
        for side in "kv":
            width = head_dim if format == "fp8" else head_dim // 2
            fields[f"{side}_codes"] = torch.zeros((*lead, width), dtype=torch.uint8, device=device)
            fields[f"{side}_row_scales"] = torch.zeros(lead, dtype=torch.float32, device=device)
            if format == "nvfp4":
                fields[f"{side}_block_scales"] = torch.zeros((*lead, head_dim // 16), dtype=torch.uint8, device=device)
        return cls(format, head_dim, **fields)

    @property
    def capacity(self) -> int:
        return int(self.k_codes.shape[2])

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (
            self.k_codes, self.v_codes, self.k_row_scales, self.v_row_scales, self.k_block_scales,
            self.v_block_scales) if t is not None)


# ------------------------------------------------------------------ rotary frequencies
def _positive(name: str, value) -> float:
    if isinstance(value, bool) or not isinstance(value, (int, float)):
        raise TypeError(f"{name} must be a real number")
    if not math.isfinite(value) or value <= 0:
        raise ValueError(f"{name} must be finite and positive, got {value}")
    return float(value)


def rope_frequencies(rotary_dim: int, rope_theta: float = 10_000.0, *, scaling: str | None = None,
                     factor: float = 1.0, original_length: int = 4096, beta_fast: float = 32.0,
                     beta_slow: float = 1.0, device="cuda") -> tuple[torch.Tensor, float]:
    """``(inv_freq, attention_factor)`` for ``cuda_apply_rope_qk``.

    Pair m of ``rotary_dim / 2`` turns by ``position * f_m``, with
    ``f_m = rope_theta ** (-2 m / rotary_dim)`` before scaling.  ``scaling``
    stretches a context of ``original_length`` by ``factor``:

    * ``None``: unscaled;
    * ``"linear"``: every ``f_m / factor`` (positions interpolated);
    * ``"ntk"``: ``rope_theta`` grows so that the slowest pair is slowed by
      exactly ``factor`` and the fastest is kept;
    * ``"yarn"``: pairs that turn more than ``beta_fast`` times within the
      original length are kept, those that turn less than ``beta_slow`` times
      are slowed by ``factor``, in between a linear ramp over m; sine and
      cosine are scaled by ``0.1 ln(factor) + 1``.

    Computed in float64 on the host, rounded once.
    """
    if isinstance(rotary_dim, bool) or not isinstance(rotary_dim, int):
        raise TypeError("rotary_dim must be an integer")
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
    theta, factor = _positive("rope_theta", rope_theta), _positive("factor", factor)
    length = _positive("original_length", original_length)
    fast, slow = _positive("beta_fast", beta_fast), _positive("beta_slow", beta_slow)
    attention_factor = 1.0
    m = torch.arange(rotary_dim // 2, dtype=torch.float64)
    if scaling == "ntk" and rotary_dim > 2:
        theta *= factor ** (rotary_dim / (rotary_dim - 2))
    freq = theta ** (-2.0 * m / rotary_dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if slow >= fast:
            raise ValueError(f"beta_slow must be below beta_fast, got {slow} and {fast}")

        def pair_of(turns: float) -> float:  # the (real) m whose pair turns so often within the length
            return rotary_dim * math.log(length / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))

        low = max(math.floor(pair_of(fast)), 0)
        high = min(math.ceil(pair_of(slow)), rotary_dim - 1)
        ramp = ((m - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        freq = freq * (1.0 - ramp) + freq / factor * ramp
        attention_factor = 1.0 if factor <= 1.0 else 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'yarn', got {scaling!r}")
    return freq.to(torch.float32).to(device), attention_factor


__all__ = ["CAPACITY_MULTIPLE", "KV_FORMATS", "QuantizedKVCache", "rope_frequencies"]

"""Storage of a paged KV cache: a pool of pages, and the table of who holds which.

A page is laid out like the cache of one sequence with the page size S as its
capacity (``quantized_kv_cache``), so ``PagedKVCache`` holds ``[N, Hkv, S, ...]``
arrays:

* ``"bf16"``: codes are the rows themselves, BF16 ``[N, Hkv, S, D]``;
* ``"fp8"``: E4M3 codes ``[N, Hkv, S, D]``, a float32 scale per row ``[N, Hkv, S]``;
* ``"nvfp4"``: packed E2M1 ``[N, Hkv, S, D/2]``, UE4M3 block-16 scales
  ``[N, Hkv, S, D/16]``, a float32 scale per row.

Slot ``s`` is row ``s % S`` of page ``s // S``, in every head.

``PageTable`` is the state of B sequences over a pool of N pages, all of it on the
device: ``pages`` int32 ``[B, M]`` names the pages of each sequence in order, -1
behind the ``held`` (int64 ``[B]``) that it has; ``free_pages`` int32 ``[N]`` is
a stack of ``free_count`` (int64 ``[1]``) pages that nobody holds.
``cuda_reserve_pages_`` and ``cuda_release_pages_`` change it.  The pools of all
layers can share one table.  A page stands once in it, in one row or on the stack:
nothing counts references, so sequences that share pages name them in a block table
of their own for the attention, and one row of the ``PageTable`` holds them.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from quantized_kv_cache import MAX_HEAD_DIM

PAGED_KV_FORMATS = ("bf16", "fp8", "nvfp4")
PAGE_SIZE_MULTIPLE = 16


def _int(name: str, v: object, least: int = 1) -> int:
    if isinstance(v, bool) or not isinstance(v, int):
        raise TypeError(f"{name} must be an integer")
    if v < least:
        raise ValueError(f"{name} must be at least {least}, got {v}")
    return v


def _page_size(v: object) -> int:
    if _int("page_size", v) % PAGE_SIZE_MULTIPLE:
        raise ValueError(f"page_size must be a multiple of {PAGE_SIZE_MULTIPLE}, got {v}")
    return v


def _check(t: object, name: str, dtype: torch.dtype, shape: tuple, device: torch.device) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must have dtype {dtype}, got {t.dtype}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if t.device != device:
        raise ValueError(f"{name} must be on device {device}, got {t.device}")


def _layout(format: str, lead: tuple, head_dim: int) -> dict:
    width = head_dim // 2 if format == "nvfp4" else head_dim
    fields = {"codes": (torch.bfloat16 if format == "bf16" else torch.uint8, (*lead, width))}
    if format != "bf16":
        fields["row_scales"] = (torch.float32, lead)
    if format == "nvfp4":
        fields["block_scales"] = (torch.uint8, (*lead, head_dim // 16))
    return fields


@dataclass(frozen=True)
class PagedKVCache:
    """A pool of pages (see the module's text for the layout).

    ``allocate`` makes an empty one; the constructor checks given arrays.  The
    operators read only the fields, so any object that has them will do.
    """

    format: str
    head_dim: int
    k_codes: torch.Tensor
    v_codes: torch.Tensor
    k_row_scales: torch.Tensor | None = None
    v_row_scales: torch.Tensor | None = None
    k_block_scales: torch.Tensor | None = None
    v_block_scales: torch.Tensor | None = None

    def __post_init__(self) -> None:
        if self.format not in PAGED_KV_FORMATS:
            raise ValueError(f"format must be one of {PAGED_KV_FORMATS}, got {self.format!r}")
        _int("head_dim", self.head_dim, 16)
        if self.head_dim > MAX_HEAD_DIM or self.head_dim % 16:
            raise ValueError(f"head_dim must be a multiple of 16 and at most {MAX_HEAD_DIM}, got {self.head_dim}")
        if not isinstance(self.k_codes, torch.Tensor) or self.k_codes.ndim != 4:
            raise TypeError("k_codes must be a rank-4 torch.Tensor")
        lead = tuple(self.k_codes.shape[:3])
        if min(lead) < 1:
            raise ValueError("cache dimensions must all be positive")
        _page_size(lead[2])
        wanted = _layout(self.format, lead, self.head_dim)
        for side in "kv":
            for field in ("codes", "row_scales", "block_scales"):
                name, t = f"{side}_{field}", getattr(self, f"{side}_{field}")
                if field in wanted:
                    _check(t, name, *wanted[field], self.k_codes.device)
                elif t is not None:
                    raise ValueError(f"a {self.format} cache has no {field.replace('_', ' ')}")

    @classmethod
    def allocate(cls, pages: int, kv_heads: int, page_size: int, head_dim: int, format: str = "bf16",
                 device="cuda") -> "PagedKVCache":
        """A pool of ``pages`` empty pages."""
        lead = (_int("pages", pages), _int("kv_heads", kv_heads), _page_size(page_size))
        _int("head_dim", head_dim)
        if format not in PAGED_KV_FORMATS:
            raise ValueError(f"format must be one of {PAGED_KV_FORMATS}, got {format!r}")
        fields = {f"{side}_{field}": torch.zeros(shape, dtype=dtype, device=device) for side in "kv"
                  for field, (dtype, shape) in _layout(format, lead, head_dim).items()}
        return cls(format, head_dim, **fields)

    @property
    def pages(self) -> int:
        return int(self.k_codes.shape[0])

    @property
    def page_size(self) -> int:
        return int(self.k_codes.shape[2])

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (
            self.k_codes, self.v_codes, self.k_row_scales, self.v_row_scales, self.k_block_scales,
            self.v_block_scales) if t is not None)


@dataclass(frozen=True)
class PageTable:
    """The pages of B sequences and the free ones (see the module's text)."""

    pages: torch.Tensor
    held: torch.Tensor
    free_pages: torch.Tensor
    free_count: torch.Tensor
    page_size: int

    def __post_init__(self) -> None:
        if not isinstance(self.pages, torch.Tensor) or self.pages.ndim != 2:
            raise TypeError("pages must be a rank-2 torch.Tensor")
        if not isinstance(self.free_pages, torch.Tensor) or self.free_pages.ndim != 1:
            raise TypeError("free_pages must be a rank-1 torch.Tensor")
        batch, most = self.pages.shape
        if min(batch, most, self.free_pages.shape[0]) < 1:
            raise ValueError("the page table's dimensions must all be positive")
        for name, dtype, shape in (("pages", torch.int32, (batch, most)), ("held", torch.int64, (batch,)),
                                   ("free_pages", torch.int32, tuple(self.free_pages.shape)),
                                   ("free_count", torch.int64, (1,))):
            _check(getattr(self, name), name, dtype, shape, self.pages.device)
        _page_size(self.page_size)

    @classmethod
    def allocate(cls, batch: int, max_pages: int, pages: int, page_size: int, device="cuda") -> "PageTable":
        """B sequences that hold nothing yet, up to ``max_pages`` each, over a pool of ``pages`` free pages."""
        shape = (_int("batch", batch), _int("max_pages", max_pages))
        n = _int("pages", pages)
        return cls(torch.full(shape, -1, dtype=torch.int32, device=device),
                   torch.zeros((batch,), dtype=torch.int64, device=device),
                   torch.arange(n - 1, -1, -1, dtype=torch.int32, device=device),  # page 0 on top
                   torch.full((1,), n, dtype=torch.int64, device=device), page_size)


__all__ = ["PAGED_KV_FORMATS", "PAGE_SIZE_MULTIPLE", "PageTable", "PagedKVCache"]

"""The paged key/value cache: the description of a serving step that ``Backend.paged_plan``, ``paged_append`` and
``paged_attention`` share (``lapid_b200_paged`` in ``include/lapid_b200.h``).

A layer's cache is two buffers ``[pages][kv_heads][page_size][head_dim]``; a request's keys lie in the pages that its row of
the block table names. A step of a layer stack, with everything on the device::

    spec = PagedSpec(dtype=DType.BF16, q_heads=32, kv_heads=8, head_dim=128, page_size=16, pages=4096,
                     requests=8, tokens=8, max_blocks=512, max_new=1)
    plan = be.alloc(plan_bytes(spec))
    be.paged_plan(spec, new_lens, cached_lens, table, slots, positions, kv_lens, used, plan, free_pages=free, n_free=n)
    for layer in layers:
        ...                                                     # q, k, v projections (f32 rows)
        be.paged_append(spec, DType.F32, q, k, v, slots, positions, layer.k, layer.v, q_half, rope=table_of_angles, rope_rows=8192, rot=128)
        be.paged_attention(spec, plan, q_half, layer.k, layer.v, table, mixed)
        ...                                                     # o projection, a_dtype = DType.BF16

``tp.PagedLayers`` is that step over whole decoder layers.
"""
from __future__ import annotations

import ctypes as C
import enum
from dataclasses import dataclass

import numpy as np

from . import _lib
from ._lib import check
from .backend import DType


class Mask(enum.IntEnum):
    """Which keys a new token sees: all, those up to its own, or the cached ones only."""
    FULL = 0
    CAUSAL = 1
    CROSS = 2


@dataclass(frozen=True)
class PagedSpec:
    """``lapid_b200_paged``: the cache's shape and the bounds of a step (``tokens`` rows of q, k, v and out; no request has more
    than ``max_new`` of them; ``max_blocks`` columns of the block table). ``scale`` 0: ``1 / sqrt(head_dim)``."""
    dtype: DType
    q_heads: int
    kv_heads: int
    head_dim: int
    page_size: int
    pages: int
    requests: int
    tokens: int
    max_blocks: int
    max_new: int
    mask: Mask = Mask.CAUSAL
    window: int = 0
    scale: float = 0.0

    def to_c(self) -> _lib.PagedC:
        c = _lib.PagedC()
        c.dtype, c.mask, c.scale = int(self.dtype), int(self.mask), float(self.scale)
        for name in ("q_heads", "kv_heads", "head_dim", "page_size", "pages", "requests", "tokens", "max_blocks", "max_new", "window"):
            v = int(getattr(self, name))
            if v < 0 or v >= 1 << (32 if name in ("q_heads", "kv_heads", "head_dim", "page_size") else 63):
                raise _lib.LapidError(1, "invalid_argument", f"PagedSpec.{name} = {v} is out of range")
            setattr(c, name, v)
        return c

    def cache_bytes(self) -> int:
        """Bytes of one layer's keys (its values take as many)."""
        return self.pages * self.kv_heads * self.page_size * self.head_dim * 2


def plan_bytes(spec: PagedSpec) -> int:
    """Bytes of the plan buffer of such a step (``lapid_b200_paged_plan_bytes``); needs no device."""
    n = C.c_uint64(0)
    c = spec.to_c()
    check(_lib.lib().lapid_b200_paged_plan_bytes(C.byref(c), C.byref(n)))
    return int(n.value)


def rope_table(positions: int, rot: int, base: float = 10000.0) -> np.ndarray:
    """``[positions, rot]`` f32 for ``paged_append``: the cosines of ``p * base ** (-2 i / rot)``, then their sines, rounded from f64."""
    angle = np.arange(positions, dtype=np.float64)[:, None] * base ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)[None, :]
    return np.concatenate([np.cos(angle), np.sin(angle)], axis=1).astype(np.float32)

"""A speculative step over the 4-bit cache (eg_rope_table, eg_rope, eg_verify_drafts; with
``Kv4Cache.attend_tree`` and ``Kv4Cache.keep`` of kv4.py; semantics and limits: include/enargeia_hip.h). No
counterpart in the reference, which decodes one token at a time.

Drafted tokens of several sequences run through the model together. A sequence's rows are its last token - row 0,
decided but not yet cached - and its drafts, as a tree (``parents``) or a chain. With ``pages`` a ``PageTable``, a step is

  ``pages.grow(seq, rows)`` for every sequence; lengths = positions with the rows
  per layer: ``rope`` (q and k at the rows' depths after starts = lengths - rows), ``cache.append`` (k, v, no rope),
  ``cache.attend_tree``
  ``verify`` (the accepted branch and the next token), ``cache.keep`` (the branch's rows together, all layers)
  ``pages.shrink(seq, rows - count)`` once the host knows the counts

and the next token is the next step's row 0.
"""

from __future__ import annotations

import struct

import numpy as np

from . import _lib
from ._lib import EG_ERR_INVALID, EgError, check
from .kernels import Device
from .kv4 import _address, _element, _packed

SCALINGS = {"none": 0, "linear": 1, "base": 2, "turns": 3, "log_turns": 4}  # eg_rope_scaling
LAYOUTS = {"half": 0, "interleaved": 1}  # eg_rope_layout
NO_ROW = 0xFFFFFFFF

# eg_rope_table_dims, eg_rope_dims, eg_verify_dims, field by field
_TABLE_DIMS = struct.Struct("3Ii6d").pack  # positions, first, rotary_dim, scaling, theta .. amplitude
# rows, heads, kv_heads, head_dim, rotary_dim, four strides, table_positions, sequences, layout, in_type, out_type
_ROPE_DIMS = struct.Struct("11I3i").pack
_VERIFY_DIMS = struct.Struct("6Ii").pack  # sequences, rows, max_rows, vocab, logits_stride, draft_stride, type


def _named(names: dict, name: str, what: str) -> int:
    e = names.get(name)
    if e is None:
        raise EgError(EG_ERR_INVALID, f"{what} {name!r}: one of {', '.join(names)}")
    return e


def rope_table(device: Device, table, *, positions: int, rotary_dim: int, theta: float = 10000.0, first: int = 0,
               scaling: str = "none", factor: float = 1.0, context: float = 0.0, low: float = 1.0, high: float = 4.0,
               amplitude: float = 1.0) -> None:
    """eg_rope_table: (cos, sin) of `positions` positions from `first` on, f32 [positions][rotary_dim / 2][2]."""
    ctx = device.ctx
    check(_lib.load().eg_rope_table(ctx, _address(table),
                                    _packed(_TABLE_DIMS, positions, first, rotary_dim, _named(SCALINGS, scaling, "scaling"),
                                            theta, factor, context, low, high, amplitude)), ctx)


def rope(device: Device, table, *, rows: int, head_dim: int, table_positions: int, rotary_dim: int = 0, q=None,
         q_out=None, heads: int = 0, k=None, k_out=None, kv_heads: int = 0, positions=None, offsets=None, starts=None,
         sequences: int = 0, layout: str = "half", in_type: str = "f32", out_type: str = "f32", q_stride: int = 0,
         k_stride: int = 0, q_out_stride: int = 0, k_out_stride: int = 0) -> None:
    """eg_rope: rows of q and k rotated at positions of their own."""
    ctx = device.ctx
    status = _lib.load().eg_rope(
        ctx, _address(q), _address(k), _address(table), _address(positions), _address(offsets), _address(starts),
        _address(q_out), _address(k_out),
        _packed(_ROPE_DIMS, rows, heads, kv_heads, head_dim, rotary_dim, q_stride, k_stride, q_out_stride, k_out_stride,
                table_positions, sequences, _named(LAYOUTS, layout, "layout"), _element(in_type), _element(out_type)))
    if status:
        check(status, ctx)


def verify(device: Device, logits, tokens, offsets, path, counts, next, *, sequences: int, rows: int, max_rows: int,
           vocab: int, parents=None, draft=None, accept=None, draws=None, temperatures=None, type: str = "f32",
           logits_stride: int = 0, draft_stride: int = 0) -> None:
    """eg_verify_drafts: from the rows' logits the branch that is accepted and the next token."""
    ctx = device.ctx
    status = _lib.load().eg_verify_drafts(
        ctx, _address(logits), _address(tokens), _address(offsets), _address(parents), _address(draft),
        _address(accept), _address(draws), _address(temperatures), _address(path), _address(counts), _address(next),
        _packed(_VERIFY_DIMS, sequences, rows, max_rows, vocab, logits_stride, draft_stride, _element(type)))
    if status:
        check(status, ctx)


def depths(parents) -> np.ndarray:
    """How far below its root each row of one sequence's tree lies (u32): its position past the first row's."""
    out = np.zeros(len(parents), np.uint32)
    for i, p in enumerate(parents):
        if 0 <= int(p) < i:
            out[i] = out[int(p)] + 1
    return out


__all__ = ["LAYOUTS", "NO_ROW", "SCALINGS", "depths", "rope", "rope_table", "verify"]

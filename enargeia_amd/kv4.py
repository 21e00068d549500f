"""Serving several sequences over a paged cache held in 4 bits (the eg_kv4_* entry points, the
attention over that cache and the attention over packed prompts; formats, semantics and limits:
include/enargeia_hip.h). No counterpart in the reference, whose cache is one sequence's.

``Kv4Cache`` is the pool and the launches over it. ``PageTable`` is the host's bookkeeping of which
page holds what: sequences grow, fork (sharing whole pages, copying the partial one), are freed, and
the used pages are moved together. Buffers are bound as elsewhere in this package (a ``Buffer``, a
``Binding`` or anything with ``ptr`` or ``data_ptr``); offsets, starts, lengths and tables are u32
in device memory, read when the launch runs.

A prompt: ``append`` (q, k, v of the packed rows; q rotated comes back, and k and v in the operands'
type if asked for), then ``attention_packed``. A chunk after earlier rows: ``append``, ``read`` all of
the sequences' rows, ``attention_packed`` with more keys than queries. A decode step: ``append`` one row
per sequence, ``attend``.
"""

from __future__ import annotations

import ctypes
import struct
from operator import index

import numpy as np

from . import _lib
from ._lib import EG_ERR_INVALID, EG_ERR_RANGE, EG_ERR_STATE, EgError, EgRangeError, check
from .kernels import Buffer, Device, _ptr

ELEMENTS = {"f32": 0, "f16": 1, "bf16": 2}  # eg_element
NO_PAGE = 0xFFFFFFFF
_MOST = 0xFFFFFFFF  # of a u32


def _element(name: str) -> int:
    e = ELEMENTS.get(name)
    if e is None:
        raise EgError(EG_ERR_INVALID, f"element type {name!r}: one of {', '.join(ELEMENTS)}")
    return e


def _address(ref) -> int | None:
    """What ctypes takes for a device pointer. (A launch's host path is most of a small call's time: these
    functions pass plain integers and the dims as packed bytes, 2.5 us less per call of eleven pointers
    than a c_void_p each and a Structure.)"""
    data_ptr = getattr(ref, "data_ptr", None)
    if data_ptr is not None:
        return data_ptr()
    return None if ref is None else _ptr(ref)


class Kv4Dims(ctypes.Structure):
    """eg_kv4_dims"""
    _fields_ = [("kv_heads", ctypes.c_uint32), ("head_dim", ctypes.c_uint32), ("page_size", ctypes.c_uint32),
                ("pages", ctypes.c_uint32), ("page_stride", ctypes.c_uint64), ("sequences", ctypes.c_uint32),
                ("max_pages", ctypes.c_uint32)]


# eg_kv4_append_dims, eg_attention_kv4_dims, eg_attention_packed_dims, field by field
_APPEND_DIMS = struct.Struct("6I2i").pack  # rows, heads, q_stride, k_stride, v_stride, rope_positions, in_type, out_type
_ATTENTION_KV4_DIMS = struct.Struct("3Iif").pack  # heads, q_stride, out_stride, type, scale
# sequences, rows, key_rows, heads, kv_heads, head_dim, q_stride, k_stride, v_stride, out_stride, type, out_type, scale
_ATTENTION_PACKED_DIMS = struct.Struct("10I2if").pack


def _packed(pack, *values) -> bytes:
    try:
        return pack(*values)
    except struct.error as e:
        raise EgRangeError(EG_ERR_RANGE, f"kv4: a dimension out of range ({e})") from None


def _fits(bits: int = 32, **values: int) -> None:
    """Refuses what does not fit its field (ctypes would keep the low bits of it)."""
    for name, x in values.items():
        if not 0 <= x < 1 << bits:
            raise EgRangeError(EG_ERR_RANGE, f"kv4: a dimension out of range ({name} {x}: 0 to 2^{bits} - 1)")


def page_bytes(kv_heads: int, head_dim: int, page_size: int) -> int:
    """Bytes of one layer's page."""
    _fits(kv_heads=kv_heads, head_dim=head_dim, page_size=page_size)
    out = ctypes.c_uint64()
    check(_lib.load().eg_kv4_page_bytes(ctypes.byref(Kv4Dims(kv_heads, head_dim, page_size, 0, 0, 0, 0)),
                                        ctypes.byref(out)), None)
    return out.value


class Kv4Cache:
    """A pool of pages, each of all layers ([pages][layers][page bytes]), and the launches over it.
    ``pool`` binds memory the caller owns (contents as they are); without it the cache allocates."""

    def __init__(self, device: Device, kv_heads: int, head_dim: int, pages: int, page_size: int = 64,
                 layers: int = 1, pool=None):
        if pages < 1 or layers < 1:
            raise EgRangeError(EG_ERR_RANGE, f"kv4: a pool of {pages} pages of {layers} layers")
        pages, layers = index(pages), index(layers)  # (numpy's would wrap in the products below)
        self.device = device
        self.layer_bytes = page_bytes(kv_heads, head_dim, page_size)
        _fits(pages=pages)
        _fits(64, pool_bytes=self.layer_bytes * layers * pages)
        self.dims = Kv4Dims(kv_heads, head_dim, page_size, pages, self.layer_bytes * layers, 0, 0)
        self._dims = ctypes.byref(self.dims)
        lib = _lib.load()  # (bound once: a small call's time is its host path)
        self._append, self._read, self._attend = lib.eg_kv4_append, lib.eg_kv4_read, lib.eg_attention_decode_kv4
        self.layers = layers
        size = self.dims.page_stride * pages
        held = pool.size if isinstance(pool, Buffer) else getattr(pool, "nbytes", None)
        if held is not None and held < size:
            raise EgRangeError(EG_ERR_RANGE, f"kv4: a pool of {held} bytes for {pages} pages of {self.dims.page_stride}")
        self.owned = device.buffer(size, "kv4 pool") if pool is None else None
        self.pool = self.owned if pool is None else pool

    def _at(self, layer: int) -> int:
        if not 0 <= layer < self.layers:
            raise EgRangeError(EG_ERR_RANGE, f"kv4: layer {layer} of {self.layers}")
        base = _address(self.pool)
        if not base:  # (an offset from nowhere would not be NULL)
            raise EgError(EG_ERR_STATE, "kv4: the pool has been released")
        return base + index(layer) * self.layer_bytes

    def _for(self, sequences: int, max_pages: int):
        if not (0 <= sequences <= _MOST and 0 <= max_pages <= _MOST):
            _fits(sequences=sequences, max_pages=max_pages)
        d = self.dims
        d.sequences, d.max_pages = sequences, max_pages
        return self._dims

    def append(self, k, v, offsets, starts, table, *, rows: int, sequences: int, max_pages: int, layer: int = 0,
               q=None, q_out=None, k_out=None, v_out=None, heads: int = 0, rope=None, rope_positions: int = 0,
               in_type: str = "f32", out_type: str = "f32", q_stride: int = 0, k_stride: int = 0,
               v_stride: int = 0) -> None:
        """eg_kv4_append: the batch's new rows rotated and stored."""
        ctx = self.device.ctx
        status = self._append(
            ctx, _address(q), _address(k), _address(v), _address(rope), _address(offsets), _address(starts),
            _address(table), self._at(layer), _address(q_out), _address(k_out), _address(v_out),
            self._for(sequences, max_pages),
            _packed(_APPEND_DIMS, rows, heads, q_stride, k_stride, v_stride, rope_positions, _element(in_type),
                    _element(out_type)))
        if status:
            check(status, ctx)

    def read(self, k_out, v_out, offsets, starts, table, *, rows: int, sequences: int, max_pages: int,
             layer: int = 0, out_type: str = "f16") -> None:
        """eg_kv4_read: cached rows as packed rows."""
        ctx = self.device.ctx
        if not 0 <= rows <= _MOST:
            _fits(rows=rows)
        status = self._read(ctx, _address(offsets), _address(starts), _address(table), self._at(layer),
                            _address(k_out), _address(v_out), rows, _element(out_type),
                            self._for(sequences, max_pages))
        if status:
            check(status, ctx)

    def attend(self, q, lengths, table, out, *, heads: int, sequences: int, max_pages: int, layer: int = 0,
               type: str = "f32", scale: float = 0.0, q_stride: int = 0, out_stride: int = 0) -> None:
        """eg_attention_decode_kv4: one token per sequence against its cached positions."""
        ctx = self.device.ctx
        status = self._attend(ctx, _address(q), _address(lengths), _address(table), self._at(layer), _address(out),
                              self._for(sequences, max_pages),
                              _packed(_ATTENTION_KV4_DIMS, heads, q_stride, out_stride, _element(type), scale))
        if status:
            check(status, ctx)

    def copy_pages(self, pairs, count: int) -> None:
        """eg_kv4_copy_pages: page pairs[i][0] to page pairs[i][1], all layers."""
        ctx = self.device.ctx
        _fits(count=count)
        check(_lib.load().eg_kv4_copy_pages(ctx, self._at(0), _address(pairs), count, self._for(0, 0)), ctx)

    def release(self) -> None:
        if self.owned is not None:
            self.owned.release()
            self.owned = self.pool = None


def attention_packed(device: Device, q, k, v, out, q_offsets, k_offsets, *, sequences: int, rows: int, key_rows: int,
                     heads: int, kv_heads: int, head_dim: int, type: str = "f16", out_type: str | None = None,
                     scale: float = 0.0, q_stride: int = 0, k_stride: int = 0, v_stride: int = 0,
                     out_stride: int = 0) -> None:
    """eg_attention_packed: causal attention over packed sequences of different lengths."""
    t = _element(type)
    ctx = device.ctx
    check(_lib.load().eg_attention_packed(
        ctx, _address(q), _address(k), _address(v), _address(q_offsets), _address(k_offsets), _address(out),
        _packed(_ATTENTION_PACKED_DIMS, sequences, rows, key_rows, heads, kv_heads, head_dim, q_stride, k_stride,
                v_stride, out_stride, t, t if out_type is None else _element(out_type), scale)), ctx)


class PageTable:
    """Which page holds which positions, on the host: pages are shared between forks by count, a page
    that more than one sequence names is never written (a fork gets its own copy of the partial last
    page), and the lowest free page is given out first. ``copies`` collects the (from, to) pairs that
    the pool still has to copy (take them with ``take_copies`` before the next launch over the pool)."""

    def __init__(self, pages: int, page_size: int):
        if page_size not in (32, 64, 128, 256):
            raise EgError(EG_ERR_INVALID, f"page_size {page_size} is not supported (32, 64, 128, 256)")
        self.pages, self.page_size = pages, page_size
        self.users = [0] * pages
        self.held: dict[int, list[int]] = {}  # sequence id -> pages
        self.length: dict[int, int] = {}
        self.copies: list[tuple[int, int]] = []
        self._next = 0

    @property
    def free_pages(self) -> int:
        """Pages that can be given out now: the sources of pending copies are not, until those are taken."""
        return len(self._free())

    def _free(self) -> list[int]:
        sources = {a for a, _ in self.copies}  # (still to be read, whoever held them)
        return [p for p, n in enumerate(self.users) if n == 0 and p not in sources]

    def _take(self, count: int) -> list[int]:
        free = self._free()[:count]
        if len(free) < count:
            raise EgRangeError(EG_ERR_RANGE, f"kv4: {count} pages wanted, {len(free)} of {self.pages} free")
        for p in free:
            self.users[p] = 1
        return free

    def create(self) -> int:
        """A new sequence of no positions; its id."""
        seq, self._next = self._next, self._next + 1
        self.held[seq], self.length[seq] = [], 0
        return seq

    def grow(self, seq: int, rows: int) -> int:
        """Room for `rows` more positions; the first one's position. (A sequence never shrinks: its next rows
        could then lie in a page that a fork shares.)"""
        rows = index(rows)  # (of an unsigned numpy integer the rounding up below would wrap)
        if rows < 0:
            raise EgRangeError(EG_ERR_RANGE, f"kv4: sequence {seq} cannot grow by {rows} rows")
        start = self.length[seq]
        need = -(-(start + rows) // self.page_size) - len(self.held[seq])
        if need > 0:
            self.held[seq] += self._take(need)
        self.length[seq] = start + rows
        return start

    def fork(self, seq: int) -> int:
        """A sequence with the same positions: whole pages shared, the partial last one copied."""
        tail = self.length[seq] % self.page_size != 0
        own = self._take(1) if tail else []
        held = self.held[seq][:-1] if tail else list(self.held[seq])
        for p in held:
            self.users[p] += 1
        if tail:  # (a page that is itself still to be copied: from where it comes)
            last = self.held[seq][-1]
            self.copies.append((next((a for a, b in self.copies if b == last), last), own[0]))
        new = self.create()
        self.held[new], self.length[new] = held + own, self.length[seq]
        return new

    def free(self, seq: int) -> None:
        """The sequence ends; its pages that no fork shares are free again."""
        for p in self.held.pop(seq):
            self.users[p] -= 1
        del self.length[seq]
        # a copy into a page that is free again has nobody to read it
        self.copies = [(a, b) for a, b in self.copies if self.users[b]]

    def compact(self) -> int:
        """The used pages moved together at the pool's beginning (into `copies`); how many they are."""
        if self.copies:
            raise EgError(EG_ERR_STATE, "kv4: copies of forks are pending (take_copies first)")
        used = [p for p, n in enumerate(self.users) if n]
        holes = [p for p in range(len(used)) if not self.users[p]]
        moved = dict(zip([p for p in used if p >= len(used)], holes))
        for a, b in moved.items():
            self.users[b], self.users[a] = self.users[a], 0
        for held in self.held.values():
            held[:] = [moved.get(p, p) for p in held]
        self.copies = list(moved.items())
        return len(used)

    def take_copies(self) -> np.ndarray:
        """The pending (from, to) pairs, u32 [count][2], for one copy_pages: no page is copied to twice,
        or both from and to."""
        pairs, self.copies = np.array(self.copies, np.uint32).reshape(-1, 2), []
        return pairs

    def table(self, seqs, max_pages: int | None = None) -> np.ndarray:
        """The page table of the given sequences, u32 [sequences][max_pages]."""
        width = max_pages or max([len(self.held[s]) for s in seqs] + [1])
        out = np.full((len(seqs), width), NO_PAGE, np.uint32)
        for i, s in enumerate(seqs):
            if len(self.held[s]) > width:
                raise EgRangeError(EG_ERR_RANGE, f"kv4: sequence {s} has {len(self.held[s])} pages, the table {width}")
            out[i, : len(self.held[s])] = self.held[s]
        return out

    def lengths(self, seqs) -> np.ndarray:
        return np.array([self.length[s] for s in seqs], np.uint32)


__all__ = ["ELEMENTS", "Kv4Cache", "Kv4Dims", "NO_PAGE", "PageTable", "attention_packed", "page_bytes"]

"""Several new tokens per sequence of a paged cache: drafted tokens, in chains
or trees, that one step checks (speculative decoding).

The operators work on the caller's tensors, as those of paged.py do:

* `paged_plan`        -- where the new tokens go: rows, positions, slots, pages
                         taken from a list of free ones, and for trees the
                         places and masks of the nodes; one launch (two where
                         very many rows take pages);
* `paged_tree_decode` -- attention of every new token over the cached tokens
                         and its own ancestors; two launches;
* `paged_keep`        -- the rows of the accepted tokens moved to where they
                         stay, in every layer; one launch.

All three read lengths, rows and tables on the device only, so a round of
plan, `rotary`, `paged_append`, `paged_tree_decode` and `paged_keep` can be
captured in a graph that serves growing sequences. `PagePool.extend` with
`PagedBatch.tree` and `.keep` is the same round with pages managed by the pool.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

from . import SDPlan, _check, paged as _p
from .paged import KVPages, _arg, _count, _handle, _like

MAX_NODES = 64
_WORKSPACE: dict = {}  # bytes of paged_tree_decode's workspace


class TokenPlan:
    """A step's new tokens as packed rows, sequence by sequence.

    first [batch + 1]: rows before each sequence; ends [batch]: lengths with
    the new tokens; seq, positions, slots [n_rows]: a row's sequence, the
    position where it is stored (-1: nowhere) and page * page_size + slot;
    places [n_rows]: its position for the rotation (positions, without a
    tree); masks [n_rows]: the nodes that it sees (None without a tree)."""

    __slots__ = ("first", "ends", "seq", "positions", "slots", "places", "masks")


def _on(stream):
    return _p.torch.cuda.stream(stream)


def paged_plan(lengths, new, tables, page_size: int, n_rows: int, *, parents=None, held=None, free=None, taken=None,
               flags=None, stream=None) -> TokenPlan:
    """Plan a step in which sequence b, of lengths[b] tokens, gets new[b] more.

    lengths, new [batch], tables [batch, width]: int32; n_rows: rows of the
    outputs, those behind the last new token hold -1 (masks 0). parents: int32
    [nodes] (one tree for all) or [batch, nodes]: node i's parent, a node
    before it or -1; below -1 there is no such node, nor any below it.

    held [batch], free [n], taken [1]: int32, all or none: pages that each
    sequence has, the list of free pages and how many of it are taken. Pages
    that the new tokens need are taken in the order of the sequences and
    written into tables, held and taken.

    What does not fit is cut from the new tokens, which first and ends tell,
    and sets bit 2 of flags."""
    if _p.torch is None:
        _p._load()
    torch, dev = _p.torch, _p._device()
    i32 = _p._I32
    if tables.dim() != 2 or tables.dtype is not i32:
        raise ValueError("tables must be int32 [batch, width]")
    batch, width = tables.shape
    n_rows = _count(n_rows, "n_rows")
    if n_rows < 0:
        raise ValueError("n_rows must not be negative")
    if (held is None) != (free is None) or (held is None) != (taken is None):
        raise ValueError("held, free and taken come together")
    nodes = stride = n_free = 0
    if parents is not None:
        if parents.dim() == 1:
            nodes = parents.shape[0]
        elif parents.dim() == 2 and parents.shape[0] == batch:
            nodes = stride = parents.shape[1]
        else:
            raise ValueError("parents must be [nodes] or [batch, nodes]")
    if free is not None:
        if free.dim() != 1:
            raise ValueError("free must be [n]")
        n_free = _count(free.shape[0], "free")
    if stream is not None:
        with _on(stream):
            p = _new_plan(torch, batch, n_rows, parents is not None, tables)
    else:
        p = _new_plan(torch, batch, n_rows, parents is not None, tables)
    tree = parents is not None
    g = SDPlan(_arg(lengths, "lengths", i32, dev, (batch,)), _arg(new, "new", i32, dev, (batch,)),
               _arg(tables, "tables", i32, dev), _count(batch, "batch"), _count(width, "width"), page_size, n_rows,
               _arg(held, "held", i32, dev, (batch,)), _arg(free, "free", i32, dev), _arg(taken, "taken", i32, dev, (1,)),
               n_free, _count(nodes, "nodes"), _arg(parents, "parents", i32, dev), stride, p.first.data_ptr(),
               p.ends.data_ptr(), p.seq.data_ptr(), p.positions.data_ptr(), p.slots.data_ptr(),
               p.places.data_ptr() if tree else None, p.masks.data_ptr() if tree else None)
    _check(_p._L.sd_paged_plan(g, _arg(flags, "flags", i32, dev), _handle(stream, dev)))
    return p


def _new_plan(torch, batch: int, n_rows: int, tree: bool, like) -> TokenPlan:
    p, new, i64 = TokenPlan(), like.new_empty, torch.int64  # an allocation each: cutting one up costs the host more
    p.first, p.ends, p.seq, p.positions = new(batch + 1), new(batch), new(n_rows), new(n_rows)
    p.slots = new(n_rows, dtype=i64)
    p.places, p.masks = (new(n_rows), new(n_rows, dtype=i64)) if tree else (p.positions, None)
    return p


def paged_tree_decode(q, pages: KVPages, tables, lengths, first, masks=None, scale: Optional[float] = None, *,
                      places=None, layer: int = 0, window: int = 0, sinks=None, out=None, flags=None, stream=None):
    """Attention of a step's new tokens: q [n_rows, Hq, D] (contiguous, on a
    16-byte boundary), rows first[b] .. first[b + 1] of sequence b, whose
    lengths[b] tokens count them and are all stored. A row sees the tokens
    before the step and those of its sequence's new ones that its mask names
    (None: the ones up to itself; `first` must not fall: then all rows give
    zeros, with bit 2 of flags); with a window, of these the ones whose place
    is above its own less `window`. Rows from first[batch] on are left as they
    are; a row that sees nothing gives zeros.

    tables [batch, width], lengths [batch], first [batch + 1], places [n_rows]:
    int32, masks [n_rows]: int64, as `paged_plan` makes them; sinks: fp32 [Hq].
    At most 64 new tokens per sequence; Hq / Hkv: 1 .. 16."""
    dev, dt, dim = pages.here(), pages.dtype, pages.head_dim
    shape, (batch, width) = q.shape, tables.shape
    if len(shape) != 3 or shape[2] != dim:
        raise ValueError(f"q must be [n_rows, Hq, {dim}]")
    n, hq, i32 = shape[0], shape[1], _p._I32
    torch = _p.torch
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    _count(n, "n_rows"), _count(batch, "batch")
    key = (dev, pages.n_kv_heads, dim, pages.dtype, pages.bits, hq, n, batch)
    need = _WORKSPACE.get(key)
    if need is None:
        size = ctypes.c_int64()
        _check(_p._L.sd_paged_tree_workspace(pages.struct, batch, n, hq, size))
        if len(_WORKSPACE) >= 4096:
            _WORKSPACE.clear()
        need = _WORKSPACE[key] = size.value
    if out is None:
        out = _like(q, stream)
    if stream is None:
        work = torch.empty(need, dtype=_p._U8, device=pages.torch_device)
    else:
        with _on(stream):
            work = torch.empty(need, dtype=_p._U8, device=pages.torch_device)
    _check(_p._L.sd_paged_tree_decode(
        pages.struct, _count(layer, "layer"), _arg(q, "q", dt, dev), n, batch, hq, _arg(tables, "tables", i32, dev),
        _count(width, "width"), _arg(lengths, "lengths", i32, dev, (batch,)), _arg(first, "first", i32, dev, (batch + 1,)),
        _arg(masks, "masks", torch.int64, dev, (n,)), _arg(places, "places", i32, dev, (n,)), scale,
        _count(window, "window"), _arg(sinks, "sinks", _p._F32, dev, (hq,)), _arg(out, "out", dt, dev, shape),
        work.data_ptr(), need, _arg(flags, "flags", i32, dev), _handle(stream, dev)))
    return out


def paged_keep(pages: KVPages, tables, ends, first, path, kept, *, lengths=None, flags=None, stream=None):
    """Keep kept[b] of the new tokens of each sequence, the nodes path[b, :kept[b]]
    in rising order: their rows move, in every layer, to the places after the
    tokens before the step. Returns the new lengths [batch], in `lengths` when
    it is given (the lengths that the plan was made from, say; none of the
    inputs here).

    tables [batch, width], ends [batch], first [batch + 1], path [batch, up to
    64], kept [batch]: int32. An entry that is no node, or does not rise, ends
    its sequence's path and sets bit 2 of flags. That a path goes down the tree
    from a root and names no absent node is the caller's (`PagedBatch.keep`
    checks it): rows move as they are."""
    dev, i32 = pages.here(), _p._I32
    if tables.dim() != 2 or path.dim() != 2 or path.shape[0] != tables.shape[0]:
        raise ValueError("tables must be [batch, width] and path [batch, nodes]")
    batch, width = tables.shape
    if lengths is None:
        lengths = _like(ends, stream)
    _check(_p._L.sd_paged_keep(
        pages.struct, _arg(tables, "tables", i32, dev), _count(batch, "batch"), _count(width, "width"),
        _arg(ends, "ends", i32, dev, (batch,)), _arg(first, "first", i32, dev, (batch + 1,)),
        _arg(path, "path", i32, dev), _count(path.shape[1], "nodes"), _arg(kept, "kept", i32, dev, (batch,)),
        _arg(lengths, "lengths", i32, dev, (batch,)), _arg(flags, "flags", i32, dev), _handle(stream, dev)))
    return lengths

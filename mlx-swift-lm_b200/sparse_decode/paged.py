"""Paged serving cache: rotary positions, page appends and copies, and decode
attention of many sequences of different lengths over one pool of pages.

The operators (each one launch, decode two) work on the caller's tensors and
keep nothing between calls:

* `rotary`        -- per-head RMS norm (optional) and rotary positions of
                     queries and keys;
* `paged_append`  -- the same, with keys and values stored into their pages
                     (quantized for 4/8-bit pools);
* `copy_pages`    -- whole pages copied inside a pool, in every layer;
* `paged_decode`  -- attention of one new token per sequence over its pages.

`PagePool` owns a pool and the map of sequences to pages (fork, copy-on-write,
trim, free, compaction); `PagedBatch` is one step's view of some sequences,
whose layers `attention_with_cache_update` takes as caches.

All calls run on the current device; `stream` defaults to the current stream.
Tensors last used on another stream must be ordered before the call by the
caller, as for any torch operation.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence

from . import DTYPES, SDError, SDPages, SDRotation, SDRows, _check, _torch_dtype, lib

# torch, its names used per call and the library, bound at the first call: the
# calls here take a few microseconds on the GPU, so the host's share counts.
torch = None
_device = _raw_stream = None
_CODE: dict = {}
_I32 = _F32 = _U8 = None
_L: Optional[ctypes.CDLL] = None
_WORKSPACE: dict = {}  # bytes of paged_decode's workspace, which depend on the device and the heads alone


def _load() -> None:
    global torch, _device, _raw_stream, _I32, _F32, _U8, _L
    import torch as t
    _L = lib()
    t.cuda.init()
    _device, _raw_stream = t.cuda.current_device, t._C._cuda_getCurrentRawStream
    _I32, _F32, _U8 = t.int32, t.float32, t.uint8
    _CODE.update({_torch_dtype(n): c for n, c in DTYPES.items()})
    torch = t


def _dtype_code(dtype) -> int:
    code = _CODE.get(dtype)
    if code is None:
        raise TypeError(f"unsupported dtype {dtype}: float32, float16 or bfloat16")
    return code


def _arg(t, name: str, dtype, dev: int, shape=None) -> Optional[int]:
    """Device pointer of a contiguous tensor argument (None passes NULL)."""
    if t is None:
        return None
    if t.get_device() != dev:
        raise ValueError(f"{name} must be a CUDA tensor on the current device")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype} (got {t.dtype})")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)} (got {tuple(t.shape)})")
    return t.data_ptr()


def _count(n: int, name: str) -> int:
    """A number that goes into a 32-bit argument: ctypes would keep its low bits."""
    if not -(1 << 31) <= n < 1 << 31:
        raise ValueError(f"{name} must be below 2^31 (got {n})")
    return n


def _rows(t, name: str, dtype, dev: int, dim: int) -> tuple:
    """sd_rows of [tokens, heads, D] or [batch, heads, tokens, D] with any
    strides but the last, as (struct, batch, tokens, heads)."""
    if t.get_device() != dev:
        raise ValueError(f"{name} must be a CUDA tensor on the current device")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype} (got {t.dtype})")
    shape, st = t.shape, t.stride()
    if shape[-1] != dim:
        raise ValueError(f"{name} has head_dim {shape[-1]}, expected {dim}")
    if st[-1] != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    if max(shape) >= 1 << 31:
        raise ValueError(f"{name} must have fewer than 2^31 tokens and heads (got {tuple(shape)})")
    if len(shape) == 3:
        return SDRows(t.data_ptr(), 0, st[0], st[1]), 1, shape[0], shape[1]
    if len(shape) == 4:
        return SDRows(t.data_ptr(), st[0], st[2], st[1]), shape[0], shape[2], shape[1]
    raise ValueError(f"{name} must be [tokens, heads, D] or [batch, heads, tokens, D]")


def _like(x, stream):
    """A new dense tensor of x's shape for work on `stream`."""
    if stream is None:
        y = torch.empty_like(x)
        return y if y.stride(-1) == 1 else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    with torch.cuda.stream(stream):
        return _like(x, None)


def _out(x, out, name: str, dtype, dev: int, dim: int, stream) -> tuple:
    """The output for x's rows -- `out`, or a new tensor -- and its sd_rows."""
    if out is not None:
        if out.shape != x.shape:
            raise ValueError(f"{name} must have its input's shape")
        return out, _rows(out, name, dtype, dev, dim)[0]
    out = _like(x, stream)
    st = out.stride()
    if len(st) == 3:
        return out, SDRows(out.data_ptr(), 0, st[0], st[1])
    return out, SDRows(out.data_ptr(), st[0], st[2], st[1])


def _refuse_capture(stream) -> None:
    with torch.cuda.stream(stream):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("host lists and tables cannot be copied in a captured graph")


def _upload(host, stream):
    """Pinned host tensor -> device, queued on `stream` (None: the current one) without waiting; the allocator keeps
    the host memory until it is copied. A graph would read it again at every replay, when it holds something else."""
    _refuse_capture(stream)
    with torch.cuda.stream(stream):
        return host.to("cuda", non_blocking=True)


def _handle(stream, dev: int) -> int:
    return _raw_stream(dev) if stream is None else stream.cuda_stream


def _rotation(inv_freq, traditional, factor, q_norm, k_norm, eps, dtype, dev: int, dim: int) -> SDRotation:
    rot = 0
    if inv_freq is not None:
        if inv_freq.dim() != 1:
            raise ValueError("inv_freq must be [rot_dim / 2]")
        rot = _count(2 * inv_freq.shape[0], "rot_dim")
    return SDRotation(_arg(inv_freq, "inv_freq", _F32, dev), _arg(q_norm, "q_norm", dtype, dev, (dim,)),
                      _arg(k_norm, "k_norm", dtype, dev, (dim,)), eps, factor, rot, 1 if traditional else 0)


# The keys of a rope_scaling dict that each kind's formula has, and those that every kind's dict may have: the lengths,
# which some formulas read, and what says nothing about the angles (rope_theta is checked against the base).
_SCALING_KEYS = {
    "default": (),
    "linear": ("factor",),
    "llama3": ("factor", "low_freq_factor", "high_freq_factor"),
    "yarn": ("factor", "beta_fast", "beta_slow", "truncate", "attention_factor", "mscale", "mscale_all_dim"),
    "longrope": ("factor", "long_factor", "short_factor", "attention_factor"),
}
_SCALING_KEYS["su"] = _SCALING_KEYS["longrope"]
_COMMON_KEYS = ("type", "rope_type", "rope_theta", "partial_rotary_factor", "finetuned", "max_position_embeddings",
                "original_max_position_embeddings")


def rotary_frequencies(rot_dim: int, base: float = 10000.0, scaling: Optional[dict] = None, device="cuda", *,
                       max_position_embeddings: Optional[int] = None,
                       original_max_position_embeddings: Optional[int] = None):
    """(inv_freq [rot_dim / 2] fp32 on `device`, factor) for `rotary` and
    `paged_append`: base^(-2i / rot_dim), computed in 64 bits, with the
    positions stretched for long contexts by `scaling`, a model
    configuration's rope_scaling dict:

    * linear:   angles divided by `factor`;
    * llama3:   only wavelengths beyond original_max_position_embeddings /
                low_freq_factor are divided, those below .../high_freq_factor
                are kept, a linear blend between;
    * yarn:     the same blend by the number of turns over the original
                context (beta_fast, beta_slow; between whole pairs unless
                `truncate` is false), and the rotated part scaled by
                0.1 ln(factor) + 1 (or by the mscale pair's ratio);
    * longrope: each angle divided by its own entry of long_factor (of
                short_factor when `factor` is at most 1), rotated part scaled
                by sqrt(1 + ln(factor) / ln(original)) or attention_factor.
                Where the dict has no `factor`, it is max_position_embeddings
                / original_max_position_embeddings, which such configurations
                keep outside of it: pass them here.

    A missing `factor` or original length is refused, and so is a key that the
    formula does not have; low_ and high_freq_factor are 1 and 4, beta_fast
    and beta_slow 32 and 1 where they are not given. What the dict says comes
    before the parameters; None counts as not given.
    """
    import torch
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError("rot_dim must be even and at least 2")
    inv = base ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim)
    mult = 1.0
    if scaling is not None:
        scaling = {k: v for k, v in scaling.items() if v is not None}
        kind = scaling.get("rope_type", scaling.get("type", "default"))
        if kind not in _SCALING_KEYS:
            raise ValueError(f"unknown rope scaling {kind!r}")
        other = [k for k in scaling if k not in _SCALING_KEYS[kind] and k not in _COMMON_KEYS]
        if other:
            raise ValueError(f"{kind} rope scaling does not have {', '.join(other)}")
        if float(scaling.get("rope_theta", base)) != float(base):
            raise ValueError(f"rope_theta is {scaling['rope_theta']}, the base {base}")
        f = float(scaling.get("factor", 1.0))
        known = scaling.get("original_max_position_embeddings", original_max_position_embeddings)
        most = scaling.get("max_position_embeddings", max_position_embeddings)
        if kind in ("linear", "llama3", "yarn") and "factor" not in scaling:
            raise ValueError(f"{kind} rope scaling needs factor")
        if kind in ("llama3", "yarn") and known is None:
            raise ValueError(f"{kind} rope scaling needs original_max_position_embeddings")
        old = float(known or 0)
        if kind == "linear":
            inv = inv / f
        elif kind == "llama3":
            lo, hi = float(scaling.get("low_freq_factor", 1.0)), float(scaling.get("high_freq_factor", 4.0))
            if hi <= lo:
                raise ValueError("high_freq_factor must be above low_freq_factor")
            turns = old * inv / (2 * math.pi)
            keep = ((turns - lo) / (hi - lo)).clamp(0, 1)
            inv = inv * (keep + (1 - keep) / f)
        elif kind == "yarn":
            def dim_of(turns: float) -> float:  # the pair that makes `turns` turns over the original context
                return rot_dim * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(base))
            lo, hi = dim_of(float(scaling.get("beta_fast", 32.0))), dim_of(float(scaling.get("beta_slow", 1.0)))
            if scaling.get("truncate", True):
                lo, hi = math.floor(lo), math.ceil(hi)
            lo, hi = max(lo, 0), min(hi, rot_dim - 1)
            i = torch.arange(rot_dim // 2, dtype=torch.float64)
            stretch = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
            inv = inv * (1 - stretch) + inv / f * stretch

            def mscale(m: float) -> float:
                return 0.1 * m * math.log(f) + 1.0 if f > 1 else 1.0
            if "attention_factor" in scaling:
                mult = float(scaling["attention_factor"])
            elif ("mscale" in scaling) != ("mscale_all_dim" in scaling):
                raise ValueError("mscale and mscale_all_dim come together")
            elif scaling.get("mscale") and scaling.get("mscale_all_dim"):
                mult = mscale(float(scaling["mscale"])) / mscale(float(scaling["mscale_all_dim"]))
            else:
                mult = mscale(1.0)
        elif kind in ("longrope", "su"):
            if "factor" not in scaling:
                if known is None or most is None:
                    raise ValueError("longrope needs factor, or max_ and original_max_position_embeddings")
                f = most / known
            name = "long_factor" if f > 1 else "short_factor"
            each = scaling.get(name)
            if each is None or len(each) != rot_dim // 2:
                raise ValueError(f"longrope needs {rot_dim // 2} numbers in {name}")
            inv = inv / torch.tensor(each, dtype=torch.float64)
            if "attention_factor" in scaling:
                mult = float(scaling["attention_factor"])
            elif f > 1:
                if known is None:
                    raise ValueError("longrope needs original_max_position_embeddings or attention_factor")
                mult = math.sqrt(1 + math.log(f) / math.log(known))
    return inv.to(torch.float32).to(device), mult


def rotary(q, k, positions, inv_freq, *, traditional: bool = False, factor: float = 1.0, q_norm=None, k_norm=None,
           eps: float = 1e-6, q_out=None, k_out=None, stream=None):
    """Rotary positions of queries and keys, with a per-head RMS norm before
    them when q_norm / k_norm ([D] weights) are given, in one pass.

    q, k: [tokens, heads, D] or [batch, heads, tokens, D] (any strides but the
    last; either may be None); positions: int32 [tokens] or [batch, tokens].
    inv_freq: fp32 [rot_dim / 2] (`rotary_frequencies`); the first rot_dim
    elements of a head are rotated, in pairs (i, i + rot_dim / 2), or
    neighbours when `traditional`. Returns (q_out, k_out), new dense tensors
    unless given; a given one may be its input."""
    if torch is None:
        _load()
    ref = q if q is not None else k
    if ref is None:
        raise ValueError("q or k is required")
    dev, dt, dim = _device(), ref.dtype, ref.shape[-1]
    code = _dtype_code(dt)
    qr = qo = kr = ko = None
    hq = hk = 0
    if q is not None:
        qr, batch, tokens, hq = _rows(q, "q", dt, dev, dim)
        q_out, qo = _out(q, q_out, "q_out", dt, dev, dim, stream)
    if k is not None:
        kr, b, n, hk = _rows(k, "k", dt, dev, dim)
        if q is None:
            batch, tokens = b, n
        elif b != batch or n != tokens or k.dim() != q.dim():
            raise ValueError("q and k must have the same tokens")
        k_out, ko = _out(k, k_out, "k_out", dt, dev, dim, stream)
    pos = _arg(positions, "positions", _I32, dev, (tokens,) if ref.dim() == 3 else (batch, tokens))
    rot = _rotation(inv_freq, traditional, factor, q_norm, k_norm, eps, dt, dev, dim)
    _check(_L.sd_rotary(rot, code, dim, batch, tokens, pos, hq, qr, qo, hk, kr, ko, _handle(stream, dev)))
    return (q_out if q is not None else None), (k_out if k is not None else None)


class KVPages:
    """The device arrays of a pool: k, v [n_pages, Hkv, page_size, D], or with
    a leading n_layers dimension. 4/8-bit pools (`bits`): k, v int32 codes
    [..., D * bits / 32] with scales and biases [..., D / 64] (the affine tuple
    of a quantized cache)."""

    def __init__(self, k, v, k_scales=None, k_biases=None, v_scales=None, v_biases=None, bits: int = 0):
        if torch is None:
            _load()
        dev, shape = k.get_device(), k.shape
        if dev < 0:
            raise ValueError("pool arrays must be CUDA tensors")
        if len(shape) == 4:
            n_layers, (n_pages, hkv, page, dim) = 1, shape
        elif len(shape) == 5:
            n_layers, n_pages, hkv, page, dim = shape
        else:
            raise ValueError("pool arrays must be [n_pages, Hkv, page_size, .] or [n_layers, n_pages, Hkv, page_size, .]")
        small = (k_scales, k_biases, v_scales, v_biases)
        if bits:
            if k_scales is None or k_biases is None or v_scales is None or v_biases is None:
                raise ValueError("a quantized pool needs k/v scales and biases")
            dt, dim = k_scales.dtype, dim * 32 // bits
            each = k_scales.shape
            if each[:-1] != shape[:-1] or each[-1] != dim // 64:
                raise ValueError(f"k_scales must have shape {(*shape[:-1], dim // 64)} (got {tuple(each)})")
            ptrs = (_arg(k, "k", _I32, dev), _arg(v, "v", _I32, dev, shape), _arg(k_scales, "k_scales", dt, dev),
                    _arg(k_biases, "k_biases", dt, dev, each), _arg(v_scales, "v_scales", dt, dev, each),
                    _arg(v_biases, "v_biases", dt, dev, each))
        else:
            if small != (None, None, None, None):
                raise ValueError("scales and biases need bits")
            dt = k.dtype
            ptrs = (_arg(k, "k", dt, dev), _arg(v, "v", dt, dev, shape), None, None, None, None)
        self.k, self.v = k, v
        self.k_scales, self.k_biases, self.v_scales, self.v_biases = small
        self.bits, self.device, self.torch_device, self.dtype = bits, dev, k.device, dt
        self.n_layers, self.n_pages = n_layers, n_pages
        self.n_kv_heads, self.page_size, self.head_dim = hkv, page, dim
        self.struct = SDPages(*ptrs, n_pages, n_layers, hkv, dim, page, _dtype_code(dt), bits, 64 if bits else 0, 0)

    def here(self) -> int:
        """The current device, which must be the pool's."""
        dev = _device()
        if dev != self.device:
            raise ValueError(f"the pool is on cuda:{self.device}, the current device is cuda:{dev}")
        return dev


def paged_append(pages: KVPages, k, v, tables, positions, *, seq=None, layer: int = 0, q=None, inv_freq=None,
                 traditional: bool = False, factor: float = 1.0, q_norm=None, k_norm=None, eps: float = 1e-6,
                 q_out=None, flags=None, stream=None):
    """Store new tokens k, v [tokens, Hkv, D] into layer `layer` of the pool:
    token n of sequence seq[n] (None: n) at positions[n] lands in page
    tables[seq[n], position // page_size]; a negative position stores nothing.
    With inv_freq or a norm the keys are normed and rotated on the way, and so
    are queries q [tokens, Hq, D], which are returned (else None). Quantized
    pools store codes of the rotated rows rounded to the pool's type.

    tables [batch, width], positions [tokens], seq [tokens]: int32. flags: an
    int32 tensor that receives bit 2 when an index is out of range (nothing is
    stored for that token)."""
    dev, dt, dim = pages.here(), pages.dtype, pages.head_dim
    kr, b, n, h = _rows(k, "k", dt, dev, dim)
    vr, vb, vn, vh = _rows(v, "v", dt, dev, dim)
    if k.dim() != 3 or v.dim() != 3 or vn != n or vh != h or h != pages.n_kv_heads:
        raise ValueError(f"k and v must be [tokens, {pages.n_kv_heads}, {dim}]")
    if tables.dim() != 2:
        raise ValueError("tables must be [batch, width]")
    rot = qr = qo = None
    hq = 0
    if q is not None:
        qr, qb, qn, hq = _rows(q, "q", dt, dev, dim)
        if q.dim() != 3 or qn != n:
            raise ValueError("q must have k's tokens")
        q_out, qo = _out(q, q_out, "q_out", dt, dev, dim, stream)
    if q is not None or inv_freq is not None or q_norm is not None or k_norm is not None:
        rot = _rotation(inv_freq, traditional, factor, q_norm, k_norm, eps, dt, dev, dim)
    batch, width = _count(tables.shape[0], "batch"), _count(tables.shape[1], "width")
    _check(_L.sd_paged_append(pages.struct, _count(layer, "layer"), n, kr, vr, _arg(tables, "tables", _I32, dev), batch,
                              width, _arg(positions, "positions", _I32, dev, (n,)), _arg(seq, "seq", _I32, dev, (n,)),
                              rot, hq, qr, qo, _arg(flags, "flags", _I32, dev), _handle(stream, dev)))
    return q_out if q is not None else None


def copy_pages(pages: KVPages, src, dst, *, flags=None, stream=None) -> None:
    """Page dst[i] = page src[i] in every layer and array of the pool. src,
    dst: int32 CUDA tensors, or sequences of ints (checked here). The dst
    pages must be distinct and none of them a src."""
    dev = pages.here()
    if not isinstance(src, torch.Tensor):
        src, dst = [int(i) for i in src], [int(i) for i in dst]
        if len(src) != len(dst):
            raise ValueError("src and dst must have the same length")
        if any(not 0 <= i < pages.n_pages for i in src + dst):
            raise ValueError("page out of range")
        if len(set(dst)) != len(dst) or set(dst) & set(src):
            raise ValueError("dst pages must be distinct and none of them a src")
        both = _upload(torch.tensor([src, dst], dtype=_I32, pin_memory=True), stream)
        src, dst = both[0], both[1]
    if src.dim() != 1:
        raise ValueError("src and dst must be [n]")
    _check(_L.sd_copy_pages(pages.struct, _arg(src, "src", _I32, dev), _arg(dst, "dst", _I32, dev, src.shape),
                            _count(src.shape[0], "n"), _arg(flags, "flags", _I32, dev), _handle(stream, dev)))


def paged_decode(q, pages: KVPages, tables, lengths, scale: Optional[float] = None, *, layer: int = 0, window: int = 0,
                 sinks=None, out=None, flags=None, stream=None):
    """Attention of one new token per sequence over its pages: q
    [batch, Hq, D] (contiguous, on a 16-byte boundary) -> [batch, Hq, D], softmax(scale q K^T) V over the last
    `window` (0: all) of lengths[b] tokens. A length of 0 gives zeros.

    tables [batch, width] and lengths [batch]: int32, read on the device only,
    so a captured call serves growing sequences. sinks: fp32 [Hq] logits that
    join the denominators. Hq / Hkv: 1 .. 16."""
    dev, dt, dim = pages.here(), pages.dtype, pages.head_dim
    shape, (batch, width) = q.shape, tables.shape
    if len(shape) != 3 or shape[0] != batch or shape[2] != dim:
        raise ValueError(f"q must be [batch, Hq, {dim}] and tables [batch, width]")
    hq = shape[1]
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    need = _WORKSPACE.get((dev, pages.n_kv_heads, dim, hq))
    if need is None:
        n = ctypes.c_int64()
        _check(_L.sd_paged_workspace(pages.struct, 1, hq, n))
        need = _WORKSPACE[dev, pages.n_kv_heads, dim, hq] = n.value
    if out is None:
        out = _like(q, stream)
    if stream is None:
        work = torch.empty(need, dtype=_U8, device=pages.torch_device)
    else:
        with torch.cuda.stream(stream):
            work = torch.empty(need, dtype=_U8, device=pages.torch_device)
    _check(_L.sd_paged_decode(pages.struct, _count(layer, "layer"), _arg(q, "q", dt, dev), batch, hq,
                              _arg(tables, "tables", _I32, dev), _count(width, "width"),
                              _arg(lengths, "lengths", _I32, dev, (batch,)), scale, _count(window, "window"),
                              _arg(sinks, "sinks", _F32, dev, (hq,)), _arg(out, "out", dt, dev, shape), work.data_ptr(),
                              need, _arg(flags, "flags", _I32, dev), _handle(stream, dev)))
    return out


class PagePool:
    """A pool of KV pages for every layer of a model, and the sequences in it.

    Sequences are named by the ids that `add` and `fork` return. Forking shares
    every page; the first token that a sequence adds to a page it shares moves
    it to a copy of its own (`extend` launches that copy). Pages are freed when
    no sequence holds them."""

    def __init__(self, n_layers: int, n_pages: int, n_kv_heads: int, head_dim: int, page_size: int = 64,
                 dtype: str = "bf16", kv_bits: int = 0):
        if torch is None:
            _load()
        if kv_bits not in (0, 4, 8):
            raise ValueError("kv_bits must be 0, 4 or 8")
        lead = (n_layers, n_pages, n_kv_heads, page_size)
        tdt = _torch_dtype(dtype)
        new = lambda last, dt: torch.zeros((*lead, last), dtype=dt, device="cuda")  # noqa: E731
        if kv_bits:
            data = [new(head_dim * kv_bits // 32, torch.int32) for _ in "kv"]
            small = [new(head_dim // 64, tdt) for _ in range(4)]
            self.pages = KVPages(*data, *small, bits=kv_bits)
        else:
            self.pages = KVPages(new(head_dim, tdt), new(head_dim, tdt))
        self.flags = torch.zeros(1, dtype=torch.int32, device="cuda")
        h = ctypes.c_void_p()
        _check(lib().sd_pagemap_create(n_pages, page_size, ctypes.byref(h)))
        self._h = h

    def close(self) -> None:
        if getattr(self, "_h", None) is not None and self._h.value:
            lib().sd_pagemap_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # -- sequences -------------------------------------------------------------
    def add(self) -> int:
        s = ctypes.c_int64()
        _check(lib().sd_pagemap_add(self._h, ctypes.byref(s)))
        return s.value

    def fork(self, seq: int) -> int:
        s = ctypes.c_int64()
        _check(lib().sd_pagemap_fork(self._h, seq, ctypes.byref(s)))
        return s.value

    def free(self, seq: int) -> None:
        _check(lib().sd_pagemap_free(self._h, seq))

    def trim(self, seq: int, n: int) -> int:
        t = ctypes.c_int64()
        _check(lib().sd_pagemap_trim(self._h, seq, n, ctypes.byref(t)))
        return t.value

    def length(self, seq: int) -> int:
        t = ctypes.c_int64()
        _check(lib().sd_pagemap_length(self._h, seq, ctypes.byref(t)))
        return t.value

    @property
    def free_pages(self) -> int:
        n = ctypes.c_int64()
        _check(lib().sd_pagemap_free_pages(self._h, ctypes.byref(n)))
        return n.value

    def compact(self, stream=None) -> int:
        """Move pages so that the used ones are the lowest; returns how many
        moved. Batches made before are stale afterwards."""
        _refuse_capture(stream)
        n = ctypes.c_int32()
        room = self.pages.n_pages // 2
        src, dst = (ctypes.c_int32 * max(room, 1))(), (ctypes.c_int32 * max(room, 1))()
        _check(lib().sd_pagemap_compact(self._h, src, dst, room, ctypes.byref(n)))
        if n.value:
            copy_pages(self.pages, src[:n.value], dst[:n.value], flags=self.flags, stream=stream)
        return n.value

    # -- steps -----------------------------------------------------------------
    def extend(self, seqs: Sequence[int], n_tokens, stream=None) -> "PagedBatch":
        """Make room for n_tokens (an int, or one per sequence) more tokens of
        each sequence and return the batch that appends them. All or nothing:
        when the pool has too few free pages, or anything else is refused, no
        sequence grows. Page copies and the batch's tables are issued on
        `stream`, on which the step's calls must then run or wait."""
        each = [int(n_tokens)] * len(seqs) if isinstance(n_tokens, int) else [int(n) for n in n_tokens]
        if len(each) != len(seqs):
            raise ValueError("n_tokens must be an int or one per sequence")
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence may be named once per batch")
        if any(not -(1 << 63) <= i < 1 << 63 for i in [*seqs, *each]):  # what ctypes would keep the low bits of
            raise ValueError("a sequence or its number of tokens does not fit 64 bits")
        _refuse_capture(stream)
        src, dst, n = ctypes.c_int32(), ctypes.c_int32(), ctypes.c_int32()
        copies, grown = [], []
        try:
            for s, k in zip(seqs, each):
                _check(lib().sd_pagemap_extend(self._h, s, k, ctypes.byref(src), ctypes.byref(dst), ctypes.byref(n)))
                grown.append((s, k))
                if n.value:
                    copies.append((src.value, dst.value))
            batch = PagedBatch(self, list(seqs), each, stream)
        except BaseException:
            try:  # the pages already copied-on-write stay with their sequences, so their contents must follow
                if copies:
                    copy_pages(self.pages, *zip(*copies), flags=self.flags, stream=stream)
            finally:
                for s, k in grown:
                    self.trim(s, k)
            raise
        if copies:
            copy_pages(self.pages, *zip(*copies), flags=self.flags, stream=stream)
        return batch

    def batch(self, seqs: Sequence[int], stream=None) -> "PagedBatch":
        """The sequences as they are, with no new tokens."""
        return PagedBatch(self, list(seqs), [0] * len(seqs), stream)

    def check_device(self) -> int:
        """Read and clear the device error bits (synchronises)."""
        f = int(self.flags.item())
        self.flags.zero_()
        return f


class PagedBatch:
    """One step of some sequences of a pool: `tables` [batch, width] and
    `lengths` [batch] with the step's new tokens counted in, and for the new
    tokens, sequence by sequence, `positions` and `seq`. Built on the host and
    copied to the device once, for every layer of the step."""

    def __init__(self, pool: PagePool, seqs: list, new: list, stream=None):
        self.pool, self.seqs, self.new = pool, seqs, new
        n = len(seqs)
        ids = (ctypes.c_int64 * max(n, 1))(*seqs)
        width = ctypes.c_int32()
        _check(lib().sd_pagemap_width(pool._h, ids, n, ctypes.byref(width)))
        w = width.value
        tokens = sum(new)
        host = torch.empty(n * w + n + 2 * tokens, dtype=torch.int32, pin_memory=True)
        i32p = ctypes.POINTER(ctypes.c_int32)
        at = lambda k: ctypes.cast(host.data_ptr() + 4 * k, i32p)  # noqa: E731
        _check(lib().sd_pagemap_tables(pool._h, ids, n, w, at(0), at(n * w)))
        lengths = host[n * w:n * w + n].tolist()
        pos = [p for t, k in zip(lengths, new) for p in range(t - k, t)]
        seq = [b for b, k in enumerate(new) for _ in range(k)]
        host[n * w + n:] = torch.tensor(pos + seq, dtype=torch.int32)
        dev = _upload(host, stream)
        self.tables = dev[:n * w].view(n, w)
        self.lengths = dev[n * w:n * w + n]
        self.positions = dev[n * w + n:n * w + n + tokens]
        self.seq = dev[n * w + n + tokens:]
        self.host_lengths = lengths

    def append(self, layer: int, k, v, q=None, **rotation):
        """`paged_append` of this step's new tokens [tokens, heads, D]."""
        return paged_append(self.pool.pages, k, v, self.tables, self.positions, seq=self.seq, layer=layer, q=q,
                            flags=self.pool.flags, **rotation)

    def decode(self, layer: int, q, scale: Optional[float] = None, **kw):
        """`paged_decode` of one query token per sequence [batch, Hq, D]."""
        return paged_decode(q, self.pool.pages, self.tables, self.lengths, scale, layer=layer, flags=self.pool.flags,
                            **kw)

    def layer(self, layer: int, *, window: int = 0, **rotation) -> "PagedLayer":
        """Layer `layer` of this step as a cache for attention_with_cache_update;
        `window`: each new token sees the last `window` tokens up to itself
        (0: all); `rotation`: the keyword arguments of `paged_append` that norm
        and rotate queries and keys (none: they come in rotated)."""
        return PagedLayer(self, layer, rotation, window)


class PagedLayer:
    """What attention_with_cache_update needs of a paged step's layer."""

    def __init__(self, batch: PagedBatch, layer: int, rotation: dict, window: int = 0):
        if window < 0:
            raise ValueError("window must not be negative")
        self.batch, self.index, self.rotation, self.window = batch, layer, rotation, window

    @property
    def offset(self):
        """Tokens of each sequence before this step."""
        return [t - n for t, n in zip(self.batch.host_lengths, self.batch.new)]

    def attend(self, queries, keys, values, scale: float, mask=None, sinks=None):
        """Append keys/values [B, Hkv, L, D] and attend with queries
        [B, Hq, L, D]; every sequence has L new tokens. L == 1 takes the decode
        kernel; longer prompts are attended densely, sequence by sequence, with
        `mask` as for the other caches: None hides nothing, "causal" the tokens
        after each one; a tensor (bool, or numbers to add) is broadcast to
        [B, Hq, L, T], T the longest sequence's tokens, and column t is token t
        of every sequence. A layer with a window takes several tokens with
        "causal" only."""
        from .cache import _dense_attention
        b = self.batch
        B, Hq, L, D = queries.shape
        if any(n != L for n in b.new) or len(b.new) != B:
            raise ValueError(f"the step holds {b.new} new tokens, the queries {[L] * B}")
        if L == 1 and mask is not None and not isinstance(mask, str):
            raise ValueError("a single-token step takes no mask but \"causal\", which hides nothing there")
        masks = self._masks(mask, B, Hq, L)
        flat = lambda x: x.transpose(1, 2).reshape(B * L, x.shape[1], D)  # noqa: E731
        q = flat(queries)
        if self.rotation:
            q = b.append(self.index, flat(keys), flat(values), q=q, **self.rotation)
        else:
            b.append(self.index, flat(keys), flat(values))
        if L == 1:
            sinks = None if sinks is None else sinks.detach().float().contiguous()
            return b.decode(self.index, q.contiguous(), scale, window=self.window, sinks=sinks).view(B, Hq, 1, D)
        q = q.view(B, L, Hq, D).transpose(1, 2)
        out = torch.empty_like(queries)
        for i in range(B):
            k, v = self.dense(i)
            out[i] = _dense_attention(q[i:i + 1], k, v, scale, masks[i], sinks)[0]
        return out

    def _masks(self, mask, B: int, Hq: int, L: int) -> list:
        """The mask of each sequence."""
        lengths = self.batch.host_lengths
        if mask is None or isinstance(mask, str):
            if mask not in (None, "causal"):
                raise ValueError(f"unknown mask {mask!r}")
            if not self.window or L == 1:  # a single token's window is the kernel's
                return [mask] * B
        if self.window and not isinstance(mask, str):
            raise ValueError("a layer with a window takes several tokens with mask \"causal\"")
        if self.window:
            dev = self.batch.tables.device
            back = [torch.arange(n - L, n, device=dev)[:, None] - torch.arange(n, device=dev) for n in lengths]
            return [(x >= 0) & (x < self.window) for x in back]
        shape = (B, Hq, L, max(lengths))
        if not 2 <= mask.dim() <= 4 or any(n not in (1, m) for n, m in zip(reversed(mask.shape), reversed(shape))):
            raise ValueError(f"mask must broadcast to {shape} (got {tuple(mask.shape)})")
        mask = mask.expand(shape)
        return [mask[i:i + 1, ..., :n] for i, n in enumerate(lengths)]

    def dense(self, i: int):
        """Keys and values of the batch's sequence i, [1, Hkv, tokens, D]."""
        from .cache import _dequantize
        b, p = self.batch, self.batch.pool.pages
        n = b.host_lengths[i]
        at = b.tables[i, :-(-n // p.page_size)].long()

        def rows(x):
            x = x[self.index, at]
            return x.transpose(0, 1).flatten(1, 2)[None, :, :n]
        if not p.bits:
            return rows(p.k), rows(p.v)
        return (_dequantize(rows(p.k), rows(p.k_scales), rows(p.k_biases), p.bits),
                _dequantize(rows(p.v), rows(p.v_scales), rows(p.v_biases), p.bits))

"""The paged serving cache without a GPU: struct layouts, argument checks that
answer before any CUDA call, the page map, and rotary frequencies."""
from __future__ import annotations

import ctypes
import math
import random

import pytest

import sparse_decode as sdp
from sparse_decode import paged

from test_abi import _c_layout


@pytest.fixture(scope="module")
def native():
    if not sdp.LIB_PATH.exists():
        from sparse_decode import build as b
        b.build()
    return sdp.lib()


@pytest.mark.parametrize("cls,cname", [(paged.SDPages, "sd_pages"), (paged.SDRows, "sd_rows"),
                                       (paged.SDRotation, "sd_rotation")])
def test_struct_layout_matches_header(cls, cname):
    names = [f[0] for f in cls._fields_]
    lay = _c_layout(cname, names)
    assert lay["sizeof"] == ctypes.sizeof(cls)
    for n in names:
        assert lay[n] == getattr(cls, n).offset, n


# -- refusals ---------------------------------------------------------------

def _pages(**kw):
    base = dict(k_data=256, v_data=512, k_scales=None, k_biases=None, v_scales=None, v_biases=None, n_pages=8,
                n_layers=2, n_kv_heads=2, head_dim=128, page_size=64, dtype=2, kv_bits=0, group_size=0, reserved=0)
    base.update(kw)
    return paged.SDPages(**base)


BAD_POOLS = [
    (dict(k_data=None), "SD_ERR_INVALID_ARG"),
    (dict(v_data=520), "SD_ERR_INVALID_ARG"),           # not 16-byte aligned
    (dict(n_pages=0), "SD_ERR_INVALID_ARG"),
    (dict(n_layers=0), "SD_ERR_INVALID_ARG"),
    (dict(n_kv_heads=0), "SD_ERR_INVALID_ARG"),
    (dict(head_dim=96), "SD_ERR_SHAPE"),
    (dict(page_size=48), "SD_ERR_SHAPE"),
    (dict(page_size=8), "SD_ERR_SHAPE"),
    (dict(dtype=3), "SD_ERR_INVALID_ARG"),
    (dict(kv_bits=2, group_size=64), "SD_ERR_SHAPE"),
    (dict(kv_bits=8, group_size=32), "SD_ERR_SHAPE"),
    (dict(group_size=64), "SD_ERR_SHAPE"),              # a dense pool has no groups
    (dict(kv_bits=8, group_size=64), "SD_ERR_INVALID_ARG"),  # no scales
    (dict(n_pages=1 << 24), "SD_ERR_SHAPE"),            # 2^31 rows
    (dict(n_pages=1 << 62), "SD_ERR_SHAPE"),
    (dict(reserved=1), "SD_ERR_INVALID_ARG"),
]


@pytest.mark.parametrize("kw,status", BAD_POOLS)
def test_every_call_refuses_a_bad_pool(native, kw, status):
    g = _pages(**kw)
    rows = paged.SDRows(256, 0, 256, 128)
    n = ctypes.c_int64()
    calls = [native.sd_paged_workspace(g, 1, 8, ctypes.byref(n)),
             native.sd_copy_pages(g, 256, 512, 1, None, None),
             native.sd_paged_append(g, 0, 1, rows, rows, 256, 1, 1, 256, None, None, 0, None, None, None, None),
             native.sd_paged_decode(g, 0, 256, 1, 8, 256, 1, 256, 1.0, 0, None, 256, 256, 1 << 30, None, None)]
    assert [sdp.STATUS[c] for c in calls] == [status] * 4
    assert native.sd_last_error()


def _decode(native, **kw):
    a = dict(g=_pages(), layer=0, q=256, batch=2, heads=8, tables=256, width=4, lengths=256, scale=0.1, window=0,
             sinks=None, out=256, work=256, bytes=1 << 30, flags=None)
    a.update(kw)
    return sdp.STATUS[native.sd_paged_decode(*a.values(), None)]


@pytest.mark.parametrize("kw,status", [
    (dict(g=None), "SD_ERR_INVALID_ARG"), (dict(layer=2), "SD_ERR_INVALID_ARG"), (dict(layer=-1), "SD_ERR_INVALID_ARG"),
    (dict(batch=-1), "SD_ERR_SHAPE"), (dict(batch=5000), "SD_ERR_SHAPE"), (dict(heads=7), "SD_ERR_SHAPE"),
    (dict(heads=0), "SD_ERR_SHAPE"), (dict(heads=34), "SD_ERR_SHAPE"),  # 17 per kv head
    (dict(q=None), "SD_ERR_INVALID_ARG"), (dict(q=264), "SD_ERR_INVALID_ARG"), (dict(out=None), "SD_ERR_INVALID_ARG"),
    (dict(work=None), "SD_ERR_INVALID_ARG"), (dict(tables=258), "SD_ERR_INVALID_ARG"),
    (dict(lengths=None), "SD_ERR_INVALID_ARG"), (dict(scale=math.nan), "SD_ERR_INVALID_ARG"),
    (dict(scale=math.inf), "SD_ERR_INVALID_ARG"), (dict(window=-1), "SD_ERR_INVALID_ARG"),
    (dict(width=0), "SD_ERR_INVALID_ARG"), (dict(width=1 << 26), "SD_ERR_SHAPE"),
    (dict(flags=258), "SD_ERR_INVALID_ARG"), (dict(sinks=257), "SD_ERR_INVALID_ARG")])
def test_decode_refusals(native, kw, status):
    assert _decode(native, **kw) == status


def test_empty_calls_are_fine(native):
    assert _decode(native, batch=0) == "SD_OK"
    g, rows = _pages(), paged.SDRows(256, 0, 256, 128)
    assert native.sd_copy_pages(g, None, None, 0, None, None) == 0
    assert native.sd_paged_append(g, 0, 0, rows, rows, None, 0, 0, None, None, None, 0, None, None, None, None) == 0
    rot = paged.SDRotation(256, None, None, 1e-6, 1.0, 128, 0)
    assert native.sd_rotary(rot, 2, 128, 1, 0, None, 8, rows, rows, 2, rows, rows, None) == 0


def _rotary(native, rot_kw=None, **kw):
    r = dict(inv_freq=256, q_norm=None, k_norm=None, eps=1e-6, factor=1.0, rot_dim=128, traditional=0)
    r.update(rot_kw or {})
    rows = paged.SDRows(256, 0, 1024, 128)
    a = dict(rot=paged.SDRotation(**r), dtype=2, dim=128, batch=1, tokens=3, pos=256, hq=8, q=rows, qo=rows, hkv=2,
             k=rows, ko=rows)
    a.update(kw)
    return sdp.STATUS[native.sd_rotary(*a.values(), None)]


@pytest.mark.parametrize("kw", [
    dict(rot=None), dict(dtype=9), dict(batch=-1), dict(tokens=-1), dict(hq=-1), dict(pos=None), dict(pos=257),
    dict(q=None), dict(qo=None), dict(ko=None), dict(k=paged.SDRows(None, 0, 1, 1)), dict(k=paged.SDRows(257, 0, 1, 1)),
    dict(rot_kw=dict(inv_freq=None)), dict(rot_kw=dict(factor=math.nan)), dict(rot_kw=dict(eps=-1.0)),
    dict(rot_kw=dict(q_norm=257))])
def test_rotary_refuses_bad_arguments(native, kw):
    assert _rotary(native, **kw) == "SD_ERR_INVALID_ARG"


@pytest.mark.parametrize("kw", [
    dict(dim=0), dict(dim=127), dict(dim=258), dict(rot_kw=dict(rot_dim=130)), dict(rot_kw=dict(rot_dim=-2)),
    dict(rot_kw=dict(rot_dim=63)), dict(hq=70000)])
def test_rotary_refuses_bad_shapes(native, kw):
    assert _rotary(native, **kw) == "SD_ERR_SHAPE"


def test_append_and_copy_refusals(native):
    g, rows = _pages(), paged.SDRows(256, 0, 256, 128)
    rot = paged.SDRotation(256, None, None, 1e-6, 1.0, 128, 0)

    def append(layer=0, n=1, k=rows, v=rows, tables=256, batch=1, width=1, pos=256, seq=None, rot=None, hq=0, q=None,
               qo=None, flags=None):
        return sdp.STATUS[native.sd_paged_append(g, layer, n, k, v, tables, batch, width, pos, seq, rot, hq, q, qo,
                                                 flags, None)]
    inv = "SD_ERR_INVALID_ARG"
    assert append(layer=2) == inv and append(n=-1) == inv and append(k=None) == inv and append(v=None) == inv
    assert append(tables=None) == inv and append(pos=None) == inv and append(pos=258) == inv and append(seq=257) == inv
    assert append(hq=8, q=rows, qo=rows) == inv                     # queries need a rotation
    assert append(hq=8, q=rows, rot=rot) == inv                     # no place for the rotated queries
    assert append(rot=paged.SDRotation(256, None, None, 1e-6, 1.0, 130, 0)) == "SD_ERR_SHAPE"
    for args in ((None, 512, 1, None), (256, None, 1, None), (256, 512, -1, None), (257, 512, 1, None),
                 (256, 512, 1, 258)):
        assert sdp.STATUS[native.sd_copy_pages(g, *args, None)] == inv


# -- the page map -------------------------------------------------------------

class Map:
    """sd_pagemap through the C ABI."""

    def __init__(self, L, n_pages, page):
        self.L, self.n, self.page = L, n_pages, page
        self.h = ctypes.c_void_p()
        assert L.sd_pagemap_create(n_pages, page, ctypes.byref(self.h)) == 0

    def _id(self, f, *a):
        v = ctypes.c_int64()
        rc = f(self.h, *a, ctypes.byref(v))
        assert rc == 0, self.L.sd_last_error()
        return v.value

    def add(self):
        return self._id(self.L.sd_pagemap_add)

    def fork(self, s):
        return self._id(self.L.sd_pagemap_fork, s)

    def length(self, s):
        return self._id(self.L.sd_pagemap_length, s)

    def trim(self, s, n):
        return self._id(self.L.sd_pagemap_trim, s, n)

    def free(self, s):
        assert self.L.sd_pagemap_free(self.h, s) == 0

    def free_pages(self):
        return self._id(self.L.sd_pagemap_free_pages)

    def extend(self, s, n):
        src, dst, c = (ctypes.c_int32() for _ in range(3))
        rc = self.L.sd_pagemap_extend(self.h, s, n, ctypes.byref(src), ctypes.byref(dst), ctypes.byref(c))
        return sdp.STATUS[rc], ([(src.value, dst.value)] if c.value else [])

    def table(self, s, width=64):
        out, ln = (ctypes.c_int32 * width)(), ctypes.c_int32()
        ids = (ctypes.c_int64 * 1)(s)
        assert self.L.sd_pagemap_tables(self.h, ids, 1, width, out, ctypes.byref(ln)) == 0
        n = -(-ln.value // self.page)
        assert list(out[n:]) == [-1] * (width - n)
        return list(out[:n])

    def compact(self, room):
        src, dst, n = (ctypes.c_int32 * max(room, 1))(), (ctypes.c_int32 * max(room, 1))(), ctypes.c_int32()
        assert self.L.sd_pagemap_compact(self.h, src, dst, room, ctypes.byref(n)) == 0
        return list(zip(src[:n.value], dst[:n.value]))


def test_fork_shares_and_copies_on_write(native):
    m = Map(native, 8, 16)
    a = m.add()
    assert m.extend(a, 40) == ("SD_OK", []) and m.free_pages() == 5
    b = m.fork(a)
    assert m.table(b) == m.table(a) and m.free_pages() == 5 and m.length(b) == 40
    last = m.table(a)[-1]
    st, copies = m.extend(b, 1)              # token 41 lands in the shared third page
    assert st == "SD_OK" and copies == [(last, m.table(b)[-1])] and m.table(b)[:2] == m.table(a)[:2]
    assert m.extend(a, 1) == ("SD_OK", [])   # a holds its page alone now
    m.free(a)
    assert m.free_pages() == 4 + 1           # only a's third page was its own
    m.free(b)
    assert m.free_pages() == 8


def test_no_copy_at_a_page_boundary(native):
    m = Map(native, 8, 16)
    a = m.add()
    m.extend(a, 32)
    b = m.fork(a)
    assert m.extend(b, 1) == ("SD_OK", []) and m.extend(a, 1) == ("SD_OK", [])
    assert m.table(a)[:2] == m.table(b)[:2] and m.table(a)[2] != m.table(b)[2]


def test_trim_into_a_shared_page_copies_it(native):
    m = Map(native, 8, 16)
    a = m.add()
    m.extend(a, 32)
    b = m.fork(a)
    assert m.trim(b, 20) == 20 and m.length(b) == 12 and len(m.table(b)) == 1
    st, copies = m.extend(b, 1)
    assert copies == [(m.table(a)[0], m.table(b)[0])]
    assert m.trim(b, 100) == 13 and m.table(b) == []


def test_a_full_pool_refuses_and_changes_nothing(native):
    m = Map(native, 3, 16)
    a = m.add()
    m.extend(a, 40)
    b = m.fork(a)
    assert m.extend(b, 1)[0] == "SD_ERR_CAPACITY"       # its copy needs a page
    assert m.extend(a, 1000)[0] == "SD_ERR_CAPACITY"
    assert m.length(a) == m.length(b) == 40 and m.table(a) == m.table(b) and m.free_pages() == 0
    m.free(a)
    assert m.extend(b, 8) == ("SD_OK", [])              # the rest of the page is its own now


def test_pagemap_refusals(native):
    L = native
    h = ctypes.c_void_p()
    inv = "SD_ERR_INVALID_ARG"
    for n, p in ((0, 16), (8, 0), (1 << 31, 16)):
        assert sdp.STATUS[L.sd_pagemap_create(n, p, ctypes.byref(h))] == inv and not h.value
    assert sdp.STATUS[L.sd_pagemap_create(8, 16, None)] == inv
    assert L.sd_pagemap_destroy(None) == 0
    m = Map(L, 8, 16)
    v, i = ctypes.c_int64(), ctypes.c_int32()
    for f in (L.sd_pagemap_fork, L.sd_pagemap_length):
        assert sdp.STATUS[f(m.h, 5, ctypes.byref(v))] == "SD_ERR_STATE"
    assert sdp.STATUS[L.sd_pagemap_free(m.h, 0)] == "SD_ERR_STATE"
    a = m.add()
    assert m.extend(a, -1)[0] == inv and m.extend(a, 1 << 40)[0] == "SD_ERR_CAPACITY"
    assert m.extend(a, 0) == ("SD_OK", []) and m.table(a) == []
    assert sdp.STATUS[L.sd_pagemap_trim(m.h, a, -1, None)] == inv
    m.extend(a, 40)
    ids = (ctypes.c_int64 * 1)(a)
    out = (ctypes.c_int32 * 4)()
    assert sdp.STATUS[L.sd_pagemap_tables(m.h, ids, 1, 2, out, None)] == "SD_ERR_SHAPE"  # three pages
    assert sdp.STATUS[L.sd_pagemap_tables(m.h, ids, 1, 0, out, None)] == inv
    assert L.sd_pagemap_width(m.h, ids, 1, ctypes.byref(i)) == 0 and i.value == 3
    assert L.sd_pagemap_width(m.h, ids, 0, ctypes.byref(i)) == 0 and i.value == 1
    assert sdp.STATUS[L.sd_pagemap_compact(m.h, None, None, -1, ctypes.byref(i))] == inv


@pytest.mark.parametrize("seed", range(6))
def test_random_histories_keep_every_token(native, seed):
    """Pages hold their tokens in a host model of the pool; the copies that the
    map asks for are made, and every sequence still reads its own tokens."""
    r = random.Random(seed)
    page, n_pages = 16, 40
    m = Map(native, n_pages, page)
    store = [[None] * page for _ in range(n_pages)]
    text: dict = {}
    stamp = 0

    def read(s):
        return [store[p][j] for p in m.table(s) for j in range(page)][:m.length(s)]

    for _ in range(400):
        move = r.random()
        if move < 0.15 or not text:
            text[m.add()] = []
        elif move < 0.65:
            s, n = r.choice(list(text)), r.choice([1, 1, 2, r.randrange(1, 60)])
            before = m.table(s)
            st, copies = m.extend(s, n)
            if st == "SD_OK":
                for src, dst in copies:
                    store[dst] = list(store[src])
                t = m.table(s)
                for k in range(n):
                    stamp += 1
                    at = len(text[s])
                    store[t[at // page]][at % page] = stamp
                    text[s].append(stamp)
            else:
                assert m.table(s) == before and not copies
        elif move < 0.75:
            s = r.choice(list(text))
            text[m.fork(s)] = list(text[s])
        elif move < 0.85:
            s = r.choice(list(text))
            n = r.randrange(0, 40)
            got = m.trim(s, n)
            assert got == min(n, len(text[s]))
            text[s] = text[s][:len(text[s]) - got]
        elif move < 0.95:
            s = r.choice(list(text))
            m.free(s)
            del text[s]
        else:
            pairs = m.compact(r.choice([0, 2, n_pages]))
            srcs, dsts = {a for a, _ in pairs}, {b for _, b in pairs}
            assert len(dsts) == len(pairs) and not srcs & dsts
            for a, b in pairs:
                store[b] = list(store[a])
                store[a] = [None] * page
        used = {p for s in text for p in m.table(s)}
        assert m.free_pages() == n_pages - len(used)
        for s in text:
            assert read(s) == text[s]
    m.compact(n_pages)
    used = {p for s in text for p in m.table(s)}
    assert used == set(range(len(used)))


# -- rotary frequencies ---------------------------------------------------------

def _freq(*a, **kw):
    inv, mult = sdp.rotary_frequencies(*a, **kw, device="cpu")
    return inv.tolist(), mult


def test_plain_and_linear_frequencies():
    inv, mult = _freq(64, 10000.0)
    assert mult == 1.0 and inv == pytest.approx([10000 ** (-2 * i / 64) for i in range(32)], rel=1e-7)
    lin, _ = _freq(64, 10000.0, {"type": "linear", "factor": 4.0})
    assert lin == pytest.approx([x / 4 for x in inv], rel=1e-7)
    assert _freq(64, 10000.0, {"rope_type": "default"})[0] == inv


def test_llama3_frequencies_blend_by_wavelength():
    s = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
         "original_max_position_embeddings": 8192}
    base, _ = _freq(128, 500000.0)
    got, mult = _freq(128, 500000.0, s)
    assert mult == 1.0
    for x, y in zip(base, got):
        wave = 2 * math.pi / x
        if wave < 8192 / 4:
            assert y == pytest.approx(x, rel=1e-6)
        elif wave > 8192:
            assert y == pytest.approx(x / 8, rel=1e-6)
        else:
            blend = (8192 / wave - 1) / 3
            assert y == pytest.approx((1 - blend) * x / 8 + blend * x, rel=1e-6)


def test_yarn_frequencies_and_factor():
    s = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
    base, _ = _freq(128, 1e6)
    got, mult = _freq(128, 1e6, s)
    assert mult == pytest.approx(0.1 * math.log(4) + 1)
    ratio = [y / x for x, y in zip(base, got)]
    assert ratio[0] == pytest.approx(1) and ratio[-1] == pytest.approx(0.25)
    assert all(a >= b - 1e-7 for a, b in zip(ratio, ratio[1:]))
    # pairs that turn more than beta_fast times over the original context keep their frequency, and those that turn
    # less than once are divided in full
    for x, q in zip(base, ratio):
        turns = 32768 * x / (2 * math.pi)
        if turns > 40:
            assert q == pytest.approx(1, abs=1e-6)
        if turns < 0.8:
            assert q == pytest.approx(0.25, abs=1e-6)


def test_longrope_frequencies_and_factor():
    each = [1 + 0.1 * i for i in range(16)]
    s = {"type": "longrope", "factor": 32.0, "original_max_position_embeddings": 4096, "long_factor": each,
         "short_factor": [1.0] * 16}
    base, _ = _freq(32, 10000.0)
    got, mult = _freq(32, 10000.0, s)
    assert got == pytest.approx([x / f for x, f in zip(base, each)], rel=1e-6)
    assert mult == pytest.approx(math.sqrt(1 + math.log(32) / math.log(4096)))


def test_frequency_refusals():
    for bad in (0, 31):
        with pytest.raises(ValueError):
            _freq(bad)
    with pytest.raises(ValueError):
        _freq(64, 1e4, {"type": "unheard-of"})
    with pytest.raises(ValueError):
        _freq(64, 1e4, {"type": "longrope", "factor": 2.0, "long_factor": [1.0]})

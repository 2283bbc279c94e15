"""The paged serving cache's operators on the GPU against plain computations in
64 bits.

Tolerances. Decode: the framework's output tolerance (_util.assert_close); the
64-bit reference reads what the pool stores (codes, scales and biases of
quantized pools included), so only the attention's own rounding is measured.
Rotary: the fp32 steps -- a norm factor (rsqrt 2 ulp, a sum of at most 256
squares), cos and sin (2 ulp, and an angle good to 2^-24 of a turn, at most
4e-7), two products and a sum -- leave at most 2e-6 of the pair's length, and
the output type's rounding half an ulp. Appends and page copies: bit for bit.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

import oracle
from sparse_decode.synth import DTYPE_CODE

from _util import assert_close

pytestmark = pytest.mark.gpu

TORCH = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}
HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # of the power of two below a value


def tdt(torch, name):
    return getattr(torch, TORCH[name])


def gen(torch, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


# ---------------------------------------------------------------------------
# rotary
# ---------------------------------------------------------------------------

def rotary64(x, pos, inv, traditional, factor, w, eps):
    """x [..., tokens, heads, D] and pos [..., tokens] -> rotated rows in fp64."""
    import torch
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    r = inv.shape[0]
    ang = (pos.double()[..., None] * inv.double())[..., None, :]
    c, s = torch.cos(ang) * factor, torch.sin(ang) * factor
    i = torch.arange(r, device=x.device)
    ia, ib = (2 * i, 2 * i + 1) if traditional else (i, i + r)
    y = x.clone()
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ib] * c + x[..., ia] * s
    size = x.abs()
    size[..., ia] = size[..., ib] = torch.hypot(x[..., ia], x[..., ib]) * abs(factor)
    return y, size


def check_rows(torch, out, ref, size, dtype):
    ulp = torch.exp2(torch.floor(torch.log2(ref.abs().clamp(min=1e-30))))
    tiny = 2.0 ** -25 if dtype == "f16" else 0.0
    bound = HALF_ULP[dtype] * ulp * 1.001 + 2e-6 * size + tiny
    bad = (out.double() - ref).abs() > bound
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((out.double() - ref).abs() - bound).max()):.3g}"


ROTARY = [  # dtype, tokens, q heads, kv heads, D, rot, traditional, norms
    ("bf16", 1, 32, 8, 128, 128, False, "qk"),
    ("bf16", 37, 5, 1, 128, 64, False, ""),
    ("bf16", 130, 7, 7, 64, 58, False, "q"),       # an odd number of pairs: single-element accesses
    ("f16", 65, 8, 2, 64, 32, True, "qk"),
    ("f16", 33, 3, 3, 80, 20, False, "k"),         # ten pairs: two-element accesses
    ("f32", 129, 8, 2, 128, 122, True, "qk"),
    ("f32", 17, 2, 1, 256, 256, False, "qk"),
    ("f32", 9, 4, 4, 96, 0, False, "qk"),          # norms alone
    ("bf16", 300, 1, 0, 256, 254, False, "q"),
    ("bf16", 300, 0, 1, 2, 2, True, ""),           # queries absent, the smallest head
    ("f16", 3, 130, 66, 64, 64, False, "qk"),      # more heads than a block has rows
]


@pytest.mark.parametrize("dtype,n,hq,hkv,d,rot,trad,norms", ROTARY)
def test_rotary_matches_64_bits(cuda, dtype, n, hq, hkv, d, rot, trad, norms):
    import torch
    import sparse_decode as sd
    dt, g = tdt(torch, dtype), gen(torch, 11 + n)
    qkv = torch.randn(n, hq + hkv + 3, d, generator=g, device="cuda").to(dt)
    q = qkv[:, :hq] if hq else None
    k = qkv[:, hq:hq + hkv] if hkv else None
    w = {c: (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(dt) if c in norms else None for c in "qk"}
    pos = torch.randint(0, 1 << 20, (n,), generator=g, device="cuda", dtype=torch.int32)
    pos[0] = 0
    inv = sd.rotary_frequencies(rot, 1e6)[0] if rot else torch.empty(0, device="cuda")
    before = qkv.clone()
    qo, ko = sd.rotary(q, k, pos, inv, traditional=trad, factor=1.25, q_norm=w["q"], k_norm=w["k"], eps=1e-5)
    assert torch.equal(before, qkv)
    for x, o, c in ((q, qo, "q"), (k, ko, "k")):
        if x is None:
            assert o is None
            continue
        ref, size = rotary64(x, pos, inv, trad, 1.25, w[c], 1e-5)
        check_rows(torch, o, ref, size, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rotary_layouts_strides_and_in_place(cuda, dtype):
    """[batch, heads, tokens, D] as projections leave it, rows that start off 16-byte boundaries, outputs given, in
    place: all the same values."""
    import torch
    import sparse_decode as sd
    dt, g = tdt(torch, dtype), gen(torch, 3)
    b, hq, hkv, n, d = 3, 6, 2, 21, 128
    x = torch.randn(b, n, (hq + hkv) * d + 1, generator=g, device="cuda").to(dt)[..., 1:]   # misaligned rows
    q = x[..., :hq * d].unflatten(-1, (hq, d)).transpose(1, 2)
    k = x[..., hq * d:].unflatten(-1, (hkv, d)).transpose(1, 2)
    pos = torch.randint(0, 5000, (b, n), generator=g, device="cuda", dtype=torch.int32)
    inv, _ = sd.rotary_frequencies(d, 1e4)
    qo, ko = sd.rotary(q, k, pos, inv)
    ref, size = rotary64(q.transpose(1, 2), pos, inv, False, 1.0, None, 0)
    check_rows(torch, qo.transpose(1, 2), ref, size, dtype)
    flat = lambda t: t.transpose(1, 2).reshape(b * n, -1, d).contiguous()  # noqa: E731
    q3, k3 = sd.rotary(flat(q), flat(k), pos.flatten(), inv)       # aligned, vector accesses
    assert torch.equal(q3, flat(qo)) and torch.equal(k3, flat(ko))
    given = torch.empty(b, n, hq, d, dtype=dt, device="cuda").transpose(1, 2)
    q4, _ = sd.rotary(q, k, pos, inv, q_out=given)
    assert q4 is given and torch.equal(given, qo)
    sd.rotary(q, k, pos, inv, q_out=q, k_out=k)
    assert torch.equal(q, qo) and torch.equal(k, ko)


def test_rotary_rotates_gradients_back(cuda):
    """The transpose of the rotation is the rotation by the opposite positions."""
    import torch
    import sparse_decode as sd
    g = gen(torch, 5)
    x = torch.randn(40, 3, 128, generator=g, device="cuda")
    y = torch.randn(40, 3, 128, generator=g, device="cuda")
    pos = torch.randint(0, 100000, (40,), generator=g, device="cuda", dtype=torch.int32)
    inv, _ = sd.rotary_frequencies(128)
    rx = sd.rotary(x, None, pos, inv)[0]
    ry = sd.rotary(y, None, -pos, inv)[0]
    a, b = (rx.double() * y.double()).sum(), (x.double() * ry.double()).sum()
    assert abs(float(a - b)) < 1e-5 * float(x.double().norm() * y.double().norm())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("trad", [False, True])
@pytest.mark.parametrize("d,rot", [(128, 122), (128, 2), (96, 62), (72, 70), (40, 6), (256, 250), (64, 36), (128, 120), (200, 100)])
def test_rotary_parts_that_end_inside_an_access(cuda, d, rot, trad, dtype):
    """Rotated halves and parts that are no whole number of 16-byte accesses, at lengths that fill the GPU and not."""
    import torch
    import sparse_decode as sd
    dt, inv = tdt(torch, dtype), sd.rotary_frequencies(rot, 1e5)[0]
    for n, hq in ((3, 2), (450, 9)):
        g = gen(torch, d + rot + n)
        q = torch.randn(n, hq, d, generator=g, device="cuda").to(dt)
        k = torch.randn(n, 1, d, generator=g, device="cuda").to(dt)
        w = (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(dt)
        pos = torch.randint(0, 1 << 20, (n,), generator=g, device="cuda", dtype=torch.int32)
        want = [rotary64(q, pos, inv, trad, 1.25, w, 1e-5), rotary64(k, pos, inv, trad, 1.25, None, 0)]
        got = sd.rotary(q, k, pos, inv, traditional=trad, factor=1.25, q_norm=w, eps=1e-5, q_out=q, k_out=k)  # in place
        for o, (ref, size) in zip(got, want):
            check_rows(torch, o, ref, size, dtype)


@pytest.mark.parametrize("d,rot", [(128, 128), (128, 122), (64, 32), (96, 62)])
@pytest.mark.parametrize("trad", [False, True])
def test_rotary_infinities_reach_their_partner_only(cuda, d, rot, trad):
    import torch
    import sparse_decode as sd
    x = torch.randn(2 * d, 3, d, generator=gen(torch, d + rot), device="cuda").bfloat16()
    at = torch.arange(2 * d, device="cuda")
    x[at, 1, at % d] = float("inf")
    pos = (1 + at).int()
    out = sd.rotary(x, None, pos, sd.rotary_frequencies(rot)[0], traditional=trad)[0]
    i = at % d
    if trad:
        j = i ^ 1
    else:
        j = torch.where(i < rot // 2, i + rot // 2, i - rot // 2)
    j = torch.where(i < rot, j, i)
    hit = torch.zeros(x.shape, dtype=torch.bool, device="cuda")
    hit[at, 1, i] = hit[at, 1, j] = True
    assert torch.equal(~torch.isfinite(out), hit)


def test_rotary_nan_and_inf_stay_in_their_row(cuda):
    import torch
    import sparse_decode as sd
    x = torch.randn(20, 4, 128, device="cuda", dtype=torch.bfloat16)
    x[7, 2, 5], x[9, 1, 127] = float("nan"), float("inf")
    pos = torch.arange(20, device="cuda", dtype=torch.int32)
    w = torch.ones(128, device="cuda", dtype=torch.bfloat16)
    out = sd.rotary(x, None, pos, sd.rotary_frequencies(128)[0], q_norm=w)[0]
    bad = ~torch.isfinite(out).all(-1)
    assert bad.nonzero().tolist() == [[7, 2], [9, 1]]


# ---------------------------------------------------------------------------
# pools
# ---------------------------------------------------------------------------

class Pool:
    """A pool of random pages: device arrays, and the values they stand for in fp64 [n_pages, Hkv, P, D]."""

    def __init__(self, torch, sd, dtype, bits, hkv, d, page, n_pages, seed, scale=1.0):
        g = gen(torch, seed)
        self.torch, self.dtype, self.bits, self.page = torch, dtype, bits, page
        dt = tdt(torch, dtype)
        arrays, self.values = [[], []], []
        for i in range(2):
            x = (scale * torch.randn(n_pages, hkv, page, d, generator=g, device="cuda")).to(dt)
            if not bits:
                arrays[i] = [x]
                self.values.append(x.double())
                continue
            codes = torch.randint(0, 1 << bits, (n_pages, hkv, page, d), generator=g, device="cuda", dtype=torch.int64)
            words = codes.unflatten(-1, (-1, 32 // bits))
            shift = torch.arange(32 // bits, device="cuda") * bits
            packed = (words << shift).sum(-1)
            packed = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)
            top = (1 << bits) - 1
            spread = torch.rand(n_pages, hkv, page, d // 64, generator=g, device="cuda") + 0.5
            sc = (scale * 6 * spread / top).to(dt)
            sign = torch.where(torch.rand(sc.shape, generator=g, device="cuda") < 0.5, -1.0, 1.0).to(dt)
            sc = sc * sign
            bi = (-3 * scale * spread * sign.float()).to(dt)
            arrays[i] = [packed, sc, bi]
            grow = lambda t: t.double().repeat_interleave(64, -1)  # noqa: E731
            self.values.append(codes.double() * grow(sc) + grow(bi))
        (k, *ks), (v, *vs) = arrays
        self.arrays = arrays
        self.pages = sd.KVPages(k, v, *ks, *vs, bits=bits)

    def spoil(self, keep):
        """Everything outside keep [n_pages, P] (bool) becomes not-a-number (scales or values)."""
        for a in self.arrays:
            x = a[-1]
            x.masked_fill_(~keep[:, None, :, None], float("nan"))


def tables_of(torch, lengths, page, n_pages, seed, width=None):
    need = [-(-t // page) for t in lengths]
    assert sum(need) <= n_pages
    order = torch.randperm(n_pages, generator=gen(torch, seed), device="cuda").tolist()
    w = width or max(1, max(need))
    t, at = [], 0
    for n in need:
        t.append(order[at:at + n] + [-1] * (w - n))
        at += n
    return torch.tensor(t, dtype=torch.int32, device="cuda")


def kept(torch, lengths, tables, page, n_pages, window=0):
    keep = torch.zeros(n_pages, page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lengths):
        for t in range(max(0, n - window) if window else 0, n, 1):
            keep[int(tables[b, t // page]), t % page] = True
    return keep


def decode64(q, pool, tables, lengths, scale, window=0, sinks=None):
    import torch
    B, Hq, D = q.shape
    k, v = pool.values
    hkv = k.shape[1]
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        at = tables[b, :-(-n // pool.page)].long()
        kk, vv = (x[at].permute(1, 0, 2, 3).flatten(1, 2) for x in (k, v))
        lo = max(0, n - window) if window else 0
        s = torch.einsum("hgd,htd->hgt", q[b].double().view(hkv, -1, D), kk[:, lo:n]) * scale
        if sinks is not None:
            s = torch.cat((s, sinks.double().view(hkv, -1, 1)), -1)
        p = torch.softmax(s, -1)[..., :n - lo]
        out[b] = torch.einsum("hgt,htd->hgd", p, vv[:, lo:n]).reshape(Hq, D)
    return out


def run_case(torch, dtype, bits, d, hkv, G, page, lengths, window=0, sinks=False, seed=0, scale=1.0, spare=3):
    import sparse_decode as sd
    n_pages = sum(-(-t // page) for t in lengths) + spare
    pool = Pool(torch, sd, dtype, bits, hkv, d, page, n_pages, seed + 1, scale)
    tables = tables_of(torch, lengths, page, n_pages, seed + 2)
    pool.spoil(kept(torch, lengths, tables, page, n_pages, window))
    q = (2 * torch.randn(len(lengths), hkv * G, d, generator=gen(torch, seed + 3), device="cuda")).to(tdt(torch, dtype))
    sk = torch.randn(hkv * G, generator=gen(torch, seed + 4), device="cuda") * 3 if sinks else None
    ln = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    flags = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = sd.paged_decode(q, pool.pages, tables, ln, window=window, sinks=sk, flags=flags)
    again = sd.paged_decode(q, pool.pages, tables, ln, window=window, sinks=sk, flags=flags)
    assert int(flags) == 0
    assert torch.equal(out, again)
    ref = decode64(q, pool, tables, lengths, 1 / math.sqrt(d), window, sk)
    assert torch.isfinite(out).all()
    live = [b for b, n in enumerate(lengths) if n]
    for b, n in enumerate(lengths):
        if n == 0:
            assert not out[b].any()
    if live:
        assert_close(out[live].double().cpu().numpy().reshape(-1, d), ref[live].cpu().numpy().reshape(-1, d), dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("bits", [0, 4, 8])
@pytest.mark.parametrize("d", [64, 128])
def test_decode_formats(cuda, dtype, bits, d):
    """Every format; lengths around tile and page edges, one token, none."""
    import torch
    run_case(torch, dtype, bits, d, hkv=2, G=4, page=64, lengths=[1, 63, 0, 64, 65, 127, 128, 129, 500, 31, 33], seed=d + bits)


@pytest.mark.parametrize("G", [1, 2, 3, 5, 7, 8, 9, 12, 16])
@pytest.mark.parametrize("dtype,bits", [("bf16", 0), ("f16", 4), ("bf16", 8), ("f32", 0), ("f32", 8)])
def test_decode_head_groups(cuda, G, dtype, bits):
    import torch
    run_case(torch, dtype, bits, 128, hkv=3, G=G, page=32, lengths=[5, 170, 1], seed=G)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype,bits,d", [("bf16", 0, 128), ("bf16", 8, 128), ("f16", 4, 64), ("f32", 0, 64), ("f32", 4, 128)])
def test_decode_page_sizes(cuda, page, dtype, bits, d):
    import torch
    run_case(torch, dtype, bits, d, hkv=2, G=4, page=page, lengths=[page - 1, page, page + 1, 3 * page + 7, 777], seed=page)


@pytest.mark.parametrize("window", [1, 16, 63, 64, 65, 100, 1000])
@pytest.mark.parametrize("dtype,bits", [("bf16", 0), ("bf16", 8), ("f16", 4), ("f32", 0)])
def test_decode_window_and_sinks(cuda, window, dtype, bits):
    """Tokens before the window are not-a-numbers here, so they cannot have been read."""
    import torch
    run_case(torch, dtype, bits, 128, hkv=2, G=4, page=16, lengths=[1, 64, 65, 300, 999, 0, 1000, 1001], window=window,
             sinks=True, seed=window)


@pytest.mark.parametrize("dtype,bits", [("bf16", 0), ("bf16", 8), ("f32", 0)])
def test_decode_long_split_over_all_ctas(cuda, dtype, bits):
    import torch
    run_case(torch, dtype, bits, 128, hkv=1, G=8, page=64, lengths=[40001], seed=1)
    run_case(torch, dtype, bits, 64, hkv=2, G=2, page=64, lengths=[20000, 3, 0, 0, 9000, 1], seed=2)


@pytest.mark.parametrize("dtype,bits", [("bf16", 0), ("bf16", 8), ("f16", 0), ("f16", 4), ("f32", 0), ("f32", 4), ("f32", 8)])
def test_decode_sums_stay_exact_over_long_segments(cuda, dtype, bits):
    """40 sequences over the same 100K tokens: as many (sequence, head) pairs as CTAs, so every pair is summed by one
    CTA from end to end. Small queries spread the probabilities over all tokens and the values' mean is not zero, so
    that errors that add up along the sums would show."""
    import torch
    import sparse_decode as sd
    B, hkv, G, d, page, n = 40, 8, 1, 128, 256, 100000
    n_pages = -(-n // page)
    pool = Pool(torch, sd, dtype, bits, hkv, d, page, n_pages, 61)
    v = pool.arrays[1]
    v[-1] += 2.0   # the biases of codes, or the values themselves
    if bits:
        words = v[0].long() & 0xFFFFFFFF
        codes = torch.stack([(words >> (bits * j)) & ((1 << bits) - 1) for j in range(32 // bits)], -1).flatten(-2)
        grow = lambda t: t.double().repeat_interleave(64, -1)  # noqa: E731
        pool.values[1] = codes.double() * grow(v[1]) + grow(v[2])
    else:
        pool.values[1] = v[0].double()
    tables = tables_of(torch, [n], page, n_pages, 62).repeat(B, 1).contiguous()
    q = (0.05 * torch.randn(B, hkv * G, d, generator=gen(torch, 63), device="cuda")).to(tdt(torch, dtype))
    ln = torch.full((B,), n, dtype=torch.int32, device="cuda")
    out = sd.paged_decode(q, pool.pages, tables, ln)
    some = [0, 13, 39]
    ref = decode64(q[some], pool, tables[some], [n] * 3, 1 / math.sqrt(d))
    assert_close(out[some].double().cpu().numpy().reshape(-1, d), ref.cpu().numpy().reshape(-1, d), dtype)


@pytest.mark.parametrize("dtype,bits", [("bf16", 0), ("f16", 4), ("f32", 0)])
def test_decode_many_short_sequences(cuda, dtype, bits):
    import torch
    rng = np.random.default_rng(3)
    lengths = [int(x) for x in rng.integers(0, 90, 700)]
    run_case(torch, dtype, bits, 64, hkv=2, G=2, page=16, lengths=lengths, seed=9)


@pytest.mark.parametrize("dtype,bits", [("bf16", 0), ("bf16", 8), ("f32", 0)])
def test_decode_largest_batch_and_group(cuda, dtype, bits):
    """4096 sequences and 16 heads per kv head leave the fewest stages of shared memory."""
    import torch
    rng = np.random.default_rng(5)
    run_case(torch, dtype, bits, 128, hkv=1, G=16, page=16, lengths=[int(x) for x in rng.integers(0, 24, 4096)], seed=3)


@pytest.mark.parametrize("dtype,bits,d,hkv,G", [("bf16", 0, 128, 3, 7), ("f16", 4, 64, 2, 16), ("bf16", 8, 128, 8, 3), ("f32", 0, 64, 5, 5)])
@pytest.mark.parametrize("long", [700, 21000])
def test_decode_many_heads_beside_a_long_sequence(cuda, dtype, bits, d, hkv, G, long):
    """More query heads than one wave of blocks joins one by one; the long sequence has many segments, the others one or
    two, some none, and the heads of a sequence do not divide by eight."""
    import torch
    rng = np.random.default_rng(long + G)
    lengths = [int(x) for x in rng.integers(0, 200, 44)]
    lengths[5] = lengths[43] = 0
    lengths[17] = long
    run_case(torch, dtype, bits, d, hkv=hkv, G=G, page=32, lengths=lengths, sinks=True, seed=G)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bits", [4, 8])
def test_decode_queries_below_every_power_of_two(cuda, dtype, bits):
    """Queries of 2^-130, subnormal: every score is zero to all digits, the output is the mean of the values."""
    import torch
    import sparse_decode as sd
    pool = Pool(torch, sd, dtype, bits, 2, 128, 64, 6, 21)
    lengths = [200, 3]
    tables = tables_of(torch, lengths, 64, 6, 22)
    q = (torch.ones(2, 8, 128, device="cuda", dtype=torch.float64) * 2.0 ** -130).to(tdt(torch, dtype))
    assert float(q.double().abs().min()) == 2.0 ** -130
    out = sd.paged_decode(q, pool.pages, tables, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    ref = decode64(q, pool, tables, lengths, 1 / math.sqrt(128))
    assert_close(out.double().cpu().numpy().reshape(-1, 128), ref.cpu().numpy().reshape(-1, 128), dtype)


@pytest.mark.parametrize("scale", [1e-4, 1e3])
@pytest.mark.parametrize("bits", [0, 4, 8])
def test_decode_small_and_large_values(cuda, scale, bits):
    """Values and scales far from 1: large keys make one-hot probabilities, small ones uniform; p times a tiny scale
    must not sink into fp16's subnormals."""
    import torch
    run_case(torch, "bf16", bits, 128, hkv=2, G=4, page=64, lengths=[300, 77], scale=scale, seed=4)


def test_decode_scales_that_grow_along_the_sequence(cuda):
    """Value scales rise by 2^24 over the sequence, and fall in another: the common power of two has to follow."""
    import torch
    import sparse_decode as sd
    n_pages = 2 * 20 + 1
    pool = Pool(torch, sd, "bf16", 8, 2, 128, 64, n_pages, 5)
    lengths = [20 * 64, 20 * 64 - 5]
    tables = tables_of(torch, lengths, 64, n_pages, 6)
    for b in range(2):
        for j in range(20):
            f = 2.0 ** ((j if b == 0 else 19 - j) * 1.25 - 12)
            pg = int(tables[b, j])
            for a in pool.arrays[1][1:]:
                a[pg] *= f
    grow = lambda t: t.double().repeat_interleave(64, -1)  # noqa: E731
    words = pool.arrays[1][0].long() & 0xFFFFFFFF
    codes = torch.stack([(words >> (8 * j)) & 255 for j in range(4)], -1).flatten(-2).double()
    pool.values[1] = codes * grow(pool.arrays[1][1]) + grow(pool.arrays[1][2])
    q = torch.randn(2, 8, 128, generator=gen(torch, 7), device="cuda").bfloat16()
    ln = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = sd.paged_decode(q, pool.pages, tables, ln)
    ref = decode64(q, pool, tables, lengths, 1 / math.sqrt(128))
    assert_close(out.double().cpu().numpy().reshape(-1, 128), ref.cpu().numpy().reshape(-1, 128), "bf16")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bits", [4, 8])
def test_decode_scales_that_jump_while_the_maximum_lags(cuda, dtype, bits):
    """The running maximum may lag the true one by 8 (log2 units): p up to 256 meets value scales that jump 2^7-fold
    between tiles, so p times the scaled s_v comes near fp16's largest number."""
    import torch
    import sparse_decode as sd
    d, page, n = 128, 64, 64 * 12
    pool = Pool(torch, sd, dtype, bits, 1, d, page, 13, 15)
    tables = tables_of(torch, [n], page, 13, 16)
    # every key of page j: codes equal, so that the score is a constant of the page, rising by 7.5 after page 3
    q = torch.ones(1, 4, d, device="cuda", dtype=tdt(torch, dtype))
    kc, ks, kb = pool.arrays[0]
    kc.zero_(), ks.fill_(1.0)
    vs, vb = pool.arrays[1][1:]
    vs.abs_(), vb.copy_(-vs)
    for j in range(12):
        pg = int(tables[0, j])
        kb[pg] = 0.0 if j < 4 else 7.5 * math.log(2) / math.sqrt(d)
        for r in range(2):
            vs[pg, ..., r] *= 2.0 ** -7 if j < 8 - 4 * r else 1.0
        vb[pg] = -vs[pg]
    words = pool.arrays[1][0].long() & 0xFFFFFFFF
    codes = torch.stack([(words >> (bits * j)) & ((1 << bits) - 1) for j in range(32 // bits)], -1).flatten(-2).double()
    grow = lambda t: t.double().repeat_interleave(64, -1)  # noqa: E731
    pool.values = [grow(kb), codes * grow(vs) + grow(vb)]
    out = sd.paged_decode(q, pool.pages, tables, torch.tensor([n], dtype=torch.int32, device="cuda"))
    ref = decode64(q, pool, tables, [n], 1 / math.sqrt(d))
    assert_close(out.double().cpu().numpy().reshape(-1, d), ref.cpu().numpy().reshape(-1, d), dtype)


@pytest.mark.parametrize("dtype,bits", [("bf16", 0), ("bf16", 8), ("f32", 0)])
def test_decode_nan_in_a_valid_token_reaches_its_heads_only(cuda, dtype, bits):
    import torch
    import sparse_decode as sd
    pool = Pool(torch, sd, dtype, bits, 2, 128, 64, 40, 8)
    lengths = [1000, 900]
    tables = tables_of(torch, lengths, 64, 40, 9)
    pool.arrays[0][-1][int(tables[1, 3]), 1, 5] = float("nan")  # a key (or its bias) of kv head 1, sequence 1
    q = torch.randn(2, 8, 128, device="cuda").to(tdt(torch, dtype))
    out = sd.paged_decode(q, pool.pages, tables, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    bad = torch.isnan(out).all(-1)
    assert bad[1, 4:].all() and int(bad.sum()) == 4 and int(torch.isnan(out).any(-1).sum()) == 4


def test_decode_shared_pages_and_equal_scores(cuda):
    """Two sequences over the same pages give the same bits; equal keys average the values."""
    import torch
    import sparse_decode as sd
    pool = Pool(torch, sd, "bf16", 0, 2, 128, 64, 12, 10)
    lengths = [640, 640]
    row = tables_of(torch, [640], 64, 12, 11)
    tables = row.repeat(2, 1).contiguous()
    q = torch.randn(1, 8, 128, device="cuda").bfloat16().repeat(2, 1, 1)
    ln = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = sd.paged_decode(q, pool.pages, tables, ln)
    assert torch.allclose(out[0].float(), out[1].float(), rtol=1e-2, atol=1e-3)
    pool.arrays[0][0].zero_()
    pool.values[0].zero_()
    out = sd.paged_decode(q, pool.pages, tables, ln)
    ref = decode64(q, pool, tables, lengths, 1 / math.sqrt(128))
    assert_close(out.double().cpu().numpy().reshape(-1, 128), ref.cpu().numpy().reshape(-1, 128), "bf16")


def test_decode_reports_bad_indexes_and_reads_nothing_there(cuda):
    import torch
    import sparse_decode as sd
    for dtype, bits in (("bf16", 0), ("bf16", 8), ("f32", 0)):
        pool = Pool(torch, sd, dtype, bits, 2, 128, 64, 9, 12)
        tables = torch.tensor([[0, 1, 2], [3, 100, 5], [6, -1, 7], [1 << 30, 2, 2]], dtype=torch.int32, device="cuda")
        q = torch.randn(4, 8, 128, device="cuda").to(tdt(torch, dtype))
        flags = torch.zeros(1, dtype=torch.int32, device="cuda")
        ln = torch.tensor([192] * 4, dtype=torch.int32, device="cuda")
        out = sd.paged_decode(q, pool.pages, tables, ln, flags=flags)
        assert int(flags) == 2 and torch.isfinite(out).all()
        ref = decode64(q[:1], pool, tables[:1], [192], 1 / math.sqrt(128))
        assert_close(out[:1].double().cpu().numpy().reshape(-1, 128), ref.cpu().numpy().reshape(-1, 128), dtype)
        # lengths out of range: clamped to the table, or to nothing
        flags.zero_()
        ok = torch.tensor([[0, 1, 2]] * 3, dtype=torch.int32, device="cuda")
        ln = torch.tensor([-5, 1 << 30, 192], dtype=torch.int32, device="cuda")
        out = sd.paged_decode(q[:1].repeat(3, 1, 1), pool.pages, ok, ln, flags=flags)
        assert int(flags) == 2 and not out[0].any() and torch.isfinite(out).all()
        assert_close(out[1:].double().cpu().numpy().reshape(-1, 128), ref.repeat(2, 1, 1).cpu().numpy().reshape(-1, 128), dtype)


# ---------------------------------------------------------------------------
# appends and copies
# ---------------------------------------------------------------------------

APPEND = [  # dtype, bits, D, q heads, kv heads, page, rot, traditional, norms, tokens per sequence
    ("bf16", 0, 128, 32, 8, 64, 128, False, "qk", [1] * 5),
    ("f16", 0, 64, 6, 2, 16, 32, True, "", [3, 17, 1, 40]),
    ("f32", 0, 128, 4, 4, 32, 122, False, "k", [2, 33]),
    ("bf16", 8, 128, 8, 2, 64, 128, False, "qk", [1, 70, 5]),
    ("bf16", 4, 64, 7, 1, 16, 58, False, "q", [9, 1, 20]),
    ("f16", 8, 64, 4, 2, 128, 64, True, "", [130, 2]),
    ("f32", 4, 128, 2, 1, 16, 64, False, "qk", [31]),
    ("f32", 8, 64, 0, 3, 16, 0, False, "", [8, 8]),
    ("bf16", 0, 128, 0, 2, 16, 0, False, "", [1, 40]),
]


@pytest.mark.parametrize("dtype,bits,d,hq,hkv,page,rot,trad,norms,counts", APPEND)
def test_append_stores_what_rotary_and_quantize_give(cuda, dtype, bits, d, hq, hkv, page, rot, trad, norms, counts):
    """q_out and the stored rows are, bit for bit, rotary's (quantized by the oracle); nothing else is touched."""
    import torch
    import sparse_decode as sd
    dt, g = tdt(torch, dtype), gen(torch, d + len(counts))
    held = [7 * i for i in range(len(counts))]
    lengths = [h + c for h, c in zip(held, counts)]
    n_pages = sum(-(-t // page) for t in lengths) + 2
    pool = Pool(torch, sd, dtype, bits, hkv, d, page, n_pages, 21)
    tables = tables_of(torch, lengths, page, n_pages, 22)
    pos = torch.tensor([h + i for h, c in zip(held, counts) for i in range(c)], dtype=torch.int32, device="cuda")
    seq = torch.tensor([b for b, c in enumerate(counts) for _ in range(c)], dtype=torch.int32, device="cuda")
    n = pos.numel()
    qkv = torch.randn(n, hq + 2 * hkv, d, generator=g, device="cuda").to(dt)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    w = {c: (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(dt) if c in norms else None for c in "qk"}
    turn = dict(inv_freq=sd.rotary_frequencies(rot, 1e4)[0], traditional=trad, factor=1.1, q_norm=w["q"],
                k_norm=w["k"]) if rot else {}
    before = [[a.clone() for a in x] for x in pool.arrays]
    flags = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = sd.paged_append(pool.pages, k, v, tables, pos, seq=seq, q=q if hq else None, flags=flags, **turn)
    assert int(flags) == 0
    qr, kr = sd.rotary(q if hq else None, k, pos, **turn) if rot else (None, k)
    assert out is None if not hq else torch.equal(out, qr)
    at = tables[seq.long(), (pos // page).long()].long()
    slot = (pos % page).long()
    code = DTYPE_CODE[dtype]
    for arrays, old, rows in zip(pool.arrays, before, (kr, v)):
        if not bits:
            new = [rows]
        else:
            host = rows.reshape(-1, d).contiguous().cpu()
            host = host.view(torch.int16).numpy().view(np.uint16) if dtype == "bf16" else host.numpy()
            cq, sc, bi = oracle.quantize(host, code, d, bits)
            back = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(  # noqa: E731
                np.int16) if dtype == "bf16" else np.ascontiguousarray(a)).cuda().view(dt).view(n, hkv, d // 64)
            new = [torch.from_numpy(np.ascontiguousarray(cq).view(np.int32)).cuda().view(n, hkv, -1), back(sc), back(bi)]
        for a, o, x in zip(arrays, old, new):
            o[at, :, slot] = x.to(o.dtype)
            assert torch.equal(a.view(torch.int32 if a.element_size() == 4 else torch.int16),
                               o.view(torch.int32 if o.element_size() == 4 else torch.int16))


@pytest.mark.parametrize("bits", [0, 8])
def test_append_skips_padding_and_reports_bad_indexes(cuda, bits):
    import torch
    import sparse_decode as sd
    pool = Pool(torch, sd, "bf16", bits, 2, 128, 16, 6, 23)
    tables = torch.tensor([[0, 1], [2, 77], [3, -1]], dtype=torch.int32, device="cuda")
    x = torch.randn(7, 2, 128, device="cuda").bfloat16()
    before = [[a.clone() for a in y] for y in pool.arrays]
    flags = torch.zeros(1, dtype=torch.int32, device="cuda")

    def append(pos, seq):
        flags.zero_()
        i = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        sd.paged_append(pool.pages, x[:len(pos)], x[:len(pos)], tables, i(pos), seq=i(seq), flags=flags)
        return int(flags)
    assert append([-1, -7], [0, 1]) == 0                            # padding
    assert append([32], [0]) == 2 and append([16], [1]) == 2        # past the table, no such page
    assert append([16], [2]) == 2 and append([0], [3]) == 2 and append([0], [-1]) == 2
    for a, o in zip(pool.arrays, before):
        assert all(torch.equal(p, r) for p, r in zip(a, o))
    assert append([17, -1], [0, 0]) == 0                            # a good token beside padding is stored
    assert not torch.equal(pool.arrays[0][0][1, :, 1], before[0][0][1, :, 1])


@pytest.mark.parametrize("dtype,bits,hkv,d,page,layers,n", [
    ("bf16", 0, 8, 128, 64, 3, 5), ("f32", 8, 1, 64, 16, 1, 1), ("f16", 4, 3, 64, 16, 2, 40), ("f32", 0, 3, 128, 32, 2, 7)])
def test_copy_pages(cuda, dtype, bits, hkv, d, page, layers, n):
    import torch
    import sparse_decode as sd
    n_pages = 2 * n + 3
    pool = Pool(torch, sd, dtype, bits, hkv, d, page, layers * n_pages, 31)
    arrays = [[a.view(layers, n_pages, *a.shape[1:]) for a in x] for x in pool.arrays]
    (k, *ks), (v, *vs) = arrays
    pages = sd.KVPages(k, v, *ks, *vs, bits=bits)
    order = torch.randperm(n_pages, generator=gen(torch, 32), device="cuda").to(torch.int32)
    src, dst = order[:n].clone(), order[n:2 * n].clone()
    want = [[a.clone() for a in x] for x in arrays]
    for x in want:
        for a in x:
            a[:, dst.long()] = a[:, src.long()]
    flags = torch.zeros(1, dtype=torch.int32, device="cuda")
    sd.copy_pages(pages, src, dst, flags=flags)
    assert int(flags) == 0
    assert all(torch.equal(a, o) for x, y in zip(arrays, want) for a, o in zip(x, y))
    # pairs out of range copy nothing; host lists are checked
    sd.copy_pages(pages, torch.tensor([0, -1, n_pages], dtype=torch.int32, device="cuda"),
                  torch.tensor([n_pages, 1, 2], dtype=torch.int32, device="cuda"), flags=flags)
    assert int(flags) == 2
    assert all(torch.equal(a, o) for x, y in zip(arrays, want) for a, o in zip(x, y))
    for s, t in (([0], [n_pages]), ([0], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [])):
        with pytest.raises(ValueError):
            sd.copy_pages(pages, s, t)
    sd.copy_pages(pages, [int(dst[0])], [int(src[0])])
    assert all(torch.equal(a, o) for x, y in zip(arrays, want) for a, o in zip(x, y))


def test_offsets_past_32_bits(cuda):
    """Pages at the end of a pool whose arrays are over 4 GiB: append, copy and decode there."""
    import torch
    import sparse_decode as sd
    n_pages, hkv, page, d = 300000, 1, 64, 128
    k = torch.empty(n_pages, hkv, page, d, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    assert k.numel() * 2 > 1 << 32
    pages = sd.KVPages(k, v)
    n = 150
    tables = torch.tensor([[n_pages - 1, n_pages - 3, n_pages - 7]], dtype=torch.int32, device="cuda")
    g = gen(torch, 41)
    kk, vv = (torch.randn(n, 1, d, generator=g, device="cuda").bfloat16() for _ in "kv")
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    sd.paged_append(pages, kk, vv, tables, pos, seq=torch.zeros(n, dtype=torch.int32, device="cuda"))
    q = torch.randn(1, 4, d, generator=g, device="cuda").bfloat16()
    ln = torch.tensor([n], dtype=torch.int32, device="cuda")
    out = sd.paged_decode(q, pages, tables, ln)
    s = torch.einsum("hd,td->ht", q[0].double(), kk[:, 0].double()) / math.sqrt(d)
    ref = torch.softmax(s, -1) @ vv[:, 0].double()
    assert_close(out[0].double().cpu().numpy(), ref.cpu().numpy(), "bf16")
    sd.copy_pages(pages, tables[0].clone(), tables[0] - 10)
    assert torch.equal(sd.paged_decode(q, pages, tables - 10, ln), out)


# ---------------------------------------------------------------------------
# streams, graphs, refusals
# ---------------------------------------------------------------------------

def test_calls_on_two_streams_do_not_disturb_each_other(cuda):
    import torch
    import sparse_decode as sd
    pool = Pool(torch, sd, "bf16", 0, 2, 128, 64, 400, 51)
    cases = []
    for i, lengths in enumerate(([12000, 5, 3000], [700, 9000])):
        tables = tables_of(torch, lengths, 64, 400, 52 + i)
        q = torch.randn(len(lengths), 8, 128, generator=gen(torch, 60 + i), device="cuda").bfloat16()
        ln = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        cases.append((q, tables, ln, sd.paged_decode(q, pool.pages, tables, ln)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[], []]
    for _ in range(30):
        for i, (q, tables, ln, _) in enumerate(cases):
            outs[i].append(sd.paged_decode(q, pool.pages, tables, ln, stream=streams[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, cases[i][3]) for o in outs[i])


def test_a_captured_step_serves_growing_sequences(cuda):
    """append + decode in one CUDA graph; lengths and positions advance on the device between replays."""
    import torch
    import sparse_decode as sd
    hkv, d, page, B = 2, 128, 16, 3
    pool = Pool(torch, sd, "bf16", 0, hkv, d, page, 64, 71)
    lengths = [30, 1, 100]
    tables = tables_of(torch, [t + 40 for t in lengths], page, 64, 72)
    g = gen(torch, 73)
    qkv = torch.empty(B, 8 + 2 * hkv, d, dtype=torch.bfloat16, device="cuda")
    ln = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    pos = ln - 1
    inv, _ = sd.rotary_frequencies(d)

    def step():
        q = sd.paged_append(pool.pages, qkv[:, 8:8 + hkv], qkv[:, 8 + hkv:], tables, pos, q=qkv[:, :8], inv_freq=inv)
        return q, sd.paged_decode(q, pool.pages, tables, ln)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q_out, out = step()
    for i in range(40):
        qkv.copy_(torch.randn(qkv.shape, generator=g, device="cuda"))
        graph.replay()
        if i % 13 == 0:
            now = [t + i for t in lengths]
            pool.values = [a[0].double() for a in pool.arrays]
            ref = decode64(q_out, pool, tables, now, 1 / math.sqrt(d))
            assert_close(out.double().cpu().numpy().reshape(-1, d), ref.cpu().numpy().reshape(-1, d), "bf16")
        ln += 1
        pos += 1


def test_python_refusals(cuda):
    import torch
    import sparse_decode as sd
    pool = Pool(torch, sd, "bf16", 0, 2, 128, 16, 8, 81)
    p = pool.pages
    q = torch.randn(1, 8, 128, device="cuda").bfloat16()
    t = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    ln = torch.ones(1, dtype=torch.int32, device="cuda")
    k = q[:, :2]
    for bad in (lambda: sd.paged_decode(q.cpu(), p, t, ln), lambda: sd.paged_decode(q, p, t.cpu(), ln),
                lambda: sd.paged_decode(q[..., :64], p, t, ln), lambda: sd.paged_decode(q, p, t, ln.repeat(2)),
                lambda: sd.paged_decode(q, p, t[0], ln), lambda: sd.paged_decode(q, p, t.repeat(2, 1), ln),
                lambda: sd.paged_decode(q, p, t, ln, sinks=torch.zeros(3, device="cuda")),
                lambda: sd.paged_append(p, k, k[:, :1], t, ln), lambda: sd.paged_append(p, q, q, t, ln),
                lambda: sd.paged_append(p, k, k, t, ln.repeat(2)),
                lambda: sd.rotary(q, k.repeat(2, 1, 1), ln, torch.ones(64, device="cuda")),
                lambda: sd.rotary(None, None, ln, torch.ones(64, device="cuda")),
                lambda: sd.rotary(q.transpose(1, 2), None, ln, torch.ones(4, device="cuda")),
                lambda: sd.rotary(q, k, ln, torch.ones(64, device="cuda"), q_norm=torch.ones(64, device="cuda").bfloat16()),
                lambda: sd.KVPages(p.k, p.v, bits=8), lambda: sd.KVPages(p.k.cpu(), p.v.cpu()),
                lambda: sd.KVPages(p.k, p.v[:4]), lambda: sd.KVPages(p.k[0], p.v[0])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: sd.paged_decode(q.float(), p, t, ln), lambda: sd.paged_decode(q, p, t.long(), ln),
                lambda: sd.paged_append(p, k.float(), k.float(), t, ln),
                lambda: sd.rotary(q, k, ln, torch.ones(64, device="cuda").double()),
                lambda: sd.rotary(q.double(), None, ln, torch.ones(64, device="cuda"))):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: sd.paged_decode(q, p, t, ln, layer=1), lambda: sd.paged_decode(q, p, t, ln, window=-1),
                lambda: sd.paged_decode(q[:, :7].contiguous(), p, t, ln),
                lambda: sd.paged_decode(torch.zeros(1, 34, 128, device="cuda").bfloat16(), p, t, ln),
                lambda: sd.paged_decode(q, p, t, ln, float("nan")),
                lambda: sd.rotary(q, k, ln, torch.ones(65, device="cuda"))):
        with pytest.raises(sd.SDError):
            bad()
    assert sd.paged_decode(q[:0], p, t[:0], ln[:0]).shape == (0, 8, 128)
    assert sd.rotary(q[:0], None, ln[:0], torch.ones(64, device="cuda"))[0].shape == (0, 8, 128)


# ---------------------------------------------------------------------------
# the pool, the router, the example
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [0, 4, 8])
def test_pool_lifecycle_keeps_every_sequence(cuda, bits):
    """Random adds, forks, extends, trims, frees and compactions; every sequence's pages hold its own tokens' rows in
    both layers all along (checked by decoding against a contiguous copy)."""
    import torch
    import sparse_decode as sd
    rng = np.random.default_rng(bits + 1)
    g = gen(torch, 90 + bits)
    layers, hkv, hq, d = 2, 2, 4, 64
    pool = sd.PagePool(layers, 40, hkv, d, 16, "bf16", bits)
    rows: dict = {}   # sequence -> per layer (k, v) [tokens, Hkv, D]
    empty = lambda: [(torch.empty(0, hkv, d, device="cuda").bfloat16(),) * 2 for _ in range(layers)]  # noqa: E731

    def check(seqs):
        if not seqs:
            return
        batch = pool.batch(seqs)
        q = torch.randn(len(seqs), hq, d, generator=g, device="cuda").bfloat16()
        for layer in range(layers):
            out = batch.decode(layer, q)
            for i, s in enumerate(seqs):
                k, v = rows[s][layer]
                if len(k) == 0:
                    assert not out[i].any()
                    continue
                one = sd.PagePool(1, -(-len(k) // 16), hkv, d, 16, "bf16", bits)
                alone = one.extend([one.add()], len(k))
                alone.append(0, k, v)
                assert torch.allclose(out[i].float(), alone.decode(0, q[i:i + 1])[0].float(), rtol=2e-2, atol=2e-3)
    for move in range(60):
        r = rng.random()
        seqs = list(rows)
        if r < 0.15 or not seqs:
            rows[pool.add()] = empty()
        elif r < 0.3:
            s = int(rng.choice(seqs))
            rows[pool.fork(s)] = list(rows[s])
        elif r < 0.75:
            some = [int(s) for s in rng.permutation(seqs)[:rng.integers(1, 4)]]
            each = [int(n) for n in rng.integers(1, 40, len(some))]
            try:
                batch = pool.extend(some, each)
            except sd.SDError:
                check(seqs)
                continue
            for layer in range(layers):
                k, v = (torch.randn(sum(each), hkv, d, generator=g, device="cuda").bfloat16() for _ in "kv")
                batch.append(layer, k, v)
                at = 0
                for s, n in zip(some, each):
                    a, b = rows[s][layer]
                    rows[s] = list(rows[s])
                    rows[s][layer] = (torch.cat((a, k[at:at + n])), torch.cat((b, v[at:at + n])))
                    at += n
        elif r < 0.85:
            s = int(rng.choice(seqs))
            n = pool.trim(s, int(rng.integers(0, 30)))
            keep = [(a[:len(a) - n], b[:len(b) - n]) for a, b in rows[s]]
            rows[s] = keep
        elif r < 0.93:
            s = int(rng.choice(seqs))
            pool.free(s)
            del rows[s]
        else:
            pool.compact()
        for s in rows:
            assert pool.length(s) == len(rows[s][0][0])
        if move % 6 == 5:
            check(list(rows))
    check(list(rows))
    assert pool.check_device() == 0


@pytest.mark.parametrize("bits", [0, 8])
def test_router_takes_paged_layers(cuda, bits):
    """Prefill and decode through attention_with_cache_update equal its own dense attention over the same tokens."""
    import torch
    import sparse_decode as sd
    g = gen(torch, 95)
    B, hq, hkv, d, n = 2, 8, 2, 128, 37
    pool = sd.PagePool(1, 16, hkv, d, 16, "bf16", bits)
    seqs = [pool.add() for _ in range(B)]
    t = lambda h, L: torch.randn(B, h, L, d, generator=g, device="cuda").bfloat16()  # noqa: E731
    q, k, v = t(hq, n), t(hkv, n), t(hkv, n)
    sinks = torch.randn(hq, generator=g, device="cuda")
    out = sd.attention_with_cache_update(q, k, v, pool.extend(seqs, n).layer(0), d ** -0.5, "causal", sinks)
    want = sd.attention_with_cache_update(q, k, v, None, d ** -0.5, "causal", sinks)
    assert torch.allclose(out.float(), want.float(), rtol=5e-2, atol=5e-2 if bits else 1e-2)
    q1, k1, v1 = t(hq, 1), t(hkv, 1), t(hkv, 1)
    layer = pool.extend(seqs, 1).layer(0)
    assert layer.offset == [n, n]
    out = sd.attention_with_cache_update(q1, k1, v1, layer, d ** -0.5, None, sinks)
    want = sd.attention_with_cache_update(q1, torch.cat((k, k1), 2), torch.cat((v, v1), 2), None, d ** -0.5, None, sinks)
    assert out.shape == q1.shape and torch.allclose(out.float(), want.float(), rtol=5e-2, atol=5e-2 if bits else 1e-2)
    with pytest.raises(ValueError):
        sd.attention_with_cache_update(q, k, v, layer, d ** -0.5)   # the step holds one new token each


@pytest.mark.parametrize("bits", [0, 4, 8])
def test_example_runs(cuda, bits):
    from sparse_decode import paged_example
    pool, seqs, outs, worst = paged_example.run(kv_bits=bits, check=True)
    assert [pool.length(s) for s in seqs] == [110, 110]  # the prompt of 70 and its fork, 40 steps on
    # normwise against 64 bits over what the pool stores: bf16's own rounding (2^-8 sqrt(1/12) per element) and
    # _dequantize's rounding of the stored values to bf16
    assert worst < 4e-3

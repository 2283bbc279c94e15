"""The paged cache on the GPU where its answers are easy to lose: weights far
below the largest, scores that tie, masks of the router, steps that fail.

Bounds are stated at each test, from the kernels' arithmetic; the references
are computed in 64 bits.
"""
from __future__ import annotations

import math

import pytest

from test_gpu_paged import gen, tdt

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# decode: accuracy
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_decode_keeps_weights_far_below_the_largest(cuda, d, dtype):
    """One token of each sequence has nearly all the weight and a value of zero, as an attention sink has, so that the
    output is what the 16383 others add up to, each with a weight of e^-17.5 .. e^-19.5 of the largest. 300 sequences
    over the same pages: segments of a whole sequence.

    Bound: a weight of at most 2^8 times the running maximum's is held as two halves of the element type. In fp16 they
    reach down to half of 2^-24 at a scale of 2^7: 2^-32 of the maximum's weight at most for each token. bf16's two
    halves lose 2^-16 of a weight; the weights and their sums in fp32 2^-20 of them, and the
    rounding of the output, or of a subnormal one."""
    import torch
    import sparse_decode as sd
    dt, g = tdt(torch, dtype), gen(torch, d)
    B, page, n = 300, 256, 16384
    k = torch.zeros(n // page, 1, page, d, device="cuda")
    score = -17.5 - 2 * torch.rand(n, generator=g, device="cuda")
    score[9000] = 0.0
    k[..., 0] = score.view(n // page, 1, page)
    v = torch.rand(n, d, generator=g, device="cuda") + 0.5
    v[9000] = 0.0
    k, v = k.to(dt), v.view(n // page, page, d)[:, None].to(dt).contiguous()
    q = torch.zeros(B, 1, d, device="cuda", dtype=dt)
    q[..., 0] = 1.0
    tables = torch.arange(n // page, dtype=torch.int32, device="cuda").repeat(B, 1)
    out = sd.paged_decode(q, sd.KVPages(k, v), tables, torch.full((B,), n, dtype=torch.int32, device="cuda"), 1.0)
    p = torch.softmax(k[..., 0].double().flatten(), 0)
    ref = p @ v.double().view(n, d)
    each = {"f16": n * 2.0 ** -32 * 1.5, "bf16": 0.0}[dtype]
    rel = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8 + 2.0 ** -16}[dtype] + 2.0 ** -20 + 2.0 ** -22
    bound = each + rel * ref + (2.0 ** -25 if dtype == "f16" else 0.0)
    worst = ((out[:, 0].double() - ref).abs() / bound).max()
    assert float(worst) <= 1.0, float(worst)


@pytest.mark.parametrize("dtype,bits", [("bf16", 4), ("bf16", 8), ("f16", 4), ("f32", 4)])
@pytest.mark.parametrize("dims", ["even", "odd", "all"])
def test_decode_ties_of_wide_keys_and_queries_of_one_sign(cuda, dtype, bits, dims):
    """Two tokens per sequence with the same score to all digits: the second one's codes are the first one's in another
    order, between dims where the query is the same. Their values are +1 and -1, so the output is tanh of half the
    difference that rounding makes between the scores, and 0 without it.

    Bound, for a group of 64 dims: four mma steps, each off by at most two units (2^-23) of the largest partial sum A,
    which is sum(c |q|) plus what is left in of the offset that makes codes fp16 numbers: 1024 |q| for 8-bit codes of
    bf16 pools, 64 |q| for the odd dims of 4-bit ones, none for other pools; in fp32 pools q is cut to two halves, 2^-22
    of sum(c |q|) more. Times scale and the key's scale for either token; the difference is halved by the mean and
    doubled by there being two. Then four fp32 operations on the score and its bias part, for either token."""
    import torch
    import sparse_decode as sd
    dt, g = tdt(torch, dtype), gen(torch, bits)
    B, hkv, G, d, page, top = 256, 2, 4, 128, 16, (1 << bits) - 1
    each = 2.0 ** (7 * torch.rand(B, hkv, 1, 2, 16, generator=g, device="cuda") - 3)
    each[..., 1::2] *= dims != "even"
    each[..., 0::2] *= dims != "odd"
    f = 1 + torch.rand(B, hkv, G, 1, 1, generator=g, device="cuda")  # another query for each head
    q = (each * f).to(dt)[..., None, :].expand(B, hkv, G, 2, 4, 16).reshape(B, hkv * G, d).contiguous()
    one = torch.randint(0, top + 1, (B, hkv, 2, 4, 16), generator=g, device="cuda")
    other = one.gather(3, torch.rand(one.shape, generator=g, device="cuda").argsort(3))
    codes = torch.zeros(B, hkv, page, d, dtype=torch.int64, device="cuda")
    codes[:, :, 0], codes[:, :, 1] = one.flatten(2), other.flatten(2)
    per = 32 // bits
    words = (codes.unflatten(-1, (-1, per)) << (torch.arange(per, device="cuda") * bits)).sum(-1)
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
    s, b = 240.0 / top, -100.0
    small = torch.full((B, hkv, page, d // 64), s, device="cuda").to(dt)
    s = float(small[0, 0, 0, 0])
    vb = torch.zeros_like(small)
    vb[:, :, 0], vb[:, :, 1] = 1.0, -1.0
    pages = sd.KVPages(words, torch.zeros_like(words), small, torch.full_like(small, b), torch.ones_like(small), vb,
                       bits=bits)
    tables = torch.arange(B, dtype=torch.int32, device="cuda")[:, None]
    scale = d ** -0.5
    out = sd.paged_decode(q, pages, tables, torch.full((B,), 2, dtype=torch.int32, device="cuda"), scale)
    x = q.double().view(B, hkv, G, d).abs()
    c = torch.maximum(codes[:, :, 0], codes[:, :, 1]).double()[:, :, None]
    cq = (x * c).sum(-1)
    left = {("bf16", 8): 1024 * x.sum(-1), ("bf16", 4): 64 * x[..., 1::2].sum(-1)}.get((dtype, bits), 0.0)
    bound = 4 * 2 * 2.0 ** -23 * (cq + left) * s * scale
    if dtype == "f32":
        bound = bound + 2.0 ** -22 * cq * s * scale
    bound = bound + 2 * 4 * 2.0 ** -24 * scale * (s * cq + abs(b) * x.sum(-1)) + 1e-6
    worst = (out.double().view(B, hkv, G, d).abs().amax(-1) / bound).max()
    assert float(worst) <= 1.0, float(worst)


# ---------------------------------------------------------------------------
# the router
# ---------------------------------------------------------------------------

def prompt(torch, bits=0, lengths=(37, 37), new=None, hq=8, hkv=2, d=128, seed=0):
    """A pool with sequences of these lengths, all but the last `new` tokens (None: none of them) stored, and the
    step's q, k, v [B, heads, new, d]."""
    import sparse_decode as sd
    g = gen(torch, seed)
    B, new = len(lengths), min(lengths) if new is None else new
    pool = sd.PagePool(1, 40, hkv, d, 16, "bf16", bits)
    seqs = [pool.add() for _ in lengths]
    rows = [[torch.randn(hkv, n, d, generator=g, device="cuda").bfloat16() for n in lengths] for _ in "kv"]
    for i, n in enumerate(lengths):
        if n > new:
            step = pool.extend(seqs[i:i + 1], n - new)
            step.append(0, *(x[i][:, :n - new].transpose(0, 1) for x in rows))
    q = torch.randn(B, hq, new, d, generator=g, device="cuda").bfloat16()
    k, v = (torch.stack([y[:, -new:] for y in x]) for x in rows)
    return pool, seqs, rows, q, k, v


def attend64(q, k, v, scale, keep, sinks=None):
    """One sequence: q [Hq, L, D], k, v [Hkv, T, D], keep [.., L, T] (bool, or numbers to add)."""
    import torch
    k, v = (x.double().repeat_interleave(q.shape[0] // x.shape[0], 0) for x in (k, v))
    s = q.double() @ k.transpose(1, 2) * scale
    s = s.masked_fill(~keep, -math.inf) if keep.dtype == torch.bool else s + keep.double()
    if sinks is not None:
        s = torch.cat((s, sinks.double().view(-1, 1, 1).expand(-1, s.shape[1], 1)), -1)
    return torch.softmax(s, -1)[..., :k.shape[1]] @ v


def close(out, ref):
    """Dense attention in bf16: its probabilities and sums may be rounded to bf16, 2^-8, once or twice."""
    assert float((out.double() - ref).norm() / ref.norm()) < 2e-2


@pytest.mark.parametrize("mask", [None, "causal"])
@pytest.mark.parametrize("with_sinks", [False, True])
def test_router_without_a_mask_hides_nothing(cuda, mask, with_sinks):
    """None and "causal" mean for a paged layer what they mean for the other caches."""
    import torch
    import sparse_decode as sd
    pool, seqs, rows, q, k, v = prompt(torch, seed=1)
    sinks = torch.randn(8, generator=gen(torch, 2), device="cuda") if with_sinks else None
    out = sd.attention_with_cache_update(q, k, v, pool.extend(seqs, 37).layer(0), 0.1, mask, sinks)
    same = sd.attention_with_cache_update(q, k, v, None, 0.1, mask, sinks)
    keep = torch.ones(37, 37, dtype=torch.bool, device="cuda")
    keep = keep.tril() if mask else keep
    for b in range(2):
        ref = attend64(q[b], k[b], v[b], 0.1, keep, sinks)
        close(out[b], ref)
        close(same[b], ref)


@pytest.mark.parametrize("with_sinks", [False, True])
@pytest.mark.parametrize("kind", ["bool", "add", "heads", "shared", "2d", "3d"])
def test_router_takes_each_sequence_its_mask(cuda, kind, with_sinks):
    """Masks with a batch dimension, for sequences of different lengths: column t is token t, and the columns past a
    sequence's end are not its own."""
    import torch
    import sparse_decode as sd
    lengths, L, B, hq = [70, 37, 51], 20, 3, 8
    pool, seqs, rows, q, k, v = prompt(torch, lengths=lengths, new=L, seed=3)
    g = gen(torch, 4)
    T = max(lengths)
    shape = {"shared": (1, 1, L, T), "heads": (B, hq, L, T), "2d": (L, T), "3d": (hq, L, T)}.get(kind, (B, 1, L, T))
    mask = torch.rand(shape, generator=g, device="cuda") < 0.5
    mask[..., 0] = True
    if kind == "add":
        mask = torch.where(mask, torch.randn(shape, generator=g, device="cuda"), -math.inf).bfloat16()
    sinks = torch.randn(hq, generator=g, device="cuda") if with_sinks else None
    out = sd.attention_with_cache_update(q, k, v, pool.extend(seqs, L).layer(0), 0.1, mask, sinks)
    full = mask.expand(B, hq, L, T)
    for b, n in enumerate(lengths):
        close(out[b], attend64(q[b], rows[0][b], rows[1][b], 0.1, full[b][..., :n], sinks))


def test_router_refuses_masks_that_do_not_fit(cuda):
    import torch
    import sparse_decode as sd
    pool, seqs, rows, q, k, v = prompt(torch, lengths=[40, 30], new=10, seed=5)
    layer = pool.extend(seqs, 10).layer(0)
    z = lambda *s: torch.zeros(*s, dtype=torch.bool, device="cuda")  # noqa: E731
    for bad in (z(3, 1, 10, 40), z(2, 3, 10, 40), z(2, 1, 9, 40), z(2, 1, 10, 39), z(2, 1, 10, 41), z(10), z(1, 2, 1, 10, 40),
                "full"):
        with pytest.raises(ValueError):
            sd.attention_with_cache_update(q, k, v, layer, 0.1, bad)


def test_router_takes_causal_for_a_single_token(cuda):
    """The newest token sees all of its sequence: "causal" hides nothing."""
    import torch
    import sparse_decode as sd
    pool, seqs, rows, q, k, v = prompt(torch, lengths=[40, 30], new=1, seed=6)
    layer = pool.extend(seqs, 1).layer(0)
    a = sd.attention_with_cache_update(q, k, v, layer, 0.1, None)
    b = sd.attention_with_cache_update(q, k, v, layer, 0.1, "causal")
    assert torch.equal(a, b)
    for bad in (torch.ones(2, 1, 1, 40, dtype=torch.bool, device="cuda"), "full"):
        with pytest.raises(ValueError):
            sd.attention_with_cache_update(q, k, v, layer, 0.1, bad)


@pytest.mark.parametrize("bits", [0, 8])
@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("window", [1, 7, 16, 30, 1000])
def test_router_windows(cuda, window, new, bits):
    """A layer with a window: every token sees the last `window` tokens up to itself, whichever path its step takes."""
    import torch
    import sparse_decode as sd
    lengths = [70, 37, 20]
    pool, seqs, rows, q, k, v = prompt(torch, bits, lengths, new, seed=7)
    step = pool.extend(seqs, new)
    sinks = torch.randn(8, generator=gen(torch, 8), device="cuda")
    out = sd.attention_with_cache_update(q, k, v, step.layer(0, window=window), 0.1, "causal", sinks)
    for b, n in enumerate(lengths):
        kk, vv = step.layer(0).dense(b)
        back = torch.arange(n - new, n, device="cuda")[:, None] - torch.arange(n, device="cuda")
        close(out[b], attend64(q[b], kk[0], vv[0], 0.1, (back >= 0) & (back < window), sinks))
    if new > 1:  # a window and another mask than "causal" say two things
        for mask in (None, torch.ones(new, 70, dtype=torch.bool, device="cuda")):
            with pytest.raises(ValueError):
                sd.attention_with_cache_update(q, k, v, step.layer(0, window=window), 0.1, mask)
    with pytest.raises(ValueError):
        step.layer(0, window=-1)


# ---------------------------------------------------------------------------
# steps
# ---------------------------------------------------------------------------

def test_page_copies_of_a_step_do_not_stop_the_host(cuda):
    """Copy-on-write, compaction and copies of host lists are queued like the rest of a step."""
    import torch
    import sparse_decode as sd
    pool = sd.PagePool(2, 12, 2, 64, 16)
    a = pool.add()
    step = pool.extend([a], 40)
    x = torch.randn(40, 2, 64, device="cuda").bfloat16()
    for layer in range(2):
        step.append(layer, x, -x)
    b = pool.fork(a)
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        step = pool.extend([b], 1)                 # leaves the shared page
        sd.copy_pages(pool.pages, [0, 1], [10, 11])
        pool.free(a)
        assert pool.compact() == 1
    finally:
        torch.cuda.set_sync_debug_mode("default")
    k, v = pool.batch([b]).layer(1).dense(0)
    assert torch.equal(k[0, :, :40], x.transpose(0, 1)) and torch.equal(v[0, :, :40], -x.transpose(0, 1))
    assert torch.equal(pool.pages.k[:, 10:], pool.pages.k[:, :2])


def test_host_lists_are_refused_in_a_captured_graph(cuda):
    """A replay would copy whatever the host memory holds by then."""
    import torch
    import sparse_decode as sd
    pool = sd.PagePool(1, 12, 2, 64, 16)
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            sd.copy_pages(pool.pages, [0], [1])
    torch.cuda.synchronize()
    sd.copy_pages(pool.pages, [0], [1])


def test_a_step_cannot_be_made_in_a_captured_graph(cuda):
    """Its tables come from the host; the step's calls are what a graph may hold. No sequence grows."""
    import torch
    import sparse_decode as sd
    pool = sd.PagePool(1, 12, 2, 64, 16)
    a = pool.add()
    pool.extend([a], 5)
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            pool.extend([a], 1)
    torch.cuda.synchronize()
    assert pool.length(a) == 5
    assert pool.batch([a]).lengths.tolist() == [5]


@pytest.mark.parametrize("bad", [([0, "x"], 3), ([0, 1], [3, "x"]), ([0, 1], [3, 1 << 70]), ([0, 1 << 70], 3), ([0, 9], 3)])
def test_a_step_that_fails_leaves_every_sequence_as_it_was(cuda, bad):
    import sparse_decode as sd
    pool = sd.PagePool(1, 12, 2, 64, 16)
    a, b = pool.add(), pool.add()
    assert (a, b) == (0, 1)
    pool.extend([a, b], 5)
    with pytest.raises(Exception):
        pool.extend(*bad)
    assert (pool.length(a), pool.length(b)) == (5, 5)

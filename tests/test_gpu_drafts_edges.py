"""Calls of the operators around drafted tokens that their documentation allows
and that read or wrote, once, what they should not have."""
from __future__ import annotations

import ctypes
import math
import random

import pytest

import test_gpu_drafts as tree
from test_gpu_drafts import i32
from test_gpu_paged import Pool, gen, tables_of, tdt

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# plan
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("take", [False, True])
@pytest.mark.parametrize("B,at", [(2, 0), (2, 1), (5, 2), (700, 300), (4096, 4095)])
@pytest.mark.parametrize("length,added", [(100, 0), (100, 3), (65, 0), (64, 1), ((1 << 31) - 1, 64)])
def test_plan_of_a_length_past_its_table(cuda, B, at, length, added, take, tree):
    """Sequence `at` has more tokens than its table's 4 pages of 16 hold (64, one more: the new one does not fit): it gets
    neither tokens nor pages, the others theirs, and nothing is written behind its row or behind the tables."""
    import sparse_decode as sd
    torch = cuda
    W, page = 4, 16
    lengths, new, held = [3] * B, [14] * B, [1] * B  # a second page each
    lengths[at], new[at], held[at] = length, added, 4
    room = torch.full((B * W + 64,), -7, dtype=torch.int32, device="cuda")
    tables = room[:B * W].view(B, W)
    tables.copy_(torch.arange(B * W, device="cuda").view(B, W))
    want = tables.clone()
    free = torch.arange(5 * B, 9 * B, dtype=torch.int32, device="cuda")
    h, taken, flags = i32(torch, held), i32(torch, [0]), i32(torch, [0])
    grow = dict(held=h, free=free, taken=taken) if take else {}
    others = [b for b in range(B) if b != at]
    if take:
        want[others, 1] = free[:B - 1]
    up = i32(torch, list(range(-1, 63))) if tree else None
    p = sd.paged_plan(i32(torch, lengths), i32(torch, new), tables, page, 14 * B + 9, parents=up, flags=flags, **grow)
    assert int(flags) == 2
    assert torch.equal(tables, want) and (room[B * W:] == -7).all()
    if take:
        assert h.tolist() == [4 if b == at else 2 for b in range(B)] and taken.tolist() == [B - 1]
    first = [0]
    for b in range(B):
        first.append(first[-1] + (0 if b == at else 14))
    assert p.first.tolist() == first
    assert p.ends.tolist() == [length if b == at else 17 for b in range(B)]
    assert p.seq.tolist() == [b for b in others for _ in range(14)] + [-1] * 23
    assert p.positions.tolist() == [t for _ in others for t in range(3, 17)] + [-1] * 23
    slot = want[others][:, :2].long().repeat_interleave(16, 1)[:, 3:17] * page + torch.arange(3, 17, device="cuda") % page
    assert torch.equal(p.slots[:14 * (B - 1)], slot.flatten())


# ---------------------------------------------------------------------------
# tree attention: rows that cannot be
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,bits,hkv,G,first", [
    ("bf16", 0, 8, 4, [0, 60] * 3),                      # few columns on average: the 16-column kernel
    ("f32", 0, 8, 4, [0, 60] * 3), ("f16", 4, 8, 4, [0, 60] * 3), ("bf16", 8, 2, 16, [0, 64] * 32 + [0]),
    ("bf16", 0, 8, 16, [0, 60, 0, 60]), ("f16", 0, 2, 16, [0, 64, 0, 64]),  # the tile kernel
    ("bf16", 4, 2, 16, [0, 64, 0, 64]), ("bf16", 8, 2, 16, [0, 64, 0, 64]),
    ("bf16", 0, 2, 4, [0, 20, 40, 39, 60]), ("bf16", 0, 2, 16, [0, 20, 40, 39, 60]), ("bf16", 4, 2, 16, [0, 60, 60, 60, 59])])
def test_tree_first_that_falls(cuda, dtype, bits, hkv, G, first):
    """Sequences with rows in common would need more than the workspace has: all rows give zeros, with the error bit, and
    nothing is written behind the workspace. A call whose first rises, in the same workspace, is right."""
    import sparse_decode as sd
    torch = cuda
    B, n, d, page, W, guard = len(first) - 1, max(first), 64, 16, 6, 1 << 22
    pool = Pool(torch, sd, dtype, bits, hkv, d, page, B * W, 3)
    tables = tables_of(torch, [page * W] * B, page, B * W, 4)
    q = torch.randn(n, hkv * G, d, generator=gen(torch, 5), device="cuda").to(tdt(torch, dtype))
    lengths, flags, size = i32(torch, [80] * B), i32(torch, [0]), ctypes.c_int64()
    L = sd.lib()
    sd._check(L.sd_paged_tree_workspace(pool.pages.struct, B, n, hkv * G, size))
    work = torch.full((size.value + guard,), 0xA5, dtype=torch.uint8, device="cuda")

    def call(rows):
        out, f = torch.full_like(q, 7.0), i32(torch, rows)
        sd._check(L.sd_paged_tree_decode(pool.pages.struct, 0, q.data_ptr(), n, B, hkv * G, tables.data_ptr(), W,
                                         lengths.data_ptr(), f.data_ptr(), None, None, 0.125, 0, None, out.data_ptr(),
                                         work.data_ptr(), size.value, flags.data_ptr(), torch.cuda.current_stream().cuda_stream))
        got = int(flags)
        flags.zero_()
        assert (work[size.value:] == 0xA5).all()
        return out, got
    out, f = call(first)
    assert f == 2 and not out[:first[-1]].any() and (out[first[-1]:] == 7).all()
    rises = [min(n, -(-n // B) * b) for b in range(B + 1)]
    out, f = call(rises)
    want = sd.paged_tree_decode(q, pool.pages, tables, lengths, i32(torch, rises), scale=0.125)
    assert f == 0 and torch.equal(out, want) and out.abs().amax((1, 2)).min() > 0


# ---------------------------------------------------------------------------
# tree attention: the same precision whatever the number of columns
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,bits,d,hkv,G,page,held,counts,more", [
    ("bf16", 0, 128, 2, 4, 64, [3000, 5, 0, 1000], [33, 20, 64, 40], {}),
    ("bf16", 0, 64, 2, 4, 64, [700, 90], [64, 20], {}),
    ("bf16", 0, 128, 2, 16, 64, [20000, 37], [33, 60], {}),
    ("bf16", 0, 128, 2, 8, 32, [400, 3, 150, 64, 0], [20, 12, 1, 64, 30], dict(window=65, sinks=True)),
    ("f16", 0, 128, 2, 4, 64, [3000, 5, 0, 1000], [33, 20, 64, 40], {}),
    ("f16", 0, 64, 3, 8, 16, [700, 90], [64, 20], dict(window=200)),
    ("f16", 0, 128, 1, 16, 64, [9000], [40], {}),
])
def test_tree_precision_does_not_go_by_the_columns(cuda, monkeypatch, dtype, bits, d, hkv, G, page, held, counts, more):
    """Calls with many columns have the framework's tolerance and the mean square of the result's own rounding, as those
    with few: weights keep 16 bits or more."""
    assert tree.uses_tiles(dtype, bits, counts, G)
    monkeypatch.setattr(tree, "uses_tiles", lambda *a: False)
    tree.run_tree(cuda, dtype, bits, d, hkv, G, page, held, counts, seed=G + d, **more)


def check_codes(torch, out, ref, size, reach, dtype, tile, bits=0):
    """Of many columns: a value of codes is two bf16 values, the first cut off, off by 2^-7 2^-8 = 2^-15 of it at most.
    So a score is off by d = 2^-15 B, B = scale sum |q k|, and the output by (e^2d - 1) A, A = sum p |v| / sum p; values,
    weights (2^-16) and the product of low halves that is left out (2^-8 p times 2^-7 v) are 2^-13 A more at most; then
    half a step of the result. Most of that cancels: in the mean square nothing but that half step shows, as with few
    columns. (Not the norm against the rounded exact result, of which one value that lies half-way makes 2e-3.)"""
    u = torch.finfo(out.dtype).eps / 2
    bound = 1.01 * u * ref.abs() + size * (torch.expm1(2.0 ** -14 * reach[0]) + 2.0 ** -13)
    off = (out.double() - ref).abs()
    assert bits and (off <= bound).all(), f"{int((off > bound).sum())} off, worst {float((off / bound).max()):.3g}"
    assert (off.pow(2).sum() / ref.pow(2).sum()).sqrt() <= 0.65 * u


@pytest.mark.parametrize("bits,d,hkv,G,page,held,counts,more", [
    (4, 128, 2, 4, 64, [3000, 5, 0, 1000], [33, 20, 64, 40], {}),
    (4, 64, 2, 16, 16, [700, 90], [64, 20], dict(window=200, sinks=True)),
    (8, 128, 2, 4, 64, [3000, 5, 0, 1000], [33, 20, 64, 40], {}),
    (8, 64, 2, 8, 32, [20000, 37], [33, 60], {}),
    (8, 64, 2, 16, 64, [700, 90], [33, 20], dict(scale=1e-3)),
])
def test_tree_precision_of_codes_does_not_go_by_the_columns(cuda, monkeypatch, bits, d, hkv, G, page, held, counts, more):
    assert tree.uses_tiles("bf16", bits, counts, G)
    monkeypatch.setattr(tree, "check_tree", check_codes)
    tree.run_tree(cuda, "bf16", bits, d, hkv, G, page, held, counts, seed=G + d, **more)


@pytest.mark.parametrize("dtype,bits,d,G", [("bf16", 0, 128, 4), ("bf16", 0, 64, 16), ("f16", 0, 128, 8), ("bf16", 4, 128, 4),
                                            ("bf16", 4, 64, 16), ("bf16", 8, 128, 8), ("bf16", 8, 64, 16)])
def test_tree_scores_of_hundreds(cuda, dtype, bits, d, G):
    """Keys and values thirty times as large: a softmax of one or a few tokens, whose weights go by errors of the scores.

    The values of codes are taken as the kernel's two halves of them, so that its sums alone are off: a score by 16 steps of
    at most 2 units 2^-23 of B, the largest scale sum |q k|, that is d = 2^-18 B, which moves the output by at most (e^2d - 1)
    A, A = sum p |v| / sum p; weights (2^-16) and the product of low halves that is left out (2^-8 p times 2^-7 v) by less
    than 2^-14 A; and half a step of the result. Weights below 2^-126 are none, and below 2^-117 their low halves lose bits: less
    than 2^-125 of a value; of fp16, whose largest weight is 2^7 at least, 2^-25 of that, 2^-32. (The framework's tolerance is
    against the rounded exact result. It does not fit here: values of codes lie half-way between two results more often than
    not.)"""
    import sparse_decode as sd
    torch = cuda
    hkv, page, held, counts = 2, 64, [700, 90], [33, 20]
    assert tree.uses_tiles(dtype, bits, counts, G)
    ends = [h + n for h, n in zip(held, counts)]
    pool = Pool(torch, sd, dtype, bits, hkv, d, page, 20, 3, 30.0)
    tables = tables_of(torch, ends, page, 20, 4)
    if bits:
        for i, x in enumerate(pool.values):
            high = (x.float().view(torch.int32) & -65536).view(torch.float32)
            pool.values[i] = high.double() + (x.float() - high).bfloat16().double()
    q = (2 * torch.randn(sum(counts), hkv * G, d, generator=gen(torch, 5), device="cuda")).to(tdt(torch, dtype))
    first = i32(torch, [0, counts[0], sum(counts)])
    out = sd.paged_tree_decode(q, pool.pages, tables, i32(torch, ends), first)
    lines = [[((2 << i) - 1, h + i) for i in range(n)] for h, n in zip(held, counts)]
    ref, size, (reach, values) = tree.tree64(q, pool, tables, held, lines, 1 / math.sqrt(d))
    u = torch.finfo(out.dtype).eps / 2
    bound = 1.01 * u * ref.abs() + size * (torch.expm1(2.0 ** -17 * reach) + 2.0 ** -14) + values * 2.0 ** (-32 if dtype == "f16" else -125)
    off = (out.double() - ref).abs()
    assert reach.min() > 150 and (off <= bound).all(), f"{int((off > bound).sum())} off, worst {float((off / bound).max()):.3g}"


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n,d", [(40, 128), (33, 64)])
def test_tree_codes_of_keys_with_large_channels(cuda, bits, n, d):
    """One channel of every group is a hundred times as large as what the others spread over, so that the scores' parts cancel."""
    import sparse_decode as sd
    torch = cuda
    hkv, G, page, held = 2, 4, 64, 4000
    pool = Pool(torch, sd, "bf16", bits, hkv, d, page, 64, 5)
    tables = tables_of(torch, [held + n], page, 64, 6)
    (k, ks, kb), top, per = pool.arrays[0], (1 << bits) - 1, 32 // bits
    g = gen(torch, 7)
    codes = torch.randint(0, 2 if bits == 4 else 6, (*ks.shape[:-1], d), generator=g, device="cuda")
    codes[..., 7::64] = top - torch.randint(0, 2 if bits == 4 else 6, codes[..., 7::64].shape, generator=g, device="cuda")
    words = (codes.unflatten(-1, (-1, per)) << (torch.arange(per, device="cuda") * bits)).sum(-1)
    k.copy_(torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32))
    ks.copy_((102 + torch.rand(ks.shape, generator=g, device="cuda")) / top)
    kb.copy_(-2 + 0.1 * torch.rand(ks.shape, generator=g, device="cuda"))
    grow = lambda t: t.double().repeat_interleave(64, -1)  # noqa: E731
    pool.values[0] = codes.double() * grow(ks) + grow(kb)
    q = torch.randn(n, hkv * G, d, generator=g, device="cuda").bfloat16()
    out = sd.paged_tree_decode(q, pool.pages, tables, i32(torch, [held + n]), i32(torch, [0, n]))
    lines = [[((2 << i) - 1, held + i) for i in range(n)]]
    ref, size, reach = tree.tree64(q, pool, tables, [held], lines, 1 / math.sqrt(d))
    tree.check_tree(torch, out, ref, size, reach, "bf16", False)


# ---------------------------------------------------------------------------
# tree attention: what a row does not see
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,bits", [("bf16", 0), ("f16", 0), ("bf16", 4), ("bf16", 8), ("f16", 4), ("f32", 8), ("f32", 0)])
@pytest.mark.parametrize("G", [2, 16])
@pytest.mark.parametrize("held", [0, 37, 200])
@pytest.mark.parametrize("x", [2.0 ** 60, -2.0 ** 60, math.inf, -math.inf, math.nan])
def test_tree_large_values_in_hidden_and_absent_nodes(cuda, dtype, bits, G, held, x):
    """Two branches from one root, and nodes that do not exist: their keys and values, finite and large or not finite, leave
    the rows alone that do not see them, bit for bit."""
    import sparse_decode as sd
    torch = cuda
    if dtype == "f16" and abs(x) < math.inf:
        x = math.copysign(2.0 ** 15, x)
    pool = Pool(torch, sd, dtype, bits, 2, 128, 16, 16, 3)
    tables = tables_of(torch, [held + 8], 16, 16, 4)
    parents = [-1, 0, 0, 1, 2, 3, -2, 6]  # 2 and 4 are the other branch, 6 and 7 absent
    masks = torch.tensor([m for m, _ in tree.lineage(parents)], dtype=torch.int64, device="cuda")
    q = torch.randn(8, 2 * G, 128, generator=gen(torch, 4), device="cuda").to(tdt(torch, dtype))
    call = lambda: sd.paged_tree_decode(  # noqa: E731
        q, pool.pages, tables, i32(torch, [held + 8]), i32(torch, [0, 8]), masks)
    clean = call()
    for arrays in (pool.arrays[:1], pool.arrays[1:], pool.arrays):
        saved = [a[-1].clone() for a in pool.arrays]
        for a in arrays:
            for node in (2, 4, 6, 7):
                t = held + node
                a[-1][int(tables[0, t // 16]), :, t % 16] = x  # all of a row, or every group's bias
        out = call()
        for a, s in zip(pool.arrays, saved):
            a[-1].copy_(s)
        for node in (0, 1, 3, 5, 6, 7):
            assert torch.equal(out[node], clean[node]), node


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("G", [4, 16])
@pytest.mark.parametrize("power", [-60, 40, 60])
def test_tree_codes_beside_tokens_of_another_size(cuda, bits, G, power):
    """A held token in every tile, and a node, whose values are 2^power of the others', with keys that give it no weight:
    the others' values keep their bits. (Calls of many columns. With few, codes are the decode kernel's, which has an error
    of 2^-28 of the largest scale.)"""
    import sparse_decode as sd
    torch = cuda
    n, held, hkv, d = 9, 300, 2, 64
    assert tree.uses_tiles("bf16", bits, [n], G)
    pool = Pool(torch, sd, "bf16", bits, hkv, d, 64, 8, 5)
    tables = tables_of(torch, [held + n], 64, 8, 6)
    q = (torch.rand(n, hkv * G, d, generator=gen(torch, 7), device="cuda") + 0.5).bfloat16()
    for t in [*range(7, held, 50), held + 2]:
        at = (int(tables[0, t // 64]), slice(None), t % 64)
        pool.arrays[0][1][at], pool.arrays[0][2][at] = 0.0, -40.0  # a score of -230 at most
        for a in pool.arrays[1][1:]:
            a[at] *= 2.0 ** power
        pool.values[0][at] = -40.0
        pool.values[1][at] *= 2.0 ** power
    out = sd.paged_tree_decode(q, pool.pages, tables, i32(torch, [held + n]), i32(torch, [0, n]))
    lines = [[((2 << i) - 1, held + i) for i in range(n)]]
    ref, size, reach = tree.tree64(q, pool, tables, [held], lines, 1 / math.sqrt(d))
    tree.check_tree(torch, out, ref, size, reach, "bf16", False)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("B", [3400, 3500, 4096])
def test_tree_codes_of_thousands_of_sequences(cuda, monkeypatch, bits, B):
    """Heads of 128: what is noted of that many sequences leaves no room for the tiles of 8-bit codes, which the other kernel takes."""
    rng = random.Random(B)

    def check(torch, out, ref, size, reach, *a):
        # The other kernel sums (p s)(c - z) and p (b + z s) apart, z the middle code: each is off by three units 2^-23 of
        # p z |s|. z |s| is half of a group's range, 1.3 times its largest |value| at most where its codes span 200 of 255, and the
        # largest A of a row a third of its tokens' largest or more: less than 2^-18 of the largest A, where A itself may
        # be next to nothing.
        check_codes(torch, out, ref, size + 2.0 ** -5 * size.amax(-1, keepdim=True), reach, *a)
    monkeypatch.setattr(tree, "check_tree", check)
    tree.run_tree(cuda, "bf16", bits, 128, 1, 16, 16, [rng.randint(0, 12) for _ in range(B)], [rng.choice([2, 3, 4]) for _ in range(B)], seed=5)


# ---------------------------------------------------------------------------
# keep
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("form", ["list", "lists", "one tensor", "tensors"])
def test_pool_refuses_paths_that_are_not_in_the_tree(cuda, form):
    """Rows are rotated for their places in the tree, and absent nodes have none: a path skips no node and ends at none that is
    absent."""
    import sparse_decode as sd
    pool = sd.PagePool(1, 30, 2, 64, 16)
    a, b = pool.add(), pool.add()
    parents = [-1, 0, 0, 1, -2, 4, -1, 6, 2]
    tree_of = {"list": parents, "lists": [parents, parents], "one tensor": i32(cuda, parents), "tensors": i32(cuda, [parents] * 2)}[form]
    step = pool.extend([a, b], [9, 7]).tree(tree_of)
    if form == "one tensor":
        tree_of.fill_(-1)  # the step has its own
    k = cuda.randn(16, 2, 64, device="cuda").bfloat16()
    step.append(0, k, k)
    for bad in ([1], [0, 3], [0, 2, 3], [0, 1, 2], [4], [0, 4], [4, 5], [0, 6], [2], [0, 1, 3, 8], [7]):
        for paths in ([bad, [0]], [[0], bad]):
            if max(paths[1]) < 7:
                with pytest.raises(ValueError, match="way down"):
                    step.keep(paths)
    assert [pool.length(s) for s in (a, b)] == [9, 7]
    step.keep([[0, 2, 8], [6]])
    assert [pool.length(s) for s in (a, b)] == [3, 1] and pool.check_device() == 0
    got = pool.batch([a]).layer(0).dense(0)[0]
    assert cuda.equal(got.reshape(2, 3, 64), k[[0, 2, 8]].transpose(0, 1))


def test_pool_refuses_paths_off_a_long_chain(cuda):
    import sparse_decode as sd
    for given in (None, i32(cuda, list(range(-1, 63)))):
        pool = sd.PagePool(1, 30, 2, 64, 16)
        a = pool.add()
        step = pool.extend([a], 64).tree(given)
        for bad in ([1], [0, 2], list(range(1, 64)), [*range(62), 63]):
            with pytest.raises(ValueError, match="way down"):
                step.keep([bad])
        step.keep([list(range(64))])
        assert pool.length(a) == 64 and pool.check_device() == 0

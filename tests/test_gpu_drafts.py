"""Drafted tokens over the paged cache on the GPU against plain computations:
plans and moved rows bit for bit against a host model, tree attention against
64 bits.

Tolerance of the attention: the framework's (_util.assert_close) where weights
keep 16 bits or more. The tile kernel (16-bit pools, and codes of bf16 ones;
more than 16 columns an average sequence, 32 of 8-bit codes) rounds a weight to
the products' type once, by at most half a step of it: u of 16-bit pools, 2^-11 of
codes. With A = sum p |v| / sum p that is u A of the output, besides u |out| for
its own rounding. Codes are fp16 values there: 2^-11 |v| more of V, another
2^-11 A, and a score is off by d = 2^-11 B at most, B = scale sum |q k| of its
token: weights become p e^x with |x| <= d, and over their sum, which is between
e^-d and e^d of what it was, p e^y with |y| <= 2 d, so the output moves by at
most (e^2d - 1) A. Scores in fp32 add less than 1e-4 of A. fp16 weights below
2^-14 are off by 2^-25 however small they are, and the largest is 2^7 at least:
2^-32 sum |v| more, which counts where the heavy tokens' values are zero.
"""
from __future__ import annotations

import math
import random

import pytest

from _util import assert_close
from test_gpu_paged import Pool, gen, tables_of, tdt

pytestmark = pytest.mark.gpu


def i32(torch, values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def random_parents(rng, n, chain=False, absent=0.0):
    p = []
    for i in range(n):
        if i and rng.random() < absent:
            p.append(-2)
        else:
            p.append(i - 1 if chain else rng.randint(max(-1, i - 6), i - 1))
    return p


def lineage(parents):
    """(mask, depth) of each node; mask 0 and depth None for an absent one."""
    got = []
    for i, up in enumerate(parents):
        if up < -1 or up >= i:
            got.append((0, None))
        elif up < 0:
            got.append((1 << i, 0))
        else:
            m, d = got[up]
            got.append((m | 1 << i, d + 1) if m else (0, None))
    return got


def signed(mask):
    return mask - (1 << 64) if mask >> 63 else mask


# ---------------------------------------------------------------------------
# plan
# ---------------------------------------------------------------------------

def plan_model(lengths, new, tables, page, n_rows, parents=None, held=None, free=None, taken=0):
    """What paged_plan makes of host lists: dict of lists, and whether anything was cut."""
    B, W = len(lengths), len(tables[0])
    tables, held_out, bad = [list(r) for r in tables], list(held) if held else None, False
    seq, pos, slots, places, masks, first, ends = [], [], [], [], [], [0], []
    for b in range(B):
        n, ln = max(0, new[b]), max(0, lengths[b])
        n = min(n, max(0, W * page - ln))
        if parents is not None:
            n = min(n, len(parents[b]))
        n = min(n, n_rows) if n > n_rows else n
        bad |= n != new[b] or ln != lengths[b]
        if held:
            need = max(0, -(-(ln + n) // page) - held[b])
            got = min(need, len(free) - taken)
            tables[b][held[b]:held[b] + got] = free[taken:taken + got]
            taken += got
            held_out[b] = held[b] + got
            if got < need:
                bad, n = True, max(0, min(n, (held[b] + got) * page - ln))
        if first[-1] + n > n_rows:
            bad, n = True, n_rows - first[-1]
        lines = lineage(parents[b][:n]) if parents is not None else [((2 << min(i, 63)) - 1, i) for i in range(n)]
        if parents is not None:
            bad |= any(up >= i for i, up in enumerate(parents[b][:n]))
        for i, (m, d) in enumerate(lines):
            at = ln + i
            seq.append(b)
            pos.append(at if m else -1)
            pg = tables[b][at // page]
            slots.append(pg * page + at % page if m and pg >= 0 else -1)
            places.append(ln + d if m else -1)
            masks.append(signed(m))
        first.append(first[-1] + n)
        ends.append(ln + n)
    pad = n_rows - first[-1]
    return dict(first=first, ends=ends, seq=seq + [-1] * pad, positions=pos + [-1] * pad, slots=slots + [-1] * pad,
                places=places + [-1] * pad, masks=masks + [0] * pad, tables=tables, held=held_out, taken=taken), bad


def check_plan(torch, lengths, new, tables, page, n_rows, parents=None, held=None, free=None, taken=0, shared=False):
    import sparse_decode as sd
    want, bad = plan_model(lengths, new, tables, page, n_rows, parents, held, free, taken)
    flags, t = i32(torch, [0]), i32(torch, tables)
    grow = dict(held=i32(torch, held), free=i32(torch, free), taken=i32(torch, [taken])) if held else {}
    up = None if parents is None else i32(torch, parents[0] if shared else parents)
    p = sd.paged_plan(i32(torch, lengths), i32(torch, new), t, page, n_rows, parents=up, flags=flags, **grow)
    for name in ("first", "ends", "seq", "positions", "slots"):
        assert getattr(p, name).tolist() == want[name], name
    if parents is None:
        assert p.places is p.positions and p.masks is None
    else:
        assert p.places.tolist() == want["places"] and p.masks.tolist() == want["masks"]
    assert t.tolist() == want["tables"]
    if held:
        assert grow["held"].tolist() == want["held"] and grow["taken"].tolist() == [want["taken"]]
    assert bool(int(flags) & 2) == bad and int(flags) in (0, 2)


def plan_case(rng, B, page, most, ctx, nodes=0, spare=4):
    lengths = [rng.choice([0, page, rng.randint(0, ctx)]) for _ in range(B)]
    new = [rng.choice([0, 1, rng.randint(0, most)]) for _ in range(B)]
    held = [-(-n // page) + rng.choice([0, 0, 1]) for n in lengths]  # one page from an earlier draft, perhaps
    W = max(max(h, -(-(n + k) // page)) for h, n, k in zip(held, lengths, new)) + 1
    ids = list(range(sum(held) + spare + sum(-(-(n + k) // page) for n, k in zip(lengths, new))))
    rng.shuffle(ids)
    tables = []
    for h in held:
        tables.append(ids[:h] + [-1] * (W - h))
        del ids[:h]
    parents = [random_parents(rng, nodes, absent=0.1) for _ in range(B)] if nodes else None
    return lengths, new, tables, held, ids, parents


@pytest.mark.parametrize("B,page,most,ctx", [(1, 64, 1, 200), (1, 16, 5000, 30), (7, 32, 90, 500), (40, 16, 700, 90),
                                             (300, 64, 3, 5000), (4096, 16, 9, 100), (2, 256, 70000, 300)])
def test_plan_takes_pages(cuda, B, page, most, ctx):
    rng = random.Random(B + page)
    lengths, new, tables, held, free, _ = plan_case(rng, B, page, most, ctx)
    for extra in (0, 5):
        check_plan(cuda, lengths, new, tables, page, sum(new) + extra, held=held, free=free)
    check_plan(cuda, lengths, new, tables, page, sum(new) + 3, held=held, free=[9, 8, 7] + free, taken=3)


@pytest.mark.parametrize("B,nodes,page", [(1, 1, 64), (1, 64, 16), (5, 33, 32), (64, 16, 64), (513, 7, 16)])
@pytest.mark.parametrize("grow", [False, True])
def test_plan_of_trees(cuda, B, nodes, page, grow):
    rng = random.Random(nodes)
    lengths, new, tables, held, free, parents = plan_case(rng, B, page, nodes, 300, nodes)
    if grow:
        check_plan(cuda, lengths, new, tables, page, B * nodes, parents, held, free)
        return
    whole, _ = plan_model(lengths, new, tables, page, B * nodes, None, held, free)
    check_plan(cuda, lengths, new, whole["tables"], page, B * nodes, parents)
    check_plan(cuda, lengths, new, whole["tables"], page, B * nodes, [parents[0]] * B, shared=True)


def test_plan_of_a_long_chain_of_parents(cuda):
    check_plan(cuda, [5, 0], [64, 64], [[0, 1], [2, 3]], 64, 130, [list(range(-1, 63))] * 2, shared=True)


def test_plan_cuts_what_does_not_fit(cuda):
    t = [[0, 1, -1, -1], [2, -1, -1, -1], [3, -1, -1, -1]]
    free = [7, 8, 9]
    # more tokens than the table holds; fewer free pages than needed; more rows than there are; none free at all
    check_plan(cuda, [20, 3, 0], [100, 4, 2], t, 16, 200, held=[2, 1, 1], free=free)
    check_plan(cuda, [20, 3, 0], [40, 40, 40], t, 16, 200, held=[2, 1, 1], free=free)
    check_plan(cuda, [20, 3, 0], [40, 40, 40], t, 16, 30, held=[2, 1, 1], free=free * 3)
    check_plan(cuda, [32, 3, 0], [1, 1, 17], t, 16, 30, held=[2, 1, 1], free=free, taken=3)
    # negative numbers; a tree that is smaller than its tokens; parents that do not come before their nodes
    check_plan(cuda, [-4, 3, 0], [2, -1, 5], t, 16, 20, held=[2, 1, 1], free=free)
    check_plan(cuda, [20, 3, 0], [3, 5, 2], t, 16, 20, [[-1, 0, 0]] * 3, held=[2, 1, 1], free=free)
    check_plan(cuda, [1, 3, 0], [4, 4, 4], t, 16, 20, [[-1, 1, 0, 2], [0, -1, 7, 2], [-1, -1, 0, -3]], held=[2, 1, 1], free=free)


def test_plan_marks_positions_without_a_page(cuda):
    check_plan(cuda, [14, 3], [4, 2], [[0, -1], [2, -1]], 16, 8)


def test_plan_without_rows_or_sequences(cuda):
    import sparse_decode as sd
    p = sd.paged_plan(i32(cuda, []), i32(cuda, []), cuda.empty((0, 3), dtype=cuda.int32, device="cuda"), 16, 5)
    assert p.first.tolist() == [0] and p.positions.tolist() == [-1] * 5 and p.seq.tolist() == [-1] * 5
    p = sd.paged_plan(i32(cuda, [4]), i32(cuda, [0]), i32(cuda, [[1]]), 16, 0)
    assert p.first.tolist() == [0, 0] and p.ends.tolist() == [4]


def test_plan_outputs_that_start_between_wide_accesses(cuda):
    """One tree for all read through a strided view is refused; outputs of odd sizes are written to the last row."""
    import sparse_decode as sd
    for n in (1, 2, 3, 5, 7):
        check_plan(cuda, [3], [n], [[0, 1]], 16, n)
    with pytest.raises(ValueError):
        sd.paged_plan(i32(cuda, [3]), i32(cuda, [1]), i32(cuda, [[0]]), 16, 1, parents=i32(cuda, [[-1, 0]] * 2)[:, 0])


# ---------------------------------------------------------------------------
# keep
# ---------------------------------------------------------------------------

def check_keep(torch, sd, arrays, bits, tables, page, ends, counts, paths, want_paths=None, flag=0, lengths=None):
    first = [0]
    for n in counts:
        first.append(first[-1] + n)
    want = [[a.clone() for a in half] for half in arrays]
    for half in want:
        for a in half:
            x = a if a.dim() == 5 else a[None]
            for b, path in enumerate(want_paths if want_paths is not None else paths):
                h = ends[b] - counts[b]
                for i, j in enumerate(path):
                    (tp, ts), (fp, fs) = divmod(h + i, page), divmod(h + j, page)
                    x[:, tables[b][tp], :, ts] = x[:, tables[b][fp], :, fs].clone()
    (k, *ks), (v, *vs) = arrays
    T = max(map(len, paths))
    flags = i32(torch, [0])
    path = torch.tensor([p[:T] + [-9] * (T - len(p)) for p in paths], dtype=torch.int32, device="cuda").view(len(paths), T)
    got = sd.paged_keep(sd.KVPages(k, v, *ks, *vs, bits=bits), i32(torch, tables), i32(torch, ends), i32(torch, first),
                        path, i32(torch, [len(p) for p in paths]), flags=flags)
    assert int(flags) == flag
    done = want_paths if want_paths is not None else paths
    assert got.tolist() == (lengths or [e - n + len(p) for e, n, p in zip(ends, counts, done)])
    for a, b in zip(arrays, want):
        for x, y in zip(a, b):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def random_arrays(torch, seed, dtype, bits, layers, n_pages, hkv, page, d):
    g = gen(torch, seed)
    lead = (layers, n_pages, hkv, page) if layers else (n_pages, hkv, page)
    raw = lambda last, dt: torch.randint(0, 256, (*lead, last * dt.itemsize), generator=g, device="cuda",  # noqa: E731
                                         dtype=torch.uint8).view(dt)
    if bits:
        return [[raw(d * bits // 32, torch.int32), raw(d // 64, tdt(torch, dtype)), raw(d // 64, tdt(torch, dtype))]
                for _ in "kv"]
    return [[raw(d, tdt(torch, dtype))] for _ in "kv"]


@pytest.mark.parametrize("dtype,bits,hkv,d,page,layers", [
    ("bf16", 0, 8, 128, 64, 3), ("f16", 0, 3, 64, 16, 1), ("f32", 0, 2, 128, 32, 0), ("bf16", 8, 8, 128, 128, 2),
    ("f16", 4, 5, 64, 16, 2), ("f32", 8, 1, 64, 256, 0), ("f32", 4, 40, 128, 16, 1), ("bf16", 4, 2, 64, 64, 5)])
def test_keep_moves_the_accepted_rows(cuda, dtype, bits, hkv, d, page, layers):
    import sparse_decode as sd
    rng = random.Random(d + page)
    counts = [1, 64, 17, 5, 33, 2, 64]
    held = [0, page - 3, 100, page, 3 * page - 1, 0, 7]
    paths = [[0], list(range(64)), sorted(rng.sample(range(17), 9)), [], sorted(rng.sample(range(33), 20)), [1],
             sorted(rng.sample(range(64), 40))]
    ends = [h + n for h, n in zip(held, counts)]
    n_pages = sum(-(-e // page) for e in ends) + 2
    tables = tables_of(cuda, ends, page, n_pages, 5).tolist()
    arrays = random_arrays(cuda, 3, dtype, bits, layers, n_pages, hkv, page, d)
    check_keep(cuda, sd, arrays, bits, tables, page, ends, counts, paths)


def test_keep_ends_a_path_that_cannot_be(cuda):
    import sparse_decode as sd
    arrays = random_arrays(cuda, 4, "bf16", 0, 2, 20, 2, 16, 64)
    tables = [[1, 2, 3], [4, 5, 99], [7, -1, 9], [10, 11, 12], [13, 14, 15], [16, 17, 18]]
    ends, counts = [30, 40, 40, 20, 47, 49], [10, 20, 20, 5, 4, 4]
    paths = [[1, 3, 3, 4], [0, 9, 14], [1, 2], [2, 4, 5], [3, 2], [0, 1]]
    # an entry that does not rise; a page past the pool; no page; past the nodes; falling; more tokens than the table,
    # which keeps what the table holds
    done = [[1, 3], [0, 9], [], [2, 4], [3], []]
    want = [22, 22, 20, 17, 44, 48]
    check_keep(cuda, sd, arrays, 0, tables, 16, ends, counts, paths, done, flag=2, lengths=want)


def test_keep_refuses_lengths_that_are_inputs(cuda):
    import sparse_decode as sd
    (k,), (v,) = random_arrays(cuda, 4, "bf16", 0, 1, 4, 2, 16, 64)
    pages, one = sd.KVPages(k, v), i32(cuda, [[0]])
    ends, first, kept = i32(cuda, [4]), i32(cuda, [0, 2]), i32(cuda, [1])
    for bad in (ends, kept, first[:1], first[1:], one[0]):
        with pytest.raises(sd.SDError):
            sd.paged_keep(pages, one, ends, first, one, kept, lengths=bad)
    lengths = i32(cuda, [2])
    assert sd.paged_keep(pages, one, ends, first, one, kept, lengths=lengths) is lengths
    assert lengths.tolist() == [3]


# ---------------------------------------------------------------------------
# tree attention
# ---------------------------------------------------------------------------

def tree64(q, pool, tables, held, lines, scale, window=0, sinks=None):
    """(out, sum p |v| / sum p, (the largest scale sum |q k|, sum |v|)) in fp64; lines: [[(mask, place)] per node] per sequence, rows in order."""
    import torch
    k, v = pool.values
    hkv, D = k.shape[1], k.shape[-1]
    out, size = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    reach = torch.zeros(q.shape[:2] + (1,), dtype=torch.float64, device="cuda")
    values = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    row = 0
    for b, (h, nodes) in enumerate(zip(held, lines)):
        n = len(nodes)
        if not n:
            continue
        at = tables[b, :-(-(h + n) // pool.page)].long()
        kk, vv = (x[at].permute(1, 0, 2, 3).flatten(1, 2)[:, :h + n] for x in (k, v))
        place = torch.tensor(list(range(h)) + [p for _, p in nodes])
        seen = torch.zeros(n, h + n, dtype=torch.bool)
        for i, (m, p) in enumerate(nodes):
            seen[i, :h] = True
            for j in range(n):
                seen[i, h + j] = bool(m >> j & 1)
            if window:
                seen[i] &= place > p - window
        seen = seen.cuda()
        s = torch.einsum("nhgd,htd->hngt", q[row:row + n].double().view(n, hkv, -1, D), kk) * scale
        most = torch.einsum("nhgd,htd->hngt", q[row:row + n].double().abs().view(n, hkv, -1, D), kk.abs()) * abs(scale)
        most = torch.where(seen[None, :, None], most, 0.0).amax(-1).transpose(0, 1).reshape(n, -1, 1)
        reach[row:row + n] = most
        s = torch.where(seen[None, :, None], s, -math.inf)  # also not-a-numbers that are not seen
        if sinks is not None:
            s = torch.cat((s, sinks.double().view(hkv, 1, -1, 1).expand(hkv, n, -1, 1)), -1)
        top = s.amax(-1, keepdim=True).clamp(min=-1e300)
        p = torch.exp(s - top)
        p = (p / p.sum(-1, keepdim=True).clamp(min=1e-300))[..., :h + n]
        vz = torch.where(seen.any(0)[None, :, None], vv, 0.0)
        out[row:row + n] = torch.einsum("hngt,htd->nhgd", p, vz).reshape(n, -1, D)
        values[row:row + n] = (vz.abs().sum(1)[None, :, None].expand(n, hkv, q.shape[1] // hkv, D)).reshape(n, -1, D)
        size[row:row + n] = torch.einsum("hngt,htd->nhgd", p, vz.abs()).reshape(n, -1, D)
        row += n
    return out, size, (reach, values)


def check_tree(torch, out, ref, size, reach, dtype, tile, bits=0):
    assert torch.isfinite(out).all()
    if tile:
        u = torch.finfo(out.dtype).eps / 2
        w = 2.0 ** -11 if bits else u
        off = (out.double() - ref).abs()
        bound = (u * ref.abs() + w * size) * 1.01 + 1e-4 * size + (2.0 ** -24 if dtype == "f16" else 0.0) + 2.0 ** -32 * reach[1]
        if bits:
            bound += size * (2.0 ** -11 + torch.expm1(2 * 2.0 ** -11 * reach[0]))
        assert (off <= bound).all(), f"{int((off > bound).sum())} of {off.numel()} off, worst {float((off / bound).max()):.3g}"
        rel = (off.pow(2).sum() / ref.pow(2).sum().clamp(min=1e-300)).sqrt()
        if not bits:
            assert rel <= u, float(rel)  # the worst case everywhere is more than what adds up in squares
    else:
        live = ref.abs().sum(-1) > 0
        if live.any():
            d = ref.shape[-1]
            assert_close(out[live].double().cpu().numpy().reshape(-1, d), ref[live].cpu().numpy().reshape(-1, d), dtype)
        assert not out[~live].any()
        if dtype != "f32" and out.numel() >= 1000:
            # Nothing but the result's own rounding shows: an error spread evenly over a step of 2 u 2^e is u 2^e / sqrt(3)
            # in the mean square, at most 0.58 u of a value of [2^e, 2^(e+1)). A rounding of as many bits before it, of
            # the weights or of the values, adds as much again in squares and makes it 0.7 u and more where mantissas lie low.
            u = torch.finfo(out.dtype).eps / 2
            assert ((out.double() - ref).pow(2).sum() / ref.pow(2).sum().clamp(min=1e-300)).sqrt() <= 0.65 * u


def uses_tiles(dtype, bits, counts, G):
    return (dtype == "bf16" or dtype == "f16" and not bits) and -(-sum(counts) // len(counts)) * G > (32 if bits == 8 else 16)


def run_tree(torch, dtype, bits, d, hkv, G, page, held, counts, window=0, sinks=False, seed=0, scale=1.0, chain=False,
             absent=0.0, causal=False, tail=0):
    import sparse_decode as sd
    rng = random.Random(seed)
    ends = [h + n for h, n in zip(held, counts)]
    n_pages = sum(-(-t // page) for t in ends) + 3
    pool = Pool(torch, sd, dtype, bits, hkv, d, page, n_pages, seed + 1, scale)
    tables = tables_of(torch, ends, page, n_pages, seed + 2)
    lines, first = [], [0]
    for h, n in zip(held, counts):
        nodes = [((2 << i) - 1, i) for i in range(n)] if causal else lineage(random_parents(rng, n, chain, absent))
        lines.append([(m, h + (x or 0)) for m, x in nodes])
        first.append(first[-1] + n)
    # what no row sees holds not-a-numbers
    keep = torch.zeros(n_pages, page, dtype=torch.bool)
    for b, (h, nodes) in enumerate(zip(held, lines)):
        lo = max(0, min((p for _, p in nodes), default=0) + 1 - window) if window else 0
        for t in range(lo, h if nodes else 0):
            keep[int(tables[b, t // page]), t % page] = True
        for j in range(len(nodes)):
            if any(m >> j & 1 for m, _ in nodes):
                keep[int(tables[b, (h + j) // page]), (h + j) % page] = True
    pool.spoil(keep.cuda())
    N = first[-1] + tail
    q = (2 * torch.randn(N, hkv * G, d, generator=gen(torch, seed + 3), device="cuda")).to(tdt(torch, dtype))
    sk = torch.randn(hkv * G, generator=gen(torch, seed + 4), device="cuda") * 3 if sinks else None
    masks = torch.tensor([signed(m) for x in lines for m, _ in x] + [0] * tail, dtype=torch.int64, device="cuda")
    places = i32(torch, [p for x in lines for _, p in x] + [-1] * tail)
    flags = i32(torch, [0])
    call = lambda: sd.paged_tree_decode(  # noqa: E731
        q, pool.pages, tables, i32(torch, ends), i32(torch, first), None if causal else masks,
        places=None if causal else places, window=window, sinks=sk, flags=flags, out=torch.full_like(q, 7.0))
    out, again = call(), call()
    assert int(flags) == 0
    assert torch.equal(out, again)
    n = first[-1]
    assert (out[n:] == 7.0).all()
    ref, size, reach = tree64(q[:n], pool, tables, held, lines, 1 / math.sqrt(d), window, sk)
    check_tree(torch, out[:n], ref, size, reach, dtype, uses_tiles(dtype, bits, counts, G), bits)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("bits", [0, 4, 8])
@pytest.mark.parametrize("d", [64, 128])
def test_tree_formats(cuda, dtype, bits, d):
    run_tree(cuda, dtype, bits, d, 2, 4, 64, [300, 5, 0, 1000], [4, 2, 3, 1], seed=d + bits)


@pytest.mark.parametrize("dtype,bits", [("f32", 0), ("bf16", 0), ("f16", 0), ("bf16", 8), ("f16", 4), ("f32", 8)])
@pytest.mark.parametrize("G", [1, 3, 5, 8, 16])
def test_tree_head_groups(cuda, dtype, bits, G):
    run_tree(cuda, dtype, bits, 128, 3, G, 32, [70, 259, 31], [7, 1, 13], seed=G)


@pytest.mark.parametrize("dtype,bits", [("f32", 0), ("bf16", 0), ("f16", 0), ("bf16", 8), ("bf16", 4)])
@pytest.mark.parametrize("nodes", [1, 2, 31, 32, 33, 63, 64])
def test_tree_sizes(cuda, dtype, bits, nodes):
    run_tree(cuda, dtype, bits, 64, 2, 4, 64, [513, 64, 0], [nodes, max(1, nodes // 2), nodes], seed=nodes)


@pytest.mark.parametrize("dtype,bits", [("f32", 0), ("bf16", 0), ("f16", 0), ("bf16", 8)])
def test_tree_of_a_chain_and_without_masks(cuda, dtype, bits):
    run_tree(cuda, dtype, bits, 128, 2, 4, 64, [500, 0, 63], [9, 64, 20], chain=True, seed=3)
    run_tree(cuda, dtype, bits, 128, 2, 4, 64, [500, 0, 63], [9, 64, 20], causal=True, seed=4)


@pytest.mark.parametrize("dtype,bits", [("f32", 0), ("bf16", 0), ("f16", 0), ("bf16", 8), ("f16", 4), ("bf16", 4)])
@pytest.mark.parametrize("window", [1, 2, 16, 64, 65, 200])
def test_tree_windows_and_sinks(cuda, dtype, bits, window):
    run_tree(cuda, dtype, bits, 64, 2, 4, 16, [400, 3, 150, 64, 0], [20, 12, 1, 64, 30], window=window,
             sinks=window % 2 == 0, seed=window)


@pytest.mark.parametrize("dtype,bits", [("f32", 0), ("bf16", 0), ("bf16", 8)])
def test_tree_absent_nodes_and_rows_behind_the_last(cuda, dtype, bits):
    run_tree(cuda, dtype, bits, 128, 2, 3, 64, [200, 0, 77], [30, 25, 40], absent=0.2, tail=5, seed=9)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype,bits,d", [("bf16", 0, 128), ("f16", 0, 64), ("bf16", 8, 128), ("f32", 0, 64), ("f16", 4, 64), ("bf16", 4, 128)])
def test_tree_page_sizes(cuda, page, dtype, bits, d):
    run_tree(cuda, dtype, bits, d, 2, 4, page, [page, 3 * page - 1, 700, 1], [16, 5, 33, 9], seed=page)


@pytest.mark.parametrize("dtype,bits", [("bf16", 0), ("f16", 0), ("bf16", 8), ("f32", 0), ("bf16", 4)])
def test_tree_long_split_over_all_ctas(cuda, dtype, bits):
    run_tree(cuda, dtype, bits, 128, 2, 4, 64, [20000, 37], [33, 60], seed=1)
    run_tree(cuda, dtype, bits, 128, 1, 8, 64, [9000], [12], seed=2)


@pytest.mark.parametrize("dtype,bits", [("bf16", 0), ("f16", 4), ("f32", 0), ("bf16", 4)])
def test_tree_many_short_sequences(cuda, dtype, bits):
    rng = random.Random(5)
    run_tree(cuda, dtype, bits, 64, 2, 2, 16, [rng.randint(0, 90) for _ in range(300)], [rng.randint(0, 12) for _ in range(300)], seed=6)


@pytest.mark.parametrize("dtype,bits", [("bf16", 0), ("f16", 0), ("bf16", 8), ("f16", 8), ("bf16", 4)])
@pytest.mark.parametrize("G,d", [(2, 64), (8, 128)])
@pytest.mark.parametrize("window", [0, 100])
def test_tree_many_segments_per_cta(cuda, dtype, bits, G, d, window):
    """Short sequences, some of a single tile, several of them for every CTA."""
    rng = random.Random(8)
    run_tree(cuda, dtype, bits, d, 8, G, 32, [rng.choice([0, 20, 129, rng.randint(0, 700)]) for _ in range(120)],
             [rng.randint(10, 40) for _ in range(120)], window=window, seed=9)


@pytest.mark.parametrize("dtype,bits", [("bf16", 0), ("f16", 0), ("bf16", 8), ("f16", 4), ("bf16", 4)])
@pytest.mark.parametrize("scale", [1e-3, 30.0])
def test_tree_small_and_large_values(cuda, dtype, bits, scale):
    run_tree(cuda, dtype, bits, 128, 2, 4, 64, [700, 90], [33, 20], scale=scale, seed=7)
    run_tree(cuda, dtype, bits, 64, 2, 16, 64, [700, 90], [33, 20], scale=scale, seed=8)


@pytest.mark.parametrize("n", [9, 40])
@pytest.mark.parametrize("bits", [4, 8])
def test_tree_code_tiles_of_very_different_size(cuda, bits, n):
    """Scales of K and V that change from page to page by up to 2^60 (down, up, zero), so that the powers of tiles and of O
    move; queries of rows that differ as much."""
    import sparse_decode as sd
    torch = cuda
    hkv, G, d, page, held = 2, 4, 64, 64, 640
    pool = Pool(torch, sd, "bf16", bits, hkv, d, page, 14, 5)
    tables = tables_of(torch, [held + n], page, 14, 6)
    ups = [0, -20, 3, 40, -40, 8, 9, 0, -8, 16, 0]
    for j, u in enumerate(ups):
        pg = int(tables[0, j])
        for a, sign in zip(pool.arrays, (-1, 1)):  # keys and values in opposite order
            f = 2.0 ** (u * sign if sign > 0 else min(u * sign, 2)) if j != 7 else 0.0
            for x in a[1:]:
                x[pg] *= f
    for a, values in zip(pool.arrays, range(2)):
        grow = lambda t: t.double().repeat_interleave(64, -1)  # noqa: E731
        words = (a[0].long() & 0xFFFFFFFF)[..., None] >> (torch.arange(32 // bits, device="cuda") * bits)
        pool.values[values] = (words & ((1 << bits) - 1)).flatten(-2).double() * grow(a[1]) + grow(a[2])
    q = torch.randn(n, hkv * G, d, generator=gen(torch, 8), device="cuda")
    q = (q * torch.exp2(torch.arange(n, device="cuda") % 5 * -20.0)[:, None, None]).bfloat16()
    out = sd.paged_tree_decode(q, pool.pages, tables, i32(torch, [held + n]), i32(torch, [0, n]))
    lines = [[((2 << i) - 1, held + i) for i in range(n)]]
    ref, size, reach = tree64(q, pool, tables, [held], lines, 1 / math.sqrt(d))
    check_tree(torch, out, ref, size, reach, "bf16", True, bits)


def test_tree_hidden_nodes_do_not_reach_their_siblings(cuda):
    """Two branches from one root: infinities and not-a-numbers in one branch's keys and values leave the other alone."""
    import sparse_decode as sd
    torch = cuda
    for dtype, bits in (("f32", 0), ("f16", 0), ("bf16", 8), ("f16", 4), ("f32", 8), ("bf16", 4), ("bf16", 0)):
        pool = Pool(torch, sd, dtype, bits, 2, 64, 16, 8, 3)
        tables, held = i32(torch, [[1, 4, 6, 2]]), 37
        parents = [-1, 0, 0, 1, 2, 3]
        masks = torch.tensor([m for m, _ in lineage(parents)], dtype=torch.int64, device="cuda")
        q = torch.randn(6, 8, 64, generator=gen(torch, 4), device="cuda").to(tdt(torch, dtype))
        call = lambda: sd.paged_tree_decode(q, pool.pages, tables, i32(torch, [43]), i32(torch, [0, 6]), masks)  # noqa: E731
        clean = call()
        for a, x in zip(pool.arrays, (float("nan"), float("inf"))):
            for node in (2, 4):
                t = held + node
                a[-1][int(tables[0, t // 16]), :, t % 16, 0 if bits else 5] = x  # a value, or a group's bias
        out = call()
        for node in (0, 1, 3, 5):
            assert torch.equal(out[node], clean[node])
        assert not torch.isfinite(out[2]).any() and not torch.isfinite(out[4]).any()


@pytest.mark.parametrize("dtype,bits", [("bf16", 0), ("f16", 0), ("bf16", 4), ("bf16", 8), ("f16", 8), ("f32", 0), ("f32", 4)])
@pytest.mark.parametrize("G", [2, 8])
def test_tree_infinite_values_count_where_they_are_seen(cuda, dtype, bits, G):
    """Keys are finite, one value (of codes: a group of 64) of node 2 is not: rows that see the node have it, all else is as before."""
    import sparse_decode as sd
    torch = cuda
    pool = Pool(torch, sd, dtype, bits, 2, 128, 16, 8, 3)
    tables, held, parents = i32(torch, [[1, 4, 6, 2]]), 37, [-1, 0, 0, 1, 2, 3]
    masks = torch.tensor([m for m, _ in lineage(parents)], dtype=torch.int64, device="cuda")
    q = torch.randn(6, 2 * G, 128, generator=gen(torch, 4), device="cuda").to(tdt(torch, dtype))
    call = lambda: sd.paged_tree_decode(q, pool.pages, tables, i32(torch, [43]), i32(torch, [0, 6]), masks).double()  # noqa: E731
    clean = call()
    at = (int(tables[0, (held + 2) // 16]), slice(None), (held + 2) % 16)
    for x in (math.inf, -math.inf, math.nan):
        pool.arrays[1][-1][at + (1 if bits else 100,)] = x
        out = call()
        hit = slice(64, 128) if bits else slice(100, 101)
        for node in range(6):
            if node in (2, 4):
                assert torch.isnan(out[node, :, hit]).all() if x != x else (out[node, :, hit] == x).all()
                out[node, :, hit] = clean[node, :, hit]
        # the power that a tile of codes takes may be another one: fp16 values of half the bits at most, of small ones
        tol = 2.0 ** -9 if dtype == "bf16" else 2.0 ** -12
        assert torch.isfinite(out).all() and ((out - clean).abs() <= 4 * tol * clean.abs().amax()).all()
        if not bits:
            assert torch.equal(out, clean)


def test_tree_reports_sequences_that_cannot_be(cuda):
    import sparse_decode as sd
    torch = cuda
    pool = Pool(torch, sd, "bf16", 0, 2, 64, 16, 40, 3)
    good = tables_of(torch, [40, 40, 40, 40], 16, 40, 4)
    q = torch.randn(200, 8, 64, generator=gen(torch, 4), device="cuda").bfloat16()
    flags = i32(torch, [0])

    def call(tables, lengths, first):
        flags.zero_()
        out = sd.paged_tree_decode(q, pool.pages, tables, i32(torch, lengths), i32(torch, first), flags=flags,
                                   out=torch.full_like(q, 7.0))
        return out, int(flags)
    want, f = call(good, [40, 40, 40, 40], [0, 6, 12, 18, 24])
    assert f == 0 and (want[24:] == 7).all()
    # fewer tokens than nodes, more tokens than the table, more nodes than a mask has bits, rows outside the call
    for lengths, first in (([40, 5, 40, 40], [0, 6, 12, 18, 24]), ([40, 49, 40, 40], [0, 6, 12, 18, 24]),
                           ([40, -3, 40, 40], [0, 6, 12, 18, 24])):
        out, f = call(good, lengths, first)
        assert f == 2 and not out[6:12].any() and torch.equal(out[:6], want[:6]) and torch.equal(out[12:], want[12:])
    out, f = call(good, [40, 47, 40, 40], [0, 6, 77, 78, 84])
    assert f == 2 and not out[6:77].any() and torch.equal(out[:6], want[:6]) and (out[84:] == 7).all()
    out, f = call(good, [40, 40, 40, 40], [0, 6, 12, 18, 300])
    assert f == 2 and not out[18:].any() and torch.equal(out[:18], want[:18])
    # pages out of range read as zeros
    bad = good.clone()
    bad[1, 1], bad[2, 2] = 99, -1
    out, f = call(bad, [40, 40, 40, 40], [0, 6, 12, 18, 24])
    assert f == 2 and torch.isfinite(out).all()
    assert torch.equal(out[:6], want[:6]) and torch.equal(out[18:], want[18:])


# ---------------------------------------------------------------------------
# rounds
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,bits", [("bf16", 0), ("f16", 8), ("f32", 0)])
def test_a_captured_round_serves_growing_sequences(cuda, dtype, bits):
    """plan + append + attend + keep in one CUDA graph: lengths, pages and what is kept advance on the device."""
    import sparse_decode as sd
    torch = cuda
    B, hkv, G, d, page, nodes, W = 3, 2, 4, 64, 16, 7, 12
    n_pages = B * W
    pool = Pool(torch, sd, dtype, bits, hkv, d, page, n_pages, 3)
    lengths = i32(torch, [5, 31, 60])
    held, taken = i32(torch, [1, 2, 4]), i32(torch, [0])
    order = torch.randperm(n_pages, generator=gen(torch, 4), device="cuda").to(torch.int32)
    tables = torch.full((B, W), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, h in enumerate([1, 2, 4]):
        tables[b, :h] = order[at:at + h]
        at += h
    free = order[at:].clone()
    parents = i32(torch, [-1, 0, 0, 1, 2, 2, 4])
    new, path, kept = i32(torch, [7, 5, 6]), i32(torch, [[0, 2, 4, 6]] * B), i32(torch, [4, 3, 1])
    x = torch.randn(B * nodes, (G + 2) * hkv, d, generator=gen(torch, 5), device="cuda").to(tdt(torch, dtype))
    q, k, v = x[:, :G * hkv].contiguous(), x[:, G * hkv:(G + 1) * hkv], x[:, (G + 1) * hkv:]
    flags = i32(torch, [0])
    inv = (10000.0 ** (-torch.arange(0, d, 2, device="cuda") / d)).float()

    def step():
        p = sd.paged_plan(lengths, new, tables, page, B * nodes, parents=parents, held=held, free=free, taken=taken, flags=flags)
        q2, k2 = sd.rotary(q, k, p.places, inv)
        sd.paged_append(pool.pages, k2, v, tables, p.positions, seq=p.seq, flags=flags)
        out = sd.paged_tree_decode(q2, pool.pages, tables, p.ends, p.first, p.masks, places=p.places, flags=flags)
        sd.paged_keep(pool.pages, tables, p.ends, p.first, path, kept, lengths=lengths, flags=flags)
        return p, q2, out
    saved = [t.clone() for t in (lengths, tables, held, taken)]
    step()
    for t, old in zip((lengths, tables, held, taken), saved):
        t.copy_(old)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p, q2, out = step()
    now = [5, 31, 60]
    lines = [lineage([-1, 0, 0, 1, 2, 2, 4][:n]) for n in (7, 5, 6)]
    for rnd in range(4):
        x.copy_(torch.randn(x.shape, generator=gen(torch, 10 + rnd), device="cuda"))
        q.copy_(x[:, :G * hkv])
        before = [stored(torch, pool, tables, b, n) for b, n in enumerate(now)]
        g.replay()
        torch.cuda.synchronize()
        assert int(flags) == 0
        assert p.first.tolist() == [0, 7, 12, 18] and p.positions.tolist()[18:] == [-1] * 3
        assert p.ends.tolist() == [t + n for t, n in zip(now, (7, 5, 6))]
        now = [t + n for t, n in zip(now, (4, 3, 1))]
        assert lengths.tolist() == now
        for b, n in enumerate(now):
            after = stored(torch, pool, tables, b, n)
            for x0, x1 in zip(before[b], after):
                assert torch.equal(x0, x1[:, :x0.shape[1]])
        # the round's attention, from the tokens before it and the drafted ones that were stored
        row = 0
        for b, n in enumerate((7, 5, 6)):
            h = now[b] - (4, 3, 1)[b]
            keys, vals = (t[:, :h] for t in stored(torch, pool, tables, b, now[b]))
            for i in range(n):
                seen = [j for j in range(n) if lines[b][i][0] >> j & 1]
                if any(j not in (0, 2, 4, 6)[:(4, 3, 1)[b]] for j in seen):
                    continue  # a node that was dropped is overwritten by now
                new_at = [(0, 2, 4, 6).index(j) for j in seen]
                both = [torch.cat((t, s[:, [h + j for j in new_at]]), 1) for t, s in
                        zip((keys, vals), stored(torch, pool, tables, b, now[b]))]
                s = torch.einsum("hgd,htd->hgt", q2[row + i].double().view(hkv, G, d), both[0]) / math.sqrt(d)
                ref = torch.einsum("hgt,htd->hgd", torch.softmax(s, -1), both[1]).reshape(-1, d)
                tol = {"bf16": 2e-2, "f16": 3e-3, "f32": 2e-5}[dtype]
                assert float((out[row + i].double() - ref).norm() / ref.norm()) < tol
            row += n


def stored(torch, pool, tables, b, n):
    """Keys and values of a sequence's first n tokens, [Hkv, n, D] in fp64, from the pool's arrays as they are now."""
    at = tables[b, :-(-n // pool.page)].long()
    got = []
    for a in pool.arrays:
        if pool.bits:
            w = a[0][at].long() & 0xFFFFFFFF
            c = torch.stack([(w >> (pool.bits * j)) & ((1 << pool.bits) - 1) for j in range(32 // pool.bits)], -1).flatten(-2)
            x = c.double() * a[1][at].double().repeat_interleave(64, -1) + a[2][at].double().repeat_interleave(64, -1)
        else:
            x = a[0][at].double()
        got.append(x.permute(1, 0, 2, 3).flatten(1, 2)[:, :n])
    return got


@pytest.mark.parametrize("bits", [0, 8])
def test_pool_keeps_the_accepted_tokens(cuda, bits):
    """Tree steps through the router: outputs against single steps of the accepted path, and the pool afterwards."""
    import sparse_decode as sd
    from sparse_decode import attention_with_cache_update
    torch = cuda
    hq, hkv, d, page, layers = 8, 2, 64, 16, 2
    inv, factor = sd.rotary_frequencies(d, 1e4)
    turn = dict(inv_freq=inv, factor=factor)
    g = gen(torch, 1)
    rand = lambda n, h, m: torch.randn(n, h, m, d, generator=g, device="cuda").bfloat16()  # noqa: E731
    pools = [sd.PagePool(layers, 60, hkv, d, page, "bf16", bits) for _ in range(2)]
    seqs = [[p.add(), p.add()] for p in pools]
    prompt = [(rand(1, hq, n), rand(1, hkv, n), rand(1, hkv, n)) for n in (300, 29)]
    for p, ss in zip(pools, seqs):
        for s, (q, k, v) in zip(ss, prompt):
            step = p.extend([s], q.shape[2])
            assert step.positions.tolist() == list(range(q.shape[2]))
            for i in range(layers):
                attention_with_cache_update(q, k, v, step.layer(i, **turn), d ** -0.5, "causal")
    parents, paths = [-1, 0, 0, 1, 2, 4], [[0, 2, 4, 5], [0, 1]]
    q, k, v = (rand(2, h, 6) for h in (hq, hkv, hkv))
    step = pools[0].extend(seqs[0], 6).tree(parents)
    got = [attention_with_cache_update(q, k, v, step.layer(i, window=40 * i, **turn), d ** -0.5) for i in range(layers)]
    step.keep(paths)
    assert [pools[0].length(s) for s in seqs[0]] == [304, 31]
    for b, path in enumerate(paths):
        for node in path:
            one = pools[1].extend([seqs[1][b]], 1)
            for i in range(layers):
                ref = attention_with_cache_update(*(x[b:b + 1, :, node:node + 1] for x in (q, k, v)),
                                                  one.layer(i, window=40 * i, **turn), d ** -0.5)
                a, c = got[i][b, :, node].double(), ref[0, :, 0].double()
                # two roundings of the output and one of the weights
                assert float((a - c).abs().max()) <= 3 * 2.0 ** -8 * float(c.abs().max())
    for p in pools:
        assert p.check_device() == 0
    for b in range(2):
        views = [p.batch([ss[b]]).layer(1).dense(0) for p, ss in zip(pools, seqs)]
        for x, y in zip(*views):
            assert torch.equal(x, y)


def test_pool_refuses_what_a_tree_cannot_be(cuda):
    import sparse_decode as sd
    pool = sd.PagePool(1, 20, 2, 64, 16)
    a, b = pool.add(), pool.add()
    step = pool.extend([a, b], [3, 2])
    for bad in ([0, 0, 1], [[-1, 0, 0], [-1]], [[-1, 0, 2], [-1, 0]], [-1, 0]):
        with pytest.raises(ValueError):
            step.tree(bad)
    with pytest.raises(ValueError):
        step.keep([[0], [0]])
    with pytest.raises(ValueError):
        step.attend_tree(0, cuda.zeros(5, 4, 64, device="cuda").bfloat16())
    step.tree([[-1, -1, 1], [-1, 0]])
    assert step.plan.masks.tolist() == [1, 2, 6, 1, 3] and step.plan.places.tolist() == [0, 0, 1, 0, 1]
    for bad in ([[0]], [[0], [2]], [[1, 0], [0]], [[0, 0], []], [[-1], []]):
        with pytest.raises(ValueError):
            step.keep(bad)
    with pytest.raises(ValueError):
        sd.PagedLayer(step, 0, {}).attend(cuda.zeros(2, 4, 3, 64, device="cuda"), None, None, 1.0)  # ragged new tokens
    c = pool.fork(a)
    with pytest.raises(ValueError, match="forked"):
        step.keep([[0], [0]])
    pool.free(c)
    step = pool.extend([b], 65)
    with pytest.raises(ValueError):
        step.tree()
    pool.trim(b, 65)
    step = pool.extend([b], 2).tree()
    assert step.plan.masks.tolist() == [1, 3]
    q = cuda.zeros(1, 4, 2, 64, device="cuda").bfloat16()
    with pytest.raises(ValueError, match="mask"):
        step.layer(0).attend(q, q[:, :2], q[:, :2], 1.0, mask=cuda.ones(2, 4, dtype=cuda.bool, device="cuda"))
    step.layer(0).attend(q, q[:, :2], q[:, :2], 1.0, mask="causal")
    step.keep([[]])
    assert pool.length(b) == 2 and pool.check_device() == 0


def test_pool_refuses_stale_steps(cuda):
    """Pages that a step's tables name may belong to others once its sequences were trimmed, freed or moved."""
    import sparse_decode as sd
    pool = sd.PagePool(1, 20, 2, 64, 16)
    a, b = pool.add(), pool.add()
    step = pool.extend([a], 20).tree()
    pool.trim(a, 20)
    pool.extend([b], 5)
    pool.extend([a], 20)  # the length that it had
    with pytest.raises(ValueError, match="since"):
        step.keep([[0]])
    step = pool.extend([a], 3).tree()
    pool.free(b)
    assert pool.compact()
    with pytest.raises(ValueError, match="since"):
        step.keep([[0]])
    with pytest.raises(ValueError, match="since"):
        step.tree()
    step = pool.extend([a], 3).tree()
    step.keep([[0, 1]])
    with pytest.raises(ValueError, match="since"):
        step.tree()
    step = pool.extend([a], 3).tree()
    pool.free(a)
    with pytest.raises(ValueError, match="since"):
        step.keep([[0]])
    assert pool.free_pages == 20 and pool.check_device() == 0


def test_a_plan_on_the_device_gives_the_positions_of_the_host(cuda):
    import sparse_decode as sd
    from sparse_decode import paged
    pool = sd.PagePool(1, 200, 1, 64, 16)
    seqs = [pool.add() for _ in range(3)]
    pool.extend(seqs, [5, 0, 40])
    step = pool.extend(seqs, [400, 1, 0])
    assert sum(step.new) >= paged._PLAN_TOKENS
    assert step.positions.tolist() == [*range(5, 405), 0] and step.seq.tolist() == [0] * 400 + [1]
    assert step.lengths.tolist() == [405, 1, 40]


@pytest.mark.parametrize("bits", [0, 8])
def test_example_drafts(cuda, bits):
    from sparse_decode import paged_example
    pool, seqs, outs, worst = paged_example.run(layers=2, kv_bits=bits, steps=3, drafts=4, check=True)
    # prompts of 70, steps, drafts that keep three and three, or three and one, and steps again
    assert [pool.length(s) for s in seqs] == [70 + 3 + 4 * 3 + 3, 70 + 3 + 2 * (3 + 1) + 3]
    assert worst < 5e-3


# ---------------------------------------------------------------------------
# limits and refusals
# ---------------------------------------------------------------------------

def test_calls_on_two_streams_share_nothing(cuda):
    import sparse_decode as sd
    torch = cuda
    rng = random.Random(3)
    cases = []
    for i, (dtype, bits, counts) in enumerate([("bf16", 0, [30, 9, 64]), ("bf16", 8, [4, 3, 1]), ("f16", 0, [64, 64, 64])]):
        held = [2000, 31, 600]
        ends = [h + n for h, n in zip(held, counts)]
        pool = Pool(torch, sd, dtype, bits, 2, 128, 64, 60, 50 + i)
        tables = tables_of(torch, ends, 64, 60, 52 + i)
        first = [0, counts[0], counts[0] + counts[1], sum(counts)]
        masks = [signed(m) for n in counts for m, _ in lineage(random_parents(rng, n))]
        q = torch.randn(sum(counts), 8, 128, generator=gen(torch, 54 + i), device="cuda").to(tdt(torch, dtype))
        args = (q, pool.pages, tables, i32(torch, ends), i32(torch, first), torch.tensor(masks, device="cuda"))
        cases.append((args, sd.paged_tree_decode(*args), pool))
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in cases], [[] for _ in cases]
    for _ in range(6):
        for i, (args, _, _) in enumerate(cases):
            outs[i].append(sd.paged_tree_decode(*args, stream=streams[i]))
    torch.cuda.synchronize()
    for i, (_, want, _) in enumerate(cases):
        assert all(torch.equal(o, want) for o in outs[i])


def test_tree_offsets_past_32_bits(cuda):
    """A pool of 9 GB: the last pages' rows lie past 2^32 bytes."""
    import sparse_decode as sd
    torch = cuda
    n_pages, hkv, page, d = 70000, 4, 64, 128
    k, v = (torch.zeros(n_pages, hkv, page, d, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    pages = sd.KVPages(k, v)
    for counts, G in (([3], 4), ([40], 4)):
        n = counts[0]
        held = 100
        tables = i32(torch, [[n_pages - 1, n_pages - 3, n_pages - 7]])
        rows = torch.randn(held + n, hkv, 2 * d, generator=gen(torch, 3), device="cuda").bfloat16()
        pos = torch.arange(held + n, device="cuda", dtype=torch.int32)
        sd.paged_append(pages, rows[..., :d], rows[..., d:], tables, pos, seq=torch.zeros_like(pos))
        q = torch.randn(n, hkv * G, d, generator=gen(torch, 4), device="cuda").bfloat16()
        out = sd.paged_tree_decode(q, pages, tables, i32(torch, [held + n]), i32(torch, [0, n]))
        kk, vv = (x.double().transpose(0, 1) for x in (rows[..., :d], rows[..., d:]))
        s = torch.einsum("nhgd,htd->hngt", q.double().view(n, hkv, G, d), kk) / math.sqrt(d)
        s = s.masked_fill(pos[None, None, None] > (held + torch.arange(n, device="cuda"))[None, :, None, None], -math.inf)
        ref = torch.einsum("hngt,htd->nhgd", torch.softmax(s, -1), vv).reshape(n, -1, d)
        assert float((out.double() - ref).norm() / ref.norm()) < 2.0 ** -8
        kept = i32(torch, [2])
        got = sd.paged_keep(pages, tables, i32(torch, [held + n]), i32(torch, [0, n]), i32(torch, [[0, n - 1]]), kept)
        assert got.tolist() == [held + 2]
        t = held + 1
        assert torch.equal(k[int(tables[0, t // page]), :, t % page], rows[held + n - 1, :, :d])


@pytest.mark.parametrize("dtype,bits,G", [("bf16", 0, 16), ("bf16", 8, 16), ("f32", 0, 4)])
def test_tree_largest_batch(cuda, dtype, bits, G):
    rng = random.Random(7)
    run_tree(cuda, dtype, bits, 64, 1, G, 16, [rng.randint(0, 20) for _ in range(4096)], [rng.choice([0, 1, 3]) for _ in range(4096)], seed=5)


def test_tree_scales_of_either_sign_and_none(cuda):
    """Negative and zero scales reach both kernels."""
    import sparse_decode as sd
    torch = cuda
    for n in (2, 20):
        pool = Pool(torch, sd, "bf16", 0, 2, 64, 16, 30, 3)
        tables = tables_of(torch, [300 + n], 16, 30, 4)
        q = torch.randn(n, 8, 64, generator=gen(torch, 4), device="cuda").bfloat16()
        for scale in (-0.2, 0.0):
            out = sd.paged_tree_decode(q, pool.pages, tables, i32(torch, [300 + n]), i32(torch, [0, n]), None, scale)
            lines = [[((2 << i) - 1, 300 + i) for i in range(n)]]
            ref, size, reach = tree64(q, pool, tables, [300], lines, scale)
            check_tree(torch, out, ref, size, reach, "bf16", n * 4 > 16)


def test_python_refusals(cuda):
    import sparse_decode as sd
    torch = cuda
    pool = Pool(torch, sd, "bf16", 0, 2, 64, 16, 8, 3)
    q, t = torch.zeros(4, 8, 64, device="cuda").bfloat16(), i32(torch, [[0, 1]])
    ends, first = i32(torch, [20]), i32(torch, [0, 4])
    masks = torch.ones(4, dtype=torch.int64, device="cuda")
    tree = sd.paged_tree_decode
    tree(q, pool.pages, t, ends, first, masks)
    for args in ((q.float(), pool.pages, t, ends, first), (q.cpu(), pool.pages, t, ends, first), (q[..., :32], pool.pages, t, ends, first),
                 (q.transpose(0, 1), pool.pages, t, ends, first), (q, pool.pages, t.long(), ends, first),
                 (q, pool.pages, t, ends, first[:1]), (q, pool.pages, t, first, first), (q, pool.pages, t, ends, first, masks[:3]),
                 (q, pool.pages, t, ends, first, masks.int())):
        with pytest.raises((TypeError, ValueError)):
            tree(*args)
    for kw in (dict(window=-1), dict(layer=1), dict(scale=float("nan"))):
        with pytest.raises(sd.SDError):
            tree(q, pool.pages, t, ends, first, masks, **kw)
    for kw in (dict(places=ends), dict(sinks=torch.zeros(7, device="cuda")), dict(out=q.float()), dict(window=1 << 31)):
        with pytest.raises((TypeError, ValueError)):
            tree(q, pool.pages, t, ends, first, masks, **kw)
    with pytest.raises(sd.SDError):  # 17 query heads per kv head
        tree(torch.zeros(1, 34, 64, device="cuda").bfloat16(), pool.pages, t, ends, i32(torch, [0, 1]))
    plan = sd.paged_plan
    for args, kw in (((ends, ends, t[0], 16, 4), {}), ((ends, ends, t, 16, 1 << 31), {}), ((ends, first, t, 16, 4), {}),
                     ((ends, ends, t, 16, -1), {}), ((ends, ends, t, 16, 4), dict(held=ends)),
                     ((ends, ends, t, 16, 4), dict(parents=t[None])), ((ends.cpu(), ends, t, 16, 4), {}),
                     ((ends, ends, t.long(), 16, 4), {})):
        with pytest.raises((TypeError, ValueError)):
            plan(*args, **kw)
    for page, kw in ((48, {}), (16, dict(parents=i32(torch, [-1] * 65)))):
        with pytest.raises(sd.SDError):
            plan(ends, ends, t, page, 4, **kw)
    with pytest.raises(ValueError):
        sd.paged_keep(pool.pages, t, ends, first, ends, ends)
    with pytest.raises(sd.SDError):
        sd.paged_keep(pool.pages, t, ends, first, i32(torch, [[0] * 65]), ends)

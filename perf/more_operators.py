"""Workloads of drafted tokens over the paged cache, in plain torch and through sparse_decode.

Three operators, a round of speculative decoding:

* plan:  where the new tokens of many sequences go -- pages taken from a list of free ones, sequence, position, slot and
         (for a tree of drafted tokens) rotary position and mask of ancestors -- from the lengths, on the GPU;
* tree:  attention of every drafted token over its sequence's cached tokens and its own ancestors in the tree;
* keep:  the rows of the accepted tokens moved to the places where they stay, in every layer;

and `round`: plan, store, attend and keep one after the other. `run` computes a case with elementary torch operations in
32 bits, or (own = True) with the library's kernels; `exact` computes it in 64 bits from the definition.

Pages are [n_pages, kv_heads, page_size, head_dim] (4/8-bit pools: uint32-packed affine codes in groups of 64 with
scales and biases in the pool's type); a sequence's tokens lie in the pages that its row of the table names. The new
tokens of a step are rows of packed arrays, sequence by sequence: those of sequence b are rows first[b] .. first[b + 1],
and its node i is the i-th of them. Node i's parent comes before it, or is -1: the last token of the cached ones.
"""
import math
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
NODES = 64  # most nodes of a tree: the bits of a mask


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # the next token of one user: latency only
        dict(name="plan_1_user", op="plan", seqs=1, new=1, ragged=0, ctx=4096, page=64, tree=False, grow=False),
        # 64 users' trees of 32 drafted tokens, pages taken from the free list as they are needed
        dict(name="plan_64_trees", op="plan", seqs=64, new=32, ragged=3, ctx=8192, page=64, tree=True, grow=True),
        # 512 prompts of up to 2000 tokens arrive at once, small pages
        dict(name="plan_512_prompts", op="plan", seqs=512, new=2000, ragged=4, ctx=500, page=16, tree=False, grow=True),
        # the smallest tree: seven drafted tokens of one user, short context, fp32, latency only
        dict(name="tree_f32_2K", op="tree", seqs=1, ctx=2048, ragged=0, nodes=7, chain=False, page=64, q_heads=8,
             kv_heads=2, dim=64, dtype="f32", bits=0, window=0, sinks=False),
        # one user, 32K tokens, a tree of 32 nodes
        dict(name="tree_bf16_32K", op="tree", seqs=1, ctx=32768, ragged=0, nodes=32, chain=False, page=64, q_heads=32,
             kv_heads=8, dim=128, dtype="bf16", bits=0, window=0, sinks=False),
        # a serving batch in an 8-bit cache, four drafted tokens one after the other for each of 16 users
        dict(name="tree_q8_16_chains", op="tree", seqs=16, ctx=8192, ragged=5, nodes=4, chain=True, page=64, q_heads=32,
             kv_heads=8, dim=128, dtype="bf16", bits=8, window=0, sinks=False),
        # a sliding-window layer with attention sinks, small heads, ragged trees of up to 21 nodes
        dict(name="tree_f16_window", op="tree", seqs=12, ctx=16384, ragged=6, nodes=21, chain=False, page=32,
             q_heads=64, kv_heads=8, dim=64, dtype="f16", bits=0, window=1000, sinks=True),
        # four long conversations in a 4-bit cache, trees of 16
        dict(name="tree_q4_4x32K", op="tree", seqs=4, ctx=32768, ragged=0, nodes=16, chain=False, page=128, q_heads=32,
             kv_heads=8, dim=128, dtype="bf16", bits=4, window=0, sinks=False),
        # the largest trees over four long conversations
        dict(name="tree_bf16_4x32K", op="tree", seqs=4, ctx=32768, ragged=0, nodes=64, chain=False, page=64, q_heads=32,
             kv_heads=8, dim=128, dtype="bf16", bits=0, window=0, sinks=False),
        # five of 16 drafted tokens of one user are accepted
        dict(name="keep_1_user", op="keep", seqs=1, ctx=1000, ragged=0, nodes=16, layers=36, page=64, kv_heads=8,
             dim=128, dtype="bf16", bits=0),
        # up to 32 drafted tokens of each of 64 users in an 8-bit cache
        dict(name="keep_q8_64_users", op="keep", seqs=64, ctx=200, ragged=8, nodes=32, layers=36, page=64, kv_heads=8,
             dim=128, dtype="bf16", bits=8),
        # a whole round of 16 users in one layer: plan, store, attend, keep
        dict(name="round_16_users", op="round", seqs=16, ctx=4096, ragged=7, nodes=16, chain=False, page=64, q_heads=32,
             kv_heads=8, dim=128, dtype="bf16", bits=0, window=0, sinks=False, layers=1),
    ]


def _log(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(hi, max(lo, n))


def draw(rng):
    op = rng.choice(["plan", "tree", "tree", "tree", "tree", "keep", "round"])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        tree = rng.random() < 0.5
        seqs = _log(rng, 1, 512)
        return dict(op=op, seqs=seqs, new=_log(rng, 1, NODES if tree else min(2000, 500000 // seqs)),
                    ragged=rng.choice([0, rng.randrange(1, 100)]), ctx=_log(rng, 1, 4000), page=page, tree=tree,
                    grow=rng.random() < 0.7)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    dim = rng.choice([64, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8])
    seqs = _log(rng, 1, 48)
    c = dict(op=op, seqs=seqs, ragged=rng.choice([0, rng.randrange(1, 100)]), nodes=_log(rng, 1, NODES), page=page,
             kv_heads=kv_heads, dim=dim, dtype=dtype, bits=rng.choice([0, 0, 4, 8]))
    if op == "keep":
        layers = rng.choice([1, 2, 7, 24])
        c.update(layers=layers, ctx=_log(rng, 1, max(1, min(2000, (1 << 20) // (seqs * layers * kv_heads)))))
        return c
    group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])
    rows = c["nodes"] * group
    # what the plain form keeps of the scores, and the pool, stay below the largest listed case's
    most = min(32768, (1 << 20) // (seqs * kv_heads), (1 << 28) // (seqs * kv_heads * rows))
    c.update(q_heads=kv_heads * group, ctx=_log(rng, 1, max(1, most)), chain=rng.random() < 0.3,
             window=rng.choice([0, 0, _log(rng, 1, 4096)]), sinks=rng.random() < 0.3)
    if op == "round":
        c.update(bits=0, layers=1)
    return c


def _counts(case):
    """(tokens held, new tokens) of each sequence, by the case alone. Ragged batches spread over [0, ctx] and
    [1, nodes], with one at both ends; from four sequences on one has an empty cache, and one of a plan nothing new."""
    n, ctx, new = case["seqs"], case["ctx"], case.get("nodes", case.get("new"))
    if not case["ragged"]:
        return [ctx] * n, [new] * n
    r = random.Random(case["ragged"])
    held, more = [r.randint(1, ctx) for _ in range(n)], [r.randint(1, new) for _ in range(n)]
    held[0], more[0] = ctx, new
    if n >= 4:
        held[2] = 0
        if case["op"] == "plan":
            more[1] = 0
    return held, more


def _paths(case):
    """The accepted nodes of each sequence: a root first, then some after it."""
    r = random.Random(case["ragged"] * 1000 + case["nodes"])
    paths = []
    for n in _counts(case)[1]:
        most = min(n, max(1, round(n ** 0.6)))
        k = most if case["ragged"] == 0 else r.randint(0, most)
        paths.append([0, *sorted(r.sample(range(1, n), k - 1))] if k else [])
    return paths


def _row_bytes(case):
    d, e = case["dim"], BYTES[case["dtype"]]
    return d * case["bits"] // 8 + 2 * (d // 64) * e if case["bits"] else d * e


def work(case):
    held, new = _counts(case)
    if case["op"] == "plan":
        rows = case["seqs"] * case["new"]
        # lengths, new tokens, table rows of the new tokens; sequence, position, slot of each (and place and mask)
        return {"bytes": 16 * case["seqs"] + rows * (28 if case["tree"] else 16) + 8 * sum(new) / case["page"],
                "flops": 0}
    hkv = case["kv_heads"]
    moved = sum(j != i for path in _paths(case) for i, j in enumerate(path)) if case["op"] != "tree" else 0
    keep = {"bytes": 16 * case["seqs"] + 4 * moved * hkv * case.get("layers", 1) * _row_bytes(case), "flops": 0}
    if case["op"] == "keep":
        return keep
    d, hq, w = case["dim"], case["q_heads"], case["window"]
    seen = sum((min(h, w) if w else h) + n for h, n in zip(held, new))
    pairs = sum(n * (min(h, w) if w else h) + n * (n + 1) // 2 for h, n in zip(held, new))
    b = 2 * seen * hkv * _row_bytes(case) + 2 * sum(new) * hq * d * BYTES[case["dtype"]]
    if case["op"] == "round":
        b += 4 * sum(new) * hkv * _row_bytes(case) + keep["bytes"]
    return {"bytes": b, "flops": 4 * pairs * hq * d}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _i32(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _parents(case, g):
    """Parents [seqs, nodes] of random trees: node 0 a root, the others under any earlier one, mostly a near one; of a
    chain, the node before. In a plan some nodes are absent (-2)."""
    n, t = case["seqs"], case.get("nodes", case.get("new"))
    i = torch.arange(t, device="cuda")
    if case.get("chain"):
        return (i - 1).to(torch.int32).expand(n, t).contiguous()
    back = 1 + (torch.rand((n, t), generator=g, device="cuda") ** 2 * 6).long()
    p = (i - back).clamp(min=-1)
    if case["op"] == "plan":
        p = torch.where((torch.rand((n, t), generator=g, device="cuda") < 0.05) & (i > 0), -2, p)
    return p.to(torch.int32)


def _lineage(parents):
    """(bits int64 [seqs, nodes]: bit j of node i where j is i or an ancestor of it, 0 for an absent node, depth)."""
    n, t = parents.shape
    i = torch.arange(t, device="cuda")
    above = (parents[:, :, None] == i).float() + torch.eye(t, device="cuda")
    for _ in range(max(1, (t - 1).bit_length())):  # the closure doubles its reach with each product
        above = ((above @ above) > 0).float()
    absent = (above @ (parents < -1).float()[:, :, None])[..., 0] > 0
    bits = (above.long() << i).sum(-1)
    return torch.where(absent, 0, bits), above.sum(-1).long() - 1, absent


def _tables(need, width, g, spare=3):
    """A table row per sequence: its pages, anywhere in the pool, then -1; and the pages that no sequence has."""
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    counts = torch.tensor(need, device="cuda")
    col = torch.arange(width, device="cuda")
    at = ((torch.cumsum(counts, 0) - counts)[:, None] + col[None]).clamp(max=pages - 1)
    return torch.where(col[None] < counts[:, None], order[at], -1).contiguous(), order[sum(need):].clone(), pages


def _quantize(x, bits):
    """Affine codes of x [..., D] in groups of 64: (codes [..., D], scales, biases [..., D/64] in x's type)."""
    w = x.float().unflatten(-1, (-1, 64))
    lo, hi = w.amin(-1), w.amax(-1)
    scale = ((hi - lo) / ((1 << bits) - 1)).clamp(min=1e-7)
    codes = torch.round((w - lo[..., None]) / scale[..., None]).clamp(0, (1 << bits) - 1).flatten(-2)
    return codes, scale.to(x.dtype), lo.to(x.dtype)


def _pack(codes, bits):
    c = codes.to(torch.int32).unflatten(-1, (-1, 32 // bits))
    shift = torch.arange(32 // bits, device="cuda", dtype=torch.int32) * bits
    return (c << shift).sum(-1).to(torch.int32).contiguous()


def _store(case, x):
    """A pool's arrays for the values x [..., D]: [x], or [codes, scales, biases]."""
    x = x.to(DTYPES[case["dtype"]])
    if not case["bits"]:
        return [x.contiguous()]
    codes, scale, bias = _quantize(x, case["bits"])
    return [_pack(codes, case["bits"]), scale.contiguous(), bias.contiguous()]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, page = case["op"], case["page"]
    held, new = _counts(case)
    s = {"case": case, "held": _i32(held), "new": _i32(new)}
    width = max(1, max(-(-(h + n) // page) for h, n in zip(held, new)))
    if op == "plan":
        grow = case["grow"]
        need = [-(-(h if grow else h + n) // page) for h, n in zip(held, new)]
        more = sum(-(-(h + n) // page) for h, n in zip(held, new)) - sum(need)
        s["tables"], s["free"], _ = _tables(need, width, g, more + 3)
        s["pages"], s["taken"] = _i32(need), _i32([0])
        s["parents"] = _parents(case, g) if case["tree"] else None
        return s
    ends = [h + n for h, n in zip(held, new)]
    s["tables"], _, pages = _tables([-(-e // page) for e in ends], width, g)
    s["first"], s["ends"] = _i32([0] + torch.tensor(new).cumsum(0).tolist()), _i32(ends)
    if op != "tree":
        paths = _paths(case)
        s["path"] = _i32([p + [-1] * (case["nodes"] - len(p)) for p in paths])
        s["kept"] = _i32([len(p) for p in paths])
        s["lengths"] = torch.empty_like(s["held"])
    d, hkv, dt = case["dim"], case["kv_heads"], DTYPES[case["dtype"]]
    if op == "keep":
        shape = (case["layers"], pages, hkv, page)
        s["pools"] = []
        for _ in "kv":
            if case["bits"]:
                codes = torch.randint(-(1 << 31), 1 << 31, (*shape, d * case["bits"] // 32), generator=g, device="cuda",
                                      dtype=torch.int32)
                s["pools"].append([codes, *((0.02 * _normal(g, *shape, d // 64)).to(dt) for _ in range(2))])
            else:
                s["pools"].append([torch.randn((*shape, d), generator=g, device="cuda", dtype=dt)])
        return s
    # tree, round: the pool holds the context and (for a tree) the drafted tokens, the queries come packed
    hq = case["q_heads"]
    s["q"] = _normal(g, sum(new), hq, d).to(dt)
    s["sinks"] = 3 * torch.rand(hq, generator=g, device="cuda") if case["sinks"] else None
    s["parents"] = _parents(case, g)
    bits, depth, _ = _lineage(s["parents"])
    at = [(b, i) for b, n in enumerate(new) for i in range(n)]
    rows = torch.tensor(at, device="cuda")
    s["masks"] = bits[rows[:, 0], rows[:, 1]].contiguous()
    s["places"] = (s["held"].long()[rows[:, 0]] + depth[rows[:, 0], rows[:, 1]]).to(torch.int32)
    if op == "round":
        s["kv"] = _normal(g, sum(new), 2 * hkv, d).to(dt)
    k, v = _normal(g, pages, hkv, page, d), _normal(g, pages, hkv, page, d)
    # one page in 16 answers its sequence's drafted tokens, as a retrieved passage does
    t = s["tables"]
    found = ((torch.rand(t.shape, generator=g, device="cuda") < 1 / 16) & (t >= 0)).nonzero()
    want = torch.zeros((case["seqs"], hq, d), device="cuda").index_add_(0, rows[:, 0], s["q"].float())
    want = want.unflatten(1, (hkv, -1)).sum(2)
    want = want / want.norm(dim=-1, keepdim=True)
    k[t[found[:, 0], found[:, 1]].long()] += 0.5 * math.sqrt(d) * want[found[:, 0], :, None, :]
    s["pools"] = [_store(case, k), _store(case, v)]
    del k, v
    # slots past a sequence's end hold what an earlier sequence left there, not-a-numbers among it
    end = torch.arange(t.shape[1], device="cuda")[None] == (s["ends"][:, None] - 1) // page
    rows = (end & (t >= 0)).nonzero()
    past = torch.arange(page, device="cuda")[None] >= ((s["ends"][rows[:, 0]] - 1) % page + 1)[:, None]
    slots = past.nonzero()
    at = t[rows[slots[:, 0], 0], rows[slots[:, 0], 1]].long()
    for pool in s["pools"]:
        pool[-1][at, :, slots[:, 1]] = float("nan")
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _plain_plan(s, capacity, page, parents, grow):
    held, new = s["held"].long(), s["new"].long()
    ends, last = held + new, torch.cumsum(new, 0)
    first = torch.cat((torch.zeros_like(last[:1]), last))
    tables = s["tables"]
    if grow:
        have = s["pages"].long()
        need = (torch.div(ends + page - 1, page, rounding_mode="floor") - have).clamp(min=0)
        base = s["taken"].long() + torch.cumsum(need, 0) - need
        col = torch.arange(tables.shape[1], device="cuda")[None] - have[:, None]
        take = (col >= 0) & (col < need[:, None])
        pick = (base[:, None] + col).clamp(0, s["free"].shape[0] - 1)
        tables.copy_(torch.where(take, s["free"][pick], tables))
        s["pages"].copy_(have + need)
        s["taken"] += need.sum().to(torch.int32)
    row = torch.arange(capacity, device="cuda")
    live = row < last[-1]
    seq = torch.searchsorted(last, row, right=True).clamp(max=held.shape[0] - 1)
    node = row - first[seq]
    pos = torch.where(live, held[seq] + node, 0)
    slot = tables[seq, torch.div(pos, page, rounding_mode="floor")].long() * page + pos % page
    got = {"first": first.to(torch.int32), "ends": ends.to(torch.int32),
           "seq": torch.where(live, seq, -1).to(torch.int32)}
    if parents is not None:
        bits, depth, absent = _lineage(parents)
        node = node.clamp(0, parents.shape[1] - 1)
        live = live & ~absent[seq, node]
        got["places"] = torch.where(live, held[seq] + depth[seq, node], -1).to(torch.int32)
        got["masks"] = torch.where(live, bits[seq, node], 0)
    got["positions"] = torch.where(live, pos, -1).to(torch.int32)
    got["slots"] = torch.where(live, slot, -1)
    if grow:
        got.update(tables=tables, pages=s["pages"], taken=s["taken"])
    return got


def _values(case, pool, at):
    """Pages `at` of a pool's K or V in fp32."""
    if not case["bits"]:
        return pool[0][at].float()
    per, bits = 32 // case["bits"], case["bits"]
    shift = torch.arange(per, device="cuda", dtype=torch.int32) * bits
    codes = ((pool[0][at][..., None] >> shift) & ((1 << bits) - 1)).flatten(-2).float().unflatten(-1, (-1, 64))
    return (codes * pool[1][at].float()[..., None] + pool[2][at].float()[..., None]).flatten(-2)


def _plain_tree(s, q, ends, first, masks, places):
    c = s["case"]
    hkv, page, d, most = c["kv_heads"], c["page"], c["dim"], c["nodes"]
    first, ends = first.long(), ends.long()
    at = s["tables"].clamp(min=0).long()
    n, width = at.shape
    # the packed rows as [sequences, nodes]
    node = torch.arange(most, device="cuda")[None]
    count = first[1:] - first[:-1]
    live = node < count[:, None]
    row = torch.where(live, first[:-1, None] + node, 0)
    held = (ends - count)[:, None, None]
    t = torch.arange(width * page, device="cuda")[None, None]
    drafted = (masks[row][..., None] >> (t - held).clamp(0, 63)) & 1
    seen = (t < held) | ((t < ends[:, None, None]) & (drafted > 0))
    if c["window"]:
        place = places.long()[row]
        # the place of token t: t itself while cached, then its node's
        its = torch.where(t < held, t, place.gather(1, (t - held)[:, 0].clamp(0, most - 1))[:, None])
        seen = seen & (its > place[..., None] - c["window"])
    seen = (seen & live[..., None])[:, None, :, None]
    k = _values(c, s["pools"][0], at).transpose(1, 2).reshape(n, hkv, width * page, d)
    x = (q.float() / math.sqrt(d))[row].unflatten(2, (hkv, -1)).permute(0, 2, 1, 3, 4)
    group = x.shape[3]
    score = (x.reshape(n, hkv, most * group, d) @ k.transpose(2, 3)).unflatten(2, (most, group))
    del k
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(score - top)
    del score
    total = p.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(s["sinks"].reshape(1, hkv, 1, group, 1) - top)
    v = _values(c, s["pools"][1], at).transpose(1, 2).reshape(n, hkv, width * page, d)
    v = torch.where((t < ends[:, None, None])[:, 0, :, None][:, None], v, 0.0)
    out = (p.flatten(2, 3) @ v).unflatten(2, (most, group)) / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 2, 1, 3, 4).reshape(n * most, hkv * group, d).to(q.dtype)
    # each row of the output from its place among [sequences, nodes]
    r = torch.arange(q.shape[0], device="cuda")
    seq = torch.searchsorted(first[1:], r, right=True)
    return out[seq * most + r - first[seq]]


def _plain_keep(s, ends, first):
    c = s["case"]
    page, t = c["page"], s["path"].shape[1]
    held = ends.long() - (first[1:] - first[:-1]).long()
    # past the accepted ones the last of them moves again, and where none is, the first row onto itself
    i = torch.minimum(torch.arange(t, device="cuda")[None], s["kept"][:, None] - 1).clamp(min=0)
    src = held[:, None] + torch.where(s["kept"][:, None] > 0, s["path"].gather(1, i), 0)
    to = held[:, None] + i
    at = [s["tables"].long().gather(1, torch.div(x, page, rounding_mode="floor")) for x in (src, to)]
    for pool in s["pools"]:
        for array in pool:
            if array.dim() == 4:
                array = array[None]
            array[:, at[1], :, to % page] = array[:, at[0], :, src % page]
    s["lengths"].copy_(held + s["kept"])
    return s["lengths"]


def _plain(s):
    c = s["case"]
    if c["op"] == "plan":
        return _plain_plan(s, c["seqs"] * c["new"], c["page"], s["parents"], c["grow"])
    if c["op"] == "tree":
        return _plain_tree(s, s["q"], s["ends"], s["first"], s["masks"], s["places"])
    if c["op"] == "keep":
        return _plain_keep(s, s["ends"], s["first"]), s["pools"]
    p = _plain_plan(s, s["q"].shape[0], c["page"], s["parents"], False)
    at, hkv = torch.div(p["slots"], c["page"], rounding_mode="floor"), c["kv_heads"]
    for pool, rows in zip(s["pools"], (s["kv"][:, :hkv], s["kv"][:, hkv:])):
        pool[0][at, :, p["slots"] % c["page"]] = rows
    out = _plain_tree(s, s["q"], p["ends"], p["first"], p["masks"], p["places"])
    return out, _plain_keep(s, p["ends"], p["first"]), s["pools"]


def _own(s):
    if "mlx-swift-lm_b200" not in sys.path:
        sys.path.insert(0, "mlx-swift-lm_b200")
    import sparse_decode as sd

    c = s["case"]
    if c["op"] == "plan":
        grow = dict(held=s["pages"], free=s["free"], taken=s["taken"]) if c["grow"] else {}
        p = sd.paged_plan(s["held"], s["new"], s["tables"], c["page"], c["seqs"] * c["new"], parents=s["parents"], **grow)
        got = {"first": p.first, "ends": p.ends, "seq": p.seq, "positions": p.positions, "slots": p.slots}
        if c["tree"]:
            got.update(places=p.places, masks=p.masks)
        if c["grow"]:
            got.update(tables=s["tables"], pages=s["pages"], taken=s["taken"])
        return got
    (k, *ks), (v, *vs) = s["pools"]
    pages = sd.KVPages(k, v, *ks, *vs, bits=c["bits"])
    if c["op"] == "keep":
        return sd.paged_keep(pages, s["tables"], s["ends"], s["first"], s["path"], s["kept"], lengths=s["lengths"]), s["pools"]
    seen = dict(window=c["window"], sinks=s["sinks"])
    if c["op"] == "tree":
        return sd.paged_tree_decode(s["q"], pages, s["tables"], s["ends"], s["first"], s["masks"], places=s["places"],
                                    **seen)
    hkv = c["kv_heads"]
    p = sd.paged_plan(s["held"], s["new"], s["tables"], c["page"], s["q"].shape[0], parents=s["parents"])
    sd.paged_append(pages, s["kv"][:, :hkv], s["kv"][:, hkv:], s["tables"], p.positions, seq=p.seq)
    out = sd.paged_tree_decode(s["q"], pages, s["tables"], p.ends, p.first, p.masks, places=p.places, **seen)
    return out, sd.paged_keep(pages, s["tables"], p.ends, p.first, s["path"], s["kept"], lengths=s["lengths"]), s["pools"]


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------

def _exact_sequence(s, pool, b, n):
    """The first n tokens of sequence b as [Hkv, n, D] in fp64."""
    c = s["case"]
    pages = s["tables"][b, :-(-n // c["page"])].long()
    if not c["bits"]:
        x = pool[0][pages].double()
    else:
        words, w = pool[0][pages].long() & 0xFFFFFFFF, c["bits"]
        codes = torch.stack([(words >> (w * j)) & ((1 << w) - 1) for j in range(32 // w)], -1).flatten(-2).double()
        grow = lambda y: y[pages].double().repeat_interleave(64, -1)  # noqa: E731
        x = codes * grow(pool[1]) + grow(pool[2])
    return x.permute(1, 0, 2, 3).flatten(1, 2)[:, :n]


def _exact_tree(s):
    c = s["case"]
    hkv, d, w = c["kv_heads"], c["dim"], c["window"]
    held, new = _counts(c)
    parents = s["parents"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    row = 0
    for b, (h, n) in enumerate(zip(held, new)):
        k, v = (_exact_sequence(s, pool, b, h + n) for pool in s["pools"])
        lines, place = [], []
        for i in range(n):
            up = parents[b][i]
            lines.append((lines[up] if up >= 0 else []) + [i])
            place.append(h + len(lines[i]) - 1)
        seen = torch.zeros((n, h + n), dtype=torch.bool)
        for i in range(n):
            seen[i, max(0, place[i] + 1 - w) if w else 0:h] = True
            for j in lines[i]:
                seen[i, h + j] = not w or place[j] > place[i] - w
        q = s["q"][row:row + n].double().view(n, hkv, -1, d)
        score = torch.einsum("nhgd,htd->hngt", q, k) / math.sqrt(d)
        score = score.masked_fill(~seen.to("cuda")[None, :, None], -math.inf)
        if s["sinks"] is not None:
            extra = s["sinks"].double().view(hkv, 1, -1, 1).expand(hkv, n, -1, 1)
            p = torch.softmax(torch.cat((score, extra), -1), -1)[..., :-1]
        else:
            p = torch.softmax(score, -1)
        out[row:row + n] = torch.einsum("hngt,htd->nhgd", p, v).reshape(n, -1, d)
        row += n
    return out


def _exact_keep(s, pools):
    """The pools' values with every accepted row moved, one after the other."""
    c = s["case"]
    held, _ = _counts(c)
    tables = s["tables"].tolist()
    for array in pools:
        if array is None:
            continue
        x = array if array.dim() == 5 else array[None]
        for b, path in enumerate(_paths(c)):
            for i, j in enumerate(path):
                to, src = (divmod(held[b] + y, c["page"]) for y in (i, j))
                x[:, tables[b][to[0]], :, to[1]] = x[:, tables[b][src[0]], :, src[1]]
    return pools


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "tree":
        return _exact_tree(s)
    pools = [[a.double() if a.is_floating_point() else None for a in pool] for pool in s["pools"]]
    if case["op"] == "keep":
        for pool in pools:
            _exact_keep(s, pool)
        return None, pools
    held, new = _counts(case)
    row = 0
    for b, (h, n) in enumerate(zip(held, new)):
        for i in range(n):
            page, slot = int(s["tables"][b, (h + i) // case["page"]]), (h + i) % case["page"]
            for pool, x in zip(s["pools"], s["kv"][row].split(case["kv_heads"])):
                pool[0][page, :, slot] = x
            row += 1
    out = _exact_tree(s)
    return out, None, [_exact_keep(s, [a.double() for a in pool]) for pool in s["pools"]]

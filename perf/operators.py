"""Workloads of the paged-cache operators, in plain torch and through sparse_decode.

Four operators, one decode step's worth:

* rotary:  per-head RMS norm (optional) and position rotation of queries and keys;
* append:  the same rotation, with the keys and values stored into their pages;
* copy:    whole pages copied inside a pool, in every layer (fork, compaction);
* decode:  attention of one new token per sequence over its pages;

and `step`, an append followed by the decode that reads it. `run` computes a
case with elementary torch operations in 32 bits, or (own = True) with the
library's kernels; `exact` computes it in 64 bits from the definition.

Pages are [n_pages, kv_heads, page_size, head_dim] (4/8-bit pools: uint32-packed
affine codes in groups of 64 with scales and biases in the pool's type); a
sequence's tokens lie in the pages that its row of the table names.
"""
import math
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one decoded token of one user: queries and keys normed and rotated, latency only
        dict(name="rotary_1_token", op="rotary", tokens=1, q_heads=32, kv_heads=8, dim=128, rot=128, norm=True,
             traditional=False, base=1e6, factor=1.0, dtype="bf16", last=32768),
        # a whole 32K prompt through one layer
        dict(name="rotary_prompt", op="rotary", tokens=32768, q_heads=32, kv_heads=8, dim=128, rot=128, norm=True,
             traditional=False, base=1e6, factor=1.0, dtype="bf16", last=32768),
        # a prompt of an odd length; half of each head rotated, neighbouring pairs, stretched positions
        dict(name="rotary_part_of_head", op="rotary", tokens=4099, q_heads=8, kv_heads=2, dim=64, rot=32, norm=False,
             traditional=True, base=1e4, factor=1.19, dtype="f16", last=131072),
        # the write half of a decode step of 16 users
        dict(name="append_16_users", op="append", seqs=16, per_seq=1, ctx=4096, page=64, q_heads=32, kv_heads=8,
             dim=128, rot=128, norm=True, traditional=False, base=1e6, factor=1.0, dtype="bf16"),
        # chunked prefill: 500 more tokens of each of 8 prompts, small pages
        dict(name="append_chunks", op="append", seqs=8, per_seq=500, ctx=2000, page=16, q_heads=32, kv_heads=8,
             dim=128, rot=128, norm=False, traditional=False, base=5e5, factor=1.0, dtype="f16"),
        # copy-on-write of the shared last page of one forked sequence, all layers
        dict(name="copy_one_page", op="copy", pairs=1, pages=24, layers=36, page=64, kv_heads=8, dim=128, dtype="bf16",
             bits=0),
        # compaction of an 8-bit pool: 400 live pages move to the front
        dict(name="copy_compaction", op="copy", pairs=400, pages=801, layers=36, page=64, kv_heads=8, dim=128,
             dtype="bf16", bits=8),
        # one user, short context, fp32: the smallest call, latency only
        dict(name="decode_f32_4K", op="decode", seqs=1, ctx=4096, ragged=0, page=64, q_heads=8, kv_heads=2, dim=64,
             dtype="f32", bits=0, window=0, sinks=False),
        # one user, 32K tokens
        dict(name="decode_bf16_32K", op="decode", seqs=1, ctx=32768, ragged=0, page=64, q_heads=32, kv_heads=8, dim=128,
             dtype="bf16", bits=0, window=0, sinks=False),
        # four long conversations in an 8-bit cache
        dict(name="decode_q8_4x128K", op="decode", seqs=4, ctx=131072, ragged=0, page=128, q_heads=32, kv_heads=8,
             dim=128, dtype="bf16", bits=8, window=0, sinks=False),
        # a serving batch: 16 conversations between nothing and 128K tokens
        dict(name="decode_ragged_16", op="decode", seqs=16, ctx=131072, ragged=5, page=64, q_heads=32, kv_heads=8,
             dim=128, dtype="bf16", bits=0, window=0, sinks=False),
        # a whole decode step of 16 users over an 8-bit cache: rotate, quantize, store, attend
        dict(name="step_q8_16_users", op="step", seqs=16, ctx=4096, ragged=7, page=64, q_heads=32, kv_heads=8, dim=128,
             rot=128, norm=True, traditional=False, base=1e6, factor=1.0, dtype="bf16", bits=8, window=0, sinks=False),
    ]


def _log(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = min(hi, max(lo, n))
    return n + 1 if n == 3072 else n


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    dim = rng.choice([64, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8])
    group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])
    c = dict(op=rng.choice(["rotary", "append", "copy", "decode", "decode", "decode", "step"]))
    rot = rng.choice([dim, dim, dim // 2, dim // 4, dim - 6])
    turn = dict(q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim, rot=rot, norm=rng.random() < 0.5,
                traditional=rng.random() < 0.4, base=rng.choice([1e4, 5e5, 1e6]), factor=rng.choice([1.0, 1.0, 1.19]),
                dtype=dtype)
    # fp32 positions stay short: an angle rounded to fp32 is the plain form's own error
    far = 2048 if dtype == "f32" else 131072
    if c["op"] == "rotary":
        c.update(turn, tokens=_log(rng, 1, min(far, 8192)), last=far)
    elif c["op"] == "append":
        c.update(turn, seqs=_log(rng, 1, 64), per_seq=rng.choice([1, 1, _log(rng, 2, 300)]), ctx=_log(rng, 1, 1500),
                 page=rng.choice([16, 32, 64, 128]))
    elif c["op"] == "copy":
        pairs = _log(rng, 1, 120)
        c.update(pairs=pairs, pages=2 * pairs + rng.randrange(1, 30), layers=rng.choice([1, 2, 7, 12]),
                 page=rng.choice([16, 32, 64, 128]), kv_heads=kv_heads, dim=dim, dtype=dtype,
                 bits=rng.choice([0, 0, 4, 8]))
    else:
        c.update(turn)
        for name in ("rot", "norm", "traditional", "base", "factor") if c["op"] == "decode" else ():
            del c[name]
        seqs = _log(rng, 1, 64)
        most = min(131072 if c["op"] == "decode" else far, (1 << 22) // (seqs * kv_heads))
        c.update(seqs=seqs, ctx=_log(rng, 1, max(1, most)), ragged=rng.choice([0, rng.randrange(1, 100)]),
                 page=rng.choice([16, 32, 64, 128]), bits=rng.choice([0, 0, 4, 8]),
                 window=rng.choice([0, 0, _log(rng, 1, 4096)]), sinks=rng.random() < 0.3)
    return c


def _lengths(case):
    """Tokens of each sequence, by the case alone. Ragged batches spread over [0, ctx], with one at ctx and, from
    four sequences on, an empty one (a step's sequences hold one token at least: the one just appended)."""
    n, ctx = case["seqs"], case["ctx"]
    if not case.get("ragged"):
        return [ctx] * n
    r = random.Random(case["ragged"])
    got = [r.randint(1, ctx) for _ in range(n)]
    got[0] = ctx
    if n >= 4:
        got[2] = 0
    return [max(1, t) for t in got] if case["op"] == "step" else got


def _seen(case):
    w = case["window"]
    return [min(t, w) if w else t for t in _lengths(case)]


def _row_bytes(case):
    d, e = case["dim"], BYTES[case["dtype"]]
    return d * case["bits"] // 8 + 2 * (d // 64) * e if case.get("bits") else d * e


def work(case):
    op, e, d = case["op"], BYTES[case["dtype"]], case["dim"]
    if op == "copy":
        page = case["kv_heads"] * case["page"] * _row_bytes(case)
        return {"bytes": 2 * 2 * case["pairs"] * case["layers"] * page, "flops": 0}
    hq, hkv = case["q_heads"], case["kv_heads"]
    if op == "rotary":
        return {"bytes": 2 * case["tokens"] * (hq + hkv) * d * e, "flops": 10 * case["tokens"] * (hq + hkv) * d}
    if op == "append":
        n = case["seqs"] * case["per_seq"]
        return {"bytes": 2 * n * (hq + 2 * hkv) * d * e, "flops": 10 * n * (hq + hkv) * d}
    seen = sum(_seen(case))
    attend = 2 * seen * hkv * _row_bytes(case) + 2 * case["seqs"] * hq * d * e
    flops = 4 * seen * hq * d
    if op == "step":
        attend += case["seqs"] * ((hq + 2 * hkv) * d * e + 2 * hkv * _row_bytes(case))
        flops += 10 * case["seqs"] * (hq + hkv) * d
    return {"bytes": attend, "flops": flops}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _qkv(case, g, tokens, s):
    """Queries, keys and values as the projection leaves them: slices of one [tokens, (Hq + 2 Hkv) D] product."""
    hq, hkv, d, dt = case["q_heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    qkv = _normal(g, tokens, hq + 2 * hkv, d).to(dt)
    s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]


def _turning(case, g, s):
    d, dt = case["dim"], DTYPES[case["dtype"]]
    i = torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64) / case["rot"]
    s["inv_freq"] = (case["base"] ** -i).float()
    s["q_norm"] = s["k_norm"] = None
    if case["norm"]:
        s["q_norm"] = (1 + 0.2 * _normal(g, d)).to(dt)
        s["k_norm"] = (1 + 0.2 * _normal(g, d)).to(dt)


def _tables(lengths, page, g):
    """A table row per sequence: its pages, anywhere in the pool, then -1. Some pages of the pool stay unused."""
    need = [-(-t // page) for t in lengths]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    width = max(1, max(need))
    counts = torch.tensor(need, device="cuda")
    col = torch.arange(width, device="cuda")
    first = torch.cumsum(counts, 0) - counts
    at = (first[:, None] + col[None]).clamp(max=pages - 1)
    return torch.where(col[None] < counts[:, None], order[at], -1).contiguous(), pages


def _quantize(x, bits):
    """Affine codes of x [..., D] in groups of 64: (codes [..., D] in fp32, scales, biases [..., D/64] in x's type).
    The edge of larger magnitude lies on a code; all steps in fp32."""
    w = x.float().unflatten(-1, (-1, 64))
    lo, hi = w.amin(-1), w.amax(-1)
    top = float((1 << bits) - 1)
    scale = ((hi - lo) / top).clamp(min=1e-7)
    low = lo.abs() > hi.abs()
    scale = torch.where(low, scale, -scale)
    edge = torch.where(low, lo, hi)
    q0 = torch.round(edge / scale)
    scale = torch.where(q0 != 0, edge / torch.where(q0 != 0, q0, 1.0), scale)
    bias = torch.where(q0 == 0, 0.0, edge)
    codes = torch.round((w - bias[..., None]) / scale[..., None]).clamp(0, top).flatten(-2)
    return codes, scale.to(x.dtype), bias.to(x.dtype)


def _pack(codes, bits):
    per = 32 // bits
    c = codes.to(torch.int32).unflatten(-1, (-1, per))
    out = c[..., 0]
    for j in range(1, per):
        out = out | (c[..., j] << (bits * j))
    return out.contiguous()


def _store(case, x):
    """A pool's arrays for the values x [..., D]: [x], or [codes, scales, biases]."""
    x = x.to(DTYPES[case["dtype"]])
    if not case.get("bits"):
        return [x.contiguous()]
    codes, scale, bias = _quantize(x, case["bits"])
    return [_pack(codes, case["bits"]), scale.contiguous(), bias.contiguous()]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s, op, d = {"case": case}, case["op"], case["dim"]
    if op == "copy":
        shape = (case["layers"], case["pages"], case["kv_heads"], case["page"])
        s["pools"] = []
        for _ in "kv":
            if case["bits"]:
                codes = torch.randint(-(1 << 31), 1 << 31, (*shape, d * case["bits"] // 32), generator=g, device="cuda",
                                      dtype=torch.int32)
                small = [(0.02 * _normal(g, *shape, d // 64)).to(DTYPES[case["dtype"]]) for _ in range(2)]
                s["pools"].append([codes, *small])
            else:
                s["pools"].append([_normal(g, *shape, d).to(DTYPES[case["dtype"]])])
        order = torch.randperm(case["pages"], generator=g, device="cuda").to(torch.int32)
        s["src"], s["dst"] = order[:case["pairs"]].clone(), order[case["pairs"]:2 * case["pairs"]].clone()
        return s
    if op == "rotary":
        _qkv(case, g, case["tokens"], s)
        _turning(case, g, s)
        start = max(0, case["last"] - case["tokens"])
        lowest = int(torch.randint(start // 2, start + 1, (1,), generator=g, device="cuda"))
        s["positions"] = torch.arange(lowest, lowest + case["tokens"], device="cuda", dtype=torch.int32)
        return s
    if op == "append":
        # sequence b already holds held[b] tokens, and per_seq more arrive
        held = [max(0, case["ctx"] - 37 * b) for b in range(case["seqs"])]
        lengths = [h + case["per_seq"] for h in held]
        per = torch.arange(case["per_seq"], device="cuda")
        s["positions"] = (torch.tensor(held, device="cuda")[:, None] + per[None]).flatten().to(torch.int32)
        s["seq"] = torch.arange(case["seqs"], device="cuda", dtype=torch.int32).repeat_interleave(case["per_seq"])
        _qkv(case, g, case["seqs"] * case["per_seq"], s)
        _turning(case, g, s)
        s["tables"], pages = _tables(lengths, case["page"], g)
        shape = (pages, case["kv_heads"], case["page"], d)
        s["pools"] = [[_normal(g, *shape).to(DTYPES[case["dtype"]])] for _ in "kv"]
        return s
    # decode, step: the pool holds the context (a step's newest token is still to be written)
    lengths = _lengths(case)
    hq, hkv, page = case["q_heads"], case["kv_heads"], case["page"]
    s["lengths"] = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    s["tables"], pages = _tables(lengths, page, g)
    if op == "step":
        _qkv(case, g, case["seqs"], s)
        _turning(case, g, s)
        s["positions"] = s["lengths"] - 1
    else:
        s["q"] = _normal(g, case["seqs"], hq, d).to(DTYPES[case["dtype"]])
    s["sinks"] = 3 * torch.rand(hq, generator=g, device="cuda") if case["sinks"] else None
    k, v = _normal(g, pages, hkv, page, d), _normal(g, pages, hkv, page, d)
    # one page in 16 answers its sequence's query, as a retrieved passage does
    t = s["tables"]
    found = (torch.rand(t.shape, generator=g, device="cuda") < 1 / 16) & (t >= 0)
    want = s["q"].float().unflatten(1, (hkv, -1)).sum(2)
    want = want / want.norm(dim=-1, keepdim=True)
    rows = found.nonzero()
    k[t[rows[:, 0], rows[:, 1]].long()] += 0.5 * math.sqrt(d) * want[rows[:, 0], :, None, :]
    s["pools"] = [_store(case, k), _store(case, v)]
    del k, v
    # slots past a sequence's end hold what an earlier sequence left there, not-a-numbers among it
    end = torch.arange(t.shape[1], device="cuda")[None] == (s["lengths"][:, None] - 1) // page
    rows = (end & (t >= 0)).nonzero()
    past = torch.arange(page, device="cuda")[None] >= ((s["lengths"][rows[:, 0]] - 1) % page + 1)[:, None]
    slots = past.nonzero()
    at = t[rows[slots[:, 0], 0], rows[slots[:, 0], 1]].long()
    for pool in s["pools"]:
        pool[-1][at, :, slots[:, 1]] = float("nan")
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _turn(s, x, weight, n):
    """The rows x [N, H, D] normed and rotated, in fp32."""
    c, x = s["case"], x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    angle = s["positions"][:n].float()[:, None] * s["inv_freq"]
    cos, sin = (c["factor"] * angle.cos())[:, None], (c["factor"] * angle.sin())[:, None]
    part, rest = x[..., :c["rot"]], x[..., c["rot"]:]
    if c["traditional"]:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = part[..., :c["rot"] // 2], part[..., c["rot"] // 2:]
        part = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((part, rest), -1)


def _plain_append(s):
    dt, n = s["q"].dtype, s["q"].shape[0]
    q = _turn(s, s["q"], s["q_norm"], n).to(dt)
    k = _turn(s, s["k"], s["k_norm"], n).to(dt)
    pos = s["positions"].long()
    page = s["case"]["page"]
    seq = s["seq"].long() if "seq" in s else torch.arange(n, device="cuda")
    at = s["tables"][seq, pos // page].long()
    for pool, x in zip(s["pools"], (k, s["v"])):
        for array, rows in zip(pool, _store(s["case"], x)):
            array[at, :, pos % page] = rows
    return q


def _values(case, pool, at):
    """Pages `at` of a pool's K or V in fp32."""
    if not case["bits"]:
        return pool[0][at].float()
    per, bits = 32 // case["bits"], case["bits"]
    shift = torch.arange(per, device="cuda", dtype=torch.int32) * bits
    codes = ((pool[0][at][..., None] >> shift) & ((1 << bits) - 1)).flatten(-2).float().unflatten(-1, (-1, 64))
    return (codes * pool[1][at].float()[..., None] + pool[2][at].float()[..., None]).flatten(-2)


def _plain_decode(s, q):
    c = s["case"]
    hkv, page, d = c["kv_heads"], c["page"], c["dim"]
    at = s["tables"].clamp(min=0).long()
    n, width = at.shape
    t = torch.arange(width * page, device="cuda")[None]
    live = t < s["lengths"][:, None]
    if c["window"]:
        live = live & (t >= s["lengths"][:, None] - c["window"])
    k = _values(c, s["pools"][0], at).transpose(1, 2).reshape(n, hkv, width * page, d)
    score = (q.float() / math.sqrt(d)).reshape(n, hkv, -1, d) @ k.transpose(2, 3)
    del k
    score = torch.where(live[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(s["sinks"].reshape(1, hkv, -1, 1) - top)
    v = _values(c, s["pools"][1], at).transpose(1, 2).reshape(n, hkv, width * page, d)
    v = torch.where(live[:, None, :, None], v, 0.0)
    out = (p @ v) / torch.where(total > 0, total, 1.0)
    empty = (s["lengths"] <= 0)[:, None, None, None]
    return torch.where(empty, 0.0, out).reshape(n, -1, d).to(q.dtype)


def _plain(s):
    c = s["case"]
    if c["op"] == "rotary":
        n, dt = s["q"].shape[0], s["q"].dtype
        return _turn(s, s["q"], s["q_norm"], n).to(dt), _turn(s, s["k"], s["k_norm"], n).to(dt)
    if c["op"] == "append":
        q = _plain_append(s)
        return q, s["pools"][0][0], s["pools"][1][0]
    if c["op"] == "copy":
        src, dst = s["src"].long(), s["dst"].long()
        for pool in s["pools"]:
            for array in pool:
                array[:, dst] = array[:, src]
        return s["pools"]
    if c["op"] == "decode":
        return _plain_decode(s, s["q"])
    out = _plain_decode(s, _plain_append(s))
    return out, _floats(s)


def _floats(s):
    """What a step returns of its updated pool: the values, or the scales and biases of its codes (the codes
    themselves are seen through the attention that reads them)."""
    return [pool[1:] if s["case"]["bits"] else pool for pool in s["pools"]]


def _own(s):
    if "mlx-swift-lm_b200" not in sys.path:
        sys.path.insert(0, "mlx-swift-lm_b200")
    import sparse_decode as sd

    c = s["case"]
    if c["op"] in ("rotary", "append", "step"):
        turn = dict(inv_freq=s["inv_freq"], traditional=c["traditional"], factor=c["factor"], q_norm=s["q_norm"],
                    k_norm=s["k_norm"], eps=EPS)
    if c["op"] == "rotary":
        return sd.rotary(s["q"], s["k"], s["positions"], **turn)
    (k, *ks), (v, *vs) = s["pools"]
    pages = sd.KVPages(k, v, *ks, *vs, bits=c.get("bits", 0))
    if c["op"] == "append":
        q = sd.paged_append(pages, s["k"], s["v"], s["tables"], s["positions"], seq=s["seq"], q=s["q"], **turn)
        return q, k, v
    if c["op"] == "copy":
        sd.copy_pages(pages, s["src"], s["dst"])
        return s["pools"]
    seen = dict(window=c["window"], sinks=s["sinks"])
    if c["op"] == "decode":
        return sd.paged_decode(s["q"], pages, s["tables"], s["lengths"], **seen)
    q = sd.paged_append(pages, s["k"], s["v"], s["tables"], s["positions"], q=s["q"], **turn)
    return sd.paged_decode(q, pages, s["tables"], s["lengths"], **seen), _floats(s)


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------

def _exact_turn(s, x, weight):
    c, rot, x = s["case"], s["case"]["rot"], x.double()
    if weight is not None:
        x = weight.double() * x / (x.pow(2).sum(-1, keepdim=True) / c["dim"] + EPS).sqrt()
    out = x.clone()
    first = torch.arange(rot // 2, device="cuda") * (2 if c["traditional"] else 1)
    second = first + (1 if c["traditional"] else rot // 2)
    angle = torch.outer(s["positions"].double(), s["inv_freq"].double())
    spin = torch.polar(torch.full_like(angle, c["factor"]), angle)[:, None]
    z = torch.complex(x[..., first], x[..., second]) * spin
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_pages(s, pool, pages):
    """Pages of one sequence as [Hkv, tokens, D] in fp64."""
    c = s["case"]
    if not c["bits"]:
        x = pool[0][pages].double()
    else:
        words, b = pool[0][pages].long() & 0xFFFFFFFF, c["bits"]
        codes = torch.stack([(words >> (b * j)) & ((1 << b) - 1) for j in range(32 // b)], -1).flatten(-2).double()
        grow = lambda t: t[pages].double().repeat_interleave(64, -1)  # noqa: E731
        x = codes * grow(pool[1]) + grow(pool[2])
    return x.permute(1, 0, 2, 3).flatten(1, 2)


def _exact_decode(s, q, last=None):
    """last: (k, v) rows in fp64 that stand in for each sequence's newest token."""
    c = s["case"]
    hkv, d = c["kv_heads"], c["dim"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(c)):
        if n == 0:
            continue
        pages = s["tables"][b, :-(-n // c["page"])].long()
        k, v = (_exact_pages(s, pool, pages)[:, :n] for pool in s["pools"])
        if last is not None:
            k[:, n - 1], v[:, n - 1] = last[0][b], last[1][b]
        begin = max(0, n - c["window"]) if c["window"] else 0
        score = torch.einsum("hgd,htd->hgt", q[b].double().view(hkv, -1, d), k[:, begin:]) / math.sqrt(d)
        if s["sinks"] is not None:
            score = torch.cat((score, s["sinks"].double().view(hkv, -1, 1)), -1)
        p = torch.softmax(score, -1)[..., :n - begin]
        out[b] = torch.einsum("hgt,htd->hgd", p, v[:, begin:]).reshape(-1, d)
    return out


def _exact_codes(x, bits, dtype):
    """Rows x [N, H, D] as a pool of codes reads them back, and their scales and biases before rounding."""
    groups = x.unflatten(-1, (-1, 64))
    top = 2 ** bits - 1
    least, most = groups.min(-1, keepdim=True).values, groups.max(-1, keepdim=True).values
    step = torch.maximum((most - least) / top, torch.full_like(most, 1e-7))
    edge = torch.where(-least > most, least, most)
    step = torch.where(-least > most, step, -step)
    at = (edge / step).round()
    step = torch.where(at == 0, step, edge / at)
    bias = torch.where(at == 0, torch.zeros_like(edge), edge)
    codes = ((groups - bias) / step).round().clamp(0, top)
    seen = codes * step.to(dtype).double() + bias.to(dtype).double()
    return seen.flatten(-2), step[..., 0], bias[..., 0]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":
        src, dst = s["src"].tolist(), s["dst"].tolist()
        got = []
        for pool in s["pools"]:
            moved = [a.double() if a.is_floating_point() and a.numel() < 1 << 27 else None for a in pool]
            for a in moved:
                for i, j in zip(src, dst):
                    if a is not None:
                        a[:, j] = a[:, i]
            got.append(moved)
        return got
    if case["op"] == "decode":
        return _exact_decode(s, s["q"])
    q = _exact_turn(s, s["q"], s["q_norm"])
    k = _exact_turn(s, s["k"], s["k_norm"])
    if case["op"] == "rotary":
        return q, k
    if case["op"] == "append":
        got = [q]
        for pool, rows in zip(s["pools"], (k, s["v"].double())):
            x = pool[0].double()
            for n, (b, p) in enumerate(zip(s["seq"].tolist(), s["positions"].tolist())):
                x[int(s["tables"][b, p // case["page"]]), :, p % case["page"]] = rows[n]
            got.append(x)
        return tuple(got)
    # a step's rows are read back as stored: rounded to the pool's type, as codes of that where it holds codes
    rows, got = [], []
    for pool, x in zip(s["pools"], (k, s["v"].double())):
        state, x = [a.double() for a in (pool[1:] if case["bits"] else pool)], x.to(s["q"].dtype).double()
        if case["bits"]:
            x, *new = _exact_codes(x, case["bits"], s["q"].dtype)
        else:
            new = [x]
        for b, n in enumerate(_lengths(case)):
            for a, y in zip(state, new):
                a[int(s["tables"][b, (n - 1) // case["page"]]), :, (n - 1) % case["page"]] = y[b]
        rows.append(x)
        got.append(state)
    return _exact_decode(s, q, rows), got

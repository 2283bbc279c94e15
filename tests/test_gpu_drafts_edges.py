"""Calls of the operators around drafted tokens that their documentation allows
and that read or wrote, once, what they should not have."""
from __future__ import annotations

import ctypes

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

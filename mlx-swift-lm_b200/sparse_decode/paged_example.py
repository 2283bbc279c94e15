"""A serving loop in small: python -m sparse_decode.paged_example

Two prompts of different lengths go into a paged cache; one of them is forked
(shared pages, copied when written); the three sequences decode together, each
step rotating, storing and attending in every layer; then one is freed, the
pool is compacted, and the rest decode on. Random weights stand in for a
model: what is shown is how the calls fit together. With --check, the last
step's attention is compared with a plain computation over each sequence's
own tokens.
"""
from __future__ import annotations

import argparse


def run(layers: int = 4, kv_bits: int = 0, prompts=(70, 33), steps: int = 20, page_size: int = 16, check: bool = False,
        seed: int = 0):
    """Returns (pool, sequence ids, last outputs [sequences, Hq, D] per layer, largest error or None)."""
    import torch

    from . import PagePool, attention_with_cache_update, rotary_frequencies

    hq, hkv, d, hidden = 8, 2, 128, 256
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()  # noqa: E731
    project = [rand(hidden, (hq + 2 * hkv) * d) * hidden ** -0.5 for _ in range(layers)]
    norm = [(1 + 0.1 * rand(d)) for _ in range(2)]
    inv_freq, factor = rotary_frequencies(d, 1e6, {"rope_type": "yarn", "factor": 4.0,
                                                   "original_max_position_embeddings": 32768})
    turn = dict(inv_freq=inv_freq, factor=factor, q_norm=norm[0], k_norm=norm[1])
    pool = PagePool(layers, 64, hkv, d, page_size, "bf16", kv_bits)

    def step(batch, x):
        """One forward step of the new tokens x [sequences, tokens each, hidden]."""
        outs = []
        for i in range(layers):
            q, k, v = (x @ project[i]).unflatten(-1, (-1, d)).split((hq, hkv, hkv), dim=2)
            out = attention_with_cache_update(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2),
                                              batch.layer(i, **turn), d ** -0.5, "causal" if x.shape[1] > 1 else None)
            outs.append(out[:, :, -1])
            x = (x + out.transpose(1, 2).flatten(2)[..., :hidden]).bfloat16()
        return outs

    seqs = []
    for n in prompts:  # prefill
        seqs.append(pool.add())
        step(pool.extend(seqs[-1:], n), rand(1, n, hidden))
    seqs.append(pool.fork(seqs[0]))
    for _ in range(steps):
        step(pool.extend(seqs, 1), rand(len(seqs), 1, hidden))
    pool.free(seqs.pop(1))
    pool.compact()
    last = {}
    for _ in range(steps):
        batch = pool.extend(seqs, 1)
        last = dict(batch=batch, outs=step(batch, rand(len(seqs), 1, hidden)))
    flags = pool.check_device()
    if flags:
        raise RuntimeError(f"device error bits {flags}")
    worst = None
    if check:
        worst = 0.0
        # the last layer's queries of the last step, once more, against the plain attention of each sequence
        q = rand(len(seqs), hq, d)
        got = last["batch"].decode(layers - 1, q)
        for b in range(len(seqs)):
            k, v = (t[0].double().repeat_interleave(hq // hkv, 0) for t in last["batch"].layer(layers - 1).dense(b))
            p = torch.softmax(torch.einsum("hd,htd->ht", q[b].double(), k) * d ** -0.5, -1)
            want = torch.einsum("ht,htd->hd", p, v)
            worst = max(worst, float((got[b].double() - want).norm() / want.norm()))
    return pool, seqs, last["outs"], worst


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--kv-bits", type=int, default=0, choices=(0, 4, 8))
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--check", action="store_true")
    a = ap.parse_args()
    pool, seqs, outs, worst = run(kv_bits=a.kv_bits, steps=a.steps, check=a.check)
    print(f"sequences {[pool.length(s) for s in seqs]} tokens, {pool.free_pages} of {pool.pages.n_pages} pages free, "
          f"{len(outs)} layers" + (f", relative error {worst:.1e}" if worst is not None else ""))


if __name__ == "__main__":
    main()

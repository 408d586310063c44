"""Speculative decoding with trees: several drafts of every sequence at once, in one
pass over the paged KV cache, and 4-bit weights in the MLP and the LM head.

    python examples/tree_decode.py [--cache bf16|e4m3] [--samples 3] [--rounds 8]

A round appends every sequence's tree (its last token and the drafts below it), each
node at its depth's position, attends along the branches, samples after every node, and
keeps the path that the sampled ids follow.  The drafts are the model's own likeliest
tokens, with some that are not.  At the end every sequence is recomputed without a cache
and compared.
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path[:0] = [os.path.dirname(HERE), HERE]

from chenxing_amd import PagedKVCache, W4Weight, _lib               # noqa: E402
from chenxing_amd.params import RowParams, pack_rows                  # noqa: E402
from paged_decode import BF16, HEAD_DIM, HEADS, KV_HEADS, LAYERS, VOCAB, Decoder, rms  # noqa: E402


class TreeDecoder(Decoder):
    """The decoder with 4-bit weights, and a step for trees."""

    def __init__(self, seed: int = 0) -> None:
        super().__init__(seed)
        for p in self.layers:
            for name in ("up", "down"):
                p[name] = W4Weight.of(p[name].T)
        self.head = W4Weight.of(self.head, 32)

    def forward(self, ids, attend):
        x = self.emb[ids].float()
        for i, p in enumerate(self.layers):
            qkv = (rms(x) @ p["qkv"]).view(len(ids), -1, HEAD_DIM)
            o = attend(i, *qkv.split([HEADS, KV_HEADS, KV_HEADS], 1))
            x = x + (o.reshape(len(ids), -1) @ p["out"]).float()
            a, b = p["up"](rms(x)).chunk(2, 1)
            x = x + p["down"]((torch.nn.functional.silu(a) * b).to(BF16))
        return rms(x)

    def tree(self, cache, seqs, tokens, parents):
        """Appends the trees; (hidden states of all nodes, the batch, the parents)."""
        new = [len(t) for t in tokens]
        cache.extend(seqs, new)
        batch = cache.batch(seqs, new)
        par = torch.tensor([p for x in parents for p in x], dtype=torch.int32, device="cuda")
        mask, depth = _lib.tree_masks_device(par, batch["q_start"], -(-max(new) // 64))
        rope = self.rope[:batch["table"].shape[1] * cache.page_tokens]
        meta = {k: v for k, v in batch.items() if k != "max_new"}

        def attend(i, q, k, v):
            p = self.layers[i]
            q = _lib.kv_append_device(q, k, v, cache.layer(i), **meta, rope=rope, q_norm=p["qn"],
                                      k_norm=p["kn"], depth=depth)
            return _lib.tree_attention_device(q, cache.layer(i), mask=mask,
                                              max_new=batch["max_new"], **meta)
        ids = torch.tensor([t for x in tokens for t in x], device="cuda")
        return self.forward(ids, attend), batch, par

    def draft(self, cache, seq, last, rng):
        """(tokens, parents) of a tree: the likeliest tokens two levels deep, two below
        each, and a few drawn blindly."""
        probe = cache.fork(seq)[0]
        tokens, parents, levels = [last], [-1], [0]
        for _ in range(2):
            at = levels[-1]
            h = self.step(cache, [probe], [[tokens[at]]])
            for t in self.head(h)[0].topk(3).indices.tolist():
                tokens.append(t)
                parents.append(at)
            levels.append(len(tokens) - 3)
        cache.free(probe)
        for _ in range(int(rng.integers(0, 4))):
            parents.append(int(rng.integers(0, len(tokens))))
            tokens.append(int(rng.integers(0, VOCAB)))
        return tokens, parents


def main(argv=None) -> float:
    ap = argparse.ArgumentParser()
    ap.add_argument("--cache", default="bf16", choices=("bf16", "e4m3"))
    ap.add_argument("--samples", type=int, default=3)
    ap.add_argument("--rounds", type=int, default=8)
    a = ap.parse_args(argv)
    rng = np.random.default_rng(5)
    model = TreeDecoder()
    cache = PagedKVCache(LAYERS, 128, KV_HEADS, HEAD_DIM, dtype=a.cache)
    text, seqs = {}, []
    for i in range(a.samples):
        s = cache.add()
        text[s] = rng.integers(0, VOCAB, 9 + 11 * i).tolist()
        model.step(cache, [s], [text[s][:-1]])
        seqs.append(s)

    accepted = drafted = 0
    for _ in range(a.rounds):
        trees = [model.draft(cache, s, text[s][-1], rng) for s in seqs]
        tokens, parents = [t for t, _ in trees], [p for _, p in trees]
        h, batch, par = model.tree(cache, seqs, tokens, parents)
        # an id sampled after every node; the walk takes those on the path
        logits = model.head(h)
        n = len(h)
        prm = pack_rows([RowParams(temperature=0.6, top_k=50)] * n)
        prm = torch.from_numpy(prm.view(np.uint8).copy()).cuda()
        sampled = _lib.sample_device(logits, prm, torch.from_numpy(rng.random(n)).cuda())[0]
        ids = torch.tensor([t for x in tokens for t in x], dtype=torch.int32, device="cuda")
        path, count, nxt = _lib.tree_accept_device(par, ids, sampled, 4, batch["q_start"])
        kept = cache.commit(seqs, batch, path, count)
        for s, t, way, k, t1 in zip(seqs, tokens, path.tolist(), kept, nxt.tolist()):
            text[s] += [*(t[x] for x in way[1:k]), t1]
            accepted += k - 1
            drafted += len(t) - 1

    worst = 0.0
    h = model.step(cache, seqs, [[text[s][-1]] for s in seqs])
    for s, row in zip(seqs, h.float()):
        want = model.recompute(text[s])[-1].float()
        worst = max(worst, float((row - want).norm() / want.norm()))
    print(f"{a.cache}: {a.rounds} rounds of {len(seqs)} sequences, {accepted} of {drafted} drafts kept, "
          f"hidden states within {worst:.2%} of a recomputation", flush=True)
    return worst


if __name__ == "__main__":
    # bf16 hidden states of a few layers, 8-bit keys and values
    sys.exit(0 if main() < 0.1 else 1)

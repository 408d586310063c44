"""A decoder on the GPU over the paged KV cache: a prompt prefilled, its pages
forked for several samples, a batch of decode steps with the sampler, verify
rounds with rejected drafts undone, and a compaction.

    python examples/paged_decode.py [--cache bf16|e4m3] [--samples 4] [--steps 24]

The model is small and its weights random; every sequence it continued is
recomputed at the end without a cache and compared.
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from chenxing_amd import PagedKVCache, _lib, rope_table              # noqa: E402
from chenxing_amd.params import RowParams, pack_rows                  # noqa: E402

LAYERS, HIDDEN, HEADS, KV_HEADS, HEAD_DIM, VOCAB, POSITIONS = 2, 512, 8, 2, 64, 4096, 512
BF16 = torch.bfloat16


def rms(x):
    x = x.float()
    return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)).to(BF16)


class Decoder:
    """Pre-norm layers of attention (q and k normed per head) and a gated MLP."""

    def __init__(self, seed: int = 0) -> None:
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)

        def w(*shape, scale):
            return (torch.randn(*shape, generator=g, device="cuda") * scale).to(BF16)
        n = (HEADS + 2 * KV_HEADS) * HEAD_DIM
        self.emb = w(VOCAB, HIDDEN, scale=1.0)
        self.layers = [dict(qkv=w(HIDDEN, n, scale=HIDDEN ** -0.5),
                            out=w(HEADS * HEAD_DIM, HIDDEN, scale=0.5 * HIDDEN ** -0.5),
                            up=w(HIDDEN, 2 * HIDDEN, scale=HIDDEN ** -0.5),
                            down=w(HIDDEN, HIDDEN, scale=0.5 * HIDDEN ** -0.5),
                            qn=(1 + w(HEAD_DIM, scale=0.1)), kn=(1 + w(HEAD_DIM, scale=0.1)))
                       for _ in range(LAYERS)]
        self.head = w(VOCAB, HIDDEN, scale=4 * HIDDEN ** -0.5)
        self.rope = rope_table(POSITIONS, HEAD_DIM, 1000.0)

    def forward(self, ids, attend):
        """Normed hidden states of tokens ``ids``; attend(layer, q, k, v)."""
        x = self.emb[ids].float()
        for i, p in enumerate(self.layers):
            qkv = (rms(x) @ p["qkv"]).view(len(ids), -1, HEAD_DIM)
            o = attend(i, *qkv.split([HEADS, KV_HEADS, KV_HEADS], 1))
            x = x + (o.reshape(len(ids), -1) @ p["out"]).float()
            a, b = (rms(x) @ p["up"]).chunk(2, 1)
            x = x + ((torch.nn.functional.silu(a.float()) * b.float()).to(BF16) @ p["down"]).float()
        return rms(x)

    def step(self, cache, seqs, tokens):
        """Appends tokens[i] (a list) to sequence seqs[i]; hidden states of all."""
        new = [len(t) for t in tokens]
        cache.extend(seqs, new)
        meta = cache.batch(seqs, None if max(new) == 1 else new)
        most = meta.pop("max_new")
        # positions past a sequence's end are in the table's last page
        rope = self.rope[:meta["table"].shape[1] * cache.page_tokens]

        def attend(i, q, k, v):
            p = self.layers[i]
            q = _lib.kv_append_device(q, k, v, cache.layer(i), **meta, rope=rope, q_norm=p["qn"],
                                      k_norm=p["kn"])
            return _lib.paged_attention_device(q, cache.layer(i), **meta, max_new=most)
        ids = torch.tensor([t for x in tokens for t in x], device="cuda")
        return self.forward(ids, attend)

    def recompute(self, tokens):
        """Hidden states of one sequence without a cache, attention in float32."""
        n, r = len(tokens), HEAD_DIM // 2
        cs = self.rope[:n, None]

        def turn(x, w):
            x = x.float()
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()
            a, b, c, s = x[..., :r], x[..., r:], cs[..., :r], cs[..., r:]
            return torch.cat([a * c - b * s, b * c + a * s], -1).to(BF16).float()

        def attend(i, q, k, v):
            p = self.layers[i]
            q, k = turn(q, p["qn"]), turn(k, p["kn"])
            k, v = (t.float().repeat_interleave(HEADS // KV_HEADS, 1) for t in (k, v.float()))
            x = torch.einsum("ihd,jhd->hij", q, k) * HEAD_DIM ** -0.5
            x = x.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), float("-inf"))
            return torch.einsum("hij,jhd->ihd", x.softmax(-1), v).to(BF16)
        return self.forward(torch.tensor(tokens, device="cuda"), attend)


def main(argv=None) -> float:
    ap = argparse.ArgumentParser()
    ap.add_argument("--cache", default="bf16", choices=("bf16", "e4m3"))
    ap.add_argument("--samples", type=int, default=4)
    ap.add_argument("--steps", type=int, default=24)
    a = ap.parse_args(argv)
    rng = np.random.default_rng(7)
    model = Decoder()
    cache = PagedKVCache(LAYERS, 128, KV_HEADS, HEAD_DIM, dtype=a.cache)
    prompt = rng.integers(0, VOCAB, 37).tolist()
    text = {}

    # the prompt, but for its last token, which every sample processes itself
    root = cache.add()
    model.step(cache, [root], [prompt[:-1]])
    seqs = [root, *cache.fork(root, a.samples - 1)]
    for s in seqs:
        text[s] = list(prompt)

    # sampled decode steps: one launch of each call a layer for the whole batch
    prm = pack_rows([RowParams(temperature=0.8, top_p=0.9)] * len(seqs))
    prm = torch.from_numpy(prm.view(np.uint8).copy()).cuda()
    last = [prompt[-1]] * len(seqs)
    for _ in range(a.steps):
        h = model.step(cache, seqs, [[t] for t in last])
        logits = (h @ model.head.T).float()
        u = torch.from_numpy(rng.random(len(seqs))).cuda()
        last = _lib.sample_device(logits, prm, u)[0].tolist()
        for s, t in zip(seqs, last):
            text[s].append(t)

    # greedy verify rounds of one sample: four drafted tokens (some are wrong),
    # the rejected ones undone
    s, gamma, accepted = seqs[-1], 4, 0
    for _ in range(4):
        draft = rng.integers(0, VOCAB, gamma).tolist()
        probe = cache.fork(s)[0]               # draft with the model itself, two tokens long
        t = text[s][-1]
        for i in range(2):
            t = int(_lib.lmhead_argmax_device(model.step(cache, [probe], [[t]]), model.head)[0])
            draft[i] = t
        cache.free(probe)
        h = model.step(cache, [s], [[text[s][-1], *draft]])
        target = (h @ model.head.T).float()[None]
        ids = torch.tensor([draft], dtype=torch.int32, device="cuda")
        acc, nxt, _, _ = _lib.spec_verify_device(
            target, None, ids, torch.zeros(1, gamma + 1, dtype=torch.float64, device="cuda"),
            torch.zeros(1, device="cuda"))
        n = int(acc)
        accepted += n
        cache.truncate(s, cache.length(s) - (gamma - n))
        text[s] += [*draft[:n], int(nxt)]

    # half of the samples end; the pages move together, the others go on
    gone = [s for s in seqs[1:-1:2]]
    for s in gone:
        cache.free(s)
    moved = cache.compact()
    left = [s for s in seqs if s not in gone]
    worst = 0.0
    h = model.step(cache, left, [[text[s][-1]] for s in left])
    for s, row in zip(left, h.float()):
        want = model.recompute(text[s])[-1].float()
        worst = max(worst, float((row - want).norm() / want.norm()))
    print(f"{a.cache}: {len(seqs)} samples of {len(text[left[0]]) - len(prompt)} tokens or more, "
          f"{accepted} of 16 drafts accepted, {moved} pages moved, "
          f"hidden states within {worst:.2%} of a recomputation", flush=True)
    return worst


if __name__ == "__main__":
    # bf16 hidden states of a few layers, 8-bit keys and values
    sys.exit(0 if main() < 0.1 else 1)

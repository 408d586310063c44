"""A paged KV cache on the GPU: its pages, and which sequence holds which.

The reference keeps its pages, their reference counts and the sequences' block
tables on the host (``chenxing/engine/radix_kv.py:74-273``); so does this
class, over one pool tensor that the device calls take as it is:

  ``_lib.kv_append_device``        writes a step's new tokens
  ``_lib.paged_attention_device``  attends over the pages
  ``_lib.tree_attention_device``   attends for a tree of drafted tokens
  ``_lib.kv_commit_device``        keeps the accepted ones (``commit``)
  ``_lib.kv_copy_pages_device``    copies pages over all layers

Sequences share pages: ``fork`` copies none, and the first of the sharers to
grow into a page that is not full gets a copy of it (``extend``), one launch
for all the copies of a step.  Not thread-safe.
"""
from __future__ import annotations

import heapq
import math

import numpy as np

__all__ = ["PagedKVCache", "OutOfKVCacheError", "rope_table"]


class OutOfKVCacheError(RuntimeError):
    """No free page (the reference's exception of that name, radix_kv.py)."""


def rope_table(positions: int, rotary_dim: int, theta: float = 10000.0, *, linear: float = 1.0,
               yarn: float = 1.0, original: int = 4096, beta_fast: float = 32.0,
               beta_slow: float = 1.0, device="cuda"):
    """float32 [positions, rotary_dim]: the cosines of every position's angles
    (rotary_dim / 2 of them), then the sines, computed in float64.  The append
    wants a row for every position of its table's pages: a last page counts
    whole.

    Angle j of position p is p * theta ** (-2 j / rotary_dim).  ``linear``
    divides the positions.  ``yarn`` (core/tensor.py:80-121; Peng et al. 2023)
    divides the angles that turn less than ``beta_slow`` times over
    ``original`` positions, leaves those that turn more than ``beta_fast``
    times, and scales all by 0.1 ln(yarn) + 1."""
    import torch
    if positions < 0 or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("positions must be >= 0 and rotary_dim even")
    if theta <= 0 or linear <= 0 or yarn < 1 or original < 1:
        raise ValueError("theta, linear and original must be positive and yarn >= 1")
    if yarn > 1 and theta <= 1:
        raise ValueError("yarn needs pairs that turn slower one after the other: theta > 1")
    j = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
    freq = theta ** (-2.0 * j / rotary_dim) / linear
    size = 1.0
    if yarn > 1:
        def dim(turns):                       # the (real) pair that turns so often
            return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))
        lo = max(math.floor(dim(beta_fast)), 0)
        hi = min(math.ceil(dim(beta_slow)), rotary_dim - 1)
        slow = ((j - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        freq = freq * (1 - slow) + freq / yarn * slow
        size = 0.1 * math.log(yarn) + 1.0
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return (torch.cat([angle.cos(), angle.sin()], 1) * size).float()


class PagedKVCache:
    """``pages`` pages of ``page_tokens`` tokens for every layer.

    ``pool`` is [layers, pages, kv_heads, width]: bfloat16 (dtype "bf16"), or
    uint8 holding e4m3 codes and their scales (dtype "e4m3")."""

    def __init__(self, layers: int, pages: int, kv_heads: int, head_dim: int,
                 page_tokens: int = 16, dtype: str = "bf16", device="cuda", copy=None) -> None:
        import torch
        if min(layers, pages, kv_heads) < 1:
            raise ValueError("layers, pages and kv_heads must be >= 1")
        if head_dim not in (64, 128, 256):
            raise ValueError("head_dim must be 64, 128 or 256")
        if page_tokens not in (16, 32, 64, 128, 256):
            raise ValueError("page_tokens must be 16, 32, 64, 128 or 256")
        if dtype not in ("bf16", "e4m3"):
            raise ValueError("dtype must be 'bf16' or 'e4m3'")
        width = 2 * page_tokens * head_dim + (0 if dtype == "bf16" else 8 * page_tokens)
        self.pool = torch.zeros(layers, pages, kv_heads, width, device=device,
                                dtype=torch.bfloat16 if dtype == "bf16" else torch.uint8)
        self.page_tokens = page_tokens
        self._head_dim = head_dim
        self._copy = copy
        self._free = list(range(pages))       # a heap: the lowest ids are handed out first
        self._refs = [0] * pages
        self._seqs: dict[int, list] = {}      # id -> [pages, length]
        self._next = 0

    # ---------------------------------------------------------------- sequences
    def add(self) -> int:
        """A new, empty sequence's id."""
        self._seqs[self._next] = [[], 0]
        self._next += 1
        return self._next - 1

    def length(self, seq: int) -> int:
        return self._seqs[seq][1]

    def pages_of(self, seq: int) -> list[int]:
        return list(self._seqs[seq][0])

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def extend(self, seqs, counts) -> None:
        """Room for counts[i] more tokens at the end of seqs[i], for all of them
        or (``OutOfKVCacheError``) none.  Pages that a sequence would write into
        and shares are copied first."""
        if len(set(seqs)) != len(seqs) or len(seqs) != len(counts) or min(counts, default=0) < 0:
            raise ValueError("extend takes each sequence once, with a count >= 0")
        P, need, shared = self.page_tokens, 0, {}
        for s, n in zip(seqs, counts):
            pages, length = self._seqs[s]
            need += max(0, -(-(length + n) // P) - len(pages))
            if n and length % P:
                shared[pages[length // P]] = shared.get(pages[length // P], 0) + 1
        # every sharer but the last to leave it gets a copy
        need += sum(min(k, self._refs[p] - 1) for p, k in shared.items())
        if need > len(self._free):
            raise OutOfKVCacheError(f"{need} pages needed, {len(self._free)} free")
        src, dst = [], []
        for s, n in zip(seqs, counts):
            pages, length = self._seqs[s]
            at = length // P
            if n and length % P and self._refs[pages[at]] > 1:
                src.append(pages[at])
                self._refs[pages[at]] -= 1
                pages[at] = self._take()
                dst.append(pages[at])
            while len(pages) * P < length + n:
                pages.append(self._take())
            self._seqs[s][1] = length + n
        self._move(src, dst)

    def fork(self, seq: int, n: int = 1) -> list[int]:
        """n new sequences that hold the same tokens, in the same pages."""
        out = []
        for _ in range(n):
            pages, length = self._seqs[seq]
            for p in pages:
                self._refs[p] += 1
            s = self.add()
            self._seqs[s] = [list(pages), length]
            out.append(s)
        return out

    def truncate(self, seq: int, length: int) -> None:
        """The sequence's first ``length`` tokens (rejected drafts undone)."""
        pages, have = self._seqs[seq]
        if not 0 <= length <= have:
            raise ValueError(f"length must be in [0, {have}]")
        keep = -(-length // self.page_tokens)
        for p in pages[keep:]:
            self._drop(p)
        self._seqs[seq] = [pages[:keep], length]

    def commit(self, seqs, batch, path, count) -> list[int]:
        """A round of drafted trees ends: of the last tokens of seqs[i], those that
        ``batch`` appended, path[i, :count[i]] stay, in that order (``path`` and
        ``count`` as ``_lib.tree_accept_device`` gives them); how many of each.  Of a
        row of path that does not rise, or reaches past the new tokens, those before
        that stay, and path holds -1 there afterwards.  A sequence that was forked
        after the append is refused, and so is a batch whose lengths or pages are no
        longer the sequences' (after ``compact``, make it again: the tokens have moved
        with their pages)."""
        from . import _lib
        import torch
        table, start = batch["table"], batch["q_start"]
        B, M, width = len(seqs), table.shape[1], path.shape[-1]
        if len(set(seqs)) != B or table.shape[0] != B or count.shape != (B,) or path.shape != (B, width) or \
                count.device != table.device or path.device != table.device or \
                not (start is None or start.shape == (B + 1,)):
            raise ValueError("commit takes each sequence of the batch once, and path [sequences, width] "
                             "and count [sequences] on the pool's device")
        # in one copy to the host, what the moves go by
        parts = [count, batch["kv_len"], path.flatten(), table.flatten()]
        host = torch.cat(parts if start is None else [*parts, start]).cpu().numpy()
        way = host[2 * B:(2 + width) * B].reshape(B, width)
        held, ends = host[(2 + width) * B:], host[(2 + width + M) * B:]
        kept, lens = host[:B].tolist(), host[B:2 * B].tolist()
        new = [1] * B if start is None else (ends[1:] - ends[:-1]).tolist()
        P, at, now, written = self.page_tokens, [], [], []
        for i, (s, c, n, was) in enumerate(zip(seqs, kept, new, lens)):
            pages, length = self._seqs[s]
            if not 0 <= c <= min(n, width, length):
                raise ValueError("count must be in [0, new tokens of the sequence], and path that wide")
            p0, p1 = (length - n) // P, len(pages)
            if was != length or p1 > M:
                raise ValueError("the sequences' lengths are not those of the batch")
            at += range(i * M + p0, i * M + p1)
            now += pages[p0:]
            if c:
                written += pages[p0:-(-(length - n + c) // P)]
        if held[at].tolist() != now:
            raise ValueError("the sequences' pages are not those of the batch")
        if any(self._refs[p] > 1 for p in written):
            raise ValueError("commit moves tokens in pages that another sequence holds too: "
                             "commit first, then fork")
        _lib.kv_commit_device(self.pool, self._head_dim, table, batch["kv_len"], path, count, start, P)
        moved = np.arange(width) < host[:B, None]
        rises = way < np.reshape(new, (B, 1))
        rises[:, :1] &= way[:, :1] >= 0
        rises[:, 1:] &= way[:, 1:] > way[:, :-1]
        if (moved & ~rises).any():             # the device has marked where those rows end
            kept = [min(c, [*row, -1].index(-1)) for row, c in zip(path.tolist(), kept)]
        for s, c, n in zip(seqs, kept, new):
            self.truncate(s, self._seqs[s][1] - n + c)
        return kept

    def free(self, seq: int) -> None:
        self.truncate(seq, 0)
        del self._seqs[seq]

    def compact(self) -> int:
        """Moves the pages in use to the lowest ids; how many moved."""
        used = sum(r > 0 for r in self._refs)
        dst = sorted(p for p in self._free if p < used)
        src = [p for p in range(used, len(self._refs)) if self._refs[p]]
        to = dict(zip(src, dst))
        for s, d in to.items():
            self._refs[d], self._refs[s] = self._refs[s], 0
        for q in self._seqs.values():
            q[0] = [to.get(p, p) for p in q[0]]
        self._free = [p for p, r in enumerate(self._refs) if not r]
        self._move(src, dst)
        return len(src)

    # ---------------------------------------------------------------- device calls
    def layer(self, i: int):
        """One layer's pages, as the device calls take them."""
        return self.pool[i]

    def batch(self, seqs, new=None) -> dict:
        """The table, kv_len, q_start and most new tokens (``max_new``) of a
        pass over sequences whose last new[i] tokens are new (None: one each),
        as the device calls' keyword arguments ``table``, ``kv_len``,
        ``q_start`` and ``page_tokens``, on the pool's device."""
        import torch
        B = len(seqs)
        held = [self._seqs[s] for s in seqs]
        width = max([len(p) for p, _ in held] + [1])
        table = np.full((B, width), -1, np.int32)
        for b, (p, _) in enumerate(held):
            table[b, :len(p)] = p
        lens = np.array([n for _, n in held], np.int32)
        start = None if new is None else np.concatenate([[0], np.cumsum(new)]).astype(np.int32)

        def up(a):
            return torch.from_numpy(a).to(self.pool.device)
        return dict(table=up(table), kv_len=up(lens), q_start=None if new is None else up(start),
                    page_tokens=self.page_tokens, max_new=1 if new is None else max([1, *new]))

    # ---------------------------------------------------------------- pages
    def _take(self) -> int:
        p = heapq.heappop(self._free)
        self._refs[p] = 1
        return p

    def _drop(self, p: int) -> None:
        self._refs[p] -= 1
        if self._refs[p] == 0:
            heapq.heappush(self._free, p)

    def _move(self, src, dst) -> None:
        if not src:
            return
        import torch
        pairs = torch.tensor([src, dst], dtype=torch.int32).to(self.pool.device)
        if self._copy is None:
            from . import _lib
            _lib.kv_copy_pages_device(self.pool, pairs[0], pairs[1])
        else:
            self._copy(self.pool, pairs[0], pairs[1])

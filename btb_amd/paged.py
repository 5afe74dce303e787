"""Sequences of unlike length and age over one paged cache held in 4 bits: prompts go in beside other sequences' next tokens, a
sequence branches into others that share its pages, ended ones give theirs back.

`Paged` runs a dense stack (`DecodeStep`'s weights) through `HipCard.norm_rope_axes`, `kv4_write` and `attn_kv4`, and keeps the books of the
pages: which sequence names which, how often each is named, which are free. `pages_fork` and `pages_compact` move what the books say in all layers
at once. A page takes 134 bytes a token, kv head and layer at head_dim 128, where a bf16 cache takes 512. No counterpart in the reference.
"""

from __future__ import annotations

import math
from itertools import islice
from typing import Any, Mapping, Sequence

import torch

from .decode import StackConfig, recording, rope_axes, rope_tables


class Paged:
    """Up to `seqs` sequences over `pages` pages of `page` tokens. A pass takes up to `rows` tokens of any of them; longer ones go in by
    several passes. A sequence has at most `longest` tokens."""

    def __init__(self, card: Any, cfg: StackConfig, weights: dict[str, Any], seqs: int, pages: int, page: int = 64, rows: int = 32,
                 longest: int = 32768) -> None:
        if min(seqs, pages, rows, longest) < 1 or rows < seqs:
            raise ValueError("[paged] seqs, pages, rows and longest are 1 or more, and a pass has a row for every sequence")
        dev = torch.device("cuda")
        self.card, self.cfg, self.w = card, cfg, weights
        self.seqs, self.page, self.rows, self.longest = seqs, page, rows, longest
        self.pool = card.kv4_pool(pages, cfg.kv_heads, cfg.head_dim, page, layers=cfg.layers)
        self.cos, self.sin = rope_tables(cfg, longest, dev)
        self.axes = rope_axes([cfg.head_dim // 2], dev)
        width = -(-longest // page)
        self.tables = torch.full((seqs, width), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(seqs, dtype=torch.int32, device=dev)
        self.held: list[list[int]] = [[] for _ in range(seqs)]  # each sequence's pages
        self.length = [0] * seqs
        self.named = [0] * pages                                # how many sequences hold each page
        self._sent = True                                       # whether tables and lens are the books'
        self._narrow, self._wide = _Pass(self, seqs), _Pass(self, rows)

    @property
    def free(self) -> int:
        """pages that nobody holds"""
        return self.named.count(0)

    def _seq(self, b: int) -> int:
        if not 0 <= b < self.seqs:
            raise ValueError(f"[paged] there are {self.seqs} sequences, none of them is {b}")
        return b

    def _take(self, n: int, what: str) -> list[int]:
        """the first n free pages"""
        found = list(islice((p for p, k in enumerate(self.named) if k == 0), n))
        if len(found) < n:
            raise RuntimeError(f"[paged] {what} needs {n} pages, {len(found)} are free")
        return found

    def advance(self, tokens: Mapping[int, Sequence[int]]) -> dict[int, torch.Tensor]:
        """these sequences' next tokens (a sequence's first ones: its prompt); the logits [vocab] behind each one's last. Where a pass
        raises, the sequences keep what the passes before it brought."""
        left = {b: [int(t) for t in part] for b, part in sorted(tokens.items())}
        for b, part in left.items():
            if any(not 0 <= t < self.cfg.vocab for t in part):
                raise ValueError(f"[paged] sequence {b} was given tokens outside 0 .. {self.cfg.vocab - 1}")
            if self.length[self._seq(b)] + len(part) > self.longest or not part:
                raise ValueError(f"[paged] sequence {b} has {self.length[b]} of {self.longest} tokens, {len(part)} more were given")
        grown = {b: -(-(self.length[b] + len(part)) // self.page) - len(self.held[b]) for b, part in left.items()}
        fresh = self._take(sum(grown.values()), "a pass")
        out: dict[int, torch.Tensor] = {}
        try:
            for b, n in grown.items():
                for p in fresh[:n]:
                    self.named[p] = 1
                self.held[b] += fresh[:n]
                fresh = fresh[n:]
            if any(grown.values()) or not self._sent:
                self._books()
            while left:
                p = self._narrow if sum(len(part) for part in left.values()) <= self.seqs else self._wide
                room, now = p.T, {}
                for i, (b, part) in enumerate(left.items()):  # a row at least for each that is left
                    now[b] = part[:room - (len(left) - 1 - i)]
                    room -= len(now[b])
                logits = p.run(now)
                left = {b: part[len(now[b]):] for b, part in left.items() if len(part) > len(now[b])}
                out.update({b: logits[i].clone() for i, b in enumerate(now) if b not in left})  # (the next pass writes over them)
        except BaseException:
            for b in grown:  # pages that it has not come to need
                del self.held[b][-(-self.length[b] // self.page):]
            self.named = [0] * len(self.named)
            for row in self.held:
                for p in row:
                    self.named[p] += 1
            self._books()
            raise
        return out

    def fork(self, branches: Mapping[int, int]) -> None:
        """sequences branches[dst] = src: each dst, which holds nothing, goes on from src's tokens"""
        if not branches:
            return
        for dst, src in branches.items():
            if self.held[self._seq(dst)] or not self.length[self._seq(src)] or src in branches:
                raise ValueError(f"[paged] sequence {dst} is to be empty and {src} not, for one to go on from the other")
        parts = {dst: src for dst, src in branches.items() if self.length[src] % self.page}
        fresh = dict(zip(parts, self._take(len(parts), "a fork")))
        none = next(iter(fresh.values()), 0)
        if not self._sent:
            self._books()
        i32 = dict(dtype=torch.int32, device=self.lens.device)
        self.card.pages_fork(self.pool, self.tables, self.lens, torch.tensor(list(branches.values()), **i32),
                             torch.tensor(list(branches), **i32), torch.tensor([fresh.get(d, none) for d in branches], **i32), self.page)
        for dst, src in branches.items():
            self.length[dst] = self.length[src]
            self.held[dst] = self.held[src][:self.length[src] // self.page] + ([fresh[dst]] if dst in fresh else [])
            for p in self.held[dst]:
                self.named[p] += 1

    def end(self, b: int) -> None:
        """the sequence gives its pages back; its number can begin anew"""
        for p in self.held[self._seq(b)]:
            self.named[p] -= 1
        self.held[b], self.length[b] = [], 0
        self._books()

    def compact(self) -> int:
        """the pages in use moved to the front of the pool; how many they are"""
        if not self._sent:
            self._books()
        self.card.pages_compact(self.pool, self.tables, self.lens, self.page)
        used = [p for p, k in enumerate(self.named) if k]
        n = len(used)
        holes = [p for p in range(n) if not self.named[p]]
        goes = dict(zip([p for p in used if p >= n], holes))
        self.held = [[goes.get(p, p) for p in row] for row in self.held]
        counts = {goes.get(p, p): self.named[p] for p in used}
        self.named = [counts.get(p, 0) for p in range(len(self.named))]
        return n

    def capture(self) -> None:
        """records the pass of a token a sequence; passes of as many rows or fewer replay it from then on"""
        self._narrow.capture()

    def _books(self) -> None:
        """tables and lengths as the books have them, on the GPU; where that fails, the next call sends them"""
        self._sent = False
        width = self.tables.shape[1]
        self.tables.copy_(torch.tensor([row + [-1] * (width - len(row)) for row in self.held], dtype=torch.int32))
        self.lens.copy_(torch.tensor(self.length, dtype=torch.int32))
        self._sent = True


class _Pass:
    """up to T rows of any sequences through the stack: buffers, and the kernel sequence"""

    def __init__(self, f: Paged, T: int) -> None:
        cfg, dev = f.cfg, torch.device("cuda")
        bf, i32 = dict(dtype=torch.bfloat16, device=dev), dict(dtype=torch.int32, device=dev)
        Hk, D = cfg.kv_heads, cfg.head_dim
        self.f, self.T = f, T
        self.ids, self.slots = torch.zeros(T, **i32), torch.full((T,), -1, **i32)
        self.pos = torch.zeros(1, T, **i32)
        self.first, self.last = torch.zeros(f.seqs + 1, **i32), torch.zeros(f.seqs, **i32)
        self.h, self.x, self.y = (torch.zeros(T, cfg.hidden, **bf) for _ in range(3))
        self.ends = torch.zeros(f.seqs, cfg.hidden, **bf)
        self.qkv = torch.zeros(T, cfg.qkv_rows, **bf)
        self.q, self.att = (torch.zeros(T, cfg.q_heads * D, **bf) for _ in range(2))
        self.K, self.V = (torch.zeros(Hk, T, D, **bf) for _ in range(2))  # the pass's own, on their way to the pages
        self.gu, self.m = torch.zeros(T, 2 * cfg.intermediate, **bf), torch.zeros(T, cfg.intermediate, **bf)
        self.logits = torch.zeros(f.seqs, cfg.vocab, **bf)
        self.scratch = f.card.attn_kv4_scratch(T, f.seqs, cfg.q_heads, Hk, D, f.longest, dev)
        self.graph: torch.cuda.CUDAGraph | None = None

    def run(self, tokens: Mapping[int, Sequence[int]]) -> torch.Tensor:
        """the sequences' next tokens, in ascending order of their numbers; the logits behind each one's last, in that order"""
        f = self.f
        ids, pos, first, last, length = [], [], [0], [], list(f.length)
        for b in range(f.seqs):
            part = tokens.get(b, ())
            ids += part
            pos += range(f.length[b], f.length[b] + len(part))
            first.append(len(ids))
            if part:
                last.append(len(ids) - 1)
            length[b] += len(part)
        n = len(ids)
        for t, values in ((self.ids, ids), (self.pos[0], pos), (self.slots, list(range(n)))):
            t.copy_(torch.tensor(values + [-1 if t is self.slots else 0] * (self.T - n), dtype=torch.int32))
        self.first.copy_(torch.tensor(first, dtype=torch.int32))
        self.last.copy_(torch.tensor(last + [0] * (f.seqs - len(last)), dtype=torch.int32))
        f.lens.copy_(torch.tensor(length, dtype=torch.int32))
        if self.graph is not None:
            self.graph.replay()
        else:
            self._body()
        f.length = length
        return self.logits

    def _body(self) -> None:
        f, k, cfg, w = self.f, self.f.card, self.f.cfg, self.f.w
        Hq, Hk, D = cfg.q_heads, cfg.kv_heads, cfg.head_dim
        k.embed(w["embed"], self.ids, self.h)
        before = None
        for i in range(cfg.layers):
            L = f"layers.{i}."
            k.add_rmsnorm(self.h, before, w[L + "ln1"], cfg.eps, self.x)
            w[L + "qkv"].matvec(self.x, self.qkv)
            k.norm_rope_axes(self.qkv, w.get(L + "wq"), w.get(L + "wk"), cfg.eps, f.cos, f.sin, self.pos, f.axes, self.slots, self.K,
                             self.V, self.q, Hq, Hk, D)
            k.kv4_write(self.K.transpose(0, 1), self.V.transpose(0, 1), f.pool[i], f.tables, f.lens, first=self.first)
            self._attend(i)
            w[L + "o"].matvec(self.att, self.y)
            k.add_rmsnorm(self.h, self.y, w[L + "ln2"], cfg.eps, self.x)
            w[L + "gu"].matvec(self.x, self.gu)
            k.silu_mul(self.gu, self.m)
            w[L + "down"].matvec(self.m, self.y)
            before = self.y
        k.add_rmsnorm(self.h, before, w["norm"], cfg.eps, self.x)
        torch.index_select(self.x, 0, self.last, out=self.ends)
        w["head"].matvec(self.ends, self.logits)

    def _attend(self, i: int) -> None:
        f, cfg = self.f, self.f.cfg
        f.card.attn_kv4(self.q, f.pool[i], f.tables, f.lens, self.att, cfg.q_heads, cfg.kv_heads, cfg.head_dim, 1.0 / math.sqrt(cfg.head_dim),
                        self.scratch, first=self.first, keys_cap=f.longest)

    def capture(self) -> None:
        # with no rows at all: nothing is written to the cache, neither by the pass before the recording nor by the recording
        self.first.zero_()
        self.slots.fill_(-1)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self._body()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with recording(graph):
            self._body()
        self.graph = graph

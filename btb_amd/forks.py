"""Several continuations of one prompt over a shared, bounded cache: the prompt goes in by chunks, the keys that its attention used
least are dropped whenever the cache holds more than its budget, and rows of their own then decode over what is left, which each
pass reads once for all of them.

`Forks` runs a dense stack (`DecodeStep`'s weights) through `HipCard.norm_rope_axes`, `attn_shared`, `attn_mass` and `kv_evict`. A
layer's cache is one arena [Hk, slots, D]: the prompt's keys first, then a stretch of `steps` slots a row, which are neither weighed
nor cut: the budget is the prompt's. After a cut a key's slot is no longer its token's number and differs from head to head, so the
numbers travel beside the cache (`pos`) and new keys are roped at their own places. No counterpart in the reference.
"""

from __future__ import annotations

import math
from typing import Any, Sequence

import torch

from .decode import StackConfig, recording, rope_axes, rope_tables


class Forks:
    """`rows` continuations of up to `steps` tokens each over at most `budget` keys a head of one prompt, which goes in `chunk` tokens
    at a time and stands on any places up to `positions` less `steps`. Of its keys the first `sinks` and the newest `recent` always
    stay. `sections`: how many frequencies each position axis turns (one axis: all of them), `interleaved` as in `rope_axes`."""

    def __init__(self, card: Any, cfg: StackConfig, weights: dict[str, Any], rows: int, budget: int, steps: int, chunk: int = 32,
                 sinks: int = 4, recent: int = 64, positions: int = 32768, sections: Sequence[int] | None = None,
                 interleaved: bool = False) -> None:
        if min(rows, budget, steps, chunk) < 1 or not 0 <= sinks + recent <= budget:
            raise ValueError("[forks] rows, budget, steps and chunk are 1 or more, and the budget holds what always stays")
        sections = [cfg.head_dim // 2] if sections is None else list(sections)
        if sum(sections) != cfg.head_dim // 2:
            raise ValueError(f"[forks] the sections share {cfg.head_dim // 2} frequencies, got {sections}")
        dev = torch.device("cuda")
        self.card, self.cfg, self.w = card, cfg, weights
        self.rows, self.budget, self.steps, self.chunk, self.sinks, self.recent = rows, budget, steps, chunk, sinks, recent
        self.positions, self.scale = positions, 1.0 / math.sqrt(cfg.head_dim)
        self.held = budget + chunk  # slots of the prompt's keys: a pass more than the budget
        cap, Hk, D = self.held + rows * steps, cfg.kv_heads, cfg.head_dim
        self.kv = torch.zeros(cfg.layers, 2, Hk, cap, D, dtype=torch.bfloat16, device=dev)
        self.mass = torch.zeros(cfg.layers, Hk, self.held, dtype=torch.float32, device=dev)
        self.pos = torch.zeros(cfg.layers, Hk, self.held, dtype=torch.int32, device=dev)
        self.idx = torch.empty(cfg.layers, Hk, budget, dtype=torch.int32, device=dev)
        self.cos, self.sin = rope_tables(cfg, positions, dev)
        self.axes = rope_axes(sections, dev, interleaved)
        self.n = 0      # keys of the prompt a head holds
        self.seen = 0   # tokens of the prompt so far
        self.place = 0  # where the next token stands on every axis: one past the largest place so far
        self.taken = 0  # steps the rows have taken
        self.begun = False  # whether the rows' tokens and slots describe the cache
        self._pass = _Pass(self, chunk, self.held, chunk)
        self._step = _Pass(self, rows, self.held, steps)
        self.graph: torch.cuda.CUDAGraph | None = None

    def prompt(self, tokens: Sequence[int], places: torch.Tensor | None = None) -> torch.Tensor:
        """the prompt's next tokens, at `places` (integers [axes, tokens]) or one after the other on every axis, from one
        past the largest place so far; the last one's logits [vocab]. Rows that had begun, with no step yet, begin again."""
        if self.taken:
            raise RuntimeError("[forks] the rows have begun: the prompt is closed")
        if not tokens:
            raise ValueError("[forks] no tokens")
        low, end = self.place, self.place + len(tokens)
        if places is not None:
            axes = self._pass.pos.shape[0]
            if places.is_floating_point() or places.shape != (axes, len(tokens)):
                raise ValueError(f"[forks] places are integers [{axes}, {len(tokens)}], got {places.dtype} {list(places.shape)}")
            low, top = (int(v) for v in places.aminmax())
            end = max(self.place, top + 1)
        if low < 0 or end + self.steps > self.positions:
            raise ValueError(f"[forks] {len(tokens)} tokens on places from {low}, {self.steps} steps from {end} on: the tables hold "
                             f"{self.positions} positions")
        self.begun = False  # rows that had begun begin again, behind these tokens
        p, logits = self._pass, None
        for at in range(0, len(tokens), self.chunk):
            part = tokens[at:at + self.chunk]
            T = len(part)
            if T != p.T:
                p = _Pass(self, T, self.held, T)
            first = torch.arange(T, dtype=torch.int32, device="cuda")
            p.ids.copy_(torch.tensor(list(part), dtype=torch.int32))
            p.pos.copy_(first + self.place + at if places is None else places[:, at:at + T])
            p.slots.copy_(first + self.n)
            # a chain: every row sees the keys there are and the pass's own up to itself
            p.lay.copy_(self.card.shared_layout(0, self.n, [(self.n, t + 1) for t in range(T)]))
            p.see.copy_(first + self.n + 1)
            logits = p.run(self.n + T)
            self.pos[:, :, self.n:self.n + T] = first + self.seen
            self.n += T
            self.seen += T
            self.cut()
        self.place = end
        return logits[-1]

    def cut(self) -> None:
        """every layer's cache back to the budget, in place; one within it stays as it is"""
        if self.n <= self.budget:
            return
        K, V = self.kv[:, 0], self.kv[:, 1]
        self.n = self.card.kv_evict(self.mass, self.pos, K, V, self.n, self.budget, K, V, self.mass, self.pos, self.idx,
                                    sinks=self.sinks, recent_from=self.seen - self.recent)

    def begin(self, tokens: Sequence[int]) -> None:
        """the rows' first tokens: one a row"""
        if len(tokens) != self.rows or not self.seen:
            raise ValueError(f"[forks] {self.rows} first tokens after a prompt, got {len(tokens)} after {self.seen}")
        p = self._step
        base = [self.held + t * self.steps for t in range(self.rows)]
        p.ids.copy_(torch.tensor(list(tokens), dtype=torch.int32))
        p.pos.fill_(self.place)
        p.slots.copy_(torch.tensor(base, dtype=torch.int32))
        p.lay.copy_(self.card.shared_layout(0, self.n, [(b, 1) for b in base]))
        self.taken, self.begun = 0, True

    def step(self) -> torch.Tensor:
        """a token more in every row, the greedy picks fed forward; the logits [rows, vocab]. Recorded by `capture`: replayed."""
        self._need_rows()
        self.taken += 1
        if self.graph is not None:
            self.graph.replay()
            return self._step.logits
        return self._body()

    def _need_rows(self) -> None:
        if not self.begun:  # their slots are the prompt's first, or their layout that of a prompt before its last tokens
            raise RuntimeError("[forks] the rows have not begun behind the prompt as it is: begin first")
        if self.taken >= self.steps:  # the next slot is another row's
            raise RuntimeError(f"[forks] the rows have room for {self.steps} tokens")

    def _body(self) -> torch.Tensor:
        p = self._step
        p.run(0)
        self.card.argmax(p.logits, p.ids)
        p.pos += 1
        p.slots += 1
        p.lay[3::2] += 1
        return p.logits

    def capture(self) -> None:
        """records a step, for which the rows have room; their state is as before (`begin` first)"""
        self._need_rows()
        p = self._step
        state = [t.clone() for t in (p.ids, p.pos, p.slots, p.lay)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self._body()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with recording(g):
            self._body()
        for t, was in zip((p.ids, p.pos, p.slots, p.lay), state):
            t.copy_(was)
        self.graph = g


class _Pass:
    """T rows through the stack: buffers, and the kernel sequence"""

    def __init__(self, f: Forks, T: int, prefix_cap: int, own_cap: int) -> None:
        cfg, dev = f.cfg, torch.device("cuda")
        bf = dict(dtype=torch.bfloat16, device=dev)
        i32 = dict(dtype=torch.int32, device=dev)
        self.f, self.T, self.prefix_cap, self.own_cap = f, T, prefix_cap, own_cap
        self.ids, self.slots, self.see = (torch.zeros(T, **i32) for _ in range(3))
        self.pos = torch.zeros(int(f.axes.max()) + 1, T, **i32)
        self.lay = torch.zeros(2 + 2 * T, **i32)
        self.h, self.x, self.y = (torch.zeros(T, cfg.hidden, **bf) for _ in range(3))
        self.qkv = torch.zeros(T, cfg.qkv_rows, **bf)
        self.q, self.att = (torch.zeros(T, cfg.q_heads * cfg.head_dim, **bf) for _ in range(2))
        self.lse = torch.zeros(T, cfg.q_heads, dtype=torch.float32, device=dev)
        self.gu, self.m = torch.zeros(T, 2 * cfg.intermediate, **bf), torch.zeros(T, cfg.intermediate, **bf)
        self.logits = torch.zeros(T, cfg.vocab, **bf)
        self.scratch = f.card.attn_shared_scratch(T, cfg.q_heads, cfg.kv_heads, cfg.head_dim, prefix_cap, own_cap, dev)

    def run(self, weigh: int) -> torch.Tensor:
        """one pass; `weigh` > 0: the weight that the first so many keys receive from it is added to their mass"""
        f, k, cfg, w = self.f, self.f.card, self.f.cfg, self.f.w
        Hq, Hk, D = cfg.q_heads, cfg.kv_heads, cfg.head_dim
        k.embed(w["embed"], self.ids, self.h)
        before = None
        for i in range(cfg.layers):
            L = f"layers.{i}."
            K, V = f.kv[i, 0], f.kv[i, 1]
            k.add_rmsnorm(self.h, before, w[L + "ln1"], cfg.eps, self.x)
            w[L + "qkv"].matvec(self.x, self.qkv)
            k.norm_rope_axes(self.qkv, w.get(L + "wq"), w.get(L + "wk"), cfg.eps, f.cos, f.sin, self.pos, f.axes, self.slots, K, V,
                             self.q, Hq, Hk, D)
            k.attn_shared(self.q, K, V, self.att, self.lay, Hq, Hk, D, f.scale, self.prefix_cap, self.own_cap, self.scratch,
                          lse=self.lse)
            if weigh:
                fresh = f.mass[i, :, weigh - self.T:weigh]
                fresh.zero_()  # the pass's own keys start with none
                k.attn_mass(self.q, K, self.lse, self.see, f.mass[i], Hq, Hk, D, f.scale, weigh)
            w[L + "o"].matvec(self.att, self.y)
            k.add_rmsnorm(self.h, self.y, w[L + "ln2"], cfg.eps, self.x)
            w[L + "gu"].matvec(self.x, self.gu)
            k.silu_mul(self.gu, self.m)
            w[L + "down"].matvec(self.m, self.y)
            before = self.y
        k.add_rmsnorm(self.h, before, w["norm"], cfg.eps, self.x)
        w["head"].matvec(self.x, self.logits)
        return self.logits

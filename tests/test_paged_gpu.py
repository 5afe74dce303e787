"""`Paged` on the tiny Qwen3 fixture: every layer's attention in every pass is held against the bf16 operators' over the cache read back,
however tokens are dealt to passes and pages (two whole runs are not compared: where a bf16 step decides a 4-bit code they go apart);
sequences that branch, end and move keep their tokens; the books stay true.

Bar of the attention, w = 2^-8 half a bf16 step: the values read back are rounded once, and the outputs of both; weights go into the
products to 2^-11 and 2^-16: together less than 4 w of the largest |value| a row sees."""

from __future__ import annotations

import os

import numpy as np
import pytest
import torch

from btb_amd.load import load_stack
from btb_amd.paged import Paged
from oracle import kv4

from .helpers import GOLDEN

pytestmark = pytest.mark.gpu

PROMPT = [3, 17, 42, 5, 99, 120, 7, 7, 200, 12, 45, 8, 3, 17, 60, 61]


@pytest.fixture(scope="module")
def stack(card):
    return load_stack(card, os.path.join(GOLDEN, "tiny_qwen3"))


def _long(n, seed):
    return [(seed * i * i + 3 * i + 11) % 250 for i in range(n)]


def _books(f):
    """tables on the GPU, counts and free pages agree"""
    torch.cuda.synchronize()
    counts = [0] * f.pool.shape[1]
    for b in range(f.seqs):
        assert len(f.held[b]) == -(-f.length[b] // f.page)
        assert f.tables[b].tolist() == f.held[b] + [-1] * (f.tables.shape[1] - len(f.held[b]))
        for p in f.held[b]:
            counts[p] += 1
    assert counts == f.named and f.lens.tolist() == f.length and f.free == counts.count(0)


class _Checked(Paged):
    """the passes, each layer's attention held against `attn_shared` over every sequence's cache as it reads back in bf16"""

    def __init__(self, *a, **kw):
        super().__init__(*a, **kw)
        self.checked = 0
        for p in (self._narrow, self._wide):
            p._attend = lambda i, p=p, attend=p._attend: self._check(p, i, attend)

    def _check(self, p, i, attend):
        attend(i)
        cfg, k = self.cfg, self.card
        Hq, Hk, D = cfg.q_heads, cfg.kv_heads, cfg.head_dim
        first, lens = p.first.tolist(), self.lens.tolist()
        for b in range(self.seqs):
            r, n = first[b + 1] - first[b], lens[b]
            if not r:
                continue
            K, V = (torch.zeros(Hk, n, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
            k.kv4_read(self.pool[i], self.tables[b:b + 1], self.lens[b:b + 1], K.transpose(0, 1), V.transpose(0, 1))
            lay = k.shared_layout(0, 0, [(0, n - r + t + 1) for t in range(r)])
            q = p.q[first[b]:first[b + 1]].contiguous()
            att = torch.zeros_like(q)
            k.attn_shared(q, K, V, att, lay, Hq, Hk, D, D**-0.5, 0, n, k.attn_shared_scratch(r, Hq, Hk, D, 0, n))
            got, want = (x.float().view(r, Hk, -1, D) for x in (p.att[first[b]:first[b + 1]], att))
            most = V.float().abs().amax(dim=(1, 2))[None, :, None, None]
            assert bool(((got - want).abs() <= 4 * 2.0**-8 * most).all()), (i, b)
            self.checked += r


@pytest.mark.parametrize("rows,page", [(4, 32), (16, 64), (7, 96)])
def test_every_layer_attends_to_its_cache(card, stack, rows, page):
    cfg, w = stack
    prompts = {0: PROMPT, 2: _long(75, 7), 3: _long(33, 5)}
    f = _Checked(card, cfg, w, 4, 24, page=page, rows=rows, longest=256)
    a = f.advance(prompts)
    _books(f)
    assert sorted(a) == [0, 2, 3] and f.checked == 124 * cfg.layers
    for i in range(40):
        tokens = {s: [(13 * i + s) % 250] for s in ((0, 2, 3) if i % 3 else (0, 3))}
        if i == 5:
            tokens[1] = _long(20, 3)  # a prompt beside the others' tokens
        a = f.advance(tokens)
        assert sorted(a) == sorted(tokens) and all(bool(x.isfinite().all()) for x in a.values())
    _books(f)


def test_layer_zero_holds_its_keys(card, stack):
    """no attention comes before layer 0's keys and values: the cache holds their 4 bits at their places, whatever passes they came by"""
    cfg, w = stack
    tokens = _long(90, 9)
    pools = []
    for rows, cuts in ((3, [90]), (32, [1, 40, 90])):
        f = Paged(card, cfg, w, 1, 5, page=32, rows=rows, longest=128)
        at = 0
        for c in cuts:
            f.advance({0: tokens[at:c]})
            at = c
        torch.cuda.synchronize()
        pools.append([kv4.tokens(f.pool[0].cpu().numpy(), f.tables[0].cpu().numpy(), 90, 32, g, cfg.head_dim) for g in range(cfg.kv_heads)])
    for (K, V, there), (K2, V2, _) in zip(*pools):
        assert there.all() and np.array_equal(K, K2) and np.array_equal(V, V2)


def test_branches_ends_and_moves(card, stack):
    cfg, w = stack
    f = Paged(card, cfg, w, 5, 20, page=32, rows=16, longest=200)
    f.advance({0: _long(70, 7), 1: _long(64, 5)})
    f.fork({2: 0, 3: 0, 4: 1})
    _books(f)
    assert f.free == 20 - 3 - 2 - 2  # whole pages are shared, each branch of a partial one has its own
    same = f.advance({s: [9] for s in (0, 2, 3)})
    assert torch.equal(same[0], same[2]) and torch.equal(same[0], same[3])
    unlike = f.advance({0: [1], 2: [2], 3: [2], 1: [4], 4: [4]})
    assert torch.equal(unlike[2], unlike[3]) and torch.equal(unlike[1], unlike[4]) and not torch.equal(unlike[0], unlike[2])
    _books(f)
    # layer 0 of a branch is that of a sequence of its own
    g = Paged(card, cfg, w, 1, 8, page=64, rows=16, longest=200)
    g.advance({0: _long(70, 7) + [9, 2]})
    torch.cuda.synchronize()
    for head in range(cfg.kv_heads):
        mine = kv4.tokens(f.pool[0].cpu().numpy(), f.tables[2].cpu().numpy(), 72, 32, head, cfg.head_dim)
        own = kv4.tokens(g.pool[0].cpu().numpy(), g.tables[0].cpu().numpy(), 72, 64, head, cfg.head_dim)
        assert np.array_equal(mine[0], own[0]) and np.array_equal(mine[1], own[1])
    f.end(0)
    f.end(1)
    _books(f)
    want = f.advance({2: [8], 3: [9], 4: [10]})
    again = {2: 8, 3: 9, 4: 10}
    before = [f.pool[:, p].clone() for p in f.held[3]]
    used = f.compact()
    _books(f)
    assert used == 20 - f.free and max(p for row in f.held for p in row) == used - 1
    assert all(torch.equal(x, f.pool[:, p]) for x, p in zip(before, f.held[3]))
    f.advance({0: _long(40, 3)})
    more = f.advance({s: [t] for s, t in again.items()})
    assert not torch.equal(more[2], want[2]) and all(bool(x.isfinite().all()) for x in more.values())
    _books(f)


def test_recorded(card, stack):
    """replayed passes of unlike sequences, through new pages and a compaction, are the eager ones"""
    cfg, w = stack
    one, two = (Paged(card, cfg, w, 3, 16, page=32, rows=8, longest=160) for _ in range(2))
    for f in (one, two):
        f.advance({0: _long(30, 7), 1: _long(50, 3)})
    pool = one.pool.clone()
    one.capture()
    torch.cuda.synchronize()
    assert torch.equal(pool, one.pool)
    for i in range(36):
        tokens = {s: [(7 * i + s) % 250] for s in ([0, 1], [1], [0, 2], [0, 1, 2])[i % 4]}
        if i == 17:
            for f in (one, two):
                f.end(1)
                f.compact()
                f.advance({1: _long(21, 11)})
        a, b = one.advance(tokens), two.advance(tokens)
        assert sorted(a) == sorted(b) and all(torch.equal(a[s], b[s]) for s in a), i
    _books(one)
    assert one.length == two.length


def test_refusals(card, stack):
    cfg, w = stack
    with pytest.raises(ValueError):
        Paged(card, cfg, w, 4, 8, rows=3)
    with pytest.raises(ValueError):
        Paged(card, cfg, w, 2, 8, page=48)
    f = Paged(card, cfg, w, 2, 3, page=32, rows=8, longest=80)
    for bad in ({2: [1]}, {2: []}, {-1: [1]}, {0: []}, {0: [1] * 81}):
        with pytest.raises(ValueError):
            f.advance(bad)
    f.advance({0: [1] * 40})
    with pytest.raises(RuntimeError):
        f.advance({1: [1] * 40})  # two pages, one is free
    _books(f)
    for bad in ({0: 1}, {1: 1}, {1: 5}, {5: 0}):
        with pytest.raises(ValueError):
            f.fork(bad)
    f.fork({1: 0})
    with pytest.raises(ValueError):
        f.fork({1: 0})  # it holds something
    assert f.free == 0
    with pytest.raises(RuntimeError):
        f.advance({0: [1] * 30})
    f.end(0)
    assert f.free == 1
    with pytest.raises(RuntimeError):
        f.fork({0: 1}) if f.free == 0 else f.advance({0: [1] * 40})
    _books(f)


def test_a_pass_that_raises(card, stack):
    """the second of three passes: the sequences have the first one's tokens and its pages, and go on from there"""
    cfg, w = stack
    one, two = (Paged(card, cfg, w, 2, 12, page=32, rows=40, longest=160) for _ in range(2))
    for f in (one, two):
        f.advance({1: _long(20, 3)})
    body, calls = one._wide._body, []

    def failing():
        calls.append(0)
        if len(calls) == 2:
            raise RuntimeError("no")
        body()

    one._wide._body = failing
    with pytest.raises(RuntimeError, match="no"):
        one.advance({0: _long(90, 7), 1: [5]})
    assert one.length == [39, 21] and one.free == 12 - 2 - 1
    _books(one)
    two.advance({0: _long(90, 7)[:39], 1: [5]})
    for f in (one, two):
        f.compact()
        _books(f)
    a, b = (f.advance({0: _long(90, 7)[39:], 1: [9]}) for f in (one, two))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for bad in ([cfg.vocab], [1, -1]):
        with pytest.raises(ValueError):
            one.advance({0: bad})
    assert one.advance({}) == {}
    one.fork({})
    _books(one)


class _Broken:
    """a tensor that takes nothing"""

    def __init__(self, t):
        self.shape = t.shape

    def copy_(self, *_):
        raise RuntimeError("no")


def test_books_that_cannot_be_sent(card, stack):
    """a call whose tables do not reach the GPU leaves the books as they were, and the next one sends them"""
    cfg, w = stack
    one, two = (Paged(card, cfg, w, 3, 12, page=32, rows=40, longest=160) for _ in range(2))
    for f in (one, two):
        f.advance({0: _long(50, 7), 1: _long(20, 3)})
    real, free = one.tables, one.free

    def broken(call, *args):
        one.tables = _Broken(real)
        with pytest.raises(RuntimeError, match="no"):
            call(*args)
        one.tables = real

    broken(one.advance, {0: _long(30, 5), 2: _long(70, 9)})  # two prompts that need pages
    assert one.length == [50, 20, 0] and one.free == free and [len(h) for h in one.held] == [2, 1, 0]
    a, b = (f.advance({0: [9], 1: [8]}) for f in (one, two))  # needs none
    _books(one)
    assert all(torch.equal(a[s], b[s]) for s in a)
    for call in (lambda f: f.compact(), lambda f: f.fork({0: 1}), lambda f: f.advance({1: [4]})):
        broken(one.end, 0)
        two.end(0)
        call(one)
        call(two)
        _books(one)
        assert one.held == two.held and one.length == two.length
        for f in (one, two):
            if f.length[0]:
                f.end(0)
            f.advance({0: _long(40, 3)})
    a, b = (f.advance({0: [3], 1: [2]}) for f in (one, two))
    assert all(torch.equal(a[s], b[s]) for s in a)


def test_a_fork_without_a_free_page(card, stack):
    """a branch of a sequence that ends inside a page needs one of its own: with none free nothing changes; of whole pages it needs none"""
    cfg, w = stack
    f = Paged(card, cfg, w, 4, 4, page=32, rows=8, longest=80)
    f.advance({0: _long(40, 7), 1: _long(64, 5)})
    assert f.free == 0
    torch.cuda.synchronize()
    was = f.tables.clone(), f.lens.clone(), f.pool.clone(), [list(h) for h in f.held], list(f.length), list(f.named)
    for branches in ({2: 0}, {2: 1, 3: 0}):
        with pytest.raises(RuntimeError, match="a fork needs 1 pages, 0 are free"):
            f.fork(branches)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(was, (f.tables, f.lens, f.pool))) and was[3:] == (f.held, f.length, f.named)
        _books(f)
    f.fork({2: 1})
    _books(f)
    assert f.held[2] == f.held[1] and f.free == 0
    f.end(1)
    with pytest.raises(RuntimeError):
        f.fork({3: 0})  # (its pages are the branch's still)
    f.end(2)
    f.fork({3: 0})
    _books(f)
    assert f.held[3][0] == f.held[0][0] and f.held[3][1] != f.held[0][1] and f.free == 1
    a = f.advance({0: [5], 3: [5]})
    assert torch.equal(a[0], a[3])

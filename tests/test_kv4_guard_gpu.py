"""Writes of the 4-bit cache's operators stay inside their buffers: outputs, pools, tables and workspaces of exactly their size between
poisoned fences, at odd sizes; two calls at once on two streams keep apart."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from .helpers import gen
from .test_guard_gpu import Fenced
from .test_kv4_gpu import _check, _put

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _bytes(shape):
    """a fenced uint8 tensor (of whole words)"""
    words = Fenced((int(np.prod(shape)) // 4,), torch.int32, torch.zeros(1, dtype=torch.int32))
    return words, words.t.view(torch.uint8).view(*shape)


@pytest.mark.parametrize("lens,rows,Hk,G,D,page,cap", [
    ([33], [33], 1, 1, 64, 32, 33), ([1, 70, 0, 200], [1, 3, 2, 65], 3, 5, 128, 64, 200), ([4000, 31], [1, 1], 2, 4, 128, 96, 4000),
    ([900] * 5, [7] * 5, 1, 8, 64, 32, 900),
])
def test_rows_and_attention(card, lens, rows, Hk, G, D, page, cap):
    g = gen(11000 + sum(lens))
    counts = [-(-n // page) for n in lens]
    W = max(counts)
    tables = torch.full((len(lens), W), -1, dtype=torch.int32)
    order = torch.randperm(sum(counts), generator=g).to(torch.int32)
    for b, c in enumerate(counts):
        tables[b, :c], order = order[:c], order[c:]
    tables = tables.cuda()
    fence, pool = _bytes((sum(counts), Hk, page // 32, {64: 2176, 128: 4288}[D]))
    held = sum(min(r, max(n, 0)) for n, r in zip(lens, rows))
    first = lambda r: _i32([0, *np.cumsum(r).tolist()])
    k, v = (torch.randn(sum(lens), Hk, D, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    card.kv4_write(k, v, pool, tables, _i32(lens), first=first(lens))
    fence.check("kv4_write, all")
    T = sum(rows)
    card.kv4_write(k[:T].contiguous(), v[:T].contiguous(), pool, tables, _i32(lens), first=first(rows))
    fence.check("kv4_write")
    assert held <= T
    for dtype in (torch.float32, torch.bfloat16):
        outs = [Fenced((T, Hk, D), dtype) for _ in range(2)]
        card.kv4_read(pool, tables, _i32(lens), outs[0].t, outs[1].t, first=first(rows))
        for o in outs:
            o.check("kv4_read")
    q = torch.randn(T, Hk * G * D, generator=g).to(torch.bfloat16).cuda()
    att, lse = Fenced((T, Hk * G * D), torch.bfloat16), Fenced((T, Hk * G), torch.float32)
    floats = card.attn_kv4_scratch(T, len(lens), Hk * G, Hk, D, cap).numel()
    ws = Fenced((floats,), torch.float32)
    card.attn_kv4(q, pool, tables, _i32(lens), att.t, Hk * G, Hk, D, 0.1, ws.t, first=first(rows), lse=lse.t, keys_cap=cap)
    for o, what in ((att, "att"), (lse, "lse"), (ws, "the workspace")):
        o.check(f"attn_kv4: {what}")


@pytest.mark.parametrize("lens,rows,G,D", [([9000], 1, 3, 128), ([9000], 1, 3, 64), ([1400], 1, 1, 64), ([1400], 1, 3, 128),
                                           ([3001, 2000, 33, 900, 1, 1500, 2999], 1, 5, 128), ([2500, 40, 2100], 1, 3, 64)])
def test_an_odd_number_of_spans(card, lens, rows, G, D):
    """rows x heads x spans odd, few of them and many: the workspace of exactly its size, and the rows are the oracle's"""
    g = gen(11050 + sum(lens) + G)
    pool, tables, _, _ = _put(card, g, lens, 1, D, 64)
    T, cap = rows * len(lens), max(lens)
    q = torch.randn(T, G, D, generator=g).to(torch.bfloat16).cuda()
    att, lse = Fenced((T, G * D), torch.bfloat16), Fenced((T, G), torch.float32)
    floats = card.attn_kv4_scratch(T, len(lens), G, 1, D, cap).numel()
    ws = Fenced((floats,), torch.float32)
    assert floats > 4 and ws.t.data_ptr() % 16 == 0
    scale = D**-0.5
    card.attn_kv4(q.view(T, -1), pool, tables, _i32(lens), att.t, G, 1, D, scale, ws.t, lse=lse.t, keys_cap=cap)
    for o, what in ((att, "att"), (lse, "lse"), (ws, "the workspace")):
        o.check(f"attn_kv4: {what}")
    _check(q, pool, tables, lens, [rows] * len(lens), att.t, lse.t, scale, G, 64)


@pytest.mark.parametrize("L,pages,nb,B,W,page", [(1, 7, 16, 3, 3, 32), (3, 50, 4288, 6, 9, 64), (2, 33, 16400, 2, 20, 96)])
def test_pages(card, L, pages, nb, B, W, page):
    g = gen(11100 + pages)
    fence, pool = _bytes((L, pages, nb))
    order = torch.randperm(pages, generator=g)
    held = min((pages - 2) // 2, B * W // 2)
    table = torch.full((B, W), -1, dtype=torch.int32)
    table.view(-1)[:held] = order[:held].to(torch.int32)
    full = [min(W, max(0, held - b * W)) for b in range(B)]
    tables, lens = Fenced((B, W), torch.int32, table.cuda()), Fenced((B,), torch.int32, _i32([max(0, c * page - 3) for c in full]))
    card.pages_fork(pool, tables.t, lens.t, _i32([0]), _i32([B - 1]), order[held:held + 1].to(torch.int32).cuda(), page)
    for o, what in ((fence, "the pool"), (tables, "tables"), (lens, "lens")):
        o.check(f"pages_fork: {what}")
    out = Fenced((B, W), torch.int32)
    words = card.lib.btb_hip_pages_compact_words(pages)
    ws, used = Fenced((words,), torch.int32), Fenced((1,), torch.int32)
    card._call("btb_hip_pages_compact", pool.data_ptr(), L, pages, nb, pages * nb, nb, tables.t.data_ptr(), lens.t.data_ptr(), B, W, page,
               out.t.data_ptr(), used.t.data_ptr(), ws.t.data_ptr(), torch.cuda.current_stream().cuda_stream)
    for o, what in ((fence, "the pool"), (tables, "tables"), (out, "tables_out"), (ws, "the workspace"), (used, "used")):
        o.check(f"pages_compact: {what}")


def test_two_calls_at_once(card):
    """two batches over one pool on two streams, each with a workspace of its own"""
    g = gen(11200)
    Hk, G, D, page, n = 2, 4, 128, 64, 3000
    pages = -(-n // page)
    pool = card.kv4_pool(2 * pages, Hk, D, page)
    tables = torch.randperm(2 * pages, generator=g).to(torch.int32).view(2, pages).cuda()
    k, v = (torch.randn(2 * n, Hk, D, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    card.kv4_write(k, v, pool, tables, _i32([n, n]))
    calls = []
    for b in range(2):
        q = torch.randn(1, Hk * G * D, generator=g).to(torch.bfloat16).cuda()
        calls.append(dict(q=q, att=torch.zeros_like(q), tables=tables[b:b + 1].contiguous(), lens=_i32([n]),
                          ws=card.attn_kv4_scratch(1, 1, Hk * G, Hk, D, n)))

    def run(c):
        card.attn_kv4(c["q"], pool, c["tables"], c["lens"], c["att"], Hk * G, Hk, D, 0.1, c["ws"], keys_cap=n)

    want = []
    for c in calls:
        run(c)
        torch.cuda.synchronize()
        want.append(c["att"].clone())
        c["att"].zero_()
    streams = [torch.cuda.Stream() for _ in calls]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for c, s in zip(calls, streams):
            with torch.cuda.stream(s):
                run(c)
    torch.cuda.synchronize()
    assert all(torch.equal(c["att"], w) for c, w in zip(calls, want))

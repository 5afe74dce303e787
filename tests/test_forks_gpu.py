"""`Forks` on the tiny Qwen3 fixture: with room for the whole prompt it reproduces the reference's receipts (the bars of
tests/test_load_gpu.py: logits 3e-2 of the largest, greedy tokens equal), however the prompt is cut into passes; with less room it
keeps what it promises to keep, and layer 0's kept keys - which no attention comes before - are the unbounded run's bits at their
positions."""

from __future__ import annotations

import os

import numpy as np
import pytest
import torch

from btb_amd.forks import Forks
from btb_amd.load import load_stack

from .helpers import GOLDEN

pytestmark = pytest.mark.gpu

PROMPT = [3, 17, 42, 5, 99, 120, 7, 7, 200, 12, 45, 8, 3, 17, 60, 61]


@pytest.fixture(scope="module")
def stack(card):
    return load_stack(card, os.path.join(GOLDEN, "tiny_qwen3"))


@pytest.fixture(scope="module")
def receipts():
    return torch.load(os.path.join(GOLDEN, "receipts_qwen3.pt"), weights_only=True)


@pytest.mark.parametrize("rows,chunk,sections,captured", [(1, 16, None, False), (3, 5, None, False), (6, 7, [16, 24, 24], True)])
def test_with_room_it_is_the_model(card, stack, receipts, rows, chunk, sections, captured):
    """every row takes the receipts' greedy tokens; three axes at one place are one axis"""
    cfg, w = stack
    f = Forks(card, cfg, w, rows, budget=32, steps=12, chunk=chunk, sinks=2, recent=4, positions=512, sections=sections)
    logits = f.prompt(PROMPT)
    torch.cuda.synchronize()
    want = receipts["bf16"]["prompt_logits"].float().numpy().reshape(-1)
    got = logits.float().cpu().numpy()
    assert np.abs(got - want).max() <= 3e-2 * np.abs(want).max()
    greedy = receipts["ref"]["greedy"]
    assert int(got.argmax()) == greedy[0] and f.n == len(PROMPT)
    f.begin([greedy[0]] * rows)
    if captured:
        f.capture()
    for tok in greedy[1:]:
        out = f.step()
        torch.cuda.synchronize()
        assert out.float().argmax(-1).tolist() == [tok] * rows
    assert f.taken == len(greedy) - 1


def test_rows_go_their_own_ways(card, stack):
    """rows that begin with unlike tokens: each one's logits are those of a run with it alone"""
    cfg, w = stack
    first = [5, 77, 200, 9]
    many = Forks(card, cfg, w, 4, budget=32, steps=6, chunk=8, sinks=1, recent=4, positions=256)
    many.prompt(PROMPT)
    many.begin(first)
    together = [many.step().float().cpu().numpy().copy() for _ in range(5)]
    for r, tok in enumerate(first):
        one = Forks(card, cfg, w, 1, budget=32, steps=6, chunk=8, sinks=1, recent=4, positions=256)
        one.prompt(PROMPT)
        one.begin([tok])
        for out in together:
            alone = one.step().float().cpu().numpy()[0]
            assert np.abs(alone - out[r]).max() <= 3e-2 * np.abs(alone).max()
    assert np.abs(together[0][0] - together[0][1]).max() > 0.1 * np.abs(together[0]).max()


def test_with_less_room_it_keeps_what_it_promises(card, stack):
    cfg, w = stack
    prompt = [(7 * i * i + 3 * i + 11) % 250 for i in range(61)]
    whole = Forks(card, cfg, w, 2, budget=64, steps=4, chunk=8, sinks=2, recent=6, positions=256)
    whole.prompt(prompt)
    f = Forks(card, cfg, w, 2, budget=24, steps=4, chunk=8, sinks=2, recent=6, positions=256)
    f.prompt(prompt[:30])
    f.prompt(prompt[30:])
    torch.cuda.synchronize()
    assert f.n == 24 and f.seen == 61 and whole.n == 61
    pos = f.pos[:, :, :24].cpu()
    for i in range(cfg.layers):
        for g in range(cfg.kv_heads):
            held = sorted(pos[i, g].tolist())
            assert len(set(held)) == 24 and set(held) >= {0, 1} | set(range(55, 61))
    for kind in (0, 1):
        for g in range(cfg.kv_heads):
            assert torch.equal(f.kv[0, kind, g, :24], whole.kv[0, kind, g, pos[0, g].long().cuda()])
    # every weight a pass hands out is a key's: with no cut, a head's keys hold one a row and query head
    total = whole.mass[:, :, :61].sum(-1).cpu()
    assert torch.allclose(total, torch.full_like(total, 61.0 * cfg.q_heads / cfg.kv_heads), rtol=1e-3)
    f.begin([1, 1])
    out = f.step()
    torch.cuda.synchronize()
    assert torch.equal(out[0], out[1]) and bool(out.isfinite().all())


def test_refusals(card, stack):
    cfg, w = stack
    with pytest.raises(ValueError):
        Forks(card, cfg, w, 1, budget=8, steps=4, sinks=4, recent=5)
    with pytest.raises(ValueError):
        Forks(card, cfg, w, 1, budget=32, steps=4, sinks=1, recent=5, sections=[16, 16])
    f = Forks(card, cfg, w, 2, budget=32, steps=1, sinks=1, recent=5, positions=40)
    with pytest.raises(ValueError):
        f.begin([1, 2])  # before any prompt
    with pytest.raises(ValueError):
        f.prompt(list(range(40)))  # positions past the tables
    f.prompt([1, 2, 3])
    with pytest.raises(ValueError):
        f.begin([1])
    f.begin([1, 2])
    f.step()
    with pytest.raises(RuntimeError):
        f.step()
    with pytest.raises(RuntimeError):
        f.prompt([4])

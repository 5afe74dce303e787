"""`Forks` called out of order: what cannot be answered rightly is refused and leaves the cache and the rows as they were."""

from __future__ import annotations

import os

import pytest
import torch

from btb_amd.forks import Forks
from btb_amd.load import load_stack

from .helpers import GOLDEN

pytestmark = pytest.mark.gpu

PROMPT = [3, 17, 42, 5, 99, 120, 7, 7, 200, 12]


@pytest.fixture(scope="module")
def stack(card):
    return load_stack(card, os.path.join(GOLDEN, "tiny_qwen3"))


def _forks(card, stack, rows=3, steps=4, budget=32):
    cfg, w = stack
    return Forks(card, cfg, w, rows, budget=budget, steps=steps, chunk=8, sinks=1, recent=4, positions=128)


def _held(f):
    torch.cuda.synchronize()
    return [t.clone() for t in (f.kv, f.mass, f.pos, f._step.ids, f._step.pos, f._step.slots, f._step.lay)] + [f.n, f.seen, f.taken]


def _same(a, b):
    return all(torch.equal(x, y) if isinstance(x, torch.Tensor) else x == y for x, y in zip(a, b))


@pytest.mark.parametrize("prompted", [False, True])
def test_no_step_and_no_recording_before_the_rows_begin(card, stack, prompted):
    """the rows' slots are the prompt's first one then: a pass would write all of them there"""
    f = _forks(card, stack)
    if prompted:
        f.prompt(PROMPT)
    before = _held(f)
    with pytest.raises(RuntimeError):
        f.step()
    with pytest.raises(RuntimeError):
        f.capture()
    assert f.graph is None and _same(_held(f), before)


@pytest.mark.parametrize("captured", [False, True])
def test_a_longer_prompt_is_what_the_rows_begin_behind(card, stack, captured):
    """tokens between `begin` and the first step: the rows begin again, and are then those of the whole prompt"""
    whole, f = _forks(card, stack, budget=12), _forks(card, stack, budget=12)
    for t in (PROMPT, [60, 61, 8, 45, 3]):
        whole.prompt(t)
    f.prompt(PROMPT)
    f.begin([5, 6, 7])
    if captured:
        f.capture()
    with pytest.raises(ValueError):
        f.prompt([1] * 128)  # refused: the rows stand as they did
    f.prompt([60, 61, 8, 45, 3])
    before = _held(f)
    for call in (f.step, f.capture):
        with pytest.raises(RuntimeError):
            call()
    assert _same(_held(f), before)
    for g in (whole, f):
        g.begin([5, 6, 7])
    for _ in range(4):
        a, b = whole.step().clone(), f.step().clone()
        torch.cuda.synchronize()
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError):
        f.prompt([1])
    assert f.begun and f.taken == 4


def test_no_recording_without_room(card, stack):
    """with all steps taken, the pass that warms a recording up would write each row's next slot: the next row's first"""
    f = _forks(card, stack, steps=2)
    f.prompt(PROMPT)
    f.begin([5, 6, 7])
    f.step()
    f.step()
    before = _held(f)
    with pytest.raises(RuntimeError):
        f.capture()
    assert f.graph is None and _same(_held(f), before)
    f.begin([8, 9, 10])
    f.capture()
    f.step()
    f.step()


def test_a_cut_within_the_budget_moves_nothing(card, stack):
    f = _forks(card, stack, budget=12)
    f.cut()
    f.prompt(PROMPT)
    f.begin([5, 6, 7])
    before = _held(f)
    f.cut()
    assert _same(_held(f), before) and f.n == len(PROMPT)
    f.step()

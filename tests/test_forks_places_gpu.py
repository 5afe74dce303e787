"""`Forks` where a token's place is not its number: a prompt with a picture, whose tokens share places, then text and decoded rows
that go on one past the largest place - against the stack evaluated directly in 64 bits from the same weights (the bar of
tests/test_forks_gpu.py: logits 3e-2 of the largest)."""

from __future__ import annotations

import os

import numpy as np
import pytest
import torch

from btb_amd.decode import rope_axes, rope_tables
from btb_amd.forks import Forks
from btb_amd.load import load_stack
from oracle import shared

from .helpers import GOLDEN

pytestmark = pytest.mark.gpu

SECTIONS = [16, 24, 24]
TEXT, PICTURE = [3, 17, 42, 5], [99, 120, 7, 33, 200, 12, 45, 8, 60]


@pytest.fixture(scope="module")
def stack(card):
    return load_stack(card, os.path.join(GOLDEN, "tiny_qwen3"))


def _f64(t):
    return t.detach().double().cpu().numpy()


def _direct(cfg, w, tokens, places, sections):
    """the last token's logits: every token at its places, each seeing itself and those before it"""
    Hq, Hk, D = cfg.q_heads, cfg.kv_heads, cfg.head_dim
    cos, sin = (_f64(t)[:, :D // 2] for t in rope_tables(cfg, 256, "cpu"))
    axes, T = rope_axes(sections, "cpu").numpy(), len(tokens)
    norm = lambda x, v: x / np.sqrt((x * x).mean(-1, keepdims=True) + cfg.eps) * _f64(v)
    h = _f64(w["embed"])[np.asarray(tokens)]
    for i in range(cfg.layers):
        L = f"layers.{i}."
        qkv = (norm(h, w[L + "ln1"]) @ _f64(w[L + "qkv"].w).T).reshape(T, Hq + 2 * Hk, D)
        q = shared.norm_rope_axes(qkv[:, :Hq], _f64(w[L + "wq"]), cfg.eps, cos, sin, places, axes)
        k = shared.norm_rope_axes(qkv[:, Hq:Hq + Hk], _f64(w[L + "wk"]), cfg.eps, cos, sin, places, axes).transpose(1, 0, 2)
        v = qkv[:, Hq + Hk:].transpose(1, 0, 2)
        own = [(0, t + 1) for t in range(T)]
        att, _, _ = shared.attn_shared(q, k, v, 0, 0, own, 1.0 / np.sqrt(D))
        h = h + att.reshape(T, -1) @ _f64(w[L + "o"].w).T
        g, u = np.split(norm(h, w[L + "ln2"]) @ _f64(w[L + "gu"].w).T, 2, axis=-1)
        h = h + (g / (1.0 + np.exp(-g)) * u) @ _f64(w[L + "down"].w).T
    return (norm(h, w["norm"]) @ _f64(w["head"].w).T)[-1]


def _hold(got, want):
    assert np.abs(_f64(got) - want).max() <= 3e-2 * np.abs(want).max()


def _picture():
    """three rows of three patches behind the text: [3, 4 + 9] places, the largest of which is 6"""
    text = np.tile(np.arange(4), (3, 1))
    patch = 4 + np.stack([np.zeros(9, int), np.arange(9) // 3, np.arange(9) % 3])
    return np.concatenate([text, patch], 1)


@pytest.mark.parametrize("chunk,captured", [(32, False), (5, True)])
def test_text_and_rows_go_on_past_the_largest_place(card, stack, chunk, captured):
    cfg, w = stack
    f = Forks(card, cfg, w, 2, budget=64, steps=4, chunk=chunk, sinks=1, recent=4, positions=128, sections=SECTIONS)
    places = _picture()
    tokens = TEXT + PICTURE
    _hold(f.prompt(tokens, torch.tensor(places, dtype=torch.int32, device="cuda")), _direct(cfg, w, tokens, places, SECTIONS))
    more = [61, 7, 150]  # no places: one after the other from 7 on
    tokens, places = tokens + more, np.concatenate([places, np.tile(np.arange(7, 10), (3, 1))], 1)
    _hold(f.prompt(more), _direct(cfg, w, tokens, places, SECTIONS))
    rows = [tokens + [t] for t in (9, 77)]
    f.begin([9, 77])
    if captured:
        f.capture()
    for at in range(10, 13):
        places = np.concatenate([places, np.full((3, 1), at)], 1)
        logits = f.step()
        torch.cuda.synchronize()
        for r in range(2):
            _hold(logits[r], _direct(cfg, w, rows[r], places, SECTIONS))
            rows[r].append(int(logits[r].float().argmax()))


def test_places_that_only_shift_change_nothing(card, stack):
    """a rotation turns by differences: a prompt seven places further on, and the steps behind it, are the model's"""
    cfg, w = stack
    tokens = TEXT + PICTURE
    n = len(tokens)
    f = Forks(card, cfg, w, 1, budget=64, steps=3, chunk=8, sinks=1, recent=4, positions=128, sections=SECTIONS)
    f.prompt(tokens, torch.arange(7, 7 + n, device="cuda").expand(3, n))
    f.begin([9])
    for at in range(1, 4):
        tokens = tokens + [9 if at == 1 else int(got[0].float().argmax())]
        got = f.step()
        torch.cuda.synchronize()
        _hold(got[0], _direct(cfg, w, tokens, np.tile(np.arange(n + at), (3, 1)), SECTIONS))


def test_refusals(card, stack):
    cfg, w = stack
    f = Forks(card, cfg, w, 1, budget=32, steps=4, sinks=1, recent=5, positions=40, sections=SECTIONS)
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    for bad in (z(3, 2), z(1, 3), z(3), z(3, 3).float(), z(3, 3) - 1, z(3, 3) + 36):  # 36 and four steps: past the tables' 40
        with pytest.raises(ValueError):
            f.prompt([1, 2, 3], bad)
    f.prompt([1, 2, 3], z(3, 3) + 35)
    with pytest.raises(ValueError):
        f.prompt([4])  # at 36
    f.prompt([4], z(3, 1))
    f.begin([5])
    assert f._step.pos.flatten().tolist() == [36] * 3

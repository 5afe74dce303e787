"""How near the operators over one shared cache come to the formulas in 64 bits, in the relative 2-norm: the bars of
test_shared_cache_gpu.py bound every single value at its worst, and a path that held its weights in fewer bits would stay
below them.

Bars, from the arithmetic (u = 2^-24). Inputs are exact on both sides. A score is D products added in f32: its roundings are
independent of one another, so e = sqrt(D) u scale |q| |k| (largest norms) bounds its error in the mean square.
  att   rounding the outputs to bf16, whose own size r = |bf16(want) - want| is taken from the 64-bit outputs themselves and
        may differ by a fiftieth; two bf16 terms hold a weight to 2^-15; scores: (2^-15 + e) of |the weighted sums of |v||
  lse   e and 4 u of its largest value and of 1
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import shared

from .helpers import gen
from .test_shared_cache_gpu import INF, U, _f64, _run_shared, _shared_case

pytestmark = pytest.mark.gpu


def _norm(a):
    return float(np.linalg.norm(a))


def _score_rms(q, K, scale):
    return math.sqrt(q.shape[-1]) * U * scale * np.linalg.norm(q, axis=-1).max() * np.linalg.norm(np.nan_to_num(K), axis=-1).max()


@pytest.mark.parametrize("T,Hq,Hk,D,P,own", [
    (4, 32, 8, 128, 700, 8),     # up to 32 pairs a kv head
    (3, 8, 2, 64, 300, 0),
    (16, 32, 8, 128, 2000, 40),  # up to 64
    (12, 20, 4, 64, 1500, 30),
    (40, 16, 2, 128, 1500, 20),  # more
    (40, 16, 2, 64, 3000, 33),
    (3, 8, 2, 128, 0, 1000),     # a row's own keys alone
    (5, 6, 3, 64, 0, 700),
])
def test_attn_shared_outputs_are_the_formulas_rounded_once(card, T, Hq, Hk, D, P, own):
    g = gen(5700 + T + D)
    q, K, V, off, offs = _shared_case(g, T, Hq, Hk, D, P, [own] * T, std=3.0)
    scale, rows = 1.0 / math.sqrt(D), [(o, own) for o in offs]
    att, lse = _run_shared(card, q, K, V, off, P, rows, scale, P, own)
    qd, Kd, Vd = _f64(q), _f64(K), _f64(V)
    want, z, spread = shared.attn_shared(qd, Kd, Vd, off, P, rows, scale)
    e = _score_rms(qd, Kd, scale)
    rounding = _norm(torch.from_numpy(want).to(torch.bfloat16).double().numpy() - want)
    off_by = _norm(_f64(att) - want)
    print(f"relative 2-norm {off_by / _norm(want):.3e}, rounding {rounding / _norm(want):.3e}, spread {_norm(spread) / _norm(want):.2f}")
    assert off_by <= 1.02 * rounding + (2.0**-15 + e) * _norm(spread)
    assert _norm(_f64(lse) - z) <= (e + 4 * U * (1 + np.abs(z).max())) * math.sqrt(z.size)


@pytest.mark.parametrize("T,D", [(2, 64), (2, 128), (12, 128), (40, 64), (40, 128)])
def test_attn_shared_an_infinite_value_stays_infinite(card, T, D):
    """whatever a key weighs - all there is, the most, or 2^-60 - its infinite value is what comes out, at any width of the pass"""
    g = gen(5750 + T + D)
    Hq, Hk, P = 8, 2, 200
    q, K, V, off, offs = _shared_case(g, T, Hq, Hk, D, P, [1] * T)
    own, scale = [(o, 1) for o in offs], 1.0 / math.sqrt(D)
    V[:, offs[0], 5] = INF  # row 0 alone sees it
    att, _ = _run_shared(card, q, K, V, off, 0, own, scale, 0, 1)  # ... and nothing else: a weight of 1
    assert bool((att[0, :, 5] == INF).all()) and bool(att[0, :, :5].isfinite().all()) and bool(att[1:].isfinite().all())
    V[:, off + 130, 7] = -INF  # in every row's prefix
    att, _ = _run_shared(card, q, K, V, off, P, own, scale, P, 1)
    assert bool((att[..., 7] == -INF).all()) and bool((att[0, :, 5] == INF).all()) and bool(att[1:, :, 5].isfinite().all())
    assert bool(att[:, :, 8:].isfinite().all())
    # the prefix's infinite key far below every other: scores 60 log 2 apart
    q[:], K[:, off:off + P] = 0.0, 0.0
    q[..., 0], K[:, off + 130, 0] = 1.0, -60.0 * math.log(2.0) / scale
    att, _ = _run_shared(card, q, K, V, off, P, own, scale, P, 1)
    assert bool((att[..., 7] == -INF).all()) and bool(att[:, :, 8:].isfinite().all())

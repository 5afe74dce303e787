"""oracle/shared.py by hand cases and against mistakes: what the GPU tests of a batch over one shared cache compare with."""

from __future__ import annotations

import numpy as np
import pytest

from btb_amd.decode import StackConfig, rope_axes, rope_tables
from oracle import decode as od
from oracle import shared


def test_one_axis_is_the_decode_steps_rotation():
    """every axis at the row's position, no rounding: the rotation the step's oracle makes"""
    rng = np.random.default_rng(1)
    cfg = StackConfig(head_dim=64)
    cos, sin = (t.float().numpy() for t in rope_tables(cfg, 40, "cpu"))
    x = rng.standard_normal((3, 2, 64))
    pos = np.array([[0, 7, 39]] * 3)
    got = shared.norm_rope_axes(x, None, 0.0, cos, sin, pos, np.arange(32) % 3)
    for t, p in enumerate(pos[0]):
        rot = np.concatenate([-x[t, :, 32:], x[t, :, :32]], -1)
        np.testing.assert_allclose(got[t], x[t] * cos[p] + rot * sin[p], atol=1e-12)


def test_each_frequency_turns_by_its_own_axis():
    x = np.zeros((1, 1, 8))
    x[0, 0, :4] = 1.0  # a quarter turn moves dim i to dim i + 4
    cos = np.ones((3, 4))
    sin = np.zeros((3, 4))
    cos[2], sin[2] = 0.0, 1.0
    got = shared.norm_rope_axes(x, None, 0.0, cos, sin, np.array([[0], [2]]), np.array([0, 1, 1, 0]))[0, 0]
    assert got.tolist() == [1, 0, 0, 1, 0, 1, 1, 0]


def test_axis_maps():
    assert rope_axes([2, 1, 1], "cpu").tolist() == [0, 0, 1, 2]
    assert rope_axes([3, 2, 1], "cpu", interleaved=True).tolist() == [0, 1, 2, 0, 1, 0]
    with pytest.raises(ValueError):
        rope_axes([], "cpu")
    with pytest.raises(ValueError):
        rope_axes([2, -1], "cpu")


def test_a_shared_prefix_is_each_rows_own_attention():
    rng = np.random.default_rng(2)
    q, K, V = rng.standard_normal((3, 4, 8)), rng.standard_normal((2, 20, 8)), rng.standard_normal((2, 20, 8))
    own = [(10, 3), (13, 0), (2, -1)]
    att, lse, _ = shared.attn_shared(q, K, V, 4, 6, own, 0.3)
    want = od.attention(q[0].astype(np.float32), K[:, 4:13].astype(np.float32), V[:, 4:13].astype(np.float32), 0.3)
    np.testing.assert_allclose(att[0], want, rtol=1e-2, atol=1e-2)
    s = np.einsum("hd,hkd->hk", q[1], K[[0, 0, 1, 1], 4:10]) * 0.3
    np.testing.assert_allclose(lse[1], np.log(np.exp(s).sum(-1)))
    assert not att[2].any() and np.isinf(lse[2]).all()
    none = shared.attn_shared(q, K, V, 4, 0, [(0, 0)] * 3, 0.3)
    assert not none[0].any() and (none[1] == -np.inf).all()


def test_weights_of_all_rows_sum_to_the_heads():
    """a row's weights over the keys it sees sum to one a head; a row that saw nothing adds none; a mistake shows"""
    rng = np.random.default_rng(3)
    q, K = rng.standard_normal((2, 4, 8)), rng.standard_normal((2, 9, 8))
    seen = [5, 9]
    lse = np.stack([[shared.attention(q[t, h:h + 1], K[h // 2, :seen[t]], K[h // 2, :seen[t]], 0.4)[1][0] for h in range(4)]
                    for t in range(2)])
    out = shared.attn_mass(q, K, lse, seen, None, 0.4, 9)
    np.testing.assert_allclose(out.sum(-1), [4.0, 4.0])
    np.testing.assert_allclose(shared.attn_mass(q, K, lse, seen, out, 0.4, 9), 2 * out)
    lse[0] = -np.inf
    np.testing.assert_allclose(shared.attn_mass(q, K, lse, seen, None, 0.4, 9).sum(-1), [2.0, 2.0])
    assert abs(shared.attn_mass(q, K, lse, seen, None, 0.5, 9).sum() - 4.0) > 1e-3  # another scale than the lse's


def test_eviction_by_hand():
    inf, nan = np.inf, np.nan
    pos = np.arange(8)[None]
    # the four heaviest are slots 1, 4, 6, 7; 1 stays, the holes 0, 2, 3 are filled in order
    assert shared.evict([[0.1, 5, 0.2, 0.3, 4, 0.1, 3, 2]], pos, 8, 4).tolist() == [[4, 1, 6, 7]]
    # ties go to the lowest slot, -0 is 0, a NaN comes last
    assert shared.evict([[nan, 0.0, -0.0, 0.0, -1, -inf, 0.0, nan]], pos, 8, 3).tolist() == [[3, 1, 2]]
    # the first and the newest stay whatever they weigh
    assert shared.evict([[0, 9, 9, 9, 9, 9, 9, 0]], pos, 8, 3, sinks=1, recent_from=7).tolist() == [[0, 1, 7]]
    # ... the lowest slots of them where even they are too many
    assert shared.evict([[0, 9, 9, 9, 9, 9, 9, 0]], pos, 8, 2, sinks=2, recent_from=7).tolist() == [[0, 1]]
    assert shared.evict([[3, 1, 2]], pos, 3, 9).tolist() == [[0, 1, 2]]

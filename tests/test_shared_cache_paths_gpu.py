"""The operators over one shared cache on the paths that long passes and full caches take: loops that go round more than once, buffers
written again, tables refilled, the wide forms of the kernels. Small tests seldom get there, so each test says by which numbers
of the launch - worked out from the workspaces' sizes and the chip's compute units - its sizes do. Against oracle/shared.py in
64 bits, with the bars of test_shared_cache_gpu.py and test_shared_cache_bits_gpu.py."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _cus():
    return torch.cuda.get_device_properties(0).multi_processor_count


def _mass_parts(card, T, Hq, Hk, D, n):
    """(workgroups the pairs are cut over, their stages)"""
    parts = max(1, card.lib.btb_hip_attn_mass_floats(T, Hq, Hk, D, n) // (Hk * n))
    return parts, -(-T * (Hq // Hk) // (16384 // D))


@pytest.mark.parametrize("D", [64, 128])
def test_attn_mass_no_workgroup_without_a_stage(card, D):
    for T in list(range(1, 140, 7)) + [200, 331, 500, 1000]:
        for Hq, Hk in ((32, 8), (12, 4), (5, 1), (48, 2)):
            for n in (31, 512, 700, 2000, 4000, 16384):
                parts, stages = _mass_parts(card, T, Hq, Hk, D, n)
                assert parts == 1 or (parts - 1) * -(-stages // parts) < stages, (T, Hq, Hk, n, parts, stages)

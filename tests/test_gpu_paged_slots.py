"""GPU test that one_paged_attention counts every slot of a cache exactly once, in its output and in the
accumulated weights, over every way the work is cut."""
import math

import pytest
import torch

from conftest import cuda_ok
from slots_util import Slots

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]

SHAPES = [  # lengths, hkv, group, dh, page
    ([200], 12, 1, 64, 16), ([0, 1, 15, 16, 17, 63, 64, 65, 130, 1000], 2, 8, 32, 7), ([500, 64], 1, 20, 96, 64), ([40, 0, 1], 1, 1, 8, 5),
    ([4097, 127], 2, 7, 128, 128), ([20000, 3], 1, 8, 64, 16), ([24576, 5, 0], 1, 2, 96, 16), ([24576], 2, 1, 128, 48), ([33000], 1, 1, 64, 16),
    ([(i * 1000 + 700) % 4001 for i in range(9)], 4, 1, 64, 16), ([(i * 331) % 1001 for i in range(18)], 4, 2, 128, 16),
    ([(i * 97) % 701 for i in range(30)], 16, 1, 64, 16), ([(i * 617) % 3001 for i in range(40)], 12, 1, 64, 16),
    ([2500 - 97 * i for i in range(16)], 4, 3, 64, 48), ([(i * 89) % 261 for i in range(33)], 10, 9, 64, 32),
    ([3001 - 500 * i for i in range(6)], 4, 1, 80, 32), ([1500, 31, 600], 5, 4, 112, 24),
]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=[f"{len(s[0])}x{s[1]}x{s[2]}x{s[3]}n{max(s[0])}" for s in SHAPES])
def test_every_slot_counts_once(shape, dt):
    from one import turbo_ops as T
    lens, hkv, g, dh, page = shape
    s = Slots(lens, hkv, g, dh, page, dt, torch.Generator().manual_seed(dh + len(lens)), "cuda")
    s.check(lambda x: T.turbo_paged_attention(x.q, x.k, x.v, x.table, x.lengths, scale_factor=math.log(2.0)))
    mass = torch.zeros(len(lens), hkv, s.table.shape[1] * page, device="cuda")
    # the weights, then the output of calls that accumulate them
    T.turbo_paged_attention(s.q, s.k, s.v, s.table, s.lengths, scale_factor=math.log(2.0), mass=mass)
    want = torch.zeros_like(mass, dtype=torch.float64)
    want[..., :s.p.shape[-1]] = s.mass()
    err = (mass.double() - want).abs() - (s.tol + g * 2.0 ** -24) * want
    assert float(err.max()) <= 0, f"mass: {float(err.max()):.3g} over"
    s.check(lambda x: T.turbo_paged_attention(x.q, x.k, x.v, x.table, x.lengths, scale_factor=math.log(2.0), mass=mass))
    assert T.ops_error() == (0, 0)

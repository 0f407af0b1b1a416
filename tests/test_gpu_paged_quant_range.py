"""Attention over a cache in 4 or 8 bits where sizes lie far apart: each output dim against the 64-bit
formula, by the sizes of its own terms."""
import pytest
import torch

import quant_util as Q

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")
KINDS = [(BF, 1), (BF, 4), (BF, 6), (BF, 12), (F32, 2), (F32, 7)]  # dtype and queries per kv head: every kind of kernel


@pytest.fixture(autouse=True)
def no_device_error():
    from one import turbo_ops as T
    T.ops_error(clear=True)
    yield
    assert T.ops_error(clear=True) == (0, 0)


def ops():
    from one import turbo_ops
    return turbo_ops


def make(lengths, hkv, g, dh, page, bits, dt, seed, positive=False):
    gen = torch.Generator().manual_seed(seed)
    cache = list(Q.make_cache(lengths, hkv, dh, page, bits, gen))
    q = torch.randn(len(lengths), hkv * g, 1, dh, generator=gen)
    return cache, ((q.abs() + 0.1) if positive else q).to(dt), gen


def place(cache, b, t):
    return int(cache[3][b, t // cache[0].shape[2]]), t % cache[0].shape[2]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt,g", KINDS)
@pytest.mark.parametrize("dh,page", [(64, 16), (96, 16), (128, 16), (80, 8), (112, 5)])
def test_groups_beside_one_that_is_not_finite(bits, dt, g, dh, page):
    """A value group whose scale is NaN makes its own dims NaN; the others are as good as without it.
    Even weights, so that each slot counts."""
    cache, q, _ = make([3, 40], 2, g, dh, page, bits, dt, 81)
    for group in range(Q.groups(dh)):
        c = list(cache)
        c[2] = cache[2].clone()
        for b, at in ((0, 1), (1, 17)):
            pg, row = place(c, b, at)
            c[2][pg, :, row, 1, group] = NAN
        ref, _, mag, smax = Q.attention(q, cache, bits, 0.0)
        out = ops().turbo_paged_quant_attention(q.cuda(), *(x.cuda() for x in c), scale_factor=0.0).cpu()
        nan = torch.zeros(dh, dtype=torch.bool)
        nan[32 * group:32 * group + 32] = True
        assert bool((out.isnan() == nan).all())
        e = Q.weight_error(40, dh, smax, dt)
        d, tol = (out.double() - ref).abs(), e * mag + torch.finfo(dt).eps / 2 * ref.abs() * (1 + e)
        assert bool((d <= tol)[..., ~nan].all()), float((d / tol)[..., ~nan].max())

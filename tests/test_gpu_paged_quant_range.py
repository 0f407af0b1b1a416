"""Attention over a cache in 4 or 8 bits where sizes lie far apart: each output dim against the 64-bit
formula, by the sizes of its own terms."""
import pytest
import torch

import quant_range_util as R
import quant_util as Q

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")
KINDS = [(BF, 1), (BF, 4), (BF, 6), (BF, 12), (F32, 2), (F32, 7)]  # dtype and queries per kv head: every kind of kernel
SHAPES = [([513], 64, 16), ([300], 128, 16), ([200], 96, 5), ([9000, 700], 64, 16), ([5000], 48, 7)]  # whole groups, rows looked up; clusters, lists


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


def zero_code(bits):
    return 0x88 if bits == 4 else 128


def least_code(bits):
    return 0x11 if bits == 4 else 1


def check(q, cache, bits, scale, mass=False, floor=0.0):
    ref, tol, w, wt = R.attention(q, cache, bits, scale)
    m0 = m = None
    if mass:
        m0 = torch.rand(q.shape[0], cache[0].shape[1], cache[3].shape[1] * cache[0].shape[2], generator=torch.Generator().manual_seed(1))
        m = m0.cuda()
    out = ops().turbo_paged_quant_attention(q.cuda(), *(x.cuda() for x in cache), scale_factor=scale, mass=m)
    R.check_out(out, ref, tol, floor)
    if mass:
        R.check_mass(m, m0, w, wt, q.shape[1] // cache[0].shape[1])
    return out


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt,g", KINDS)
@pytest.mark.parametrize("lengths,dh,page", SHAPES)
def test_a_huge_value_that_nobody_attends_to(bits, dt, g, lengths, dh, page):
    """One slot of values 2^40 times the others', and a score some 50 below them: it adds 2^-30 of the output."""
    for at in (0, lengths[0] // 2, lengths[0] - 1):
        cache, q, _ = make(lengths, 2, g, dh, page, bits, dt, 11 + at, positive=True)
        pg, row = place(cache, 0, at)
        cache[0][pg, :, row] = least_code(bits)
        cache[2][pg, :, row, 0] = 50.0 / (Q.top(bits) * float(q.float().sum(-1).mean()) * dh ** -0.5)
        cache[2][pg, :, row, 1] *= 2.0 ** 40
        check(q, cache, bits, dh ** -0.5, mass=at == 0)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt,g", KINDS)
@pytest.mark.parametrize("lengths,dh,page", SHAPES)
@pytest.mark.parametrize("far", [30, 60])
def test_groups_of_values_far_apart(bits, dt, g, lengths, dh, page, far):
    """One group of 32 dims of every value is 2^far times the others: each dim by its own terms."""
    cache, q, _ = make(lengths, 2, g, dh, page, bits, dt, 21 + far)
    for group in (0, Q.groups(dh) - 1):
        c = list(cache)
        c[2] = cache[2].clone()
        c[2][..., 1, group] *= 2.0 ** far
        check(q, c, bits, dh ** -0.5)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt,g", KINDS)
@pytest.mark.parametrize("dh,page", [(64, 16), (128, 16), (80, 8)])
def test_dims_that_a_huge_value_leaves_alone(bits, dt, g, dh, page):
    """A slot like any other, of values 2^50 times the others', whose code is 0 in some dims."""
    cache, q, _ = make([400, 90], 2, g, dh, page, bits, dt, 31)
    for b, at in ((0, 0), (0, 200), (1, 89)):
        pg, row = place(cache, b, at)
        cache[1][pg, :, row, ::3] = zero_code(bits)
        cache[2][pg, :, row, 1] *= 2.0 ** 50
    check(q, cache, bits, dh ** -0.5)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt,g", KINDS)
@pytest.mark.parametrize("size", [-100, -60, 90])
def test_values_of_the_smallest_and_of_large_scales(bits, dt, g, size):
    """Scales from 2^-100 on; products of the smallest ones and of small weights end at 2^-133 (bf16's last
    step) in their last part, of at most 128 times 400."""
    cache, q, _ = make([400, 33], 2, g, 64, 16, bits, dt, 41)
    used = torch.isfinite(cache[2][..., 1, :].float())
    cache[2][..., 1, :] = torch.where(used, torch.exp2(torch.full(used.shape, float(size))).bfloat16(), cache[2][..., 1, :])
    check(q, cache, bits, 0.125, floor=2.0 ** -133 * 128 * 400)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt,g", KINDS)
@pytest.mark.parametrize("dh,page", [(64, 16), (128, 16), (80, 8)])
def test_scores_whose_terms_are_large(bits, dt, g, dh, page):
    """Small codes, sums of terms of some 2000 in all, which cancel to scores near 0: the weights show each
    score's error."""
    gen = torch.Generator().manual_seed(51)
    n, groups, top = 200, Q.groups(dh), Q.top(bits)
    q = torch.randn(1, g, 1, dh, generator=gen).to(dt)
    codes = torch.randint(-1, 2, (1 << 17, dh), generator=gen)
    ks = (torch.rand(1 << 17, groups, generator=gen) + 0.5).bfloat16()
    k = codes.double() * ks.double().repeat_interleave(32, -1)[:, :dh]
    lead = q[0, 0, 0].double()
    scale = 2000.0 / float((k.abs() @ lead.abs()).mean())
    pick = torch.argsort((k @ lead).abs())[:n]  # of the first query; the others' are what they are
    pick = pick[torch.randperm(n, generator=gen)]
    u = (codes[pick] + top + 1).to(torch.uint8)
    u = u[:, 0::2] + 16 * u[:, 1::2] if bits == 4 else u
    cache, _, _ = make([n], 1, 1, dh, page, bits, dt, 52)
    for t in range(n):
        pg, row = place(cache, 0, t)
        cache[0][pg, 0, row] = u[t]
        cache[2][pg, 0, row, 0] = ks[pick[t]]
    check(q, cache, bits, scale, mass=True)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt,g", KINDS)
@pytest.mark.parametrize("dh,page", [(64, 16), (128, 16), (80, 8)])
@pytest.mark.parametrize("far", [-45, 45])
def test_groups_of_queries_and_keys_far_apart(bits, dt, g, dh, page, far):
    """A group of the query's dims 2^far times the others, and its keys 2^-far times: ordinary scores."""
    cache, q, _ = make([300, 40], 2, g, dh, page, bits, dt, 61)
    q = q.float()
    q[..., :32] *= 2.0 ** far
    cache[2][..., 0, 0] *= 2.0 ** -far
    check(q.to(dt), cache, bits, dh ** -0.5, mass=True)


def test_scale_of_zero_and_queries_of_every_size():
    cache, q, _ = make([200, 30], 2, 3, 64, 16, 4, F32, 91)
    for dt in (BF, F32):
        for size, scale in ((1.0, 0.0), (2.0 ** 120, 2.0 ** -122), (2.0 ** -120, 2.0 ** 118), (1.0, -0.3), (2.0 ** -60, 0.125)):
            check((q * size).to(dt), cache, 4, scale, mass=True)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt,g", KINDS)
@pytest.mark.parametrize("lengths,dh,page", SHAPES)
@pytest.mark.parametrize("what", [-INF, INF, NAN])
def test_queries_that_are_not_finite_are_nan_alone(bits, dt, g, lengths, dh, page, what):
    T = ops()
    cache, q, _ = make(lengths, 2, g, dh, page, bits, dt, 71)
    dev = [x.cuda() for x in cache]
    clean = T.turbo_paged_quant_attention(q.cuda(), *dev)
    for head, d in ((0, 0), (2 * g - 1, dh - 1), (g, dh // 2)):
        x = q.clone()
        x[0, head, 0, d] = what
        out = T.turbo_paged_quant_attention(x.cuda(), *dev)
        assert bool(out[0, head].isnan().all())
        out[0, head] = clean[0, head]
        assert torch.equal(out, clean)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt,g", KINDS)
@pytest.mark.parametrize("lengths,dh,page", SHAPES)
@pytest.mark.parametrize("far", [8, 16, 20])
def test_large_dims_of_queries_that_keys_leave_alone(bits, dt, g, lengths, dh, page, far):
    """Two dims of the query 2^far times the others, where all keys have the code 0: they add nothing."""
    cache, q, _ = make(lengths, 2, g, dh, page, bits, dt, 101)
    q = q.float()
    for d in (0, dh - 1):
        q[..., d] *= 2.0 ** far
        if bits == 8:
            cache[0][..., d] = zero_code(bits)
        else:
            cache[0][..., d // 2] = cache[0][..., d // 2] & (0x0f if d % 2 else 0xf0) | (0x80 if d % 2 else 0x08)
    check(q.to(dt), cache, bits, 3 * dh ** -0.5, mass=True)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt,g", KINDS)
@pytest.mark.parametrize("lengths,dh,page", SHAPES)
def test_rows_whose_scores_are_all_minus_infinity(bits, dt, g, lengths, dh, page):
    """A query of -inf in a dim where every key is positive: nothing is attended to, as by the dense operator:
    zeros and no masses, and the other queries as ever."""
    T = ops()
    cache, q, _ = make(lengths, 2, g, dh, page, bits, dt, 71)
    if bits == 4:  # codes of 3 in dims 0, 2, ..
        cache[0] = cache[0] & 0xf0 | 0x0b
    else:  # codes of 1 and more
        cache[0] |= 0x81
    dev = [x.cuda() for x in cache]
    clean = T.turbo_paged_quant_attention(q.cuda(), *dev)
    kd, vd = T.turbo_paged_quant_read(*dev, max(lengths), dh, dtype=dt)  # a dense cache of one page per sequence
    table = torch.arange(len(lengths), dtype=torch.int32, device="cuda")[:, None]
    for none in ([0], [2 * g - 1], list(range(2 * g))):
        x = q.clone()
        x[0, none, 0, 0] = -INF
        m = torch.zeros(len(lengths), 2, cache[3].shape[1] * page, device="cuda")
        out = T.turbo_paged_quant_attention(x.cuda(), *dev, mass=m)
        assert bool((out[0, none] == 0).all())
        assert bool((T.turbo_paged_attention(x.cuda(), kd, vd, table, dev[4])[0, none] == 0).all())
        left = [h for h in range(2 * g) if h not in none]
        assert torch.equal(out[0, left], clean[0, left]) and torch.equal(out[1:], clean[1:])
        # a live query's weights sum to 1, each of n within a few roundings of it
        total = torch.tensor([sum(h // g == kv and h not in none for h in range(2 * g)) for kv in range(2)], dtype=torch.float32)
        assert torch.allclose(m[0].sum(-1).cpu(), total, rtol=0, atol=g * max(lengths) * 2.0 ** -22)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("g", [2, 7])
@pytest.mark.parametrize("lengths,dh,page", SHAPES)
def test_larger_dims_of_fp32_queries_that_keys_leave_alone(bits, g, lengths, dh, page):
    """fp32 holds dims 2^28 below their group's largest as well as a sum's own rounding."""
    test_large_dims_of_queries_that_keys_leave_alone(bits, F32, g, lengths, dh, page, 28)

"""The operators over a paged cache in 4 or 8 bits against the formulas in 64 bits."""
import itertools
import math

import pytest
import torch

import paged_util as P
import quant_util as Q

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")


@pytest.fixture(autouse=True)
def no_device_error():
    from one import turbo_ops as T
    T.ops_error(clear=True)
    yield
    assert T.ops_error(clear=True) == (0, 0)


def ops():
    from one import turbo_ops
    return turbo_ops


def gen_of(*key):
    return torch.Generator().manual_seed(hash(key) % 2 ** 31)


def cuda(ts):
    return tuple(t.cuda() for t in ts)


def same(a, b):
    """Equal bits, NaN as NaN."""
    a, b = a.cpu(), b.cpu()
    if a.dtype.is_floating_point:
        return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0, 1e30, -1e30), b.nan_to_num(0, 1e30, -1e30))
    return torch.equal(a, b)


# ------------------------------------------------------------------ quantising as it is written
def rotated(x, cos, sin):
    return (P.rotate(x, cos, sin) if cos is not None else x.double()).float()


def append_case(dt, bits, hkv, g, dh, page, starts, n, counts=None, tables=None, strided=False, cos_batch=None, special=False, offset=0):
    T, gen = ops(), gen_of(bits, hkv, dh, page, n, strided)
    B = len(starts)
    width = -(-(max(starts) + n) // page) + 1
    k0, v0, s0, table, lengths = Q.make_cache([x + n for x in starts], hkv, dh, page, bits, gen, width=width)
    lengths = torch.tensor(starts, dtype=torch.int32)

    def new(h):
        x = (torch.randn(B, n, h, dh, generator=gen) * torch.exp(torch.randn(h, dh, generator=gen))).to(dt)
        return x
    k, v, q = new(hkv), new(hkv), new(hkv * g)
    if special:  # rows of zeros, tiny, huge, infinite and NaN values, halves of steps, a lone value
        for i, row in enumerate((torch.zeros(dh), torch.full((dh,), 1e-38), torch.linspace(-3e38, 3e38, dh),
                                 torch.arange(dh) * 0.5 - 3.5, torch.eye(dh)[dh - 1] * 1e-20, torch.arange(dh) * 2.0 ** -104,
                                 torch.linspace(-1, 1, dh) * 7 * 2.0 ** -100, torch.linspace(0, 1, dh) * 2.0 ** -97)):
            k[0, i % n, i % hkv] = v[0, i % n, (i + 1) % hkv] = row.to(dt)
        v[-1, 0, 0, dh // 2], v[-1, -1, -1, 0], k[-1, -1, 0, dh - 1] = INF, -INF, NAN
    cos = sin = None
    if tables is not None:
        pos = torch.tensor(starts[:cos_batch])[:, None] + torch.arange(n)
        ang = pos[..., None].double() * 1e4 ** (-torch.arange(0, dh, 2).double() / dh)
        ang = torch.cat([ang, ang], -1)
        cos, sin = ang.cos().to(tables), ang.sin().to(tables)
    dev = [x.cuda() for x in (k, v, q)]
    if offset:  # rows that start off every vector boundary
        dev = [torch.cat([x.flatten(), x.new_zeros(8)])[:x.numel()].view(x.shape) if False else
               torch.empty(x.numel() + offset, dtype=dt, device="cuda")[offset:].view(x.shape).copy_(x) for x in dev]
    kd, vd, qd = (x.transpose(1, 2) if strided else x.transpose(1, 2).contiguous() for x in dev)
    if offset and not strided:
        kd, vd, qd = (torch.empty(x.numel() + offset, dtype=dt, device="cuda")[offset:].view(x.shape).copy_(x) for x in (kd, vd, qd))
    pools = cuda((k0, v0, s0))
    mass = torch.full((B, hkv, width * page), 7.0, device="cuda")
    cnt = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    out = T.turbo_paged_quant_append(kd, vd, *pools, table.cuda(), lengths.cuda(), cos=None if cos is None else cos.cuda(),
                                     sin=None if sin is None else sin.cuda(), q=qd, counts=cnt, mass=mass)
    # the formulas
    rk, rv = rotated(k.transpose(1, 2), cos, sin), v.transpose(1, 2).float()
    want, m = [k0.clone(), v0.clone(), s0.clone()], torch.full_like(mass.cpu(), 7.0)
    for w, x in enumerate((rk, rv)):
        codes, scales = Q.close(x, bits)
        for b in range(B):
            for t in range(n if counts is None else counts[b]):
                slot = starts[b] + t
                pg, at = int(table[b, slot // page]), slot % page
                want[w][pg, :, at] = codes[b, :, t]
                want[2][pg, :, at, w] = scales[b, :, t]
                m[b, :, slot] = 0
    for name, a, b_ in zip(("keys", "values", "scales"), pools, want):
        assert same(a, b_), name
    assert torch.equal(mass.cpu(), m)
    rq = P.rotate(q.transpose(1, 2), cos, sin) if cos is not None else q.transpose(1, 2).double()
    # fp32 (or, of two inexact products, fp64) arithmetic, then one rounding to dtype
    tol = torch.finfo(dt).eps / 2 * rq.abs() + 2.0 ** -23 * q.transpose(1, 2).abs().amax(-1, keepdim=True).double() * 2
    d = (out.cpu().double() - rq).abs()
    assert bool((d[torch.isfinite(rq)] <= tol[torch.isfinite(rq)]).all())
    return pools


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt,tables", [(BF, BF), (BF, F32), (BF, None), (F32, F32), (F32, None)])
@pytest.mark.parametrize("hkv,g,dh,page", [(2, 1, 64, 16), (3, 2, 80, 8), (1, 4, 128, 5), (5, 1, 16, 1), (4, 1, 32, 3), (2, 3, 96, 48),
                                           (2, 1, 48, 7), (1, 1, 112, 16)])
def test_append(bits, dt, tables, hkv, g, dh, page):
    append_case(dt, bits, hkv, g, dh, page, [0, 13, 5], 9, counts=[9, 0, 4], tables=tables, strided=dh in (64, 80, 32))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("dh", [32, 64, 80, 128])
def test_append_single_tokens_and_special_values(bits, dt, dh):
    append_case(dt, bits, 4, 1, dh, 16, [0, 15, 16, 31, 200, 3, 9], 1, tables=dt, strided=True)
    append_case(dt, bits, 3, 1, dh, 16, [4, 7], 8, special=True)


@pytest.mark.parametrize("offset", [1, 4, 8])
def test_append_rows_off_vector_boundaries(offset):
    for dt, strided in itertools.product((BF, F32), (True, False)):
        append_case(dt, 4, 3, 2, 64, 16, [5, 30], 6, tables=dt, strided=strided, offset=offset)


def test_append_shared_tables_and_prompts():
    append_case(BF, 4, 12, 1, 64, 16, [0, 0, 0], 333, counts=[333, 100, 257], tables=BF, strided=True, cos_batch=1)
    append_case(BF, 8, 5, 2, 128, 64, [0, 70], 200, tables=BF, strided=True)
    append_case(F32, 4, 4, 1, 96, 16, [3, 0], 150, counts=[1, 150], tables=F32, strided=True, cos_batch=1)


# ------------------------------------------------------------------ reading back
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("hkv,dh,page", [(2, 64, 16), (3, 80, 8), (1, 128, 5), (5, 16, 1), (4, 32, 3), (2, 96, 48), (1, 112, 16)])
def test_read(bits, dt, hkv, dh, page):
    T = ops()
    cache = Q.make_cache([0, 1, 37, 200, 16], hkv, dh, page, bits, gen_of(bits, dh), width=-(-200 // page) + 2)
    dev = cuda(cache)
    for n, starts in ((200, None), (1, None), (37, None), (150, [0, 0, 36, 170, 3]), (7, [5, 1, 30, 0, 16]), (230, [0, 0, 0, 0, 0])):
        st = None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda")
        got = T.turbo_paged_quant_read(*dev, n, dh, starts=st, dtype=dt)
        for w in range(2):
            want = torch.zeros(5, hkv, n, dh, dtype=torch.float64)
            for b in range(5):
                x = Q.rows(cache, w, b, int(cache[4][b]), bits, dh)[:, (starts[b] if starts else 0):][:, :n]
                want[b, :, :x.shape[1]] = x
            assert torch.equal(got[w].cpu(), want.to(dt))  # scale * code is exact in fp32, rounded once


def test_read_nothing():
    T = ops()
    k, v, s, t, n = cuda(Q.make_cache([5, 3], 2, 64, 16, 4, gen_of(1)))
    assert T.turbo_paged_quant_read(k, v, s, t, n, 0, 64)[0].shape == (2, 2, 0, 64)
    assert T.turbo_paged_quant_read(k, v, s, t[:0], n[:0], 4, 64)[1].shape == (0, 2, 4, 64)
    x = torch.zeros(2, 2, 0, 64, dtype=BF, device="cuda")
    assert T.turbo_paged_quant_append(x, x, k, v, s, t, n) is None
    assert T.turbo_paged_quant_attention(torch.zeros(0, 4, 1, 64, dtype=BF, device="cuda"), k, v, s, t[:0], n[:0]).shape == (0, 4, 1, 64)
    m, kept = T.turbo_paged_quant_evict(k, v, s, t[:0], t[:0].clone(), n[:0], torch.zeros(0, 2, 16, device="cuda"), 8)
    assert m.shape == (0, 2, 16) and kept.shape == (0, 2, 8)


def test_groups_that_are_not_finite_read_as_nan_alone():
    T, dh = ops(), 96
    k = torch.randn(1, 1, 4, dh, generator=gen_of(5)).cuda()
    x = k.clone()
    x[0, 0, 1, 40], x[0, 0, 2, 0], x[0, 0, 2, 95] = INF, NAN, -INF
    for bits in (4, 8):
        pools = T.turbo_paged_quant_pools(1, 1, 16, dh, bits)
        t, n = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        T.turbo_paged_quant_append(x, x, *pools, t, n)
        a, b = T.turbo_paged_quant_read(*pools, t, n + 4, 4, dh, dtype=F32)
        assert torch.equal(a.isnan(), b.isnan())
        want = torch.zeros(4, dh, dtype=torch.bool)
        want[1, 32:64] = want[2, :32] = want[2, 64:] = True
        assert torch.equal(a[0, 0].isnan().cpu(), want)
        # and in the attention: keys of NaN make the row NaN, values of NaN the dims of their group
        q = torch.randn(1, 1, 1, dh, device="cuda")
        T.turbo_paged_quant_append(k, x, *pools, t, n)
        out = T.turbo_paged_quant_attention(q, *pools, t, n + 2)
        assert torch.equal(out[0, 0, 0].isnan().cpu(), want[1])
        T.turbo_paged_quant_append(x, k, *pools, t, n)
        assert bool(T.turbo_paged_quant_attention(q, *pools, t, n + 2).isnan().all())
        assert bool(torch.isfinite(T.turbo_paged_quant_attention(q, *pools, t, n + 1)).all())


# ------------------------------------------------------------------ attention
def check_attention(dt, bits, hkv, g, dh, page, lengths, mass=False, scale=None, width=None, qs=1.0, seed=0, q_strided=False):
    T, gen = ops(), gen_of(bits, hkv, g, dh, page, seed)
    cache = Q.make_cache(lengths, hkv, dh, page, bits, gen, width=width)
    B, width = len(lengths), cache[3].shape[1]
    q = (torch.randn(B, hkv * g, 1, dh, generator=gen) * qs).to(dt)
    sc = dh ** -0.5 if scale is None else scale
    ref, ps, mag, smax = Q.attention(q, cache, bits, sc)
    m0 = torch.rand(B, hkv, width * page + 3, generator=gen) if mass else None
    m = None if m0 is None else m0.cuda()
    qd = q.cuda()
    if q_strided:
        qd = torch.empty(B, 1, hkv * g, dh + 8, dtype=dt, device="cuda")[..., :dh].transpose(1, 2).copy_(qd)
    out = T.turbo_paged_quant_attention(qd, *cuda(cache), scale_factor=scale, mass=m)
    n = max(max(lengths), 1)
    e = Q.weight_error(n, dh, smax, dt)
    d, tol = (out.cpu().double() - ref).abs(), e * mag + torch.finfo(dt).eps / 2 * ref.abs() * (1 + e) + 1e-30
    assert out.dtype == dt and bool((d <= tol).all()), float((d - tol).max())
    if mass:
        want = m0.double().clone()
        for b in range(B):
            want[b, :, :lengths[b]] += ps[b].view(hkv, g, -1).sum(1)
        e = Q.weight_error(n, dh, smax, F32)  # the masses' weights are in fp32 throughout
        add = want - m0.double()
        # approximate 2^x: 2^-22 relative; g sums and one sum with the mass, each rounded to fp32
        tol = (e + 2.0 ** -21) * add + (g + 1) * 2.0 ** -24 * want
        assert bool(((m.cpu().double() - want).abs() <= tol).all())
    return out


DIMS = [(64, 16), (32, 16), (128, 64), (96, 48), (80, 16), (16, 8), (48, 5), (112, 1), (64, 1), (128, 24)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("dh,page", DIMS)
def test_attention_dims_and_pages(bits, dt, dh, page):
    check_attention(dt, bits, 2, 3, dh, page, [0, 1, 7, 40, 129], mass=True)
    check_attention(dt, bits, 1, 1, dh, page, [65, 300, 1100])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("hkv,g", [(1, 1), (3, 2), (2, 4), (1, 7), (2, 8), (1, 9), (2, 12), (1, 16), (1, 17), (1, 33)])
def test_attention_heads(bits, dt, hkv, g):
    check_attention(dt, bits, hkv, g, 64, 16, [33, 500, 0], mass=True)
    check_attention(dt, bits, hkv, g, 128, 32, [200, 15])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("lengths", [[1], [15], [16], [17], [64], [255], [256], [257], [513], [3000], [5000, 1, 0, 700], [0], [0, 0, 3]])
def test_attention_lengths(bits, dt, lengths):
    check_attention(dt, bits, 2, 2, 64, 16, lengths, mass=len(lengths) % 2 == 0)
    check_attention(dt, bits, 1, 1, 128, 16, lengths, mass=len(lengths) % 2 == 1)


@pytest.mark.parametrize("dt", [BF, F32])
def test_attention_batches_of_every_cut(dt):
    check_attention(dt, 4, 4, 1, 64, 16, [(37 * i) % 500 for i in range(90)], mass=True)        # a CTA per segment
    check_attention(dt, 4, 12, 1, 64, 16, [900, 20, 1500, 0, 333, 1999] * 3)                    # a list
    check_attention(dt, 8, 2, 4, 128, 48, [4000, 100, 2500], mass=True)                         # a list, with weights
    check_attention(dt, 4, 8, 1, 32, 16, [(11 * i) % 60 for i in range(300)])
    check_attention(dt, 4, 2, 1, 64, 16, [700, 650, 800], mass=True, width=2000)                # a table far wider than its sequences


@pytest.mark.parametrize("dt", [BF, F32])
def test_attention_scales_and_peaks(dt):
    check_attention(dt, 4, 2, 2, 64, 16, [100, 300], scale=0.0)
    check_attention(dt, 4, 2, 2, 64, 16, [100, 300], scale=-0.3)
    check_attention(dt, 8, 2, 2, 64, 16, [100, 300], qs=20.0, mass=True)     # one slot takes it all
    check_attention(dt, 4, 2, 2, 64, 16, [100, 300], qs=1e-6)
    check_attention(dt, 4, 2, 2, 64, 16, [100, 300], qs=0.0)
    check_attention(dt, 4, 2, 2, 64, 16, [100, 300], qs=1e18, scale=1e-18)
    check_attention(dt, 4, 2, 3, 64, 16, [100, 300], q_strided=True)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("bits", [4, 8])
def test_attention_values_of_very_different_sizes(dt, bits):
    """Scales of values that grow and shrink by many powers of two along the sequence."""
    T, gen = ops(), gen_of(bits, 77)
    cache = list(Q.make_cache([700, 90], 2, 64, 16, bits, gen))
    size = torch.exp2(torch.randint(-30, 30, cache[2].shape[:3], generator=gen).float())
    cache[2][..., 1, :] = (cache[2][..., 1, :].float() * size[..., None]).bfloat16()
    q = torch.randn(2, 4, 1, 64, generator=gen).to(dt)
    ref, _, mag, smax = Q.attention(q, cache, bits, 0.125)
    out = T.turbo_paged_quant_attention(q.cuda(), *cuda(cache))
    e = Q.weight_error(700, 64, smax, dt)
    d, tol = (out.cpu().double() - ref).abs(), e * mag + torch.finfo(dt).eps / 2 * ref.abs() * (1 + e)
    assert bool((d <= tol).all()), float((d / tol).max())


def test_attention_rows_without_a_mask_left():
    """All scores -inf (a query of -inf times positive keys is refused by no one): NaN or 0 stay in their row."""
    T = ops()
    k, v, s, t, n = cuda(Q.make_cache([40, 33], 1, 64, 16, 4, gen_of(9)))
    q = torch.randn(2, 2, 1, 64, device="cuda").bfloat16()
    clean = T.turbo_paged_quant_attention(q, k, v, s, t, n)
    q[0, 1] = NAN
    out = T.turbo_paged_quant_attention(q, k, v, s, t, n)
    assert bool(out[0, 1].isnan().all()) and torch.equal(out[0, 0], clean[0, 0]) and torch.equal(out[1], clean[1])


# ------------------------------------------------------------------ eviction
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hkv,dh,page,lengths,budget,recent,sink", [
    (2, 64, 16, [100, 40, 0], 40, 8, 4), (3, 80, 8, [333, 20, 1], 100, 0, 0), (1, 16, 1, [50, 64], 33, 33, 0),
    (2, 128, 5, [1200, 700], 600, 100, 16), (1, 48, 16, [5000], 700, 5, 1), (4, 96, 48, [3000, 2999, 100] * 14, 1000, 64, 4),
    (1, 32, 16, [20000], 300, 10, 2), (1, 112, 16, [40000], 1000, 100, 4)])
def test_evict(bits, hkv, dh, page, lengths, budget, recent, sink):
    T, gen = ops(), gen_of(dh, page)
    B, src = len(lengths), [-(-n // page) for n in lengths]
    dst = [-(-min(n, budget) // page) for n in lengths]
    k, v, s, table, n = Q.make_cache(lengths, hkv, dh, page, bits, gen, spare=sum(dst) + 3)
    free = sorted(set(range(k.shape[0])) - set(table[table >= 0].tolist()))
    to = torch.full((B, -(-budget // page) + 1), -1, dtype=torch.int32)
    for b in range(B):
        for i in range(dst[b]):
            to[b, i] = free.pop()
    mass = torch.randint(0, 40, (B, hkv, table.shape[1] * page), generator=gen).float()
    mass[:, :, ::17] = NAN
    dev = cuda((k, v, s))
    got_mass, kept = T.turbo_paged_quant_evict(*dev, table.cuda(), to.cuda(), n.cuda(), mass.cuda(), budget, recent=recent, sink=sink)
    want = [x.clone() for x in (k, v, s)]
    want_mass, want_kept = torch.zeros(got_mass.shape), torch.full((B, hkv, budget), -1, dtype=torch.int32)
    for b in range(B):
        for h in range(hkv):
            keep = torch.tensor(P.evict(mass[b, h], lengths[b], budget, recent, sink), dtype=torch.int64)
            at = torch.arange(len(keep))
            want_kept[b, h, :len(keep)] = keep
            want_mass[b, h, :len(keep)] = mass[b, h, keep]
            for x, y in zip(want, (k, v, s)):
                x[to[b].long()[at // page], h, at % page] = y[table[b].long()[keep // page], h, keep % page]
    assert torch.equal(kept.cpu(), want_kept) and same(got_mass, want_mass)
    for a, b_ in zip(dev, want):
        assert same(a, b_)


# ------------------------------------------------------------------ bad pages and lengths
def test_bad_pages_and_lengths_are_recorded():
    T = ops()
    k, v, s, t, n = cuda(Q.make_cache([40, 30], 2, 64, 16, 4, gen_of(3)))
    pages = k.shape[0]
    q = torch.randn(2, 2, 1, 64, device="cuda").bfloat16()
    good = T.turbo_paged_quant_attention(q, k, v, s, t, n)
    for page in (-1, pages, 2 ** 31 - 1, -2 ** 31):
        bad = t.clone()
        bad[0, 1] = page
        out = T.turbo_paged_quant_attention(q, k, v, s, bad, n)
        assert T.ops_error(clear=True)[0] == 2
        assert bool(torch.isfinite(out).all()) and torch.equal(out[1], good[1])
        a, b = T.turbo_paged_quant_read(k, v, s, bad, n, 40, 64)
        assert T.ops_error(clear=True)[0] == 2
        assert bool((a[0, :, 16:32] == 0).all()) and bool((b[0, :, 16:32] == 0).all()) and bool((a[0, :, 32:] != 0).any())
        before = [x.clone() for x in (k, v, s)]
        x = torch.randn(2, 2, 1, 64, device="cuda").bfloat16()
        T.turbo_paged_quant_append(x, x, k, v, s, bad, torch.tensor([20, 48], dtype=torch.int32, device="cuda"))
        assert T.ops_error(clear=True)[0] == 2
        assert all(same(a_, b_) for a_, b_ in zip((k, v, s), before))
    wrong = torch.tensor([-5, 1000], dtype=torch.int32, device="cuda")
    out = T.turbo_paged_quant_attention(q, k, v, s, t.clamp(min=0), wrong)
    assert T.ops_error(clear=True)[0] == 2 and bool((out[0] == 0).all())
    T.turbo_paged_quant_read(k, v, s, t, n, 4, 64, starts=torch.tensor([-2, 0], dtype=torch.int32, device="cuda"))
    assert T.ops_error(clear=True)[0] == 2


# ------------------------------------------------------------------ addresses past 32 bits
@pytest.mark.parametrize("page", [16, 12])
def test_pools_past_four_gigabytes(page):
    T, hkv, dh = ops(), 8, 128
    per = hkv * page * dh // 2
    pages = (9 << 29) // per + 4  # 4.5 GB of codes
    k, v = (torch.zeros(pages, hkv, page, dh // 2, dtype=torch.uint8, device="cuda") for _ in range(2))
    s = torch.zeros(pages, hkv, page, 2, 4, dtype=BF, device="cuda")
    gen = gen_of(12)
    x, y = (torch.randn(1, hkv, 3 * page, dh, generator=gen).bfloat16().cuda() for _ in range(2))
    q = torch.randn(1, hkv, 1, dh, generator=gen).bfloat16().cuda()
    n0 = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = []
    for where in ([pages - 1, 0, pages - 2], [1, 2, 3]):
        t = torch.tensor([where], dtype=torch.int32, device="cuda")
        T.turbo_paged_quant_append(x, y, k, v, s, t, n0)
        n = n0 + 3 * page
        got.append([T.turbo_paged_quant_attention(q, k, v, s, t, n), *T.turbo_paged_quant_read(k, v, s, t, n, 3 * page, dh)])
        to = torch.tensor([[w + (5 if w < 10 else -5) for w in where]], dtype=torch.int32, device="cuda")
        mass = torch.rand(1, hkv, 3 * page, generator=torch.Generator().manual_seed(4)).cuda()
        m, kept = T.turbo_paged_quant_evict(k, v, s, t, to, n, mass, 2 * page, recent=4)
        got[-1] += [m, kept, *T.turbo_paged_quant_read(k, v, s, to, n0 + 2 * page, 2 * page, dh)]
    for a, b in zip(*got):
        assert torch.equal(a, b)
    codes, scales = Q.close(x.cpu().float(), 4)
    assert torch.equal(got[0][1].cpu(), Q.open_(codes, scales, 4, dh).bfloat16())


# ------------------------------------------------------------------ together, streams, graphs
def serve(T, steps, bits, graph, dt=BF, stream=None):
    """A prompt, decode steps with masses, an eviction, more steps: outputs of every call."""
    gen = gen_of(bits, 21)
    B, hkv, g, dh, page, slots = 3, 2, 2, 64, 16, 8
    pools = T.turbo_paged_quant_pools(2 * B * slots, hkv, page, dh, bits)
    for x in pools:
        x.zero_()
    order = torch.randperm(2 * B * slots, generator=gen).to(torch.int32)
    tables = order.view(2, B, slots).cuda()
    table, lengths = tables[0].clone(), torch.zeros(B, dtype=torch.int32, device="cuda")
    mass = torch.zeros(B, hkv, slots * page, device="cuda")
    counts = torch.tensor([50, 17, 33], dtype=torch.int32, device="cuda")

    def new(n):
        return [torch.randn(B, h, n, dh, generator=gen).to(dt).cuda() for h in (hkv, hkv, hkv * g)]
    k, v, _ = new(50)
    T.turbo_paged_quant_append(k, v, *pools, table, lengths, counts=counts, mass=mass)
    lengths += counts
    out = []
    kx, vx, qx = new(1)

    def step():
        q = T.turbo_paged_quant_append(kx, vx, *pools, table, lengths, q=qx, mass=mass)
        lengths.add_(1)
        return T.turbo_paged_quant_attention(q, *pools, table, lengths, mass=mass)
    play = step
    if graph:
        keep = [x.clone() for x in (*pools, lengths, mass)]
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y = step()
        for x, z in zip((*pools, lengths, mass), keep):
            x.copy_(z)

        def play():
            gr.replay()
            return y.clone()
    for i in range(steps):
        for x, z in zip((kx, vx, qx), new(1)):
            x.copy_(z)
        out.append(play())
        if i == steps // 2:
            m, kept = T.turbo_paged_quant_evict(*pools, table, tables[1], lengths, mass, 40, recent=8, sink=2)
            table.copy_(tables[1])
            lengths.clamp_(max=40)
            mass.copy_(m)
            out += [m, kept]
    out += list(T.turbo_paged_quant_read(*pools, table, lengths, slots * page, dh, dtype=dt))
    return out, (pools, table, lengths, mass)


@pytest.mark.parametrize("bits", [4, 8])
def test_a_run_of_them_together(bits):
    T = ops()
    plain, state = serve(T, 12, bits, False)
    again, _ = serve(T, 12, bits, False)
    graph, _ = serve(T, 12, bits, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other, _ = serve(T, 12, bits, False)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b, c, d in zip(plain, again, graph, other):
        assert same(a, b) and same(a, c) and same(a, d)
    # the last step once more, from the cache's values through the dense attention operator's formula
    (k, v, s), table, lengths, _ = state
    q = torch.randn(3, 4, 1, 64, generator=gen_of(2)).bfloat16()
    cache = tuple(x.cpu() for x in (k, v, s, table, lengths))
    ref, _, mag, smax = Q.attention(q, cache, bits, 0.125)
    out = T.turbo_paged_quant_attention(q.cuda(), k, v, s, table, lengths)
    e = Q.weight_error(128, 64, smax, BF)
    assert bool(((out.cpu().double() - ref).abs() <= e * mag + 2.0 ** -8 * ref.abs() * (1 + e)).all())


@pytest.mark.parametrize("dt", [BF, F32])
def test_attention_repeats_bit_for_bit(dt):
    T = ops()
    cache = cuda(Q.make_cache([3000, 40, 1500, 0, 999], 4, 64, 16, 4, gen_of(8)))
    q = torch.randn(5, 8, 1, 64, device="cuda").to(dt)
    m = [torch.zeros(5, 4, cache[3].shape[1] * 16, device="cuda") for _ in range(4)]
    out = [T.turbo_paged_quant_attention(q, *cache, mass=x) for x in m]
    for a, b in zip(out[1:], m[1:]):
        assert torch.equal(a, out[0]) and torch.equal(b, m[0])


def test_pages_apart_and_shared():
    """Slices of one pool, and one page in two sequences."""
    T, gen = ops(), gen_of(31)
    k, v, s, t, n = Q.make_cache([60, 60], 2, 64, 16, 4, gen)
    t[1, :2] = t[0, :2]
    big = torch.zeros(k.shape[0], 2, 2, 16, 32, dtype=torch.uint8, device="cuda")
    sc = torch.zeros(k.shape[0], 3, 2, 16, 2, 2, dtype=BF, device="cuda")
    kd, vd, sd = big[:, 0], big[:, 1], sc[:, 1]
    kd.copy_(k), vd.copy_(v), sd.copy_(s)
    q = torch.randn(2, 4, 1, 64, generator=gen).bfloat16()
    ref, _, mag, smax = Q.attention(q, (k, v, s, t, n), 4, 0.125)
    e = Q.weight_error(60, 64, smax, BF)
    out = T.turbo_paged_quant_attention(q.cuda(), kd, vd, sd, t.cuda(), n.cuda())
    assert bool(((out.cpu().double() - ref).abs() <= e * mag + 2.0 ** -8 * ref.abs() * (1 + e)).all())
    odd = torch.zeros(k.shape[0] * (2 * 16 * 32 + 8), dtype=torch.uint8, device="cuda").view(k.shape[0], -1)[:, 8:].unflatten(1, (2, 16, 32))
    odd.copy_(k)  # pages on 8-byte boundaries alone
    so = torch.zeros(k.shape[0] * (2 * 16 * 4 + 2), dtype=BF, device="cuda").view(k.shape[0], -1)[:, 2:].unflatten(1, (2, 16, 2, 2))
    so.copy_(s)
    assert torch.equal(T.turbo_paged_quant_attention(q.cuda(), odd, vd, so, t.cuda(), n.cuda()), out)
    assert same(T.turbo_paged_quant_read(odd, vd, so, t.cuda(), n.cuda(), 60, 64)[0], T.turbo_paged_quant_read(kd, vd, sd, t.cuda(), n.cuda(), 60, 64)[0])

"""GPU tests of the paged key-value cache's operators against their formulas in 64 bits."""
import math

import pytest
import torch

import paged_util as P
from conftest import cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]

BF, F32 = torch.bfloat16, torch.float32


def ops():
    from one import turbo_ops
    return turbo_ops


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    assert ops().ops_error() == (0, 0)


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def check_attention(got, q, k, v, table, lens, scale, dt, mass=None, mass0=None):
    ref, ps, mag, smax = P.attention(q, k, v, table, lens, scale)
    n, dh = int(max(lens)), q.shape[-1]
    e = P.weight_error(n, dh, smax, dt)
    err = (got.cpu().double() - ref).abs()
    tol = torch.finfo(dt).eps / 2 * ref.abs() + e * mag * (1 + torch.finfo(dt).eps)
    assert bool((err <= tol).all()), f"out: {float((err - tol).max()):.3g} over"
    if mass is not None:
        want = mass0.double().clone()
        add = torch.zeros_like(want)
        hkv = k.shape[1]
        for b, p in enumerate(ps):
            add[b, :, :p.shape[1]] = p.unflatten(0, (hkv, -1)).sum(1)
        err = (mass.cpu().double() - want - add).abs()
        tol = 2.0 ** -23 * (want + add) + 2 * e * add  # the sum's rounding, the weights'
        assert bool((err <= tol).all()), f"mass: {float((err - tol).max()):.3g} over"


LENS = [0, 1, 15, 16, 17, 63, 64, 65, 130, 1000]
SHAPES = [  # hkv, group, dh, page, lengths
    (2, 1, 64, 16, LENS), (1, 3, 64, 1, [0, 1, 5, 33]), (2, 8, 32, 7, LENS), (1, 12, 128, 48, LENS), (3, 2, 40, 16, [77, 3, 0]),
    (1, 20, 96, 64, [500, 64]), (4, 16, 64, 32, [129, 2]), (1, 1, 8, 5, [40, 0, 1]), (2, 7, 128, 128, [4097, 127]),
    (12, 1, 64, 16, [2049]), (1, 8, 64, 16, [20000, 3]), (1, 1, 16, 3, [0, 0]), (5, 4, 112, 24, [1500, 31, 600]),
    (16, 1, 64, 16, [(i * 97) % 701 for i in range(30)]), (10, 2, 32, 32, [(i * 331) % 1300 for i in range(50)]),
    (1, 4, 64, 16, [300]), (2, 9, 128, 16, [4096, 1]), (1, 2, 96, 16, [8192 * 3, 5, 0]),
    (4, 1, 64, 16, [(i * 1000 + 700) % 4001 for i in range(9)]), (4, 2, 128, 16, [(i * 331) % 1001 for i in range(18)]),
]
MANY = [(i * 89) % 261 for i in range(33)]  # more segments than are taken one by one with a deep ring
SHAPES += [(10, g, dh, page, MANY) for g, dh, page in
           [(1, 64, 16), (9, 64, 32), (2, 128, 16), (12, 128, 16), (3, 96, 16), (10, 96, 48), (1, 32, 16), (20, 32, 5), (2, 80, 16)]]


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("with_mass", [False, True], ids=["plain", "mass"])
@pytest.mark.parametrize("shape", SHAPES, ids=[f"{s[0]}x{s[1]}x{s[2]}p{s[3]}n{max(s[4])}" for s in SHAPES])
def test_attention(shape, with_mass, dt):
    hkv, g, dh, page, lens = shape
    gen = torch.Generator().manual_seed(100 * dh + hkv)
    k, v, table, ln = P.make_cache(lens, hkv, dh, page, dt, gen)
    q = (1.5 * torch.randn(len(lens), hkv * g, 1, dh, generator=gen)).to(dt)
    mass0 = torch.rand(len(lens), hkv, table.shape[1] * page + 3, generator=gen) if with_mass else None
    dq, dk, dv, dtab, dl, dm = cuda(q, k, v, table, ln, mass0)
    got = ops().turbo_paged_attention(dq, dk, dv, dtab, dl, mass=dm)
    check_attention(got, q, k, v, table, ln, dh ** -0.5, dt, dm, mass0)


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "fp32"])
def test_attention_repeats_bit_for_bit_and_takes_scales(dt):
    gen = torch.Generator().manual_seed(3)
    k, v, table, ln = P.make_cache([3000, 17, 900], 2, 64, 16, dt, gen)
    q = torch.randn(3, 8, 1, 64, generator=gen).to(dt)
    d = cuda(q, k, v, table, ln)
    for scale in (0.5, 0.0, -0.25):
        a = ops().turbo_paged_attention(*d, scale_factor=scale)
        b = ops().turbo_paged_attention(*d, scale_factor=scale)
        assert torch.equal(a, b)
        check_attention(a, q, k, v, table, ln, scale, dt)


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("n", [2500, 9000])
def test_attention_large_scores(dt, n):
    """Scores of thousands, of both signs: one slot takes the whole weight; the running maximum rises
    within and across the parts of a split sequence."""
    gen = torch.Generator().manual_seed(4)
    k, v, table, ln = P.make_cache([n], 1, 64, 16, dt, gen)
    q = (300 * torch.randn(1, 4, 1, 64, generator=gen)).to(dt)
    d = cuda(q, k, v, table, ln)
    got = ops().turbo_paged_attention(*d)
    ref, ps, mag, smax = P.attention(q, k, v, table, ln, 0.125)
    assert float(max(p.max() for p in ps)) > 0.99
    check_attention(got, q, k, v, table, ln, 0.125, dt)


def test_attention_slices_of_one_pool_and_strided_queries():
    gen = torch.Generator().manual_seed(5)
    k, v, table, ln = P.make_cache([300, 40], 2, 64, 16, BF, gen)
    pool = torch.full((3, k.shape[0], 2, *k.shape[1:]), float("nan"), dtype=BF, device="cuda")  # [layers, pages, k | v, ...]
    pool = pool.transpose(0, 1)  # pages of the layers interleaved: the page stride is not the page's size
    pool[:, 1, 0], pool[:, 1, 1] = k.cuda(), v.cuda()
    wide = torch.randn(2, 1, 3, 4, 64, generator=gen).to(BF)
    q = wide[:, :, 1].transpose(1, 2)  # [2, 4, 1, 64], rows apart
    big = torch.full((2, table.shape[1] + 5), 10 ** 6, dtype=torch.int32)
    big[:, :table.shape[1]] = table
    got = ops().turbo_paged_attention(wide.cuda()[:, :, 1].transpose(1, 2), pool[:, 1, 0], pool[:, 1, 1],
                                      big.cuda()[:, :table.shape[1]], ln.cuda())
    check_attention(got, q, k, v, table, ln, 0.125, BF)


def test_offsets_past_32_bits():
    """A pool of more than 2^32 elements whose last pages are in use: append, attention, eviction."""
    gen = torch.Generator().manual_seed(6)
    hkv, dh, page = 2, 64, 16
    n = 2 ** 32 // (hkv * page * dh) + 40
    pool = torch.empty(n, hkv, page, dh, dtype=BF, device="cuda")
    lens = [300]
    k, v, table, ln = P.make_cache(lens, hkv, dh, page, BF, gen, spare=0)
    first = n - k.shape[0]
    pool[first:] = k.cuda()
    far = (table + first).to(torch.int32)
    q = torch.randn(1, 4, 1, dh, generator=gen).to(BF)
    dq, dl, dt_ = cuda(q, ln, far)
    got = ops().turbo_paged_attention(dq, pool, pool, dt_, dl)
    check_attention(got, q, k, k, table, ln, dh ** -0.5, BF)
    new = torch.randn(1, hkv, 1, dh, generator=gen).to(BF)
    ops().turbo_paged_append(new.cuda(), new.cuda(), pool, pool, dt_, dl - 1)
    assert torch.equal(pool[int(far[0, 299 // page]), :, 299 % page].cpu(), new[0, :, 0])
    mass = torch.rand(1, hkv, far.shape[1] * page, device="cuda")
    to = torch.arange(first - 8, first - 4, dtype=torch.int32, device="cuda").view(1, 4)
    _, kept = ops().turbo_paged_evict(pool, pool, dt_, to, dl, mass, 64)
    for h in range(hkv):
        src = kept[0, h].long()
        want = pool[dt_[0].long()[src // page], h, src % page]
        t = torch.arange(64, device="cuda")
        assert torch.equal(pool[to[0].long()[t // page], h, t % page], want)


def test_scores_of_minus_infinity():
    """Slots whose score is -inf weigh nothing; a sequence of such slots alone gives zeros."""
    gen = torch.Generator().manual_seed(7)
    for dt in (BF, F32):
        k, v, table, ln = P.make_cache([100, 20], 1, 64, 16, dt, gen)
        for b, t in [(0, t) for t in range(0, 90)] + [(1, t) for t in range(20)]:
            k[table[b, t // 16], :, t % 16] = -math.inf
        q = torch.rand(2, 2, 1, 64, generator=gen).add(0.1).to(dt)
        mass = torch.zeros(2, 1, table.shape[1] * 16)
        dq, dk, dv, dtab, dl, dm = cuda(q, k, v, table, ln, mass)
        got = ops().turbo_paged_attention(dq, dk, dv, dtab, dl, mass=dm).cpu()
        assert bool((got[1] == 0).all()) and bool((dm[1] == 0).all()) and bool((dm[0, :, :90] == 0).all())
        sub, subv = P.rows(k, table, 0, 100)[:, 90:], P.rows(v, table, 0, 100)[:, 90:]
        p = torch.softmax(torch.einsum("hd,nd->hn", q[0, :, 0].double(), sub[0].double()) * 0.125, -1)
        want = p @ subv[0].double()
        assert torch.allclose(got[0, :, 0].double(), want, rtol=2.0 ** -7, atol=2.0 ** -12)


def test_bad_pages_and_lengths_are_recorded():
    gen = torch.Generator().manual_seed(8)
    k, v, table, ln = P.make_cache([64, 64], 1, 64, 16, BF, gen)
    bad = table.clone()
    bad[0, 1], bad[0, 2] = k.shape[0], -7  # slots 16 .. 47 have no page
    q = torch.randn(2, 1, 1, 64, generator=gen).to(BF)
    dq, dk, dv, dbad, dl = cuda(q, k, v, bad, ln)
    got = ops().turbo_paged_attention(dq, dk, dv, dbad, dl)
    assert ops().ops_error()[0] == 2
    two = torch.stack([table[0, 0], table[0, 3]]).view(1, 2)  # the other slots are attended
    check_attention(got[:1], q[:1], k, v, two, torch.tensor([32]), 0.125, BF)
    check_attention(got[1:], q[1:], k, v, table[1:], ln[1:], 0.125, BF)
    far = torch.tensor([65, -3], dtype=torch.int32)  # beyond the table: its slots; negative: none
    got = ops().turbo_paged_attention(dq, dk, dv, table.cuda(), far.cuda())
    assert ops().ops_error()[0] == 2
    check_attention(got[:1], q[:1], k, v, table[:1], ln[:1], 0.125, BF)
    assert bool((got[1] == 0).all())
    before = dk.clone()
    new = torch.randn(2, 1, 2, 64, generator=gen).to(BF).cuda()
    full = torch.tensor([64, -1], dtype=torch.int32).cuda()
    ops().turbo_paged_append(new, new, dk, dv, table.cuda(), full)
    assert ops().ops_error()[0] == 2
    ops().turbo_paged_append(new, new, dk, dv, dbad, torch.tensor([16, 62], dtype=torch.int32).cuda())
    assert ops().ops_error()[0] == 2
    at = int(table[1, 3])
    before[at, :, 14:] = new[1]
    assert torch.equal(torch.nan_to_num(dk), torch.nan_to_num(before))
    mass = torch.rand(2, 1, 64, device="cuda")
    to = torch.tensor([[0, k.shape[0]], [-1, -1]], dtype=torch.int32).cuda()
    spare = [p for p in range(k.shape[0]) if p not in set(table.flatten().tolist())]
    to[0, 0] = spare[0]
    _, kept = ops().turbo_paged_evict(dk, dv, table.cuda(), to, dl, mass, 32)
    assert ops().ops_error()[0] == 2
    src = kept[0, 0, :16].long().cpu()
    assert torch.equal(dk[spare[0], 0].cpu(), dk.cpu()[table[0].long()[src // 16], 0, src % 16])


# ------------------------------------------------------------------ append
APPEND = [  # hkv, hq, dh, page, starts, n, counts
    (2, 4, 64, 16, [0, 5, 31], 1, None), (1, 0, 64, 16, [0, 40], 70, [70, 1]), (12, 12, 64, 16, [100] * 5, 1, None),
    (3, 3, 40, 7, [2, 0, 13], 9, [9, 0, 4]), (1, 5, 128, 1, [3], 20, None), (2, 2, 8, 3, [1, 1], 4, [2, 9]),
    (2, 6, 24, 64, [0], 333, None), (3, 5, 80, 16, [0, 7], 40, [40, 3]), (5, 1, 48, 5, [2], 17, None), (2, 2, 112, 32, [9], 33, None),
    (7, 5, 16, 8, [3, 0], 11, [11, 2]), (4, 4, 32, 48, [47, 48], 2, [-1, 2]), (1, 1, 96, 16, [16], 5, [5]),
]


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("rope", [None, "shared", "rows"])
@pytest.mark.parametrize("case", APPEND, ids=[f"{c[0]}x{c[2]}p{c[3]}n{c[5]}" for c in APPEND])
def test_append(case, rope, dt):
    hkv, hq, dh, page, starts, n, counts = case
    B = len(starts)
    gen = torch.Generator().manual_seed(10 * dh + n)
    cnt = [n] * B if counts is None else [min(max(c, 0), n) for c in counts]
    k, v, table, _ = P.make_cache([s + n for s in starts], hkv, dh, page, dt, gen, junk=7.0)
    new = [torch.randn(B, n, h, dh, generator=gen).to(dt).transpose(1, 2) if h else None for h in (hkv, hkv, hq)]
    cos = sin = None
    if rope:
        ang = torch.rand(B if rope == "rows" else 1, n, dh, generator=gen) * 6.28
        cos, sin = ang.cos().to(dt), ang.sin().to(dt)
    mass = torch.rand(B, hkv, table.shape[1] * page + 1, generator=gen) + 0.5
    dk, dv, dtab, dl, dm = cuda(k.clone(), v.clone(), table, torch.tensor(starts, dtype=torch.int32), mass)
    dcos, dsin, dcnt = cuda(cos, sin, None if counts is None else torch.tensor(counts, dtype=torch.int32))
    # the projections' layout: [B, N, heads, dim] seen as [B, heads, N, dim]
    dnew = [None if t is None else t.transpose(1, 2).contiguous().cuda().transpose(1, 2) for t in new]
    got = ops().turbo_paged_append(dnew[0], dnew[1], dk, dv, dtab, dl, cos=dcos, sin=dsin, q=dnew[2], counts=dcnt, mass=dm)
    # two products and a sum in fp32, one rounding
    u = torch.finfo(dt).eps / 2

    def close(x, src, rotated):
        want = P.rotate(src, cos, sin) if rotated and rope else src.double()
        mag = P.rotate(src.abs(), cos.abs(), -sin.abs()).abs() + want.abs() if rotated and rope else torch.zeros_like(want)
        if rotated and rope:
            h = src.shape[-1] // 2
            a, s2 = src.double().abs(), sin.double().abs()[:, None]
            mag = a * cos.double().abs()[:, None] + torch.cat([a[..., h:], a[..., :h]], -1) * s2
        return bool(((x.cpu().double() - want).abs() <= u * want.abs() + 2.0 ** -22 * mag).all())

    if hq:
        assert got.shape == (B, hq, n, dh) and close(got, new[2], True)
    else:
        assert got is None
    wm, touched = mass.clone(), torch.zeros(k.shape[0], page, dtype=torch.bool)
    for b in range(B):
        for t in range(cnt[b]):
            s = starts[b] + t
            touched[table[b, s // page], s % page] = True
            wm[b, :, s] = 0
    assert torch.equal(dm.cpu(), wm)
    keep = ~touched[:, None, :, None].expand_as(k)
    assert torch.equal(dk.cpu()[keep], k[keep]) and torch.equal(dv.cpu()[keep], v[keep])
    for b in range(B):
        if not cnt[b]:
            continue
        s = starts[b] + torch.arange(cnt[b])
        at = table[b].long()[s // page], s % page
        ck = None if cos is None else cos[b:b + 1] if rope == "rows" else cos
        kb, vb = (x.cpu()[at[0], :, at[1]].transpose(0, 1)[None] for x in (dk, dv))
        assert torch.equal(vb[0], new[1][b, :, :cnt[b]])
        src = new[0][b:b + 1, :, :cnt[b]]
        if rope:
            sb = sin[b:b + 1] if rope == "rows" else sin
            want = P.rotate(src, ck[:, :cnt[b]], sb[:, :cnt[b]])
            h, a = dh // 2, src.double().abs()
            mag = a * ck[:, :cnt[b]].double().abs()[:, None] + torch.cat([a[..., h:], a[..., :h]], -1) * sb[:, :cnt[b]].double().abs()[:, None]
            assert bool(((kb.double() - want).abs() <= u * want.abs() + 2.0 ** -22 * mag).all())
        else:
            assert torch.equal(kb, src)


def test_append_row_strides_that_are_not_aligned():
    """Rows that start anywhere: a slice of a wider projection, an odd offset."""
    gen = torch.Generator().manual_seed(11)
    wide = torch.randn(2, 3, 2, 67, generator=gen).to(BF)
    k, v, table, _ = P.make_cache([10, 10], 2, 64, 16, BF, gen, junk=0.0)
    dw = wide.cuda()
    dk, dv, dtab = cuda(k.clone(), v.clone(), table)
    dl = torch.tensor([0, 4], dtype=torch.int32).cuda()
    src = dw[..., 3:].transpose(1, 2)
    q = ops().turbo_paged_append(src, src, dk, dv, dtab, dl, q=src)
    assert torch.equal(q, src)
    for b, s in ((0, 0), (1, 4)):
        assert torch.equal(dk[table[b, 0].item(), :, s:s + 3], src[b]) and torch.equal(dv[table[b, 0].item(), :, s:s + 3], src[b])


# ------------------------------------------------------------------ evict
EVICT = [  # hkv, dh, page, lengths, budget, recent, sink
    (2, 64, 16, [40, 33, 32, 31, 0, 1], 32, 8, 4), (1, 64, 16, [1000], 999, 0, 0), (3, 32, 7, [200, 64, 70], 64, 64, 0),
    (1, 128, 48, [5000, 2], 100, 30, 70), (2, 8, 1, [9, 3], 1, 0, 0), (1, 40, 5, [300, 299], 128, 5, 1),
    (12, 64, 16, [2049, 2048, 500], 2048, 100, 4), (1, 16, 128, [70000], 1000, 100, 0), (1, 64, 16, [50], 60, 10, 0), (2, 32, 16, [48, 3], 70, 5, 64),
    (2, 64, 16, [20000, 16384], 16000, 0, 0), (2, 16, 16, [3999, 0], 300, 9, 9), (1, 8, 16, [7777, 8000], 500, 3, 0), (1, 16, 32, [16000, 9000], 700, 0, 2),
]


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("kind", ["distinct", "ties", "odd"])
@pytest.mark.parametrize("case", EVICT, ids=[f"{c[0]}x{c[1]}p{c[2]}n{max(c[3])}to{c[4]}" for c in EVICT])
def test_evict(case, kind, dt):
    hkv, dh, page, lens, budget, recent, sink = case
    B = len(lens)
    gen = torch.Generator().manual_seed(7 * budget + dh)
    k, v, table, ln = P.make_cache(lens, hkv, dh, page, dt, gen, spare=sum(-(-min(n, budget) // page) for n in lens) + 1, junk=3.0)
    free = [p for p in range(k.shape[0]) if p not in set(table.flatten().tolist())]
    to = torch.full((B, -(-budget // page) + 1), -1, dtype=torch.int32)
    used = 0
    for b, n in enumerate(lens):
        m = -(-min(n, budget) // page)
        to[b, :m] = torch.tensor(free[used:used + m], dtype=torch.int32)
        used += m
    mass = torch.rand(B, hkv, table.shape[1] * page + 2, generator=gen)
    if kind == "ties":
        mass = torch.floor(mass * 3) / 2
    if kind == "odd":  # NaN, infinities, both zeros, negative values
        pick = torch.randint(0, 9, mass.shape, generator=gen)
        for i, x in enumerate((float("nan"), math.inf, -math.inf, -0.0, 0.0, -1.0)):
            mass[pick == i] = x
        mass[pick == 8] = -float("nan")
    dk, dv, dtab, dto, dl, dm = cuda(k.clone(), v.clone(), table, to, ln, mass)
    mo, kept = ops().turbo_paged_evict(dk, dv, dtab, dto, dl, dm, budget, recent=recent, sink=sink)
    assert mo.shape == (B, hkv, to.shape[1] * page) and kept.shape == (B, hkv, budget)
    ck, cv, ckept, cmo = dk.cpu(), dv.cpu(), kept.cpu(), mo.cpu()
    wk, wv, wmo = k.clone(), v.clone(), torch.zeros_like(cmo)
    for b, n in enumerate(lens):
        for h in range(hkv):
            s = P.evict(mass[b, h], n, budget, recent, sink)
            assert ckept[b, h].tolist() == s + [-1] * (budget - len(s))
            src, dst = torch.tensor(s, dtype=torch.long), torch.arange(len(s))
            wmo[b, h, :len(s)] = mass[b, h][src]
            wk[to[b].long()[dst // page], h, dst % page] = k[table[b].long()[src // page], h, src % page]
            wv[to[b].long()[dst // page], h, dst % page] = v[table[b].long()[src // page], h, src % page]
    assert torch.equal(ck, wk) and torch.equal(cv, wv)
    assert torch.equal(torch.nan_to_num(cmo, nan=-5.0), torch.nan_to_num(wmo, nan=-5.0))
    assert torch.equal(torch.nan_to_num(dm.cpu(), nan=-5.0), torch.nan_to_num(mass, nan=-5.0))


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("kind,hkv,b,n,budget", [
    ("ties", 50, 6, 1000, 250), ("odd", 25, 6, 2000, 700), ("distinct", 50, 6, 4090, 100), ("ties", 50, 6, 4500, 300),
    ("odd", 10, 10, 9000, 900), ("distinct", 5, 6, 17000, 4000), ("ties", 5, 5, 33000, 3333)])
def test_evict_more_than_fits_the_gpu_at_once(kind, hkv, b, n, budget):
    test_evict((hkv, 16, 16, [n - 37 * i for i in range(b)], budget, 7, 3), kind, BF)


def test_shared_prefix_pages_side_stream_and_graph():
    """Two sequences over the same prompt pages; a decode step (append, attention) captured and
    replayed on a side stream with lengths that move between replays; then an eviction, which only
    reads the shared pages."""
    gen = torch.Generator().manual_seed(12)
    hkv, hq, dh, page = 2, 4, 64, 16
    k, v, table, _ = P.make_cache([64, 32, 32], hkv, dh, page, BF, gen, spare=0)
    tab = torch.stack([torch.cat([table[0, :4], table[1, :2]]), torch.cat([table[0, :4], table[2, :2]])]).to(torch.int32)
    pad = torch.zeros(4, hkv, page, dh, dtype=BF)
    k, v = torch.cat([k, pad]), torch.cat([v, pad])
    to = torch.tensor([[8, 9], [10, 11]], dtype=torch.int32)
    dk, dv, dt_, dto = cuda(k, v, tab, to)
    dl = torch.tensor([64, 64], dtype=torch.int32, device="cuda")
    n1 = dl + 1
    mass = torch.zeros(2, hkv, 6 * page, device="cuda")
    xk, xv, xq = (torch.zeros(2, h, 1, dh, dtype=BF, device="cuda") for h in (hkv, hkv, hq))
    stream = torch.cuda.Stream()
    steps = [[torch.randn(2, h, 1, dh, generator=gen).to(BF) for h in (hkv, hkv, hq)] for _ in range(10)]

    def step():
        q = ops().turbo_paged_append(xk, xv, dk, dv, dt_, dl, q=xq, mass=mass)
        return ops().turbo_paged_attention(q, dk, dv, dt_, n1, mass=mass)

    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
        mass.zero_()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step()
    ck, cv, cm = dk.cpu(), dv.cpu(), torch.zeros(2, hkv, 6 * page, dtype=torch.float64)
    with torch.cuda.stream(stream):
        for i, (a, b, c) in enumerate(steps):
            xk.copy_(a), xv.copy_(b), xq.copy_(c)
            graph.replay()
            got = out.clone()
            n = 65 + i
            for s in range(2):
                ck[tab[s, (n - 1) // page], :, (n - 1) % page] = a[s, :, 0]
                cv[tab[s, (n - 1) // page], :, (n - 1) % page] = b[s, :, 0]
            stream.synchronize()
            check_attention(got, c, ck, cv, tab, torch.tensor([n, n]), dh ** -0.5, BF)
            _, ps, _, _ = P.attention(c, ck, cv, tab, torch.tensor([n, n]), dh ** -0.5)
            for s in range(2):
                cm[s, :, :n] += ps[s].unflatten(0, (hkv, -1)).sum(1)
            dl += 1
            n1 += 1
        assert torch.equal(dk.cpu(), ck) and torch.equal(dv.cpu(), cv)
        assert torch.allclose(mass.cpu().double(), cm, rtol=1e-4, atol=1e-7)
        mo, kept = ops().turbo_paged_evict(dk, dv, dt_, dto, dl, mass, 24, recent=6, sink=2)
        short = dl.clamp(max=24)
        got = ops().turbo_paged_attention(xq, dk, dv, dto, short, mass=mo)
        stream.synchronize()
    assert torch.equal(dk[:8].cpu(), ck[:8])
    hk = mass.cpu()
    for s in range(2):
        for h in range(hkv):
            assert kept[s, h].tolist() == P.evict(hk[s, h], 74, 24, 6, 2)
    check_attention(got, steps[-1][2], dk.cpu(), dv.cpu(), to, torch.tensor([24, 24]), dh ** -0.5, BF)


def test_two_calls_on_two_streams():
    """Calls that run at the same time share nothing."""
    gen = torch.Generator().manual_seed(13)
    cases = []
    for n in (9000, 7000):
        k, v, table, ln = P.make_cache([n], 1, 64, 16, BF, gen)
        q = torch.randn(1, 2, 1, 64, generator=gen).to(BF)
        cases.append((cuda(q, k, v, table, ln), torch.cuda.Stream()))
    alone = [ops().turbo_paged_attention(*d) for d, _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (d, s) in enumerate(cases):
            with torch.cuda.stream(s):
                got[i].append(ops().turbo_paged_attention(*d))
    torch.cuda.synchronize()
    assert all(torch.equal(x, alone[i]) for i in range(2) for x in got[i])

"""Pages that are missing and lengths that do not fit, through every path of the operators over a cache in
4 or 8 bits: what is left is attended to or moved, and the record names the operator. Page numbers and
lengths are checked by the kernels before they are used."""
import pytest
import torch

import paged_util as P
import quant_range_util as R
import quant_util as Q

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
BAD_ARG, APPEND, READ, ATTEND, EVICT = 2, 44, 45, 46, 47
DENSE_APPEND, DENSE_ATTEND, DENSE_EVICT = 42, 41, 43


def ops():
    from one import turbo_ops
    return turbo_ops


@pytest.fixture(autouse=True)
def no_device_error():
    ops().ops_error(clear=True)
    yield
    assert ops().ops_error(clear=True) == (0, 0)


def recorded():
    return ops().ops_error(clear=True)


def cuda(ts):
    return tuple(t.cuda() for t in ts)


def bad_numbers(pages):
    return [-1, pages, 2 ** 31 - 1, -2 ** 31]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt,g", [(BF, 1), (BF, 7), (BF, 12), (F32, 3), (F32, 8)])
@pytest.mark.parametrize("dh,page", [(64, 16), (64, 5), (128, 32), (80, 16), (96, 48)])
@pytest.mark.parametrize("lengths", [[200, 40, 300], [5000, 3000, 70]], ids=["clusters", "list"])
def test_attention_over_what_pages_are_left(bits, dt, g, dh, page, lengths):
    """Sequence 0 lacks its first, a middle and its last page, sequence 1 all of them, sequence 2 none."""
    cache = list(Q.make_cache(lengths, 2, dh, page, bits, torch.Generator().manual_seed(dh + page + g)))
    wrong, used = bad_numbers(cache[0].shape[0]), -(-lengths[0] // page)
    cache[3] = cache[3].clone()
    for i, at in enumerate((0, used // 2, used // 2 + 1, used - 1)):
        cache[3][0, at] = wrong[i]
    cache[3][1] = torch.tensor(wrong, dtype=torch.int32).repeat(cache[3].shape[1])[:cache[3].shape[1]]
    q = torch.randn(3, 2 * g, 1, dh, generator=torch.Generator().manual_seed(5)).to(dt)
    ref, tol, w, wt = R.attention(q, cache, bits, dh ** -0.5)
    m0 = torch.rand(3, 2, cache[3].shape[1] * page, generator=torch.Generator().manual_seed(6))
    m = m0.cuda()
    for mass in (m, None):
        out = ops().turbo_paged_quant_attention(q.cuda(), *cuda(cache), mass=mass)
        assert recorded() == (BAD_ARG, ATTEND)
        R.check_out(out, ref, tol)
        assert bool((out[1] == 0).all())
    R.check_mass(m, m0, w, wt, g)
    assert torch.equal(m[1].cpu(), m0[1])


@pytest.mark.parametrize("lengths", [[80, 40], [5040, 3000]], ids=["clusters", "list"])  # whole pages of either size
@pytest.mark.parametrize("page", [16, 5])
def test_lengths_that_do_not_fit_are_recorded_by_name(lengths, page):
    T = ops()
    k, v, s, t, n = cuda(Q.make_cache(lengths, 2, 64, page, 4, torch.Generator().manual_seed(3)))
    q = torch.randn(2, 2, 1, 64, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    full = n.clone()
    full[0] = t.shape[1] * page
    want = T.turbo_paged_quant_attention(q, k, v, s, t, full)
    for wrong, site in ((t.shape[1] * page + 1, ATTEND), (-1, ATTEND)):
        n2 = n.clone()
        n2[0] = wrong
        out = T.turbo_paged_quant_attention(q, k, v, s, t, n2)
        assert recorded() == (BAD_ARG, site)
        assert torch.equal(out[0], want[0]) if wrong > 0 else bool((out[0] == 0).all())
        T.turbo_paged_quant_read(k, v, s, t.clamp(min=0), n2, 8, 64)
        assert recorded() == (BAD_ARG, READ)
    x = torch.zeros(2, 2, 1, 64, dtype=BF, device="cuda")
    T.turbo_paged_quant_append(x, x, k, v, s, t, torch.tensor([-1, t.shape[1] * page], dtype=torch.int32, device="cuda"))
    assert recorded() == (BAD_ARG, APPEND)
    odd = torch.zeros(x.numel() + 1, dtype=BF, device="cuda")[1:].view(x.shape)
    T.turbo_paged_quant_append(odd, odd, k, v, s, t, torch.tensor([-1, t.shape[1] * page], dtype=torch.int32, device="cuda"))
    assert recorded() == (BAD_ARG, APPEND)


def evict_case(lengths, hkv, dh, page, bits, budget, seed=0):
    gen = torch.Generator().manual_seed(seed)
    k, v, s, t, n = Q.make_cache(lengths, hkv, dh, page, bits, gen, spare=len(lengths) * -(-budget // page) + 2)
    free = sorted(set(range(k.shape[0])) - set(t[t >= 0].tolist()))
    to = torch.tensor(free[:len(lengths) * -(-budget // page)], dtype=torch.int32).view(len(lengths), -1)
    mass = torch.rand(len(lengths), hkv, t.shape[1] * page, generator=gen)
    return (k, v, s), t, n, to, mass


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("lengths,hkv,dh,page,budget", [([100, 60], 2, 64, 16, 40), ([100, 60], 1, 80, 5, 33),
                                                        ([900] * 80, 4, 48, 16, 300)], ids=["one launch", "odd pages", "two launches"])
def test_eviction_from_and_to_missing_pages(bits, lengths, hkv, dh, page, budget):
    """Survivors are chosen by their masses all the same; rows from or to a page that is not there stay."""
    T = ops()
    pools, t, n, to, mass = evict_case(lengths, hkv, dh, page, bits, budget)
    pages = pools[0].shape[0]
    for i, wrong in enumerate(bad_numbers(pages)):
        src, dst = t.clone(), to.clone()
        if i % 2:
            src[0, 1] = wrong
        else:
            dst[0, 1] = wrong
        dev = cuda(pools)
        got, kept = T.turbo_paged_quant_evict(*dev, src.cuda(), dst.cuda(), n.cuda(), mass.cuda(), budget, recent=5, sink=2)
        want, lost = [x.clone() for x in pools], False
        for b in range(len(lengths)):
            for h in range(hkv):
                keep = torch.tensor(P.evict(mass[b, h], lengths[b], budget, 5, 2))
                at = torch.arange(len(keep))
                assert torch.equal(kept[b, h, :len(keep)].cpu().long(), keep)
                assert torch.equal(got[b, h, :len(keep)].cpu(), mass[b, h, keep])
                ps, pd = src[b].long()[keep // page], dst[b].long()[at // page]
                ok = (ps >= 0) & (ps < pages) & (pd >= 0) & (pd < pages)
                lost |= not bool(ok.all())
                for x, y in zip(want, pools):
                    x[pd[ok], h, at[ok] % page] = y[ps[ok], h, keep[ok] % page]
        assert recorded() == ((BAD_ARG, EVICT) if lost else (0, 0))
        for a, b_ in zip(dev, want):
            assert torch.equal(a.cpu().view(torch.uint8), b_.view(torch.uint8))


@pytest.mark.parametrize("heads", [2, 320], ids=["one launch", "two launches"])
def test_lengths_of_an_eviction_are_recorded_by_name(heads):
    T = ops()
    pools, t, n, to, mass = evict_case([100, 60], heads, 32, 16, 4, 40)
    for wrong in (-3, t.shape[1] * 16 + 1):
        n2 = n.clone()
        n2[1] = wrong
        src = torch.where(t < 0, 0, t)  # a length cut to the table reads all of it
        T.turbo_paged_quant_evict(*cuda(pools), src.cuda(), to.cuda(), n2.cuda(), mass.cuda(), 40)
        assert recorded() == (BAD_ARG, EVICT)


def test_the_dense_operators_keep_their_names():
    T = ops()
    k, v = (torch.zeros(4, 2, 16, 64, dtype=BF, device="cuda") for _ in range(2))
    t, n = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), torch.tensor([40], dtype=torch.int32, device="cuda")
    q = torch.zeros(1, 2, 1, 64, dtype=BF, device="cuda")
    T.turbo_paged_attention(q, k, v, t, n)
    assert recorded() == (BAD_ARG, DENSE_ATTEND)
    T.turbo_paged_append(q, q, k, v, t, n)
    assert recorded() == (BAD_ARG, DENSE_APPEND)
    T.turbo_paged_evict(k, v, t, torch.tensor([[2, 3]], dtype=torch.int32, device="cuda"), n, torch.zeros(1, 2, 32, device="cuda"), 8)
    assert recorded() == (BAD_ARG, DENSE_EVICT)

"""What the serving operators refuse, on the CPU: in Python before any CUDA call, and at the C entry
points before any launch."""
import pytest
import torch

import paged_util as P
from one import _capi as C
from one import turbo_ops as T
from one.engine import OneEngine, pack_token_mask, process_logits  # noqa: F401


def cache(dt=torch.bfloat16, hkv=2, dh=64, page=16):
    gen = torch.Generator().manual_seed(0)
    return P.make_cache([40, 20], hkv, dh, page, dt, gen)


def test_cpu_tensors_have_no_path():
    k, v, t, n = cache()
    q = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        T.turbo_paged_attention(q, k, v, t, n)
    with pytest.raises(RuntimeError, match="no CPU path"):
        T.turbo_paged_append(q[:, :2], q[:, :2], k, v, t, n)
    with pytest.raises(RuntimeError, match="no CPU path"):
        T.turbo_paged_evict(k, v, t, t.clone(), n, torch.zeros(2, 2, 48), 32)
    with pytest.raises(C.OneError, match="CUDA"):
        process_logits(torch.zeros(2, 10))


def bad(fn, *a, **kw):
    with pytest.raises((ValueError, C.OneError)) as e:
        fn(*a, **kw)
    assert "no CPU path" not in str(e.value) and "CUDA" not in str(e.value)


def test_attention_refusals():
    k, v, t, n = cache()
    q = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16)
    f = T.turbo_paged_attention
    bad(f, q[:1], k, v, t, n)
    bad(f, q[:, :3], k, v, t, n)
    bad(f, q[..., :32], k, v, t, n)
    bad(f, q.expand(2, 4, 2, 64), k, v, t, n)
    bad(f, q.float(), k, v, t, n)
    bad(f, q.half(), k.half(), v.half(), t, n)
    bad(f, q, k, v[:1], t, n)
    bad(f, q, k, v.float(), t, n)
    bad(f, q, k.transpose(1, 2).contiguous().transpose(1, 2), v, t, n)
    bad(f, q, k, v, t.long(), n)
    bad(f, q, k, v, t, n.long())
    bad(f, q, k, v, t.t().contiguous().t(), n)
    bad(f, q, k, v, t, n[:1])
    bad(f, q, k, v, t, n, mass=torch.zeros(2, 2, 47))
    bad(f, q, k, v, t, n, mass=torch.zeros(2, 4, 48))
    bad(f, q, k, v, t, n, mass=torch.zeros(2, 2, 48, dtype=torch.float64))
    bad(f, q, k, v, t, n, mass=torch.zeros(2, 2, 96)[..., ::2])
    bad(f, q, k, v, t, n, out=torch.zeros(2, 4, 1, 64))


def test_append_refusals():
    k, v, t, n = cache()
    x = torch.zeros(2, 2, 3, 64, dtype=torch.bfloat16)
    cs = torch.zeros(1, 3, 64)
    f = T.turbo_paged_append
    bad(f, x[:, :1], x[:, :1], k, v, t, n)
    bad(f, x, x[:, :, :2], k, v, t, n)
    bad(f, x, x.float(), k, v, t, n)
    bad(f, x, x, k, v, t, n, q=x[:, :, :1])
    bad(f, x, x, k, v, t, n, q=x.float())
    bad(f, x, x, k, v, t, n, cos=cs)
    bad(f, x, x, k, v, t, n, cos=cs, sin=cs[:, :2])
    bad(f, x, x, k, v, t, n, cos=cs.expand(3, 3, 64), sin=cs.expand(3, 3, 64))
    bad(f, x, x, k, v, t, n, counts=torch.zeros(2))
    bad(f, x, x, k, v, t, n, counts=torch.zeros(3, dtype=torch.int32))


def test_evict_refusals():
    k, v, t, n = cache()
    to, m = t.clone(), torch.zeros(2, 2, 48)
    f = T.turbo_paged_evict
    for budget, recent, sink in ((0, 0, 0), (-1, 0, 0), (32, 33, 0), (32, 20, 13), (32, -1, 0), (32, 0, -1), (49, 0, 0)):
        bad(f, k, v, t, to, n, m, budget, recent=recent, sink=sink)
    bad(f, k, v, t, t, n, m, 32)
    bad(f, k, v, t, to.long(), n, m, 32)
    bad(f, k, v, t, to[:1], n, m, 32)
    bad(f, k, v, t, to, n, None, 32)
    bad(f, k, v, t, to, n, m[:, :1], 32)


def test_logits_refusals():
    x, h = torch.zeros(2, 40), torch.zeros(2, 5, dtype=torch.int64)
    f = process_logits
    bad(f, x[0])
    bad(f, x.half())
    bad(f, x, h[:1], repetition_penalty=1.5)
    bad(f, x, h.float(), repetition_penalty=1.5)
    bad(f, x, repetition_penalty=1.5)
    bad(f, x, presence_penalty=0.5)
    bad(f, x, frequency_penalty=torch.zeros(2))
    bad(f, x, h, repetition_penalty=0.0)
    bad(f, x, h, repetition_penalty=float("nan"))
    bad(f, x, h, repetition_penalty=torch.ones(3))
    bad(f, x, h, repetition_penalty=torch.ones(2, dtype=torch.float64))
    bad(f, x, h, output_starts=torch.zeros(2))
    bad(f, x, bias=torch.zeros(41))
    bad(f, x, bias=torch.zeros(3, 40))
    bad(f, x, bias=torch.zeros(40, dtype=torch.bfloat16))
    bad(f, x, token_mask=torch.zeros(1, dtype=torch.int32))
    bad(f, x, token_mask=torch.zeros(2, dtype=torch.int64))
    bad(f, x, out=torch.zeros(2, 40, dtype=torch.bfloat16))
    bad(f, x, out=torch.zeros(2, 41))


def test_token_mask_words():
    allowed = torch.zeros(2, 70, dtype=torch.bool)
    allowed[0, [0, 31, 32, 63, 69]] = True
    w = pack_token_mask(allowed)
    assert w.shape == (2, 3) and w.dtype == torch.int32
    got = (w[:, torch.arange(70) // 32] >> (torch.arange(70) % 32)) & 1
    assert torch.equal(got.bool(), allowed)
    assert torch.equal(pack_token_mask(allowed[0]), w[0])


def test_c_entry_points_refuse_before_launching():
    """Valid-looking addresses that no launch may reach: every call here is refused by its sizes."""
    a, b = 4096, 2048

    def attention(**kw):
        d = dict(q=a, qb=256, qh=64, k=a, v=a, ks=2048, vs=2048, pages=4, ps=16, table=b, ts=3, mp=3, ln=b, B=2, hq=4, hkv=2, dh=64,
                 scale=0.1, dt=0, mass=0, mw=0, out=a, ws=a, wb=1 << 30, st=0)
        d.update(kw)
        return C.LIB.one_paged_attention(*d.values())

    for kw in (dict(q=0), dict(k=0), dict(table=0), dict(ln=0), dict(out=0), dict(ws=0), dict(wb=0), dict(dt=2), dict(hq=3),
               dict(hq=0), dict(B=0), dict(ps=0), dict(pages=0), dict(mp=0), dict(ts=2), dict(ks=2047), dict(vs=100), dict(k=a + 2),
               dict(ks=2052), dict(mass=a, mw=47)):
        assert attention(**kw) == C.ONE_ERR_INVALID, kw
    for kw in (dict(dh=60), dict(dh=136, ks=1 << 20, vs=1 << 20), dict(B=70000), dict(hkv=70000, hq=70000, ks=1 << 30, vs=1 << 30),
               dict(ps=1 << 20, mp=1 << 12, ts=1 << 12, ks=1 << 30, vs=1 << 30)):
        assert attention(**kw) == C.ONE_ERR_UNSUPPORTED, kw

    def append(**kw):
        d = dict(k=a, k1=1, k2=1, k3=1, v=a, v1=1, v2=1, v3=1, q=a, q1=1, q2=1, q3=1, cos=a, sin=a, cb=1, cnt=0, kp=a, vp=a, ks=2048,
                 vs=2048, pages=4, ps=16, table=b, ts=3, mp=3, ln=b, B=2, n=1, hq=2, hkv=2, dh=64, dt=0, mass=0, mw=0, out=a, st=0)
        d.update(kw)
        return C.LIB.one_paged_append(*d.values())

    for kw in (dict(k=0), dict(v=0), dict(out=0), dict(q=0), dict(sin=0), dict(cb=3), dict(n=0), dict(hq=0), dict(kp=0),
               dict(mass=a, mw=1)):
        assert append(**kw) == C.ONE_ERR_INVALID, kw

    def evict(**kw):
        d = dict(kp=a, vp=a, ks=2048, vs=2048, pages=4, ps=16, table=b, ts=3, mp=3, dst=a, ds=2, dm=2, ln=b, mass=a, mw=48, B=2, hkv=2,
                 dh=64, dt=0, budget=32, recent=8, sink=4, mo=b, mow=32, kept=b, st=0)
        d.update(kw)
        return C.LIB.one_paged_evict(*d.values())

    for kw in (dict(budget=0), dict(recent=30), dict(sink=-1), dict(budget=33, mow=33), dict(mow=31), dict(mw=47), dict(ds=1),
               dict(kept=0), dict(mass=0), dict(mo=0), dict(dst=0)):
        assert evict(**kw) == C.ONE_ERR_INVALID, kw

    def logits(**kw):
        d = dict(x=a, ld=100, B=2, V=100, dt=0, h=a, hl=5, T=5, hb=8, st0=0, r=0, r1=1.0, p=0, p1=0.0, f=0, f1=0.0, bias=0, bl=0,
                 mask=0, ml=0, out=b, ol=100, best=0, st=0)
        d.update(kw)
        return C.LIB.one_process_logits(*d.values())

    for kw in (dict(x=0), dict(out=0), dict(h=0), dict(ld=99), dict(ol=99), dict(hl=4), dict(hb=2), dict(dt=5), dict(r1=0.0),
               dict(r1=float("nan")), dict(bias=a, bl=99), dict(mask=a, ml=3), dict(B=0), dict(V=0), dict(T=-1)):
        assert logits(**kw) == C.ONE_ERR_INVALID, kw

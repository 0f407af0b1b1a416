"""What the serving operators refuse, on the CPU: in Python before any CUDA call, and at the C entry
points before any launch."""
import ctypes

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
    bad(f, q, k, v, t, n, out=q)


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


class Cache(ctypes.Structure):
    """one_paged_cache of include/one_b200.h, field by field."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("kp", "vp")] + [(n, ctypes.c_int64) for n in ("ks", "vs")]
                + [("table", ctypes.c_void_p), ("ts", ctypes.c_int64), ("ln", ctypes.c_void_p), ("mass", ctypes.c_void_p),
                   ("mw", ctypes.c_int64)] + [(n, ctypes.c_int32) for n in ("pages", "ps", "mp", "B", "hkv", "dh", "dt", "reserved")])


class Tokens(ctypes.Structure):
    """one_paged_tokens."""
    _fields_ = ([(n, ctypes.c_void_p) for n in "kvq"] + [(n, ctypes.c_int64 * 3) for n in ("k_s", "v_s", "q_s")]
                + [(n, ctypes.c_void_p) for n in ("cos", "sin", "counts", "out")]
                + [(n, ctypes.c_int32) for n in ("n", "hq", "cb", "reserved")])


class Rules(ctypes.Structure):
    """one_logits_rules."""
    _fields_ = ([("h", ctypes.c_void_p), ("hl", ctypes.c_int64)] + [(n, ctypes.c_void_p) for n in ("starts", "r", "p", "f", "bias")]
                + [("bl", ctypes.c_int64), ("mask", ctypes.c_void_p), ("ml", ctypes.c_int64)]
                + [(n, ctypes.c_int32) for n in ("T", "hb")] + [(n, ctypes.c_float) for n in ("r1", "p1", "f1")]
                + [("reserved", ctypes.c_int32)])


A, B_ = 4096, 2048  # valid-looking addresses that no launch may reach: every call below is refused
CACHE = dict(kp=A, vp=A, ks=2048, vs=2048, table=B_, ts=3, ln=B_, mass=0, mw=0, pages=4, ps=16, mp=3, B=2, hkv=2, dh=64, dt=0)


def packs(struct, packed, values):
    """The packed form that the package hands to the library equals the structure's."""
    x = struct(**values)
    assert bytes(x) == packed and ctypes.sizeof(struct) == len(packed)


def test_packed_structures_match_the_header():
    v = dict(zip([n for n, _ in Cache._fields_ if n != "reserved"], range(1, 17)))
    packs(Cache, C.PAGED_CACHE(*v.values()), v)
    n = [x for x, _ in Tokens._fields_ if x != "reserved"]
    flat = list(range(1, 4)) + list(range(10, 19)) + list(range(20, 27))
    v = dict(zip(n[:3], flat[:3]), k_s=(ctypes.c_int64 * 3)(10, 11, 12), v_s=(ctypes.c_int64 * 3)(13, 14, 15),
             q_s=(ctypes.c_int64 * 3)(16, 17, 18), **dict(zip(n[6:], flat[12:])))
    packs(Tokens, C.PAGED_TOKENS(*flat), v)
    v = dict(zip([x for x, _ in Rules._fields_ if x != "reserved"], range(1, 16)))
    packs(Rules, C.LOGITS_RULES(*v.values()), v)


def refused(call, base, invalid, unsupported=()):
    for kw in invalid:
        assert call(**{**base, **kw}) == C.ONE_ERR_INVALID, kw
    for kw in unsupported:
        assert call(**{**base, **kw}) == C.ONE_ERR_UNSUPPORTED, kw


def cache_of(d):
    return ctypes.byref(Cache(**{k: d[k] for k in CACHE}))


BAD_CACHE = [dict(kp=0), dict(vp=0), dict(table=0), dict(ln=0), dict(dt=2), dict(B=0), dict(ps=0), dict(pages=0), dict(mp=0),
             dict(ts=2), dict(ks=2047), dict(vs=100), dict(kp=A + 2), dict(ks=2052), dict(mass=A, mw=47)]
BIG_CACHE = [dict(dh=60), dict(dh=136, ks=1 << 20, vs=1 << 20), dict(B=70000), dict(hkv=70000, hq=70000, ks=1 << 30, vs=1 << 30),
             dict(ps=1 << 20, mp=1 << 12, ts=1 << 12, ks=1 << 30, vs=1 << 30), dict(ks=1 << 31), dict(vs=1 << 33)]


def test_c_attention_refuses_before_launching():
    def call(q, qb, qh, hq, out, ws, wb, **cache):
        return C.LIB.one_paged_attention(cache_of(cache), q, qb, qh, hq, 0.1, out, ws, wb, 0)
    base = dict(CACHE, mp=4096, ts=4096, q=A, qb=256, qh=64, hq=4, out=A, ws=A, wb=1 << 30)
    refused(call, base, [k for k in BAD_CACHE if k != dict(ts=2)] + [dict(ts=4095), dict(q=0), dict(out=0), dict(ws=0), dict(wb=64),
                                                                    dict(hq=3), dict(hq=0)], BIG_CACHE)
    assert C.LIB.one_paged_attention(None, A, 1, 1, 4, 0.1, A, A, 1 << 30, 0) == C.ONE_ERR_INVALID
    # small caches need no workspace, others do
    assert C.LIB.one_paged_attention_workspace_bytes(2, 4, 2, 64, 16, 3, 0, 0) == 0
    assert C.LIB.one_paged_attention_workspace_bytes(2, 4, 2, 64, 16, 3, 0, 1) > 0
    assert C.LIB.one_paged_attention_workspace_bytes(2, 4, 2, 64, 16, 4096, 0, 0) > 0


def test_c_append_refuses_before_launching():
    three = (ctypes.c_int64 * 3)(64, 64, 64)

    def call(k, v, q, cos, sin, out, n, hq, cb, **cache):
        t = Tokens(k=k, v=v, q=q, k_s=three, v_s=three, q_s=three, cos=cos, sin=sin, counts=0, out=out, n=n, hq=hq, cb=cb)
        return C.LIB.one_paged_append(cache_of(cache), ctypes.byref(t), 0)
    base = dict(CACHE, k=A, v=A, q=A, cos=A, sin=A, out=A, n=1, hq=2, cb=1)
    refused(call, base, BAD_CACHE + [dict(k=0), dict(v=0), dict(out=0), dict(q=0), dict(sin=0), dict(cos=0), dict(cb=3), dict(n=0),
                                     dict(hq=0)], [x for x in BIG_CACHE if "hq" not in x] + [dict(n=1 << 30)])
    assert C.LIB.one_paged_append(cache_of(CACHE), None, 0) == C.ONE_ERR_INVALID


def test_c_evict_refuses_before_launching():
    def call(dst, ds, dm, budget, recent, sink, mo, mow, kept, **cache):
        return C.LIB.one_paged_evict(cache_of(cache), dst, ds, dm, budget, recent, sink, mo, mow, kept, 0)
    base = dict(CACHE, mass=A, mw=48, dst=A, ds=2, dm=2, budget=32, recent=8, sink=4, mo=B_, mow=32, kept=B_)
    refused(call, base, [k for k in BAD_CACHE if "mass" not in k] + [
        dict(budget=0), dict(recent=30), dict(sink=-1), dict(recent=-1), dict(budget=33, mow=33), dict(mow=31), dict(mw=47), dict(ds=1),
        dict(dm=0), dict(kept=0), dict(mass=0), dict(mo=0), dict(dst=0)], [dict(dh=60), dict(B=70000), dict(mow=1 << 31)])


def test_c_logits_refuse_before_launching():
    def call(x, ld, B, V, dt, out, ol, **rules):
        return C.LIB.one_process_logits(ctypes.byref(Rules(**rules)), x, ld, B, V, dt, out, ol, 0, 0)
    base = dict(x=A, ld=100, B=2, V=100, dt=0, out=B_, ol=100, h=A, hl=5, T=5, hb=8, starts=0, r=0, r1=1.0, p=0, p1=0.0, f=0, f1=0.0,
                bias=0, bl=0, mask=0, ml=0)
    refused(call, base, [dict(x=0), dict(out=0), dict(h=0), dict(ld=99), dict(ol=99), dict(hl=4), dict(hb=2), dict(dt=5), dict(r1=0.0),
                         dict(r1=float("nan")), dict(bias=A, bl=99), dict(mask=A, ml=3), dict(B=0), dict(V=0), dict(T=-1)],
            [dict(V=1 << 30, ld=1 << 30, ol=1 << 30)])
    assert C.LIB.one_process_logits(None, A, 100, 2, 100, 0, B_, 100, 0, 0) == C.ONE_ERR_INVALID

"""What the operators over a cache in 4 or 8 bits refuse, on the CPU: in Python before any CUDA call, and
at the C entry points before any launch."""
import ctypes

import pytest
import torch

import quant_util as Q
from one import _capi as C
from one import turbo_ops as T

BF, F32 = torch.bfloat16, torch.float32


def cache(hkv=2, dh=64, page=16, bits=4):
    return Q.make_cache([40, 20], hkv, dh, page, bits, torch.Generator().manual_seed(0))


def bad(fn, *a, **kw):
    with pytest.raises((ValueError, C.OneError)) as e:
        fn(*a, **kw)
    assert "no CPU path" not in str(e.value) and "CUDA" not in str(e.value)


@pytest.mark.parametrize("bits", [4, 8])
def test_cpu_tensors_have_no_path(bits):
    c = cache(bits=bits)
    q = torch.zeros(2, 4, 1, 64, dtype=BF)
    for call in (lambda: T.turbo_paged_quant_attention(q, *c), lambda: T.turbo_paged_quant_append(q[:, :2], q[:, :2], *c),
                 lambda: T.turbo_paged_quant_read(*c, 8, 64),
                 lambda: T.turbo_paged_quant_evict(*c[:4], c[3].clone(), c[4], torch.zeros(2, 2, 48), 32)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_pools():
    k, v, s = T.turbo_paged_quant_pools(3, 2, 8, 80, 4, device="cpu")
    assert k.shape == v.shape == (3, 2, 8, 40) and s.shape == (3, 2, 8, 2, 3) and k.dtype == torch.uint8 and s.dtype == BF
    assert T.turbo_paged_quant_pools(3, 2, 8, 80, 8, device="cpu")[0].shape == (3, 2, 8, 80)
    for dh, bits in ((64, 5), (0, 4), (8, 4), (72, 4), (144, 8)):
        bad(T.turbo_paged_quant_pools, 3, 2, 8, dh, bits, device="cpu")


def test_cache_refusals():
    k, v, s, t, n = cache()
    q = torch.zeros(2, 4, 1, 64, dtype=BF)
    f = T.turbo_paged_quant_attention
    bad(f, q[..., :32], k, v, s, t, n)              # rows of another head_dim
    bad(f, q.half(), k, v, s, t, n)
    bad(f, q, k, v[:1], s, t, n)
    bad(f, q, k.view(torch.int8), v, s, t, n)
    bad(f, q, k, v, s.float(), t, n)
    bad(f, q, k, v, s[..., :1], t, n)
    bad(f, q, k, v, s[:, :, :, 0], t, n)
    bad(f, q, k, v, s[:1], t, n)
    bad(f, q, k, v, s.transpose(1, 2).contiguous().transpose(1, 2), t, n)
    bad(f, q, k.transpose(1, 2).contiguous().transpose(1, 2), v, s, t, n)
    bad(f, q, k, v, s, t.long(), n)
    bad(f, q, k, v, s, t, n.long())
    bad(f, q, k, v, s, t, n[:1])
    bad(f, q[:1], k, v, s, t, n)
    bad(f, q[:, :3], k, v, s, t, n)
    bad(f, q.expand(2, 4, 2, 64), k, v, s, t, n)
    bad(f, q, k, v, s, t, n, mass=torch.zeros(2, 2, 47))
    bad(f, q, k, v, s, t, n, out=q)
    bad(f, q, k, v, s, t, n, out=torch.zeros(2, 4, 1, 64))


def test_append_and_read_refusals():
    c = cache()
    x = torch.zeros(2, 2, 3, 64, dtype=BF)
    cs = torch.zeros(1, 3, 64)
    f = T.turbo_paged_quant_append
    bad(f, x[:, :1], x[:, :1], *c)
    bad(f, x, x[:, :, :2], *c)
    bad(f, x, x.float(), *c)
    bad(f, x.half(), x.half(), *c)
    bad(f, x, x, *c, q=x[:, :, :1])
    bad(f, x, x, *c, q=x.float())
    bad(f, x, x, *c, cos=cs)
    bad(f, x, x, *c, cos=cs, sin=cs[:, :2])
    bad(f, x, x, *c, counts=torch.zeros(2))
    bad(f, x, x, *c, mass=torch.zeros(2, 3, 48))
    f = T.turbo_paged_quant_read
    bad(f, *c, -1, 64)
    bad(f, *c, 8, 32)
    bad(f, *c, 8, 64, dtype=torch.float16)
    bad(f, *c, 8, 64, starts=torch.zeros(2))
    bad(f, *c, 8, 64, starts=torch.zeros(3, dtype=torch.int32))


def test_evict_refusals():
    k, v, s, t, n = cache()
    to, m = t.clone(), torch.zeros(2, 2, 48)
    f = T.turbo_paged_quant_evict
    for budget, recent, sink in ((0, 0, 0), (32, 33, 0), (32, 20, 13), (32, -1, 0), (32, 0, -1), (49, 0, 0)):
        bad(f, k, v, s, t, to, n, m, budget, recent=recent, sink=sink)
    bad(f, k, v, s, t, t, n, m, 32)
    bad(f, k, v, s, t, to.long(), n, m, 32)
    bad(f, k, v, s, t, to, n, None, 32)
    bad(f, k, v, s, t, to, n, m[:, :1], 32)


FIELDS = "k v s ks vs ss table ts lengths mass mw n ps mp b hkv dh bits".split()
GOOD = dict(k=4096, v=8192, s=16384, ks=1024, vs=1024, ss=128, table=64, ts=4, lengths=128, mass=0, mw=0, n=5, ps=16, mp=4, b=2,
            hkv=2, dh=64, bits=4)


def pack(**over):
    return C.PAGED_QUANT_CACHE(*(dict(GOOD, **over)[f] for f in FIELDS))


BAD = [dict(k=0), dict(s=0), dict(table=0), dict(lengths=0), dict(k=4100), dict(v=8193), dict(s=16386), dict(ks=1023), dict(ks=1028),
       dict(ss=127), dict(ss=126), dict(ss=131), dict(ts=3), dict(n=0), dict(ps=0), dict(mp=0), dict(b=0), dict(hkv=0), dict(dh=8),
       dict(dh=40), dict(dh=144, ks=1 << 20, vs=1 << 20), dict(bits=5), dict(b=65536), dict(ks=1 << 31), dict(mass=64, mw=63),
       dict(ps=1 << 30, ks=1 << 20)]


@pytest.mark.parametrize("over", BAD, ids=lambda o: "-".join(f"{k}={v}" for k, v in o.items()))
def test_c_entry_points_check_the_cache(over):
    cache_ = pack(**over)
    assert C.LIB.one_paged_quant_attention(cache_, 64, 256, 64, 4, 1.0, 0, 64, None, 0, None) in (C.ONE_ERR_INVALID, C.ONE_ERR_UNSUPPORTED)
    assert C.LIB.one_paged_quant_read(cache_, None, 4, 0, 64, 64, None) in (C.ONE_ERR_INVALID, C.ONE_ERR_UNSUPPORTED)
    tokens = C.PAGED_TOKENS(64, 64, 0, *[0] * 9, 0, 0, 0, 0, 1, 0, 1)
    assert C.LIB.one_paged_quant_append(cache_, tokens, 0, None) in (C.ONE_ERR_INVALID, C.ONE_ERR_UNSUPPORTED)
    if "mass" not in over:
        cache_ = pack(**dict(over, mass=64, mw=over.get("mp", 4) * max(over.get("ps", 16), 16)))
    assert C.LIB.one_paged_quant_evict(cache_, 64, 4, 4, 8, 0, 0, 64, 64, 64, None) in (C.ONE_ERR_INVALID, C.ONE_ERR_UNSUPPORTED)


def test_c_entry_points_check_the_rest():
    bad_rc = (C.ONE_ERR_INVALID, C.ONE_ERR_UNSUPPORTED)
    L, c = C.LIB, pack()
    tokens = lambda **o: C.PAGED_TOKENS(*(dict(dict(k=64, v=64, q=0), **o)[f] for f in "kvq"), *[0] * 9, o.get("cos", 0),
                                        o.get("sin", 0), 0, o.get("q_out", 0), o.get("n", 1), o.get("hq", 0), o.get("cb", 1))
    for o in (dict(k=0), dict(v=0), dict(q=64), dict(q_out=64), dict(q=64, q_out=64, hq=0), dict(cos=64), dict(n=0),
              dict(cos=64, sin=64, cb=3)):
        assert L.one_paged_quant_append(c, tokens(**o), 0, None) in bad_rc
    assert L.one_paged_quant_append(c, tokens(), 2, None) in bad_rc
    assert L.one_paged_quant_append(None, tokens(), 0, None) in bad_rc
    assert L.one_paged_quant_append(c, None, 0, None) in bad_rc
    for args in ((c, None, 0, 0, 64, 64), (c, None, 4, 2, 64, 64), (c, None, 4, 0, 0, 64), (c, None, 4, 0, 64, 72), (None, None, 4, 0, 64, 64)):
        assert L.one_paged_quant_read(*args, None) in bad_rc
    for hq, dt, q, out in ((3, 0, 64, 64), (0, 0, 64, 64), (4, 2, 64, 64), (4, 0, 0, 64), (4, 0, 64, 0)):
        assert L.one_paged_quant_attention(c, q, 256, 64, hq, 1.0, dt, out, None, 0, None) in bad_rc
    massed = pack(mass=64, mw=64)
    need = L.one_paged_quant_attention_workspace_bytes(2, 4, 2, 64, 16, 4, 0, 1)
    assert need > 0
    assert L.one_paged_quant_attention(massed, 64, 256, 64, 4, 1.0, 0, 64, 256, need - 1, None) == C.ONE_ERR_INVALID
    assert L.one_paged_quant_attention(massed, 64, 256, 64, 4, 1.0, 0, 64, None, need, None) == C.ONE_ERR_INVALID
    assert L.one_paged_quant_evict(c, 64, 4, 4, 8, 0, 0, 64, 64, 64, None) in bad_rc  # no masses
    assert L.one_paged_quant_attention_workspace_bytes(0, 4, 2, 64, 16, 4, 0, 1) == 0


def test_lists_past_31_bits_are_refused():
    """A list counts tiles of 32 slots, for every head of every sequence."""
    f = C.LIB.one_paged_quant_attention
    for dh in (32, 64, 128):
        c = pack(b=4096, hkv=64, dh=dh, ps=16, mp=1 << 14, ts=1 << 14, ks=1 << 20, vs=1 << 20, ss=1 << 20)
        assert f(c, 64, 4096, 64, 64, 1.0, 0, 64, None, 0, None) == C.ONE_ERR_UNSUPPORTED


def test_quantising_on_the_cpu():
    """The tests' own formulas: values come back within half a step, ties go to the even code."""
    x = torch.randn(50, 80, generator=torch.Generator().manual_seed(3)) * 3
    for bits in (4, 8):
        codes, scales = Q.close(x, bits)
        y = Q.open_(codes, scales, bits, 80)
        step = scales.double().repeat_interleave(32, -1)[:, :80]
        # half a step, and what a scale below max / m leaves of the largest value: m * 2^-9 steps
        assert bool(((y - x.double()).abs() <= step * (0.5 + Q.top(bits) * 2.0 ** -9)).all())
    t = torch.tensor([[7.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 6.5] + [0.0] * 24])
    codes, scales = Q.close(t, 4)
    assert Q.open_(codes, scales, 4, 32)[0, :8].tolist() == [7, 0, 2, 2, 0, -2, -2, 6] and float(scales) == 1.0

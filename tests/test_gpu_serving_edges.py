"""GPU tests of the serving operators at their edges: rotation tables of another type, empty batches,
rows shared by a batch, weights below the normal range, tables wider than their sequences, captured
first calls, and that every slot of a cache counts exactly once."""
import math
import os
import subprocess
import sys

import pytest
import torch

import paged_util as P
from conftest import PKG, REPO, cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]

BF, F32 = torch.bfloat16, torch.float32


def ops():
    from one import turbo_ops
    return turbo_ops


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    assert ops().ops_error() == (0, 0)


def test_generate_takes_the_repetition_penalty_of_a_generation_config():
    from transformers import GenerationConfig
    from one.configuration_one import tiny_config
    from one.initialization import init_state_dict
    from one.modeling_one import OneForCausalLM
    cfg = tiny_config()
    model = OneForCausalLM(cfg)
    model.load_state_dict(init_state_dict(cfg, 0, torch.float32), strict=False)
    model = model.to(torch.bfloat16).cuda()
    ids = torch.randint(1, cfg.vocab_size, (3, 10), generator=torch.Generator().manual_seed(23)).cuda()
    plain = model.generate(ids, max_new_tokens=16)
    want = model.generate(ids, max_new_tokens=16, repetition_penalty=0.05)
    assert not torch.equal(plain, want)
    config = GenerationConfig(repetition_penalty=0.05)
    assert torch.equal(model.generate(ids, generation_config=config, max_new_tokens=16), want)
    assert torch.equal(model.generate(ids, generation_config=config, max_new_tokens=16, repetition_penalty=1.0), plain)
    drawn = model.generate(ids, max_new_tokens=16, do_sample=True, repetition_penalty=0.05, seed=3)
    assert torch.equal(model.generate(ids, generation_config=config, max_new_tokens=16, do_sample=True, seed=3), drawn)
    with pytest.raises(ValueError, match="repetition_penalty"):
        model.generate(ids, max_new_tokens=2, repetition_penalty=0.0)
    model.generation_config = config
    assert torch.equal(model.generate(ids, max_new_tokens=16), want)


# ------------------------------------------------------------------ rotation tables
@pytest.mark.parametrize("tables", [F32, torch.float64, torch.float16, BF], ids=["fp32", "fp64", "fp16", "bf16"])
@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("dh,n,shared", [(64, 40, False), (80, 7, True), (40, 5, False), (128, 1, True), (8, 3, False)])
def test_append_rotates_by_tables_of_any_type_in_fp32(dh, n, shared, dt, tables):
    """Two products of fp32 factors and their sum, one rounding: 2^-22 of the products' magnitudes
    (three roundings, and one of the tables for fp64), half a step of the result."""
    gen = torch.Generator().manual_seed(dh + n)
    hkv, hq, page, start = 2, 3, 16, [5, 0]
    k, v, table, _ = P.make_cache([s + n for s in start], hkv, dh, page, dt, gen, junk=0.0)
    new = [torch.randn(2, h, n, dh, generator=gen).to(dt) for h in (hkv, hkv, hq)]
    ang = 6.28 * torch.rand(1 if shared else 2, n, dh, generator=gen, dtype=torch.float64)
    cos, sin = ang.cos().to(tables), ang.sin().to(tables)
    dk, dv, dtab, dl = k.cuda(), v.cuda(), table.cuda(), torch.tensor(start, dtype=torch.int32).cuda()
    got = ops().turbo_paged_append(new[0].cuda(), new[1].cuda(), dk, dv, dtab, dl, cos=cos.cuda(), sin=sin.cuda(), q=new[2].cuda())
    u, h = torch.finfo(dt).eps / 2, dh // 2

    def check(x, src):
        want, a = P.rotate(src, cos, sin), src.double().abs()
        mag = a * cos.double().abs()[:, None] + torch.cat([a[..., h:], a[..., :h]], -1) * sin.double().abs()[:, None]
        err = (x.cpu().double() - want).abs() - u * want.abs() - 2.0 ** -22 * mag
        assert bool((err <= 0).all()), float(err.max())

    check(got, new[2])
    check(torch.stack([P.rows(dk.cpu(), table, b, s + n)[:, s:] for b, s in enumerate(start)]), new[0])


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "fp32"])
def test_logits_and_history_shared_by_the_rows(dt):
    from one.engine import process_logits
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(1, 777, generator=gen).to(dt)
    hist = torch.randint(0, 777, (1, 30), generator=gen)
    rep = torch.tensor([1.5, 1.0, 2.0, 0.5])
    dx, dh, dr = x.cuda(), hist.cuda(), rep.cuda()
    want = process_logits(dx.repeat(4, 1), dh.repeat(4, 1), repetition_penalty=dr)
    assert torch.equal(process_logits(dx.expand(4, -1), dh.expand(4, -1), repetition_penalty=dr), want)
    assert torch.equal(process_logits(dx.repeat(4, 1), dh.expand(4, -1), repetition_penalty=dr), want)
    one = torch.tensor([[5]], device="cuda")
    want = process_logits(dx.repeat(4, 1), one.repeat(4, 1), repetition_penalty=dr)
    assert torch.equal(process_logits(dx.expand(4, -1), one.expand(4, -1), repetition_penalty=dr), want)


# ------------------------------------------------------------------ empty, shared rows
@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "fp32"])
def test_empty_batches_and_no_new_tokens(dt):
    from one.engine import process_logits
    gen = torch.Generator().manual_seed(1)
    k, v, table, ln = (x.cuda() for x in P.make_cache([20, 3], 2, 64, 16, dt, gen, junk=0.0))
    before, mass = k.clone(), torch.rand(2, 2, 32, device="cuda")
    m0 = mass.clone()
    q = torch.randn(2, 4, 0, 64, device="cuda").to(dt)
    got = ops().turbo_paged_append(q[:, :2], q[:, :2], k, v, table, ln, q=q, mass=mass)
    assert got.shape == (2, 4, 0, 64) and got.dtype == dt
    assert ops().turbo_paged_append(q[:, :2], q[:, :2], k, v, table, ln) is None
    cos = torch.zeros(1, 0, 64, device="cuda")
    assert ops().turbo_paged_append(q[:, :2], q[:, :2], k, v, table, ln, cos=cos, sin=cos, q=q).shape == q.shape
    none, zero = table[:0], ln[:0]
    one = torch.randn(0, 4, 1, 64, device="cuda").to(dt)
    assert ops().turbo_paged_append(one[:, :2], one[:, :2], k, v, none, zero, q=one).shape == one.shape
    assert ops().turbo_paged_attention(one, k, v, none, zero, mass=mass[:0]).shape == one.shape
    out = torch.empty_like(one)
    assert ops().turbo_paged_attention(one, k, v, none, zero, out=out) is out
    mo, kept = ops().turbo_paged_evict(k, v, none, none, zero, mass[:0], 32)
    assert mo.shape == (0, 2, 32) and kept.shape == (0, 2, 32) and kept.dtype == torch.int32
    x = torch.zeros(0, 100, device="cuda").to(dt)
    s, best = process_logits(x, torch.zeros(0, 5, dtype=torch.int64, device="cuda"), repetition_penalty=1.5, return_argmax=True)
    assert s.shape == (0, 100) and s.dtype == F32 and best.shape == (0,) and best.dtype == torch.int32
    assert process_logits(x).shape == (0, 100)
    assert torch.equal(k, before) and torch.equal(mass, m0)


# ------------------------------------------------------------------ weights
@pytest.mark.parametrize("hkv,g,n", [(1, 1, 40), (1, 4, 300), (2, 3, 9000), (40, 1, 2000)])
def test_fp32_weights_below_the_normal_range(hkv, g, n):
    """A slot 2^130 times lighter than the heaviest adds 2^-130 (a denormal) to its mass."""
    k = torch.zeros(1, hkv, n, 64)
    k[..., 0] = -130.0
    k[:, :, 3, 0] = 0.0
    page = 16
    pages = -(-n // page)
    pool = torch.zeros(pages, hkv, page, 64)
    kp = torch.nn.functional.pad(k, (0, 0, 0, pages * page - n)).view(hkv, pages, page, 64).transpose(0, 1).contiguous().cuda()
    q = torch.zeros(1, hkv * g, 1, 64)
    q[..., 0] = 1.0
    mass = torch.zeros(1, hkv, pages * page, device="cuda")
    table = torch.arange(pages, dtype=torch.int32, device="cuda").view(1, -1)
    ops().turbo_paged_attention(q.cuda(), kp, pool.cuda(), table, torch.tensor([n], dtype=torch.int32, device="cuda"),
                                scale_factor=math.log(2.0), mass=mass)
    got = mass.cpu().double()[0, :, :n]
    want = torch.full((hkv, n), g * 2.0 ** -130, dtype=torch.float64)
    want[:, 3] = g
    # one step of the denormals; an exponent of 130 is off by 130 * 2^-23 at most, the weight by 2^-16 of itself
    assert bool(((got - want).abs() <= g * 2.0 ** -149 + 2.0 ** -15 * want).all())


WIDE = [([200], 1, 1, 64, 16), ([0, 700, 33], 4, 3, 64, 16), ([1500, 2, 90, 0], 2, 8, 128, 48), ([5], 1, 20, 32, 7)]


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("with_mass", [False, True], ids=["plain", "mass"])
@pytest.mark.parametrize("lens,hkv,g,dh,page", WIDE)
def test_attention_in_a_table_for_32768_slots(lens, hkv, g, dh, page, with_mass, dt):
    from test_gpu_paged import check_attention, cuda
    gen = torch.Generator().manual_seed(9)
    k, v, table, ln = P.make_cache(lens, hkv, dh, page, dt, gen, width=32768 // page)
    q = torch.randn(len(lens), hkv * g, 1, dh, generator=gen).to(dt)
    mass0 = torch.rand(len(lens), hkv, table.shape[1] * page, generator=gen) if with_mass else None
    dq, dk, dv, dtab, dl, dm = cuda(q, k, v, table, ln, mass0)
    got = ops().turbo_paged_attention(dq, dk, dv, dtab, dl, mass=dm)
    check_attention(got, q, k, v, table, ln, dh ** -0.5, dt, dm, mass0)
    if with_mass:
        for b, n in enumerate(lens):
            assert torch.equal(dm[b, :, n:].cpu(), mass0[b, :, n:])


@pytest.mark.parametrize("width", [4096, 32768, 40000], ids=str)
@pytest.mark.parametrize("b,hkv", [(2, 3), (20, 40)])
def test_evict_and_append_in_a_wide_table(b, hkv, width):
    gen = torch.Generator().manual_seed(b)
    page, dh, budget, recent, sink = 16, 16, 100, 20, 4
    lens = [(130 + 37 * i) % 300 for i in range(b)]
    k, v, table, ln = P.make_cache([n + 1 for n in lens], hkv, dh, page, BF, gen, width=width // page, spare=b * 7, junk=3.0)
    free = [p for p in range(k.shape[0]) if p not in set(table.flatten().tolist())]
    to = torch.full((b, width // page), -1, dtype=torch.int32)
    for i in range(b):
        to[i, :7] = torch.tensor(free[7 * i:7 * i + 7], dtype=torch.int32)
    mass = torch.rand(b, hkv, width, generator=gen)
    dk, dv, dtab, dto, dm = (x.cuda() for x in (k, v, table, to, mass))
    dl = torch.tensor(lens, dtype=torch.int32).cuda()
    new = torch.randn(b, hkv, 1, dh, generator=gen).to(BF)
    ops().turbo_paged_append(new.cuda(), new.cuda(), dk, dv, dtab, dl, mass=dm)
    for i, n in enumerate(lens):
        assert torch.equal(dk[int(table[i, n // page]), :, n % page].cpu(), new[i, :, 0])
        mass[i, :, n] = 0
    assert torch.equal(dm.cpu(), mass)
    mo, kept = ops().turbo_paged_evict(dk, dv, dtab, dto, dl + 1, dm, budget, recent=recent, sink=sink)
    ck, src = dk.cpu(), kept.cpu()
    assert mo.shape == (b, hkv, width) and float(mo[..., budget:].abs().max()) == 0.0
    for i, n in enumerate(lens):
        for h in range(hkv):
            s = P.evict(mass[i, h], n + 1, budget, recent, sink)
            assert src[i, h].tolist() == s + [-1] * (budget - len(s))
            s, d = torch.tensor(s), torch.arange(len(s))
            assert torch.equal(ck[to[i].long()[d // page], h, d % page], ck[table[i].long()[s // page], h, s % page])
            assert torch.equal(mo[i, h, :len(s)].cpu(), mass[i, h][s])


FIRST = """
import sys
sys.path[:0] = sys.argv[1:3]
import torch
import paged_util as P
from one import turbo_ops as T
from one.engine import process_logits
gen = torch.Generator().manual_seed(0)
k, v, t, n = (x.cuda() for x in P.make_cache([900, 40], 2, 64, 16, torch.bfloat16, gen, spare=80, junk=0.0))
free = [p for p in range(k.shape[0]) if p not in set(t.flatten().tolist())]
to = torch.tensor(free[:16], dtype=torch.int32).view(2, 8).cuda()
q = torch.randn(2, 4, 1, 64, generator=gen).bfloat16().cuda()
mass = torch.rand(2, 2, t.shape[1] * 16, device="cuda")
x, hist = torch.randn(2, 5000, device="cuda"), torch.randint(0, 5000, (2, 9), device="cuda")
long = torch.arange(4, dtype=torch.int32, device="cuda").repeat(2, 512)
m = torch.tensor([20000, 5], dtype=torch.int32, device="cuda")
last = n - 1
calls = [lambda: T.turbo_paged_append(q[:, :2], q[:, :2], k, v, t, last, q=q),
         lambda: T.turbo_paged_attention(q, k, v, t, n, mass=mass.clone()),
         lambda: T.turbo_paged_attention(q, k, v, long, m),
         lambda: T.turbo_paged_evict(k, v, t, to, n, mass, 128)[1],
         lambda: process_logits(x, hist, repetition_penalty=1.5)]
torch.cuda.synchronize()
graphs = []
for f in calls:
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = f()
    graphs.append((g, got))
for (g, got), f in zip(graphs, calls):
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, f())
assert T.ops_error() == (0, 0)
print("captured")
"""


def test_the_first_call_of_a_process_may_be_captured():
    done = subprocess.run([sys.executable, "-c", FIRST, PKG, os.path.join(REPO, "tests")], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]

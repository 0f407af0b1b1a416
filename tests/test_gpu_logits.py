"""GPU tests of process_logits against its formula in 64 bits, and of generate() with it."""
import math

import pytest
import torch

import paged_util as P
from conftest import cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]


def check(got, ref, x, dt):
    """Each of the three steps rounds once in fp32 (a product or quotient, the frequency product and
    the differences, the bias sum): five half-steps of the largest magnitude on the way, which is at
    most 2 |x| (a penalty of at most 2), the result, and 12 for the bias and the presence penalty."""
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf])
    ok = torch.isfinite(ref)
    mag = torch.nan_to_num(x.double().abs(), posinf=0.0) * 2 + torch.nan_to_num(ref.abs(), posinf=0.0) + 12
    assert bool(((got - ref).abs()[ok] <= 5 * 2.0 ** -24 * mag[ok]).all())


def check_best(best, got):
    s = torch.nan_to_num(got.cpu(), nan=-math.inf)
    top = s.max(-1, keepdim=True).values
    want = torch.where(top.squeeze(-1) == -math.inf, 0, (s == top).int().argmax(-1))
    assert torch.equal(best.cpu().long(), want.long())


CASES = [(1, 1, 0), (3, 33, 5), (2, 1000, 1), (4, 32000, 300), (1, 50257, 5000), (5, 8192, 64), (2, 8193, 17),
         (1, 160001, 40), (300, 70, 9), (2, 40000, 32767), (1, 40000, 33000), (148, 5001, 33)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("ids", [torch.int32, torch.int64], ids=["i32", "i64"])
@pytest.mark.parametrize("rows", [False, True], ids=["shared", "rows"])
@pytest.mark.parametrize("case", CASES, ids=["x".join(map(str, c)) for c in CASES])
def test_process_logits(case, rows, ids, dt):
    from one.engine import pack_token_mask, process_logits
    B, V, T = case
    g = torch.Generator().manual_seed(B + V + T)
    x = (3 * torch.randn(B, V, generator=g)).to(dt)
    hist = (V * torch.rand(B, T, generator=g) ** 3).to(ids)
    if T > 4:  # padding of every kind
        hist[:, 1], hist[:, 2], hist[0, 4:] = -1, V, torch.iinfo(ids).min
    starts = torch.randint(-1, T + 2, (B,), generator=g, dtype=torch.int32)
    rep, pres, freq = (torch.rand(B, generator=g) + 0.5 for _ in range(3))
    bias = torch.randn(*((B, V) if rows else (V,)), generator=g)
    allowed = torch.rand(*((B, V) if rows else (1, V)), generator=g) < 0.7
    allowed[0] = allowed[0] & (B == 1)  # a grammar with nothing left
    pen = (rep, pres, freq) if rows else (torch.full((B,), 1.25), torch.full((B,), 0.5), torch.full((B,), 0.125))
    arg = [p.cuda() for p in pen] if rows else [1.25, 0.5, 0.125]
    out, best = process_logits(x.cuda(), hist.cuda(), starts.cuda(), *arg, bias=bias.cuda(),
                               token_mask=pack_token_mask(allowed).cuda(), return_argmax=True)
    ref = P.logits(x, hist, starts, *pen, bias, allowed.expand(B, V))
    check(out, ref, x, dt)
    check_best(best, out)


@pytest.mark.parametrize("case,dt", [((297, 33001, 20), torch.bfloat16), ((299, 40, 32800), torch.float32)], ids=["slices", "ids"])
def test_more_rows_than_fit_at_once(case, dt):
    test_process_logits(case, True, torch.int32, dt)


def test_each_part_alone_and_nothing():
    from one.engine import pack_token_mask, process_logits
    g = torch.Generator().manual_seed(1)
    B, V = 3, 5000
    x = torch.randn(B, V, generator=g)
    x[0, 7], x[1, 7], x[2, 9], x[0, 100] = math.nan, math.inf, -math.inf, -0.0
    hist = torch.randint(0, V, (B, 50), generator=g)
    hist[:, :4] = torch.tensor([7, 9, 100, 7])
    one, zero = torch.ones(B), torch.zeros(B)
    dx, dh = x.cuda(), hist.cuda()
    out, best = process_logits(dx, return_argmax=True)
    assert torch.equal(torch.nan_to_num(out.cpu(), nan=5.5), torch.nan_to_num(x, nan=5.5))
    check_best(best, out)
    check(process_logits(dx, dh, repetition_penalty=1.5), P.logits(x, hist, None, one * 1.5, zero, zero, None, None), x, None)
    check(process_logits(dx, dh, presence_penalty=-0.5), P.logits(x, hist, None, one, one * -0.5, zero, None, None), x, None)
    check(process_logits(dx, dh, frequency_penalty=0.75), P.logits(x, hist, None, one, zero, one * 0.75, None, None), x, None)
    allowed = torch.zeros(B, V, dtype=torch.bool)
    allowed[:, 4999] = True
    out, best = process_logits(dx, token_mask=pack_token_mask(allowed).cuda(), return_argmax=True)
    assert best.tolist() == [4999] * 3 and int(torch.isfinite(out).sum()) == 3
    nothing = torch.full((2, 100), math.nan).cuda()
    _, best = process_logits(nothing, return_argmax=True)
    assert best.tolist() == [0, 0]
    ties = torch.zeros(2, 70000)
    ties[0, [69999, 40000, 12345]] = 2.0
    ties[1, 0] = -0.0
    _, best = process_logits(ties.cuda(), return_argmax=True)
    assert best.tolist() == [12345, 0]


def test_counts_past_15_and_16_bits():
    from one.engine import process_logits
    for n in (32767, 32768, 70000):
        hist = torch.full((1, n), 5, dtype=torch.int32)
        hist[0, 0] = 4  # before the output, beside the token that fills its count
        x = torch.zeros(1, 64)
        starts = torch.tensor([1], dtype=torch.int32)
        out = process_logits(x.cuda(), hist.cuda(), starts.cuda(), frequency_penalty=1.0, presence_penalty=0.5,
                             repetition_penalty=2.0).cpu()
        want = torch.zeros(64)
        want[5] = -(n - 1) - 0.5
        assert torch.equal(out[0], want)


def test_in_place_strided_rows_and_graph():
    from one.engine import process_logits
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(4, 1030, generator=g)
    hist = torch.randint(0, 1000, (4, 64), generator=g, dtype=torch.int32)
    bias = torch.randn(8, 1001, generator=g)
    dw, dh, db = wide.cuda(), hist.cuda(), bias.cuda()
    x = dw[:, 5:1005]
    want = P.logits(wide[:, 5:1005], hist[:, 3:40], None, torch.full((4,), 2.0), torch.zeros(4), torch.zeros(4), bias[::2, 1:], None)
    out = process_logits(x, dh[:, 3:40], repetition_penalty=2.0, bias=db[::2, 1:])
    check(out, want, wide[:, 5:1005], None)
    graph = torch.cuda.CUDAGraph()
    src = torch.empty_like(x.contiguous())
    with torch.cuda.graph(graph):
        got, best = process_logits(src, dh[:, 3:40], repetition_penalty=2.0, bias=db[::2, 1:], return_argmax=True)
    src.copy_(x)
    graph.replay()
    assert torch.equal(got, out)
    check_best(best, out)
    same = process_logits(x, dh[:, 3:40], repetition_penalty=2.0, bias=db[::2, 1:], out=x)
    assert same.data_ptr() == x.data_ptr() and torch.equal(x, out)
    assert torch.equal(dw[:, :5].cpu(), wide[:, :5]) and torch.equal(dw[:, 1005:].cpu(), wide[:, 1005:])


def _model():
    from one.configuration_one import tiny_config
    from one.initialization import init_state_dict
    from one.modeling_one import OneForCausalLM
    cfg = tiny_config()
    model = OneForCausalLM(cfg)
    model.load_state_dict(init_state_dict(cfg, 0, torch.float32), strict=False)
    return cfg, model.to(torch.bfloat16).cuda()


def test_generate_with_penalties():
    """Greedy choice with each penalty equals a loop over the model's own logits and transformers'
    RepetitionPenaltyLogitsProcessor (or the formula); a token mask and a bias hold; sampling with a
    seed repeats; without any of them nothing changes."""
    from transformers.generation.logits_process import RepetitionPenaltyLogitsProcessor
    from one.engine import pack_token_mask
    cfg, model = _model()
    ids = torch.randint(1, cfg.vocab_size, (3, 10), generator=torch.Generator().manual_seed(23)).cuda()

    def loop(process, steps=8):
        eng = model.engine(max_batch=3, max_tokens=30)
        lg, seq = eng.prefill(ids, logits="last"), ids
        for i in range(steps):
            tok = process(seq, lg.float()).argmax(-1)
            seq = torch.cat([seq, tok[:, None]], 1)
            lg, _ = eng.step(tok, logits=True, next_ids=False)
        return seq

    plain = model.generate(ids, max_new_tokens=8)
    same = model.generate(ids, max_new_tokens=8, repetition_penalty=1.0, presence_penalty=0.0)
    assert torch.equal(plain, same)
    hf = RepetitionPenaltyLogitsProcessor(1.5)
    got = model.generate(ids, max_new_tokens=8, repetition_penalty=1.5)
    assert torch.equal(got, loop(lambda s, x: hf(s, x)))

    def counted(s, x):
        c = torch.zeros_like(x).scatter_add_(1, s[:, 10:], torch.ones_like(s[:, 10:], dtype=x.dtype))
        return x - (0.25 * c + 0.5 * (c > 0))
    got = model.generate(ids, max_new_tokens=8, presence_penalty=0.5, frequency_penalty=0.25)
    assert torch.equal(got, loop(counted))
    allowed = torch.zeros(cfg.vocab_size, dtype=torch.bool)
    allowed[100:200] = True
    mask = pack_token_mask(allowed).cuda()
    bias = torch.zeros(cfg.vocab_size)
    bias[150] = 1e4
    got = model.generate(ids, max_new_tokens=4, token_mask=mask, logit_bias=bias.cuda())
    assert bool((got[:, 10:] == 150).all())
    a = model.generate(ids, max_new_tokens=6, do_sample=True, token_mask=mask, repetition_penalty=1.2, seed=4)
    b = model.generate(ids, max_new_tokens=6, do_sample=True, token_mask=mask, repetition_penalty=1.2, seed=4)
    assert torch.equal(a, b) and bool(((a[:, 10:] >= 100) & (a[:, 10:] < 200)).all())

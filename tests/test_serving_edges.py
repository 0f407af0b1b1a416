"""What the serving operators answer at their edges, on the CPU: sizes whose lists do not fit 31 bits,
outputs that overlap the inputs, empty batches."""
import ctypes

import pytest
import torch

from conftest import cuda_ok
from one import _capi as C
from one import turbo_ops as T
from one.engine import process_logits
from test_serving_refusals import A, B_, CACHE, Tokens, cache, cache_of


def overlap(fn, *a, **kw):
    with pytest.raises((ValueError, C.OneError), match="overlap"):
        fn(*a, **kw)


def test_packed_tokens_with_fp32_tables():
    """The two packed forms differ in the last field of one_paged_tokens alone."""
    plain, fp32 = C.PAGED_TOKENS(*range(1, 20)), C.PAGED_TOKENS_FP32_TABLES(*range(1, 20), 1)
    assert len(plain) == len(fp32) == ctypes.sizeof(Tokens) and Tokens.reserved.offset == len(plain) - 4
    assert plain[-4:] == bytes(4) and fp32 == plain[:-4] + (1).to_bytes(4, "little")


def test_attention_refuses_an_out_that_overlaps_q():
    k, v, t, n = cache()
    buf = torch.zeros(4096, dtype=torch.bfloat16)
    q = buf[:512].view(2, 4, 1, 64)
    f = T.turbo_paged_attention
    overlap(f, q, k, v, t, n, out=q.view(2, 4, 1, 64))
    overlap(f, q, k, v, t, n, out=buf[8:520].view(2, 4, 1, 64))
    overlap(f, q, k, v, t, n, out=buf[504:1016].view(2, 4, 1, 64))
    rows = buf.view(2, 4, 8, 64)[:, :, 1:2]  # rows of a wider projection
    overlap(f, rows, k, v, t, n, out=buf[:512].view(2, 4, 1, 64))
    for out in (buf[512:1024], buf[3584:]):  # beside q, and behind its rows
        with pytest.raises(RuntimeError, match="no CPU path"):
            f(q, k, v, t, n, out=out.view(2, 4, 1, 64))
    apart = buf.as_strided((2, 4, 1, 64), (2048, 64, 64, 1))  # rows 0 .. 255 and 2048 .. 2303
    with pytest.raises(RuntimeError, match="no CPU path"):
        f(apart, k, v, t, n, out=buf[256:768].view(2, 4, 1, 64))
    overlap(f, apart, k, v, t, n, out=buf[1600:2112].view(2, 4, 1, 64))


def test_logits_refuse_an_out_that_overlaps_them_otherwise_than_in_place():
    buf = torch.zeros(3, 100)
    x = buf[:, :40]
    overlap(process_logits, x, out=buf[:, 1:41])
    overlap(process_logits, x, out=buf[:, 39:79])
    overlap(process_logits, buf[:2, :40], out=buf[1:, :40])
    half = buf.view(torch.bfloat16)  # the same bytes, read as 200 a row
    overlap(process_logits, half[:, :40], out=buf[:, :40])
    for out in (x, buf[:, 40:80], buf[:, :40].view(3, 40), torch.zeros(3, 40)):  # in place, between the rows, elsewhere
        with pytest.raises(C.OneError, match="CUDA"):
            process_logits(x, out=out)


def test_empty_inputs_have_no_cpu_path_either():
    k, v, t, n = cache()
    q = torch.zeros(0, 4, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        T.turbo_paged_attention(q, k, v, t[:0], n[:0])
    with pytest.raises(C.OneError, match="CUDA"):
        process_logits(torch.zeros(0, 10))


@pytest.mark.skipif(cuda_ok(), reason="its addresses are no memory: where the call were not refused it must not launch")
def test_attention_refuses_lists_that_its_shares_would_carry_past_31_bits():
    """2^31 - 383 tiles rounded up to equal shares pass 2^31."""
    heads, tiles = 255, 8421503
    big = dict(CACHE, B=heads, hkv=1, ps=64, mp=tiles, ts=tiles, ks=64 * 64, vs=64 * 64)
    call = lambda **c: C.LIB.one_paged_attention(cache_of(c), A, 64, 64, 1, 0.1, B_, A, 1 << 40, 0)
    assert heads * (tiles + 1) <= 0x7fffffff and heads * tiles + 443 > 0x7fffffff
    assert call(**big) == C.ONE_ERR_UNSUPPORTED

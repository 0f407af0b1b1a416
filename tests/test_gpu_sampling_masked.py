"""Scores of -inf (tokens that a mask forbids, logits that are NaN) are never drawn, whatever the
variate; scores of +inf take the whole draw."""
import math

import pytest
import torch

from conftest import cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]

# (seed, offset) whose 24-bit variate of row 0 is 0: the draw takes the first token of any weight
ZERO = [(2, 7487565), (3, 4595281), (12, 3490575), (12, 4261844)]


def philox4x32_10(offset, row, seed):
    """First output word for the counter (offset, row), key seed (Salmon et al., SC 2011)."""
    c = [offset & 0xffffffff, offset >> 32, row, 0]
    k = [seed & 0xffffffff, seed >> 32]
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xffffffff, (a >> 32) ^ c[3] ^ k[1], a & 0xffffffff]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
    return c[0]


def test_the_variates_are_zero():
    assert philox4x32_10(0, 0, 0) == 0x6627e8d5  # the paper's known answer
    assert all(philox4x32_10(o, 0, s) >> 8 == 0 for s, o in ZERO)


WARPS = [(1.0, 0, 1.0), (0.7, 0, 1.0), (1.0, 50, 1.0), (1.0, 0, 0.9), (1.3, 60, 0.95), (1.0, 31999, 1.0), (1.0, 5, 1.0)]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("hidden", [-math.inf, math.nan], ids=["masked", "nan"])
@pytest.mark.parametrize("T,k,p", WARPS)
def test_hidden_tokens_are_never_drawn(T, k, p, hidden, dt):
    from one.engine import sample_tokens
    x = torch.full((1, 32000), hidden)
    allowed = torch.arange(20000, 20010)
    x[0, allowed] = torch.linspace(-1, 1, 10)
    dx = x.to(dt).cuda()
    first = 20000 if k != 5 and p == 1.0 else None
    for seed, offset in ZERO:
        got = int(sample_tokens(dx, T, k, p, seed=seed, offset=offset))
        assert 20000 <= got < 20010
        if first is not None:
            assert got == first  # a variate of 0 takes the first token that may be drawn
    for offset in range(20):
        assert 20000 <= int(sample_tokens(dx, T, k, p, seed=7, offset=offset)) < 20010


def test_a_row_with_nothing_left_gives_token_0():
    from one.engine import sample_tokens
    x = torch.full((3, 100), -math.inf)
    x[1] = math.nan
    x[2, 60] = -3.0
    for k, p in ((0, 1.0), (7, 1.0), (0, 0.5), (7, 0.5)):
        assert sample_tokens(x.cuda(), 1.0, k, p, seed=1, offset=0).tolist() == [0, 0, 60]


def test_scores_behind_the_mask_draw_as_they_did():
    """What may be drawn keeps its place on the line of weights: one masked token in front changes
    nothing but its own."""
    from one.engine import sample_tokens
    g = torch.Generator().manual_seed(3)
    x = torch.randn(64, 1000, generator=g)
    x[:, 0] = -100.0  # weight 2^-32, the least there is
    y = x.clone()
    y[:, 0] = -math.inf
    for offset in range(4):
        a, b = (sample_tokens(t.cuda(), 1.0, 0, 1.0, seed=5, offset=offset).cpu() for t in (x, y))
        assert int((a != b).sum()) <= 1


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("T,k,p", WARPS)
def test_scores_of_plus_infinity_take_the_draw(T, k, p, dt):
    """A bias of +inf forces a token; several share the draw."""
    from one.engine import sample_tokens
    x = torch.randn(200, 32000, generator=torch.Generator().manual_seed(4))
    x[:, 17000] = math.inf
    x[:, 3] = -math.inf
    x[100:, 31000] = math.inf
    got = sample_tokens(x.to(dt).cuda(), T, k, p, seed=2, offset=7487565).cpu()
    assert bool((got[:100] == 17000).all())
    assert bool(((got[100:] == 17000) | (got[100:] == 31000)).all())
    # 100 draws of two equal tokens: 5 standard deviations of a binomial
    assert 25 <= int((got[100:] == 31000).sum()) <= 75


def test_generate_is_forced_by_an_infinite_bias():
    from one.configuration_one import tiny_config
    from one.initialization import init_state_dict
    from one.modeling_one import OneForCausalLM
    cfg = tiny_config()
    model = OneForCausalLM(cfg)
    model.load_state_dict(init_state_dict(cfg, 0, torch.float32), strict=False)
    model = model.to(torch.bfloat16).cuda()
    ids = torch.randint(1, cfg.vocab_size, (3, 6), generator=torch.Generator().manual_seed(1)).cuda()
    bias = torch.zeros(cfg.vocab_size)
    bias[77] = math.inf
    for sample in (False, True):
        got = model.generate(ids, max_new_tokens=5, do_sample=sample, logit_bias=bias.cuda(), seed=1)
        assert bool((got[:, 6:] == 77).all())

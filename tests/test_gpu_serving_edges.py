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

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

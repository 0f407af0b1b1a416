"""The check of slots_util finds what it is for, on the CPU: a lost or doubled slot or group of slots."""
import pytest
import torch

from slots_util import Slots, oracle


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lens,dh", [([700, 0, 33], 64), ([12288, 5], 96)], ids=["700", "12288"])
def test_the_check_takes_the_formula_and_nothing_less(lens, dh, dt):
    s = Slots(lens, 1, 3, dh, 16, dt, torch.Generator().manual_seed(5))
    s.check(oracle)
    for lost, twice in (([0], []), ([lens[0] - 1], []), (range(320, 336), []), ([], [319]), ([], range(64, 80)), ([17], [18])):
        with pytest.raises(AssertionError, match="over"):
            s.check(lambda x: oracle(x, lost, twice))

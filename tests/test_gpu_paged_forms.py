"""Forms of the paged attention beyond the common ones, against the evaluation in 64 bits of test_gpu_paged.py and with its bounds."""
import pytest
import torch

import aha_amd  # noqa: F401
from test_gpu_paged import check_attention, filled, gen, ints, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hints", [dict(max_q=2 ** 31), dict(max_len=2 ** 32 + 1), dict(max_q=2 ** 40, max_len=2 ** 64)])
def test_hints_of_any_width(hints):
    c = filled([700, 90], 16, 28, 4, 128, "bf16", 17)
    check_attention(c, randn(gen(18), 132, 28, 128).bfloat16(), ints([0, 1]), ints([0, 131, 132]), **hints)

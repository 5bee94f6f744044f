"""The bound of test_gpu_paged_precision.py on the CPU, in 64 bits: probabilities as two bf16 halves keep it, rounded once to bf16 they break it - so a
kernel that lost its second half would fail those tests."""
import pytest
import torch

from test_gpu_paged_precision import U, tight


def attend(q, k, v, halves):
    """softmax(q k^T / sqrt(D)) v with P in so many bf16 halves (0: as it is), rounded once at the end -> (out, exact, sum p |v|, size)."""
    scale = q.shape[-1] ** -0.5
    s = q @ k.T * scale
    p = (s - s.amax(-1, keepdim=True)).exp()
    l, exact = p.sum(-1, keepdim=True), torch.softmax(s, -1)
    if halves:
        hi = p.bfloat16().double()
        p = hi + ((p - hi).bfloat16().double() if halves == 2 else 0)
        l = p.sum(-1, keepdim=True)
    return (p @ v / l).bfloat16().double(), exact @ v, exact @ v.abs(), float((q.abs() @ k.abs().T * scale).max())


@pytest.mark.parametrize("dim", [16, 48, 64, 80, 128])
@pytest.mark.parametrize("keys", [5, 17, 33, 70, 700])
def test_one_rounding_of_p_breaks_the_bound_and_two_halves_keep_it(dim, keys):
    g = torch.Generator().manual_seed(dim + keys)
    q, k, v = ((torch.randn(n, dim, generator=g, dtype=torch.float64) * f).bfloat16().double() for n, f in ((28, 1.5), (keys, 1), (keys, 1)))
    for halves, kept in ((0, True), (2, True), (1, False)):
        out, exact, mag, size = attend(q, k, v, halves)
        off = (out - exact).abs() - U * exact.abs() - tight(dim, size, keys) * mag
        assert (float(off.max()) <= 0) == kept, (halves, float(off.max()), int((off > 0).sum()))


def test_no_handle_no_choice():
    from aha_amd import lib
    assert lib.get().aha_paged_set_precise(None, 1) == -22

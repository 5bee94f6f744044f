"""How exact the attention is where the probabilities go into the second product as two bf16 halves: the bound has no room for one rounding to bf16.

|out - o| <= 2^-8 |o| (the output's rounding) + e sum_j p_j |v_j|, with e =
  2 * D * 2^-24 * max_j sum_d |q_d k_jd| * scale     the scores, fp32 sums of D products (numerator and denominator)
  + 2 * 2^-17                                        the halves: what the first leaves is 2^-8 of p at most, half its step 2^-17 (both)
  + 4 * L * 2^-24                                    the sums over two halves of L keys, a rounding an addition (both)
  + 2^-21                                            exp2, the weights of the join, the division: a few units of 2^-24
test_paged_bound.py shows that one rounding breaks it."""
import pytest
import torch

import aha_amd  # noqa: F401
from test_gpu_paged import DEV, LAYOUTS, U, attention64, close, filled, gen, ints, randn

pytestmark = pytest.mark.gpu


def tight(dim, size, keys):
    return 2 * dim * 2.0 ** -24 * size + 2.0 ** -16 + 4 * keys * 2.0 ** -24 + 2.0 ** -21


def check_tight(c, q, seqs, cu, window=0, **hints):
    got = c.attention(0, q, seqs, cu, window=window, **hints)
    want, mag, size = attention64(c, q, seqs, cu, window)
    close(got, want, U * want.abs() + tight(q.shape[-1], size, int(c.lens.max())) * torch.nan_to_num(mag), "attention")
    return got


@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_single_tokens(heads, kv_heads, dim, kind):
    """Short and long sequences, whole and cut, with the hints and without."""
    lens = [1, 2, 5, 17, 33, 70, 700]
    c = filled(lens, 16, heads, kv_heads, dim, kind, heads + dim)
    q = (randn(gen(1), 7, heads, dim) * 1.5).bfloat16()
    seqs, cu = ints(range(7)), ints(range(8))
    check_tight(c, q, seqs, cu, max_q=1, max_len=700)
    check_tight(c, q, seqs, cu)
    check_tight(c, q, seqs, cu, window=20, max_q=1)


@pytest.mark.parametrize("heads,kv_heads,dim,T", [(8, 2, 64, 4), (7, 1, 128, 2), (4, 4, 16, 16), (6, 3, 80, 8)])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_few_tokens_of_a_small_group(heads, kv_heads, dim, T, kind):
    """Up to sixteen rows a key-value head."""
    lens = [T, T + 3, 33, 70, 700]
    c = filled(lens, 32, heads, kv_heads, dim, kind, dim + T)
    q = (randn(gen(2), 5 * T, heads, dim) * 1.5).bfloat16()
    check_tight(c, q, ints(range(5)), ints(range(0, 5 * T + 1, T)), max_q=T)


@pytest.mark.parametrize("kind,L", [("bf16", 3001), ("e4m3", 2500)])
def test_a_token_over_a_long_sequence(kind, L):
    c = filled([L, 40], 64, 28, 4, 128, kind, L)
    check_tight(c, randn(gen(3), 2, 28, 128).bfloat16(), ints([0, 1]), ints([0, 1, 2]), max_q=1, max_len=L)

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


def precisely(c):
    c._chk(c.lib.aha_paged_set_precise(c.handle, 1))
    return c


@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_a_precise_pool_keeps_the_bound_with_many_rows(heads, kv_heads, dim, kind):
    """Drafts, frames and prompts, cut and whole, in tiles of 64 and of 128 rows, with a window and without."""
    lens = [150, 36, 700, 300, 5, 129, 3]
    counts = [2, 36, 131, 0, 5, 49, 5]                                       # (the last has more tokens than keys)
    c = precisely(filled(lens, 32, heads, kv_heads, dim, kind, dim))
    cu = ints([0] + torch.tensor(counts).cumsum(0).tolist())
    q = (randn(gen(2), sum(counts), heads, dim) * 1.5).bfloat16()
    whole = check_tight(c, q, ints(range(7)), cu, max_q=131, max_len=256)
    check_tight(c, q, ints(range(7)), cu)
    check_tight(c, q, ints(range(7)), cu, window=40, max_q=131)
    few = torch.cat([q[cu[i]:cu[i] + 5] for i in (1, 2, 4)])
    check_tight(c, few, ints([1, 2, 4]), ints([0, 5, 10, 15]), max_q=5)
    assert torch.equal(c.attention(0, q, ints(range(7)), cu, max_q=131, max_len=256), whole)


@pytest.mark.parametrize("T,L,kind", [(5, 3000, "bf16"), (36, 2500, "bf16"), (36, 2500, "e4m3"), (300, 1500, "e4m3")])
def test_a_precise_pool_over_long_sequences(T, L, kind):
    c = precisely(filled([L, 40], 64, 28, 4, 128, kind, L))
    n = T + 1
    check_tight(c, randn(gen(3), n, 28, 128).bfloat16(), ints([0, 1]), ints([0, T, n]), max_q=T, max_len=L)


@pytest.mark.parametrize("T,kind", [(6, "bf16"), (40, "bf16"), (140, "e4m3")])
def test_a_value_that_is_not_finite_in_a_precise_pool(T, kind):
    """Reaches the rows that see its key, no others."""
    L = 200
    c = precisely(filled([L], 16, 7, 1, 128, kind, 11))
    raw = c.v_pages.view(torch.uint8 if kind == "e4m3" else torch.int16)
    for j in (L - 2, L - T // 2 - 1):
        raw[0, int(c.block_table[0, j // 16]), 0, j % 16, 3] = 0x7f if kind == "e4m3" else 0x7fc0
    got = check_tight(c, randn(gen(7), T, 7, 128).bfloat16(), ints([0]), ints([0, T]), window=20, max_q=T)
    assert bool(torch.isnan(got[-1, 0, 3])) and not bool(torch.isnan(got[0].float()).any())


def test_the_choice_is_the_handles():
    """Two handles over the same memory, one precise: each keeps its own, a token has the same bits in both, and it can be switched off again."""
    from aha_amd.paged import PagedKVCache
    a = filled([700, 300], 16, 28, 4, 128, "bf16", 5)
    b = PagedKVCache(a.n_pages, 16, 4, 128, 2, a.max_blocks, device=DEV, k_pages=a.k_pages, v_pages=a.v_pages, block_table=a.block_table, lens=a.lens,
                     free_pages=a.free_pages, n_free=a.n_free, precise=True)
    seqs, cu, one = ints([0, 1]), ints([0, 40, 80]), ints([0, 1, 2])
    q = randn(gen(9), 80, 28, 128).bfloat16()
    rounded, exact = a.attention(0, q, seqs, cu, max_q=40), check_tight(b, q, seqs, cu, max_q=40)
    assert not torch.equal(rounded, exact)
    assert torch.equal(a.attention(0, q[:2], seqs, one, max_q=1), b.attention(0, q[:2], seqs, one, max_q=1))
    b._chk(b.lib.aha_paged_set_precise(b.handle, 0))
    assert torch.equal(b.attention(0, q, seqs, cu, max_q=40), rounded)

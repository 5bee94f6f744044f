"""Forms of the paged attention beyond the common ones, against the evaluation in 64 bits of test_gpu_paged.py and with its bounds."""
import pytest
import torch

import aha_amd  # noqa: F401
from aha_amd.paged import PagedKVCache
from aha_amd.runtime import AhaError
from test_gpu_paged import DEV, check_attention, filled, gen, ints, pool, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hints", [dict(max_q=2 ** 31), dict(max_len=2 ** 32 + 1), dict(max_q=2 ** 40, max_len=2 ** 64)])
def test_hints_of_any_width(hints):
    c = filled([700, 90], 16, 28, 4, 128, "bf16", 17)
    check_attention(c, randn(gen(18), 132, 28, 128).bfloat16(), ints([0, 1]), ints([0, 131, 132]), **hints)


@pytest.mark.parametrize("T", [1, 3, 40, 150])
@pytest.mark.parametrize("window", [0, 70])
def test_a_head_whose_scale_is_zero(T, window):
    """Its keys are all zero, so every visible key weighs the same; hidden ones still nothing.  Another head's values are zero."""
    c = filled([700, 90, T], 16, 12, 4, 128, "e4m3", 41 + T)
    c.k_scale[0, 1], c.v_scale[0, 2] = 0.0, 0.0
    q = (randn(gen(42), 3 * T, 12, 128) * 1.5).bfloat16()
    got = check_attention(c, q, ints([0, 1, 2]), ints([0, T, 2 * T, 3 * T]), window=window, max_q=T)
    assert not bool(got.view(-1, 4, 3, 128)[:, 2].any())


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("scale", [1e-38, 2e-45])
def test_scales_whose_product_is_below_the_least_float(T, scale):
    c = filled([700, 90], 16, 8, 2, 64, "e4m3", 43)
    c.k_scale.fill_(1e-12)
    check_attention(c, randn(gen(44), 2 * T, 8, 64).bfloat16(), ints([0, 1]), ints([0, T, 2 * T]), scale=scale, max_q=T)


def test_append_with_a_scale_of_zero_stores_zero():
    c = pool(1, 16, 1, 1, 2, 16, dtype=torch.float8_e4m3fn, k_scale=torch.tensor([[0.0, 0.5]], device=DEV), v_scale=torch.tensor([[0.5, 0.0]], device=DEV))
    x = torch.tensor([[0.0, -0.0, 3.0, -1e4, float("inf"), -float("inf"), float("nan"), 2 ** -20] * 4], device=DEV).bfloat16()
    c.append(0, None, x, x, ints([0]))
    for pages, zero in ((c.k_pages, 0), (c.v_pages, 1)):
        got = pages[0, 0, :, 0].float()
        nan = torch.isnan(x.view(2, 16)[0])
        assert torch.equal(torch.isnan(got[zero]), nan) and not bool(got[zero][~nan].any())
        other = (x.view(2, 16)[1 - zero].float() / 0.5).clamp(-448, 448)
        assert torch.equal(got[1 - zero][~nan], other[~nan].to(torch.float8_e4m3fn).float())


@pytest.mark.parametrize("heads,kv_heads,dim", [(17, 1, 64), (64, 2, 128), (71, 1, 48), (130, 1, 128), (256, 2, 16)])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_groups_of_more_than_sixteen_heads(heads, kv_heads, dim, kind):
    """A token alone then fills a tile of 64 or 128 rows, or several; in place, with a window, and with a few more tokens."""
    lens = [1, 700, 33, 64, 0, 65, 2500]
    c = filled(lens, 16, heads, kv_heads, dim, kind, heads)
    q = (randn(gen(1), 7, heads, dim) * 1.5).bfloat16()
    seqs, cu = ints([3, 1, -1, 0, 6, 4, 2]), ints(range(8))
    want = check_attention(c, q, seqs, cu, max_q=1, max_len=2500)
    check_attention(c, q, seqs, cu)
    check_attention(c, q, seqs, cu, window=100, max_q=1)
    got = q.clone()
    c.attention(0, got, seqs, cu, max_q=1, max_len=2500, out=got)
    assert torch.equal(torch.cat((got[:2], got[3:])), torch.cat((want[:2], want[3:]))) and torch.equal(got[2], q[2])
    q = randn(gen(2), 12, heads, dim).bfloat16()
    check_attention(c, q, ints([6, 1, 2]), ints([0, 5, 9, 12]), max_q=5)


@pytest.mark.parametrize("page", [256, 512, 1024])
@pytest.mark.parametrize("T", [1, 6, 40, 150])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_large_pages(page, T, kind):
    lens = [page - 1, page, page + 1, 2 * page + 77, T, 3 * page]
    c = filled(lens, page, 14, 2, 64, kind, page + T)
    q = randn(gen(5), 6 * T, 14, 64).bfloat16()
    seqs, cu = ints([5, 0, 1, 4, 2, 3]), ints(range(0, 6 * T + 1, T))
    check_attention(c, q, seqs, cu, max_q=T, max_len=3 * page)
    check_attention(c, q, seqs, cu, window=page // 2, max_q=T)


@pytest.mark.parametrize("kv_heads", [128, 300, 600])
@pytest.mark.parametrize("T", [1, 20])
def test_more_key_value_heads_than_workgroups_run_at_once(kv_heads, T):
    """A long sequence is then cut in few chunks or none."""
    c = filled([3000, 70], 32, kv_heads, kv_heads, 16, "bf16", kv_heads)
    q = randn(gen(6), 2 * T, kv_heads, 16).bfloat16()
    check_attention(c, q, ints([0, 1]), ints([0, T, 2 * T]), max_q=T)


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_sequences_that_fill_their_tables(page, kind):
    """No entry is left behind the last page, of the last sequence no table either; not one token more is reserved."""
    lens = [5 * page, 3, 5 * page - 1, 5 * page]
    c = filled(lens, page, 14, 2, 64, kind, page, spare=0)
    c = PagedKVCache(c.n_pages, page, 2, 64, 4, 5, dtype=c.dtype, device=DEV, k_pages=c.k_pages, v_pages=c.v_pages, block_table=c.block_table[:, :5].contiguous(),
                     lens=c.lens, k_scale=c.k_scale, v_scale=c.v_scale)
    c.n_free.zero_()
    for T in (1, 7, 40):
        q = randn(gen(T), 4 * T, 14, 64).bfloat16()
        check_attention(c, q, ints([3, 1, 2, 0]), ints(range(0, 4 * T + 1, T)), max_q=T)
        check_attention(c, q, ints([3, 1, 2, 0]), ints(range(0, 4 * T + 1, T)), window=page + 5, max_q=T)
    assert c.reserve(ints([2]), ints([1]), 1)[3].tolist() == [0, 0] and c.reserve(ints([2]), ints([1]), 1)[3].tolist() == [16, 0]
    assert c.lens.tolist() == [5 * page, 3, 5 * page, 5 * page]


@pytest.mark.parametrize("T,L", [(1, 300), (1, 3000), (6, 300), (40, 3000), (150, 300)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_query_that_is_no_number_stays_alone(T, L, bad):
    c = filled([L, L - 70], 16, 14, 2, 64, "bf16", 51)
    q = randn(gen(52), 2 * T, 14, 64).bfloat16()
    seqs, cu = ints([0, 1]), ints([0, T, 2 * T])
    want = c.attention(0, q, seqs, cu, max_q=T)
    q[T // 2, 9, 5] = bad                                                    # times keys of both signs: no row of numbers either way
    got = c.attention(0, q, seqs, cu, max_q=T)
    assert bool(torch.isnan(got[T // 2, 9]).all())
    got[T // 2, 9] = want[T // 2, 9]
    assert torch.equal(got, want)


def test_calls_from_two_threads():
    """Each on a stream of its own over one pool; a refusal's message is its thread's."""
    import threading
    c = filled([900, 700], 16, 14, 2, 64, "bf16", 53)
    qs = [randn(gen(54 + i), 2, 14, 64).bfloat16() for i in range(2)]
    seqs, cu = ints([0, 1]), ints([0, 1, 2])
    want, wrong = [c.attention(0, q, seqs, cu, max_q=1) for q in qs], []
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = c.attention(0, qs[i], seqs, cu, max_q=1)
                try:
                    c.attention(0 if i else 7, qs[i], seqs, cu, scale=-1.0 if i else None)
                except AhaError as e:
                    wrong.extend([] if ("scale" if i else "layer") in str(e) else [str(e)])
                torch.cuda.current_stream().synchronize()
                wrong.extend([] if torch.equal(got, want[i]) else ["values"])

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]

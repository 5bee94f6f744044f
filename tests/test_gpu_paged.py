"""The paged key-value cache against plain evaluations in 64 bits: block tables and slot maps, rotation and storage, attention.

Bounds, u = 2^-8 being half a bf16 step relative to the value (torch.finfo(torch.bfloat16).eps / 2):
  tables     whole numbers, equal
  append     one rounding of an fp32 result: u |x| + 2^-22 (|x1| + |x2|) (two products, exact in fp32, and a sum); e4m3: 2^-4 |x| (half its step), and
             half of its least step 2^-9 below the smallest normal number
  attention  u |o| (the output) + e sum_j p_j |v_j|, e being what p may be off by: 2 * D * 2^-24 * max_j sum_d |q_d k_jd| * scale from the fp32 scores
             (numerator and denominator) + 2^-12 for exp2, the sums over the keys (each lane adds at most L / 16 terms, in fp32) and the
             remainder of P's two bf16 halves (2^-17); + u where P is rounded to one bf16 (tiles of many rows).
"""
import math
import random

import pytest
import torch

import aha_amd  # noqa: F401
from aha_amd.paged import PagedKVCache
from aha_amd.runtime import AhaError, rope_table

pytestmark = pytest.mark.gpu
U = 2.0 ** -8
DEV = "cuda:0"


def ints(x):
    return torch.tensor(list(x), dtype=torch.int32, device=DEV)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


# ---- tables -------------------------------------------------------------------------------------------------------------------------
class Tables:
    """The tables of a pool, one request after the other in whole numbers."""

    def __init__(self, n_pages, page, max_seqs, max_blocks):
        self.page, self.n_pages, self.max_blocks = page, n_pages, max_blocks
        self.free, self.lens, self.pages = list(range(n_pages - 1, -1, -1)), [0] * max_seqs, [[] for _ in range(max_seqs)]

    def reserve(self, seqs, counts, n_tokens):
        slots, positions, cu = [], [], [0]
        for s, c in zip(seqs, counts):
            if s >= 0:
                for p in range(self.lens[s], self.lens[s] + c):
                    if p // self.page == len(self.pages[s]):
                        self.pages[s].append(self.free.pop())
                    slots.append(self.pages[s][p // self.page] * self.page + p % self.page)
                    positions.append(p)
                self.lens[s] += c
            cu.append(len(slots))
        pad = [-1] * (n_tokens - len(slots))
        return slots + pad, positions + pad, cu

    def truncate(self, seqs, lens):
        taken = []
        for s, n in zip(seqs, lens):
            if s >= 0:
                keep = -(-n // self.page)
                taken += self.pages[s][keep:]
                del self.pages[s][keep:]
                self.lens[s] = n
        self.free += taken[::-1]

    def same(self, c):
        assert c.lens.tolist() == self.lens
        n = int(c.n_free)
        assert c.free_pages[:n].tolist() == self.free
        t = c.block_table.tolist()
        for s, p in enumerate(self.pages):
            assert t[s][:len(p)] == p, s


def pool(n_pages, page, max_seqs, max_blocks, kv_heads=1, dim=16, **kw):
    return PagedKVCache(n_pages, page, kv_heads, dim, max_seqs, max_blocks, device=DEV, **kw)


@pytest.mark.parametrize("page,max_seqs,n,most,steps", [(16, 3, 1, 1, 40), (16, 40, 17, 60, 6), (64, 300, 257, 40, 4), (32, 1500, 1300, 9, 3), (128, 70, 64, 700, 2),
                                                        (1024, 5, 5, 3000, 2)])
def test_tables_follow_the_plain_bookkeeping(page, max_seqs, n, most, steps):
    """Random steps: growth (some by nothing), padding entries, spare slots, truncation and release, whole state compared after each."""
    rng = random.Random(page * 7 + n)
    blocks = -(-most * steps // page) + 1
    c, t = pool(max_seqs * blocks, page, max_seqs, blocks), Tables(max_seqs * blocks, page, max_seqs, blocks)
    for _ in range(steps):
        seqs = rng.sample(range(max_seqs), n)
        for i in range(0, n, 5):
            if n > 4 and rng.random() < 0.5:
                seqs[i] = -1
        counts = [rng.choice((0, 1, most, rng.randint(0, most))) for _ in range(n)]
        total = sum(k for s, k in zip(seqs, counts) if s >= 0)
        room = total + rng.choice((0, 3))
        slots, positions, cu, status = c.reserve(ints(seqs), ints(counts), room)
        ws, wp, wc = t.reserve(seqs, counts, room)
        assert status.tolist() == [0, 0]
        assert cu.tolist() == wc and slots.tolist() == ws and positions.tolist() == wp
        t.same(c)
        back = rng.sample(range(max_seqs), max(1, n // 2))
        lens = [rng.choice((0, t.lens[s], rng.randint(0, t.lens[s]))) for s in back]
        assert c.truncate(ints(back), ints(lens)).tolist() == [0, 0]
        t.truncate(back, lens)
        t.same(c)


def state(c):
    return [x.clone() for x in (c.block_table, c.lens, c.free_pages, c.n_free)]


@pytest.mark.parametrize("n,most", [(1, 1), (9, 200), (70, 3000)])
def test_truncate_is_the_inverse_of_reserve(n, most):
    rng = random.Random(n)
    c = pool(n * (most // 16 + 8), 16, n, most // 16 + 8)
    seqs = ints(rng.sample(range(n), n))
    c.check(c.reserve(seqs, ints(rng.randint(0, 50) for _ in range(n)), 50 * n)[3])
    before, held = state(c), c.lens[seqs.long()].contiguous()
    c.check(c.reserve(seqs, ints(rng.randint(0, most) for _ in range(n)), most * n)[3])
    c.check(c.truncate(seqs, held))
    free = int(before[3])
    assert torch.equal(c.free_pages[:free], before[2][:free])
    assert torch.equal(c.lens, before[1]) and torch.equal(c.n_free, before[3]) and torch.equal(c.block_table, before[0])


@pytest.mark.parametrize("what,seqs,counts,room,code,missing", [
    ("pages", [0, 1], [16, 16 * 9], 500, 1, 1), ("tokens", [0, 1], [5, 6], 10, 2, 0), ("sequence", [0, 4], [1, 1], 10, 4, 0), ("twice", [2, 1, 2], [1, 1, 1], 10, 8, 0),
    ("long", [0], [16 * 12 + 1], 500, 16, 0), ("longest count", [0], [2 ** 31 - 1], 500, 16, 0), ("negative", [0, 1], [3, -1], 10, 32, 0),
    ("two reasons", [0, 0], [-1, 1], 10, 40, 0)])
def test_a_reserve_that_cannot_be_done_changes_nothing(what, seqs, counts, room, code, missing):
    c = pool(12, 16, 4, 12)
    c.check(c.reserve(ints([3]), ints([33]), 33)[3])                        # three of the twelve pages
    before = state(c)
    slots, positions, cu, status = c.reserve(ints(seqs), ints(counts), room)
    assert status.tolist() == [code, missing]
    assert cu.tolist() == [0] * (len(seqs) + 1) and set(slots.tolist()) == {-1} and set(positions.tolist()) == {-1}
    assert all(torch.equal(a, b) for a, b in zip(before, state(c)))
    with pytest.raises(AhaError):
        c.check(status)


@pytest.mark.parametrize("seqs,lens,code", [([3], [34], 32), ([3], [-1], 32), ([3, 3], [1, 1], 8), ([4], [0], 4)])
def test_a_truncate_that_cannot_be_done_changes_nothing(seqs, lens, code):
    c = pool(12, 16, 4, 12)
    c.check(c.reserve(ints([3]), ints([33]), 33)[3])
    before = state(c)
    assert c.truncate(ints(seqs), ints(lens)).tolist() == [code, 0]
    assert all(torch.equal(a, b) for a, b in zip(before, state(c)))


def test_tables_of_no_request():
    c = pool(12, 16, 4, 12)
    slots, positions, cu, status = c.reserve(ints([]), ints([]), 3)
    assert slots.tolist() == [-1] * 3 and cu.tolist() == [0] and status.tolist() == [0, 0]
    assert c.truncate(ints([]), ints([])).tolist() == [0, 0] and int(c.n_free) == 12
    c.check(c.reserve(ints([-1, -7]), ints([5, 6]), 0)[3])                  # nothing but padding, no slots asked for
    assert int(c.n_free) == 12


# ---- append -------------------------------------------------------------------------------------------------------------------------
def close(got, want, bound, what):
    """Elementwise; where `want` is not finite, got is the same."""
    got, want, bound = got.double(), want.double(), torch.as_tensor(bound, device=got.device).double().expand_as(want)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    off = ((got - want).abs() - bound)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, (what, float(off.max()), int((off > 0).sum()))


LAYOUTS = [(28, 4, 128), (8, 2, 64), (4, 4, 16), (6, 3, 80), (7, 1, 128), (5, 1, 48)]


@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("n", [1, 37])
def test_append_rotates_and_stores(heads, kv_heads, dim, kind, n):
    """Strided rows of a fused projection; some tokens without a slot; the rest of the pool stays as it was."""
    g = gen(heads * dim + n)
    page, pages, layers = 16, 9, 2
    cos, sin = (t.to(DEV) for t in rope_table(4096, dim, 1e6))
    scales = {} if kind == "bf16" else dict(k_scale=torch.rand((layers, kv_heads), generator=g, device=DEV) + 0.01, v_scale=torch.rand((layers, kv_heads), generator=g, device=DEV) * 1e-3)
    dtype = torch.bfloat16 if kind == "bf16" else torch.float8_e4m3fn
    c = pool(pages, page, 4, 4, kv_heads, dim, layers=layers, dtype=dtype, rope=(cos, sin), **scales)
    for p in (c.k_pages, c.v_pages):
        p.view(torch.uint8).copy_(torch.randint(0, 256, p.view(torch.uint8).shape, generator=g, device=DEV))       # anything, NaN among it
    was = [p.clone() for p in (c.k_pages, c.v_pages)]
    qkv = (randn(g, n, (heads + 2 * kv_heads) * dim) * 2).bfloat16()
    q, k, v = qkv.split((heads * dim, kv_heads * dim, kv_heads * dim), -1)
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:n].int()
    if n > 5:
        slots[3], slots[4] = -1, pages * page                                # no slot, one behind the pool
    positions = torch.randint(0, 4096, (n,), generator=g, device=DEV).int()
    got = c.append(1, q, k, v, slots, positions)
    q2 = qkv.clone()[:, :heads * dim]
    assert torch.equal(c.append(1, q2, k, v, slots, positions, q_out=q2).reshape_as(got), got)                      # in place, and twice the same
    cc, ss = cos[positions.long()].double()[:, None], sin[positions.long()].double()[:, None]

    def turn(x):
        x = x.double().reshape(n, -1, dim)
        r = torch.cat((-x[..., dim // 2:], x[..., :dim // 2]), -1)
        return x * cc + r * ss, (x * cc).abs() + (r * ss).abs()

    want, mag = turn(q)
    close(got, want, U * want.abs() + 2.0 ** -22 * mag, "q")
    kr, km = turn(k)
    ok = (slots >= 0) & (slots < pages * page)
    for pages_t, old, x, mag, scale, what in ((c.k_pages, was[0], kr, km, scales.get("k_scale"), "k"),
                                              (c.v_pages, was[1], v.double().reshape(n, -1, dim), torch.zeros_like(km), scales.get("v_scale"), "v")):
        assert torch.equal(pages_t[0].view(torch.uint8), old[0].view(torch.uint8)), what                             # the other layer
        now, then = (t[1].transpose(1, 2).reshape(pages * page, kv_heads, dim) for t in (pages_t.view(torch.uint8).view(dtype), old))
        s = slots[ok].long()
        if kind == "e4m3":
            y = x[ok] / scale[1].double()[:, None]
            clamped = y.clamp(-448, 448)
            close(now.view(torch.uint8)[s].view(dtype).float(), clamped, clamped.abs() / 16 * (1 + 2 ** -18) + 2.0 ** -10 + 2.0 ** -22 * mag[ok] / scale[1].double()[:, None], what)
        else:
            close(now[s], x[ok], U * x[ok].abs() + 2.0 ** -22 * mag[ok], what)
        keep = torch.ones(pages * page, dtype=torch.bool, device=DEV)
        keep[s] = False
        assert torch.equal(now.view(torch.uint8)[keep], then.view(torch.uint8)[keep]), what


def test_append_without_rotation_or_queries_keeps_the_bits():
    g = gen(5)
    c = pool(4, 16, 1, 4, 2, 32)
    k, v = randn(g, 7, 2, 32).bfloat16(), randn(g, 7, 2, 32).bfloat16()
    k[2, 1, 3], v[1, 0, 0], v[6, 1, 31] = float("nan"), float("inf"), -float("inf")
    assert c.append(0, None, k, v, ints(range(20, 27))) is None
    flat = [p[0].transpose(1, 2).reshape(64, 2, 32)[20:27] for p in (c.k_pages, c.v_pages)]
    for a, b in zip(flat, (k, v)):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_e4m3_clamps_and_keeps_nan():
    c = pool(1, 16, 1, 1, 1, 16, dtype=torch.float8_e4m3fn)
    v = torch.tensor([[1e4, -1e4, 448, 449, 464, 465, float("inf"), -float("inf"), float("nan"), 0, -0.0, 2 ** -9, 2 ** -10, 3 * 2 ** -11, 17, 19]], device=DEV).bfloat16()
    c.append(0, None, v, v, ints([0]))
    want = v.float().clamp(-448, 448).to(torch.float8_e4m3fn)
    assert torch.equal(c.v_pages[0, 0, 0, 0].view(torch.uint8), want[0].view(torch.uint8)) or torch.equal(
        torch.nan_to_num(c.v_pages[0, 0, 0, 0].float(), 7.5), torch.nan_to_num(want[0].float(), 7.5))


# ---- attention ----------------------------------------------------------------------------------------------------------------------
def filled(lens, page, heads, kv_heads, dim, kind, seed, spare=3, rubbish=True):
    """A pool whose sequences have these lengths, pages in a random order; every slot that no sequence owns, and every page that none has,
    holds NaN and infinities."""
    g = gen(seed)
    blocks = [-(-n // page) for n in lens]
    n_pages, wide = sum(blocks) + spare, max(max(blocks), 1) + 1
    dtype = torch.bfloat16 if kind == "bf16" else torch.float8_e4m3fn
    scales = {} if kind == "bf16" else dict(k_scale=torch.rand((1, kv_heads), generator=g, device=DEV) * 0.02 + 0.01, v_scale=torch.rand((1, kv_heads), generator=g, device=DEV) * 0.02 + 0.01)
    c = pool(n_pages, page, len(lens), wide, kv_heads, dim, dtype=dtype, **scales)
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    at = 0
    for s, b in enumerate(blocks):
        c.block_table[s, :b] = ints(order[at:at + b])
        at += b
    c.lens.copy_(ints(lens))
    for p in (c.k_pages, c.v_pages):
        x = randn(g, *p.shape)
        p.copy_(x.to(dtype) if kind == "bf16" else (x * 60).clamp(-448, 448).to(dtype))
    if rubbish:
        owned = torch.zeros((n_pages, page), dtype=torch.bool, device=DEV)
        for s, n in enumerate(lens):
            t = torch.arange(n, device=DEV)
            owned[c.block_table[s][t // page].long(), t % page] = True
        hole = ~owned[None, :, None, :, None].expand_as(c.k_pages)
        raw = torch.uint8 if kind == "e4m3" else torch.int16
        for p, bits in ((c.k_pages, 0x7f if kind == "e4m3" else 0x7fc0), (c.v_pages, 0xff if kind == "e4m3" else 0x7f80)):
            p.view(raw)[hole] = bits
    return c


def attention64(c, q, seqs, cu, window=0, scale=None, layer=0):
    """(what it is, sum p |v|, the largest sum |q k| scale) in 64 bits; rows of no request are NaN."""
    n, heads, d = q.shape
    hk, page = c.kv_heads, c.page_size
    scale = d ** -0.5 if scale is None else scale
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device=q.device)
    mag, size = out.clone(), 0.0
    cu, lens = cu.tolist(), c.lens.tolist()
    for i, s in enumerate(seqs.tolist()):
        if s < 0 or cu[i] == cu[i + 1]:
            continue
        L, T = lens[s], cu[i + 1] - cu[i]
        rows = slice(cu[i], cu[i + 1])
        out[rows], mag[rows] = 0.0, 0.0
        if L == 0:
            continue
        t = torch.arange(L, device=q.device)
        pages = c.block_table[s].long()[t // page]
        good = (pages >= 0) & (pages < c.n_pages)
        pages = pages.clamp(0, c.n_pages - 1)

        def take(p, sc):
            x = p[layer].view(torch.uint8)[pages, :, t % page].view(c.dtype).double()
            return x if sc is None else x * sc[layer].double()[:, None]

        k, v = take(c.k_pages, c.k_scale), take(c.v_pages, c.v_scale)                           # [L, hk, d]
        pos = L - T + torch.arange(T, device=q.device)[:, None]
        see = (t <= pos) & good
        if window:
            see &= t > pos - window
        for h in range(heads):
            kh, vh = k[:, h * hk // heads], v[:, h * hk // heads]
            sc = (q[rows, h].double() @ kh.T * scale).masked_fill(~see, -math.inf)
            p = torch.softmax(sc, -1).masked_fill(~see, 0.0)
            p = torch.where(see.any(-1, keepdim=True), p, torch.zeros_like(p))
            fine = torch.isfinite(vh)
            vz = torch.where(fine, vh, torch.zeros_like(vh))
            o, m = p @ vz, p @ vz.abs()
            if not bool(fine.all()):                                                            # a value that is not finite reaches the rows that see it
                w = torch.where(see[:, :, None], p[:, :, None] * vh[None], torch.zeros((), dtype=torch.float64, device=q.device)).sum(1)
                o = torch.where((see.double() @ (~fine).double()) > 0, w, o)
            out[rows, h], mag[rows, h] = o, m
            reach = (q[rows, h].double().abs() @ torch.where(torch.isfinite(kh), kh, torch.zeros_like(kh)).abs().T * scale)[see]
            size = max(size, float(reach.max()) if reach.numel() else 0.0)
    return out, mag, size


def slack(dim, size, rounded_p):
    return 2 * dim * 2.0 ** -24 * size + 2.0 ** -12 + (U if rounded_p else 0.0)


def check_attention(c, q, seqs, cu, window=0, scale=None, **hints):
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=DEV)
    got = c.attention(0, q, seqs, cu, window=window, scale=scale, out=out, **hints)
    want, mag, size = attention64(c, q, seqs, cu, window, scale)
    nobody = torch.ones(q.shape[0], dtype=torch.bool, device=DEV)
    for i, s in enumerate(seqs.tolist()):
        if s >= 0:
            nobody[int(cu[i]):int(cu[i + 1])] = False
    assert bool((got[nobody] == 7.0).all()), "rows of no request were written"
    rows = ~nobody
    close(got[rows], want[rows], U * want[rows].abs() + slack(q.shape[-1], size, True) * torch.nan_to_num(mag[rows]), "attention")
    return got


@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
@pytest.mark.parametrize("kind,page", [("bf16", 16), ("bf16", 64), ("e4m3", 16), ("e4m3", 128)])
def test_attention_of_single_tokens(heads, kv_heads, dim, kind, page):
    lens = [1, 700, 17, 64, 0, 65, 333]
    c = filled(lens, page, heads, kv_heads, dim, kind, heads + page)
    seqs, cu = ints([3, 1, -1, 0, 6, 4, 2]), ints([0, 1, 2, 3, 4, 5, 6, 7])
    q = (randn(gen(1), 7, heads, dim) * 1.5).bfloat16()
    check_attention(c, q, seqs, cu, max_q=1, max_len=700)
    check_attention(c, q, seqs, cu)                                          # nothing known


@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_attention_of_ragged_tokens(heads, kv_heads, dim, kind):
    """Drafts, frames and prompts in one call, one that is its whole sequence, one request of no token, padding rows behind the last."""
    lens = [150, 36, 700, 300, 5, 129]
    counts = [2, 36, 131, 0, 5, 49]
    c = filled(lens, 32, heads, kv_heads, dim, kind, dim)
    cu = ints([0] + torch.tensor(counts).cumsum(0).tolist())
    q = (randn(gen(2), sum(counts) + 4, heads, dim) * 1.5).bfloat16()
    check_attention(c, q, ints(range(6)), cu, max_q=131, max_len=700)
    check_attention(c, q, ints(range(6)), cu)


@pytest.mark.parametrize("T", [1, 2, 3, 9, 40, 150])
@pytest.mark.parametrize("L", [1, 63, 64, 65, 128, 129, 1000])
def test_attention_lengths(T, L):
    """Every tile edge; more tokens than keys (the first rows see nothing and are zero)."""
    c = filled([L], 16, 14, 2, 64, "bf16", T * 1000 + L)
    q = randn(gen(3), T, 14, 64).bfloat16()
    check_attention(c, q, ints([0]), ints([0, T]), max_q=T, max_len=L)


@pytest.mark.parametrize("window", [1, 16, 63, 64, 100, 5000])
@pytest.mark.parametrize("T,heads,kv_heads,dim,kind", [(1, 8, 2, 64, "bf16"), (5, 7, 1, 128, "e4m3"), (90, 8, 2, 64, "bf16"), (150, 7, 1, 128, "bf16"), (49, 4, 2, 80, "e4m3")])
def test_attention_with_a_window(window, T, heads, kv_heads, dim, kind):
    """Keys before the window are gone: their pages are not even in the table."""
    lens = [1200, 260, T]
    c = filled(lens, 16, heads, kv_heads, dim, kind, window + T)
    for s, n in enumerate(lens):
        gone = max(0, n - T + 1 - window) // 16
        c.block_table[s, :gone] = -1
    q = randn(gen(4), 3 * T, heads, dim).bfloat16()
    check_attention(c, q, ints([0, 1, 2]), ints([0, T, 2 * T, 3 * T]), window=window, max_q=T, max_len=1200)


@pytest.mark.parametrize("T", [1, 4, 60])
def test_attention_hides_the_keys_of_entries_that_are_no_page(T):
    c = filled([300, 200], 16, 7, 1, 128, "bf16", 9)
    c.block_table[0, 3], c.block_table[0, 7], c.block_table[1, 0] = -1, c.n_pages, 2 ** 30
    q = randn(gen(6), 2 * T, 7, 128).bfloat16()
    check_attention(c, q, ints([0, 1]), ints([0, T, 2 * T]), max_q=T, max_len=300)


@pytest.mark.parametrize("T,heads,kv_heads,dim,kind", [(3, 7, 1, 128, "bf16"), (6, 4, 4, 64, "bf16"), (40, 7, 1, 128, "bf16"), (140, 8, 2, 64, "bf16"), (40, 7, 1, 128, "e4m3")])
@pytest.mark.parametrize("window", [0, 20])
def test_a_value_that_is_not_finite_stays_with_the_rows_that_see_it(T, heads, kv_heads, dim, kind, window):
    L = 200
    c = filled([L], 16, heads, kv_heads, dim, kind, 11)
    nan = 0x7f if kind == "e4m3" else 0x7fc0
    raw = c.v_pages.view(torch.uint8 if kind == "e4m3" else torch.int16)
    for j in (L - 2, L - T // 2 - 1):                                        # keys that the first of the new tokens do not see
        raw[0, int(c.block_table[0, j // 16]), 0, j % 16, 3] = nan
    q = randn(gen(7), T, heads, dim).bfloat16()
    got = check_attention(c, q, ints([0]), ints([0, T]), window=window, max_q=T, max_len=L)
    assert bool(torch.isnan(got[-1, 0, 3])) and not bool(torch.isnan(got[0].float()).any())


@pytest.mark.parametrize("dim", [80, 128])
@pytest.mark.parametrize("T", [1, 3, 40, 140])
def test_a_key_at_minus_infinity_weighs_nothing(T, dim):
    """As one at a score so low that its exponential is zero, bit for bit; also where the head is narrower than the kernel's tiles."""
    c = filled([300], 16, 4, 2, dim, "bf16", 13)
    q = randn(gen(14), T, 4, dim).bfloat16()
    q[..., dim - 1] = 1.0
    for j in (5, 100, 299 - T // 2):
        c.k_pages[0, int(c.block_table[0, j // 16]), :, j % 16, dim - 1] = -1e5
    seqs, cu = ints([0]), ints([0, T])
    want = check_attention(c, q, seqs, cu, max_q=T, max_len=300)
    c.k_pages[c.k_pages == c.k_pages.new_tensor(-1e5)] = float("-inf")
    assert bool(torch.isinf(c.k_pages).any())
    assert torch.equal(c.attention(0, q, seqs, cu, max_q=T, max_len=300), want)


@pytest.mark.parametrize("T", [1, 20])
def test_a_window_beyond_every_length_is_none(T):
    c = filled([5, 400], 16, 4, 2, 64, "bf16", 15)
    q = randn(gen(16), 2 * T, 4, 64).bfloat16()
    seqs, cu = ints([0, 1]), ints([0, T, 2 * T])                             # (more rows than the first has keys: they are zero)
    want = check_attention(c, q, seqs, cu, max_q=T)
    for window in (c.max_blocks * c.page_size, 2 ** 31 - 1, 2 ** 31, 2 ** 40 + 1):
        assert torch.equal(c.attention(0, q, seqs, cu, max_q=T, window=window), want)


def test_the_workspace_does_not_grow_with_the_tokens():
    import ctypes as C
    c = filled([100], 16, 28, 4, 128, "bf16", 25)
    need = []
    for tokens in (2048, 16384, 131072):
        b = C.c_size_t()
        c._chk(c.lib.aha_paged_attention_workspace(c.handle, 28, tokens, 1, tokens, 0, C.byref(b)))
        need.append(b.value)
    assert need[0] == need[1] == need[2]


def test_attention_scale_strides_and_sharp_rows():
    """Rows of a fused projection in, strided rows out; a query that puts all its weight on one key returns that key's value."""
    c = filled([500], 64, 14, 2, 128, "bf16", 21, rubbish=False)
    g = gen(22)
    qkv = randn(g, 3, 18 * 128).bfloat16()
    keys, values = c.export_kv(0, 0), c.export_kv(0, 0, True)
    qkv.view(3, 18, 128)[2, 0] = keys[0, 257] * 8
    buf = torch.zeros((3, 20 * 128), dtype=torch.bfloat16, device=DEV)
    q = qkv[:, :14 * 128]
    got = c.attention(0, q, ints([0]), ints([0, 3]), scale=0.5, max_q=3, out=buf[:, 128:15 * 128]).view(3, 14, 128)
    want, mag, size = attention64(c, q.reshape(3, 14, 128), ints([0]), ints([0, 3]), scale=0.5)
    close(got, want, U * want.abs() + slack(128, size, True) * mag, "strided")
    assert torch.equal(got[2, 0], values[0, 257])
    assert not bool(buf[:, :128].any()) and not bool(buf[:, 15 * 128:].any())


@pytest.mark.parametrize("hints", [dict(max_q=1, max_len=1), dict(max_q=1), dict(max_len=16), dict(max_q=2, max_len=100), dict(max_q=10 ** 6, max_len=10 ** 9)])
def test_wrong_hints_cost_time_not_results(hints):
    lens, counts = [700, 90, 1500], [131, 1, 9]
    c = filled(lens, 16, 28, 4, 128, "bf16", 17)
    cu = ints([0, 131, 132, 141])
    check_attention(c, randn(gen(18), 141, 28, 128).bfloat16(), ints(range(3)), cu, **hints)


@pytest.mark.parametrize("T", [1, 6, 60])
def test_attention_in_place_and_twice_over_one_sequence(T):
    """out is q; the same sequence listed twice (each time its last tokens are meant)."""
    c = filled([900, 33], 32, 14, 2, 64, "bf16", 19)
    q = randn(gen(20), 2 * T + 1, 14, 64).bfloat16()
    seqs, cu = ints([0, 1, 0]), ints([0, T, T + 1, 2 * T + 1])
    want = check_attention(c, q, seqs, cu, max_q=T)
    got = q.clone()
    assert c.attention(0, got, seqs, cu, max_q=T, out=got) is got
    assert torch.equal(got, want)


def test_a_workspace_that_is_too_small_is_refused():
    import ctypes as C
    c = filled([4000], 16, 28, 4, 128, "bf16", 23)
    q = randn(gen(24), 1, 28, 128).bfloat16()
    need = C.c_size_t()
    c._chk(c.lib.aha_paged_attention_workspace(c.handle, 28, 1, 1, 1, 4000, C.byref(need)))
    assert need.value > 0
    ws = torch.empty(need.value, dtype=torch.uint8, device=DEV)

    def call(p, size):
        s, cu, out = ints([0]), ints([0, 1]), torch.empty_like(q)
        rc = c.lib.aha_paged_attention(c.handle, 0, q.data_ptr(), 28 * 128, 28, s.data_ptr(), cu.data_ptr(), 1, 1, 1, 4000, 0, 0.1, out.data_ptr(), 28 * 128, p, size, c._stream())
        torch.cuda.synchronize()
        return rc

    assert call(ws.data_ptr(), need.value - 1) == -34 and call(None, need.value) == -34 and call(ws.data_ptr() + 4, need.value) == -22
    assert call(ws.data_ptr(), need.value) == 0


def test_many_requests():
    """More requests than a workgroup has threads: the split is worked out over several rounds."""
    rng = random.Random(3)
    n = 700
    lens = [rng.choice((0, 1, rng.randint(1, 90))) for _ in range(n)]
    lens[650] = 3000
    c = filled(lens, 16, 4, 2, 64, "bf16", 31)
    counts = [rng.choice((1, 1, 1, 0, 3)) for _ in range(n)]
    order = rng.sample(range(n), n)
    cu = ints([0] + torch.tensor(counts).cumsum(0).tolist())
    q = randn(gen(32), sum(counts), 4, 64).bfloat16()
    check_attention(c, q, ints(order), cu, max_q=3, max_len=3000)


@pytest.mark.parametrize("n,T", [(100, 1), (100, 20), (300, 1), (300, 40)])
def test_many_requests_of_which_some_are_cut(n, T):
    """Short requests between long ones: the partial results of the cut ones lie one behind the other."""
    lens = [40 + i % 7 for i in range(n)]
    for i in (0, 63, 64, n // 2, n - 1):
        lens[i] = 5000 + 777 * (i % 3)
    c = filled(lens, 64, 4, 2, 64, "bf16", 33)
    q = randn(gen(34), n * T, 4, 64).bfloat16()
    got = check_attention(c, q, ints(range(n)), ints(range(0, n * T + 1, T)), max_q=T)
    assert torch.equal(c.attention(0, q, ints(range(n)), ints(range(0, n * T + 1, T)), max_q=T), got)


def test_one_token_over_as_many_chunks_as_workgroups():
    c = filled([80000], 128, 8, 1, 64, "bf16", 35)
    check_attention(c, randn(gen(36), 1, 8, 64).bfloat16(), ints([0]), ints([0, 1]), max_q=1)
    check_attention(c, randn(gen(37), 3, 8, 64).bfloat16(), ints([0]), ints([0, 3]), max_q=3)


@pytest.mark.parametrize("T,L,kind", [(1, 30001, "bf16"), (1, 20000, "e4m3"), (5, 9000, "bf16"), (36, 6000, "bf16"), (700, 1500, "e4m3")])
def test_long_sequences_and_the_same_bits_twice(T, L, kind):
    c = filled([L, 40], 64, 28, 4, 128, kind, L)
    n = T + 1
    q = randn(gen(41), n, 28, 128).bfloat16()
    got = check_attention(c, q, ints([0, 1]), ints([0, T, n]), max_q=T, max_len=L)
    for _ in range(3):
        assert torch.equal(c.attention(0, q, ints([0, 1]), ints([0, T, n]), max_q=T, max_len=L), got)


def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 bytes (and 2^31 elements) each for K and V; sequences on its last pages."""
    pages, page, hk, d = 70000, 64, 4, 128
    c = pool(pages, page, 2, 8, hk, d)
    g = gen(51)
    c.n_free.fill_(pages)
    c.free_pages.copy_(torch.arange(pages, dtype=torch.int32))               # taken from the end: the last pages first
    seqs = ints([0, 1])
    slots, positions, cu, status = c.reserve(seqs, ints([200, 77]), 277)
    c.check(status)
    assert int(slots.min()) * hk * d > 2 ** 31
    q, k, v = randn(g, 277, 8, d).bfloat16(), randn(g, 277, hk, d).bfloat16(), randn(g, 277, hk, d).bfloat16()
    c.append(0, q, k, v, slots, positions)
    assert torch.equal(c.export_kv(0, 0), k[:200].transpose(0, 1)) and torch.equal(c.export_kv(0, 1, True), v[200:].transpose(0, 1))
    check_attention(c, q, seqs, cu, max_q=200, max_len=200)
    check_attention(c, q[:2], seqs, ints([0, 1, 2]), max_q=1, max_len=200)


# ---- together -----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_a_server_steps_admits_drafts_and_releases(kind):
    """Prompts admitted, frames and tokens appended, drafts rejected, a request released and its pages taken by the next: the attention of
    every step against an evaluation of all that the sequences hold, kept aside in full."""
    heads, kv_heads, dim, layers = 14, 2, 64, 2
    cos, sin = (t.to(DEV) for t in rope_table(2048, dim, 1e6))
    dtype = torch.bfloat16 if kind == "bf16" else torch.float8_e4m3fn
    scales = {} if kind == "bf16" else dict(k_scale=torch.full((layers, kv_heads), 0.02, device=DEV), v_scale=torch.full((layers, kv_heads), 0.02, device=DEV))
    c = pool(24, 32, 4, 16, kv_heads, dim, layers=layers, dtype=dtype, rope=(cos, sin), **scales)
    c.k_pages.view(torch.uint8).fill_(0x7f)
    c.v_pages.view(torch.uint8).fill_(0x7f)
    held = [[[], []] for _ in range(4)]                                      # per sequence and layer: the new tokens' (k, v) as given
    g = gen(61)
    steps = [([0, 1], [70, 5]), ([2, 0], [36, 1]), ([0, 1, 2], [1, 1, 1]), ([1, 0], [8, 4])]
    drop = {3: ([1, 0], [4, 4])}                                             # rejected drafts
    for n, (seqs, counts) in enumerate(steps + [([3, 0, 1], [300, 36, 1])]):
        if n == 4:
            c.check(c.truncate(ints([2]), ints([0])))                        # released
            held[2] = [[], []]
        total = sum(counts)
        slots, positions, cu, status = c.reserve(ints(seqs), ints(counts), total)
        c.check(status)
        for layer in range(layers):
            qkv = randn(g, total, (heads + 2 * kv_heads) * dim).bfloat16()
            q, k, v = qkv.split((heads * dim, kv_heads * dim, kv_heads * dim), -1)
            qr = c.append(layer, q, k, v, slots, positions)
            got = c.attention(layer, qr, ints(seqs), cu, max_q=max(counts))
            want, mag, size = attention64(c, qr, ints(seqs), cu, layer=layer)
            close(got, want, U * want.abs() + slack(dim, size, True) * mag, (n, layer))
            at = 0
            for s, k_ in zip(seqs, counts):
                held[s][layer].append((k[at:at + k_], v[at:at + k_]))
                at += k_
        if n in drop:
            back = [int(c.lens[s]) - r for s, r in zip(*drop[n])]
            c.check(c.truncate(ints(drop[n][0]), ints(back)))
            for s, r in zip(*drop[n]):
                for layer in range(layers):
                    k, v = held[s][layer].pop()
                    if r < len(k):
                        held[s][layer].append((k[:-r], v[:-r]))
    assert c.lens.tolist() == [sum(len(k) for k, _ in h[0]) for h in held]
    for s in range(4):
        for layer in range(layers):
            if held[s][layer]:
                k, v = (torch.cat(x).reshape(-1, kv_heads, dim).transpose(0, 1).double() for x in zip(*held[s][layer]))
                n = k.shape[1]
                cc, ss = cos[:n].double(), sin[:n].double()
                k = k * cc + torch.cat((-k[..., dim // 2:], k[..., :dim // 2]), -1) * ss
                rel, least = (U, 2.0 ** -20) if kind == "bf16" else (2.0 ** -4 * (1 + 2.0 ** -18), 0.02 * 2.0 ** -10 + 2.0 ** -20)
                close(c.export_kv(layer, s), k, rel * k.abs() + least, ("k", s))
                close(c.export_kv(layer, s, True), v, rel * v.abs() + least, ("v", s))
    c.check(c.truncate(ints([0, 1, 2, 3]), ints([0] * 4)))
    assert int(c.n_free) == 24 and sorted(c.free_pages.tolist()) == list(range(24))


def test_the_pages_give_what_the_ring_gives():
    """The same rotated keys, values and queries through a stream's ring (aha_cache_update, aha_attention_forward) and through pages."""
    from aha_amd.config import preset
    from aha_amd.runtime import Runtime
    from aha_amd.synth import make_weights
    cfg = preset("tiny128")
    rt = Runtime(cfg, make_weights(cfg, dtype=torch.bfloat16), max_step_tokens=64, max_vit_frames=1, max_positions=1024)
    c = rt.open_paged(40, 2, page_size=16)
    assert (c.layers, c.kv_heads, c.head_dim, c.max_blocks) == (2, 1, 128, 64) and c.cos.shape == (1024, 128)
    c.cos = c.sin = None
    c._rope = (None, None, 0)                                                # the keys come rotated
    st = rt.open_stream(None, capacity=600)
    g = gen(71)
    for T in (36, 1, 36, 20, 1):
        slots, positions, cu, status = c.reserve(ints([1]), ints([T]), T)
        c.check(status)
        for layer in range(2):
            k, v, q = randn(g, 1, T, 128).bfloat16(), randn(g, 1, T, 128).bfloat16(), randn(g, T, 7, 128).bfloat16()
            kr, vr = rt.cache_update(st, layer, k[None], v[None])
            c.append(layer, None, k[0], v[0], slots)
            assert torch.equal(c.export_kv(layer, 1), kr[0]) and torch.equal(c.export_kv(layer, 1, True), vr[0])
            ring = rt.attention([st], q.reshape(1, T, -1), layer).view(T, 7, 128)
            got = c.attention(layer, q, ints([1]), cu, max_q=T)
            want, mag, size = attention64(c, q, ints([1]), cu, layer=layer)
            bound = U * want.abs() + slack(128, size, True) * mag
            close(got, want, bound, "paged")
            close(ring, want, bound, "ring")
    st.close()
    c.close()
    rt.close()


def test_steps_in_a_graph():
    """A step's calls captured once and replayed: the lengths live on the device, so every replay is the next step.  Two graphs of the same pool
    with workspaces of their own, eager work and synchronizations between the replays."""
    heads, kv_heads, dim = 28, 4, 128
    cos, sin = (t.to(DEV) for t in rope_table(4096, dim, 1e6))
    made = []
    for _ in range(2):                                                       # one for the graphs, one stepped eagerly
        c = pool(200, 16, 3, 64, kv_heads, dim, rope=(cos, sin))
        g = gen(81)
        first = c.reserve(ints([0, 1, 2]), ints([500, 3, 170]), 673)
        c.check(first[3])
        kv = randn(g, 673, 2, kv_heads * dim).bfloat16()
        c.append(0, None, kv[:, 0], kv[:, 1], first[0], first[1])
        made.append(c)
    c, e = made
    seqs = ints([2, 0, -1, 1])
    counts = {"token": ints([1, 1, 0, 1]), "frame": ints([36, 2, 0, 36])}
    rooms = {"token": 4, "frame": 76}
    x = {k: torch.zeros((n, 36 * dim), dtype=torch.bfloat16, device=DEV) for k, n in rooms.items()}
    outs = {k: torch.zeros((n, heads, dim), dtype=torch.bfloat16, device=DEV) for k, n in rooms.items()}

    def step(cache, kind, out):
        slots, positions, cu, status = cache.reserve(seqs, counts[kind], rooms[kind])
        q, k, v = x[kind].split((heads * dim, kv_heads * dim, kv_heads * dim), -1)
        q = cache.append(0, q, k, v, slots, positions)
        return cache.attention(0, q, seqs, cu, max_q=36 if kind == "frame" else 1, max_len=1024, out=out), status

    graphs, status = {}, {}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for kind in rooms:
            graphs[kind] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graphs[kind], stream=side):
                _, status[kind] = step(c, kind, outs[kind])
    torch.cuda.current_stream().wait_stream(side)
    for n, kind in enumerate(("token", "frame", "token", "token", "frame", "token")):
        x[kind].copy_(randn(gen(90 + n), *x[kind].shape))
        graphs[kind].replay()
        want, st = step(e, kind, torch.zeros_like(outs[kind]))
        assert status[kind].tolist() == [0, 0] and st.tolist() == [0, 0]
        assert torch.equal(outs[kind], want), (n, kind)
        assert torch.equal(c.lens, e.lens) and torch.equal(c.block_table, e.block_table)
        assert torch.equal(c.export_kv(0, 1), e.export_kv(0, 1))


def test_two_streams_at_once():
    """Calls on two streams that run at the same time share nothing but the pool they read."""
    c = filled([5000, 4000, 300], 64, 28, 4, 128, "bf16", 91)
    qa, qb = randn(gen(92), 2, 28, 128).bfloat16(), randn(gen(93), 90, 28, 128).bfloat16()
    a, b = (ints([0, 1]), ints([0, 1, 2])), (ints([2, 1]), ints([0, 50, 90]))
    want = c.attention(0, qa, *a, max_q=1), c.attention(0, qb, *b, max_q=50)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(s1):
            g1 = c.attention(0, qa, *a, max_q=1)
        with torch.cuda.stream(s2):
            g2 = c.attention(0, qb, *b, max_q=50)
        torch.cuda.synchronize()
        assert torch.equal(g1, want[0]) and torch.equal(g2, want[1])

"""Table entries that are no page (callers may drop the pages before a window, and attention hides the keys of such entries): they are given back
to nobody when their sequence is cut or released, and no new token is sent to one.  Whole numbers, equal to a bookkeeping in Python."""
import random

import pytest
import torch

import aha_amd  # noqa: F401
from aha_amd.runtime import AhaError
from test_gpu_paged import filled, ints, pool, state

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,blocks,share", [(1, 3, 0.5), (1, 3, 1.0), (5, 400, 0.3), (70, 9, 0.5), (300, 30, 0.02), (1300, 4, 0.5), (2100, 3, 1.0)])
def test_a_truncate_passes_over_entries_that_are_no_page(n, blocks, share):
    """`share` of the entries are -1 or lie outside the pool; requests on both sides of a workgroup's threads, entries too."""
    rng = random.Random(n * 100 + blocks)
    c = pool(n * blocks + 7, 16, n + 2, blocks)
    seqs = rng.sample(range(n + 2), n)
    lens = [rng.randint(1, blocks * 16) for _ in seqs]
    c.check(c.reserve(ints(seqs), ints(lens), sum(lens))[3])
    table, free = c.block_table.tolist(), c.free_pages[:int(c.n_free)].tolist()
    for s, length in zip(seqs, lens):
        for b in range(-(-length // 16)):
            if rng.random() < share:
                table[s][b] = rng.choice((-1, c.n_pages, 2 ** 30, -2 ** 31))
    c.block_table.copy_(torch.tensor(table, dtype=torch.int32))
    order = rng.sample(range(n), n)
    cut = [rng.choice((0, 0, rng.randint(0, lens[i]))) for i in order]
    assert c.truncate(ints(seqs[i] for i in order), ints(cut)).tolist() == [0, 0]
    back = []
    for i, keep in zip(order, cut):
        for b in range(-(-keep // 16), -(-lens[i] // 16)):
            if 0 <= table[seqs[i]][b] < c.n_pages:
                back.append(table[seqs[i]][b])
            table[seqs[i]][b] = -1
    free += back[::-1]
    assert int(c.n_free) == len(free) and c.free_pages[:len(free)].tolist() == free
    assert c.block_table.tolist() == table
    want = c.lens.tolist()
    assert [want[seqs[i]] for i in order] == cut


def test_a_released_window_leaves_pages_that_can_be_taken():
    """A sequence whose pages before the window were dropped (and handed back by its owner) is released; the next one gets its other pages and no -1."""
    c = pool(6, 16, 2, 6)
    c.check(c.reserve(ints([0]), ints([96]), 96)[3])
    gone = c.block_table[0, :4].clone()
    c.block_table[0, :4] = -1
    c.free_pages[:4] = gone                                                  # its owner puts them on the list, which was empty
    c.n_free.fill_(4)
    assert c.truncate(ints([0]), ints([0])).tolist() == [0, 0]
    assert int(c.n_free) == 6 and sorted(c.free_pages.tolist()) == list(range(6))
    slots, positions, cu, status = c.reserve(ints([1]), ints([96]), 96)
    assert status.tolist() == [0, 0] and sorted(slots.tolist()) == list(range(96))


def test_more_pages_than_the_pool_has_are_still_refused():
    c = filled([96, 40], 16, 1, 1, 16, "bf16", 3, spare=0)
    c.n_free.fill_(1)                                                        # a list that claims a page that a table holds
    c.block_table[0, 0] = -1
    assert c.truncate(ints([0, 1]), ints([0, 0])).tolist() == [0, 0]         # eight pages and one claimed: the missing entry makes room
    c = filled([96, 40], 16, 1, 1, 16, "bf16", 3, spare=0)
    c.n_free.fill_(1)
    before = state(c)
    assert c.truncate(ints([0, 1]), ints([0, 0])).tolist() == [4, 0]
    assert all(torch.equal(a, b) for a, b in zip(before, state(c)))


@pytest.mark.parametrize("pages,at", [(1, 0), (9, 8), (300, 299), (300, 0), (2500, 1024), (2500, 2499), (5000, 4100)])
@pytest.mark.parametrize("entry", [-1, "n_pages", 2 ** 30])
def test_a_reserve_does_not_hand_out_an_entry_that_is_no_page(pages, at, entry):
    """`at`: how far from the list's end the entry lies, up to the last page that is asked for; one page less is done."""
    c = pool(pages + 3, 16, 4, pages)
    c.free_pages[c.n_pages - 1 - at] = c.n_pages if entry == "n_pages" else entry
    before = state(c)
    room = pages * 16
    slots, positions, cu, status = c.reserve(ints([1, 2]), ints([(pages - 1) * 16, 5]), room)
    assert status.tolist() == [64, 0] and cu.tolist() == [0, 0, 0]
    assert bool((slots == -1).all()) and bool((positions == -1).all())
    assert all(torch.equal(a, b) for a, b in zip(before, state(c)))
    with pytest.raises(AhaError, match="free list"):
        c.check(status)
    if at:
        slots, positions, cu, status = c.reserve(ints([1, 2]), ints([at * 16 - 3, 0]), at * 16)
        assert status.tolist() == [0, 0]
        want = range(at)                                                     # page 0 is at the end of the list
        assert slots.tolist() == [p * 16 + k for p in want for k in range(16)][:at * 16 - 3] + [-1] * 3


@pytest.mark.parametrize("n", [1, 70, 1300])
@pytest.mark.parametrize("entry", [-1, 2 ** 30])
def test_a_reserve_does_not_fill_an_entry_that_is_no_page(n, entry):
    """The page that a sequence's next token goes to was dropped: refused.  No token, or one at a page's border, does not need it."""
    c = pool(3 * n, 16, n, 4)
    lens = [20] * n
    lens[n // 2] = 32
    c.check(c.reserve(ints(range(n)), ints(lens), sum(lens))[3])
    c.block_table[:, 0] = -1                                                 # before a window: no token goes there
    c.block_table[n // 2, 1] = entry                                         # full
    c.check(c.reserve(ints(range(n)), ints([1] * n), n)[3])
    s = n - 1
    c.block_table[s, 2 if s == n // 2 else 1] = entry
    before = state(c)
    slots, positions, cu, status = c.reserve(ints(range(n)), ints([1] * n), n)
    assert status.tolist() == [64, 0] and bool((slots == -1).all()) and not bool(cu.any())
    assert all(torch.equal(a, b) for a, b in zip(before, state(c)))
    counts = [1] * n
    counts[s] = 0
    c.check(c.reserve(ints(range(n)), ints(counts), n)[3])

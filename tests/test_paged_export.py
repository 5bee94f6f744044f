"""What a look at a sequence of the paged key-value cache gives, on the CPU: its keys from its pages, zeros for entries that are no page."""
import pytest
import torch

import aha_amd  # noqa: F401
from aha_amd.paged import PagedKVCache
from aha_amd.runtime import AhaError


def small(kind):
    dtype = torch.bfloat16 if kind == "bf16" else torch.float8_e4m3fn
    more = {} if kind == "bf16" else dict(k_scale=torch.tensor([[0.5, 2.0], [1.0, 3.0]]))
    c = PagedKVCache(5, 16, 2, 32, 3, 4, layers=2, dtype=dtype, device="cpu", **more)
    g = torch.Generator().manual_seed(1)
    for p in (c.k_pages, c.v_pages):
        p.copy_(torch.randn(p.shape, generator=g).to(dtype))
    c.block_table[1] = torch.tensor([4, 0, 3, -1])
    c.lens[1] = 41
    return c


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("entry", [None, -1, 5, 2 ** 30, -2 ** 31])
@pytest.mark.parametrize("block", [0, 1, 2])
def test_the_keys_of_a_sequence(kind, entry, block):
    c = small(kind)
    want = torch.zeros(2, 41, 32)
    for j in range(41):
        if entry is None or j // 16 != block:
            want[:, j] = c.k_pages[1, int(c.block_table[1, j // 16]), :, j % 16].float()
    if kind == "e4m3":
        want *= c.k_scale[1][:, None, None]
    if entry is not None:
        c.block_table[1, block] = entry
    got = c.export_kv(1, 1)
    assert got.dtype == (torch.bfloat16 if kind == "bf16" else torch.float32) and torch.equal(got.float(), want)


def test_an_empty_sequence_and_what_is_none():
    c = small("bf16")
    assert c.export_kv(0, 0).shape == (2, 0, 32) and c.export_kv(0, 2, True).shape == (2, 0, 32)
    for layer, seq in ((-1, 1), (2, 1), (0, -1), (0, 3)):
        with pytest.raises(ValueError, match="out of range"):
            c.export_kv(layer, seq)
    for length in (-1, 65, 2 ** 31 - 1):
        c.lens[1] = length
        with pytest.raises(AhaError, match="corrupt length"):
            c.export_kv(0, 1)

"""Numbers that do not fit the library's 32-bit arguments are refused, or mean what they say: the bits above are never cut off.  On the CPU: the
checks are made before anything is enqueued."""
import pytest
import torch

import aha_amd  # noqa: F401
from aha_amd.paged import PagedKVCache
from aha_amd.runtime import AhaError

WIDE = (2 ** 32, 2 ** 31, 2 ** 64, -2 ** 32, -2 ** 40)


@pytest.fixture
def c(monkeypatch):
    monkeypatch.setattr(PagedKVCache, "_stream", lambda self: 0)
    return PagedKVCache(8, 16, 2, 32, 4, 4, device="cpu")


class NoneNeeded(dict):
    def get(self, key):
        return 0


@pytest.mark.parametrize("layer", WIDE)
def test_a_layer(c, layer):
    kv, q = torch.zeros((3, 2, 32), dtype=torch.bfloat16), torch.zeros((3, 4, 32), dtype=torch.bfloat16)
    ints = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(AhaError, match="layer out of range"):
        c.append(layer, q, kv, kv, ints)
    c._workspace = NoneNeeded()
    with pytest.raises(AhaError, match="layer out of range"):
        c.attention(layer, q, ints[:2], ints)


@pytest.mark.parametrize("low", [-1, -2 ** 31, -2 ** 32, -2 ** 32 + 5, -2 ** 64 + 5])
@pytest.mark.parametrize("name", ["window", "max_q", "max_len"])
def test_a_window_and_hints(c, name, low):
    q, ints = torch.zeros((3, 4, 32), dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    c._workspace = NoneNeeded()
    with pytest.raises(AhaError, match="negative"):
        c.attention(0, q, ints[:2], ints, **{name: low})


@pytest.mark.parametrize("tokens", [2 ** 31, 2 ** 31 - 4096, 2 ** 32, 2 ** 32 + 4, 2 ** 64])
def test_tokens_of_a_reserve(c, tokens):
    ints = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="n_tokens"):                        # before the slots are allocated
        c.reserve(ints, ints, tokens)


@pytest.mark.parametrize("name", ["n_pages", "page_size", "kv_heads", "head_dim", "max_seqs", "max_blocks", "layers"])
def test_a_pools_sizes(name):
    sizes = dict(n_pages=8, page_size=16, kv_heads=2, head_dim=32, max_seqs=4, max_blocks=4, layers=1)
    for wide in (2 ** 31, 2 ** 32 + sizes[name]):
        with pytest.raises(ValueError, match="2\\^31"):                      # before anything is allocated
            PagedKVCache(device="cpu", **{**sizes, name: wide})

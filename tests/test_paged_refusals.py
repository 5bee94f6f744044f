"""What the paged key-value cache refuses, on the CPU: every check is made before anything is enqueued, so none of this needs a GPU."""
import ctypes as C

import pytest
import torch

import aha_amd  # noqa: F401
from aha_amd import lib as L
from aha_amd.paged import PagedKVCache
from aha_amd.runtime import AhaError


def make(**kw):
    a = dict(n_pages=8, page_size=16, kv_heads=2, head_dim=32, max_seqs=4, max_blocks=4, device="cpu")
    a.update(kw)
    return PagedKVCache(**a)


@pytest.mark.parametrize("bad", [dict(n_pages=0), dict(page_size=8), dict(page_size=48), dict(page_size=2048), dict(kv_heads=0), dict(kv_heads=2000),
                                 dict(head_dim=24), dict(head_dim=144), dict(max_seqs=0), dict(max_seqs=70000), dict(max_blocks=0), dict(layers=0),
                                 dict(dtype=torch.float16), dict(max_blocks=1 << 28), dict(k_scale=torch.ones(1, 2)), dict(k_pages=torch.zeros(3)),
                                 dict(lens=torch.zeros(4)), dict(block_table=torch.zeros((4, 5), dtype=torch.int32)), dict(free_pages=torch.zeros(8, dtype=torch.int32)),
                                 dict(dtype=torch.float8_e4m3fn, v_scale=torch.ones(2, 2)), dict(rope=(torch.zeros(9, 32), torch.zeros(9, 32))),
                                 dict(rope=(torch.zeros((9, 32), dtype=torch.bfloat16), torch.zeros((8, 32), dtype=torch.bfloat16)))])
def test_a_pool_that_is_none(bad):
    if bad.get("max_blocks") == 1 << 28:                                     # too long a sequence; its table is not made
        d = L.PagedDesc(*([16] * 6 + [None] * 2), 1, 8, 16, 2, 32, 0, 4, 1 << 28)
        h = C.c_void_p()
        assert L.get().aha_paged_create(C.byref(d), 0, C.byref(h)) == -34 and b"tokens" in L.get().aha_paged_last_error()
        return
    with pytest.raises((ValueError, AhaError)):
        make(**bad)


def test_a_pool_of_more_slots_than_an_index_holds():
    d = L.PagedDesc(*([16] * 6 + [None] * 2), 1, 1 << 27, 16, 2, 32, 0, 4, 4)
    h = C.c_void_p()
    assert L.get().aha_paged_create(C.byref(d), 0, C.byref(h)) == -34 and b"slots" in L.get().aha_paged_last_error()
    d.n_pages, d.k_pages = 8, 24
    assert L.get().aha_paged_create(C.byref(d), 0, C.byref(h)) == -22 and b"aligned" in L.get().aha_paged_last_error()
    d.k_pages, d.kv_type = 16, 2
    assert L.get().aha_paged_create(C.byref(d), 0, C.byref(h)) == -22
    assert L.get().aha_paged_create(None, 0, C.byref(h)) == -22 and L.get().aha_paged_create(C.byref(d), -1, C.byref(h)) == -22


I = torch.int32                                                              # noqa: E741


def test_tables_refuse_what_is_not_theirs(monkeypatch):
    c = make()
    monkeypatch.setattr(PagedKVCache, "_stream", lambda self: 0)
    seqs, counts = torch.zeros(2, dtype=I), torch.ones(2, dtype=I)
    for args in ((seqs.long(), counts, 4), (seqs, counts.float(), 4), (seqs, counts[:1], 4), (seqs[:, None], counts, 4), (seqs, counts, -1),
                 (torch.zeros(4, dtype=I)[::2], counts, 4)):
        with pytest.raises(ValueError):
            c.reserve(*args)
    with pytest.raises(ValueError):
        c.truncate(seqs, counts[:1])
    with pytest.raises(AhaError):
        c.reserve(torch.zeros(200000, dtype=I), torch.zeros(200000, dtype=I), 1)
    lib, p = c.lib, seqs.data_ptr()
    assert lib.aha_paged_reserve(None, p, p, 2, p, p, 4, p, p, None) == -22
    assert lib.aha_paged_reserve(c.handle, None, p, 2, p, p, 4, p, p, None) == -22
    assert lib.aha_paged_reserve(c.handle, p, p, 2, None, p, 4, p, p, None) == -22
    assert lib.aha_paged_reserve(c.handle, p, p, -1, p, p, 4, p, p, None) == -22
    assert lib.aha_paged_reserve(c.handle, p, p, 2, p, p, 4, None, p, None) == -22
    assert lib.aha_paged_truncate(c.handle, p, None, 2, p, None) == -22 and lib.aha_paged_truncate(c.handle, p, p, 2, None, None) == -22


def test_append_refuses(monkeypatch):
    monkeypatch.setattr(PagedKVCache, "_stream", lambda self: 0)
    rope = tuple(torch.zeros((64, 32), dtype=torch.bfloat16) for _ in range(2))
    c = make(rope=rope)
    kv = torch.zeros((3, 2, 32), dtype=torch.bfloat16)
    q = torch.zeros((3, 4, 32), dtype=torch.bfloat16)
    s = torch.zeros(3, dtype=I)
    for args, kw in (((0, q.float(), kv, kv, s, s), {}), ((0, q, kv[:, :1], kv, s, s), {}), ((0, q, kv, kv[:2], s, s), {}), ((0, q[:2], kv, kv, s, s), {}),
                     ((0, q, kv, kv, s[:2], s), {}), ((0, q, kv, kv, s, s.long()), {}), ((0, q, kv, kv, s), {}), ((0, q[..., :24], kv, kv, s, s), {}),
                     ((0, q, kv, kv, s, s), dict(q_out=q[:, :2])), ((0, q, kv, kv, s, s), dict(q_out=q[:2])),
                     ((0, q, kv, kv, s, s), dict(q_out=torch.zeros((3, 4, 64), dtype=torch.bfloat16)[..., ::2]))):
        with pytest.raises(ValueError):
            c.append(*args, **kw)
    for layer in (-1, 1):
        with pytest.raises(AhaError, match="layer"):
            c.append(layer, q, kv, kv, s, s)
    wide = torch.zeros((3, 132), dtype=torch.bfloat16)
    with pytest.raises(AhaError, match="multiples of 8"):
        c.append(0, wide[:, :128], kv, kv, s, s)
    wide = torch.zeros((3, 136), dtype=torch.bfloat16)
    with pytest.raises(AhaError, match="aligned"):
        c.append(0, wide[:, 4:132], kv, kv, s, s)
    p = kv.data_ptr()
    call = c.lib.aha_paged_append
    assert call(None, 0, p, 128, 4, p, 128, p, 64, p, 64, p, p, 3, None, None, 0, None) == -22
    assert call(c.handle, 0, p, 128, 4, p, 128, None, 64, p, 64, p, p, 3, None, None, 0, None) == -22
    assert call(c.handle, 0, p, 64, 4, p, 128, p, 64, p, 64, p, p, 3, None, None, 0, None) == -34          # a stride shorter than its row
    assert call(c.handle, 0, p, 128, 4, p, 136, p, 64, p, 64, p, p, 3, None, None, 0, None) == -22         # in place with two strides
    assert call(c.handle, 0, p, 128, 4, p, 128, p, 64, p, 64, p, p, 3, p, None, 9, None) == -22            # cos without sin
    assert call(c.handle, 0, p, 128, 4, p, 128, p, 64, p, 64, p, None, 3, p, p, 9, None) == -22            # rotation without positions
    assert call(c.handle, 0, p, 128, 4, p, 128, p, 64, p, 64, p, p, -1, None, None, 0, None) == -22
    assert call(c.handle, 0, None, 0, 0, None, 0, None, 0, None, 0, None, None, 0, None, None, 0, None) == 0   # no token: nothing to do


def test_attention_refuses(monkeypatch):
    monkeypatch.setattr(PagedKVCache, "_stream", lambda self: 0)
    c = make()
    q = torch.zeros((3, 4, 32), dtype=torch.bfloat16)
    seqs, cu = torch.zeros(2, dtype=I), torch.zeros(3, dtype=I)
    for args, kw in (((0, q.float(), seqs, cu), {}), ((0, q, seqs, cu[:2]), {}), ((0, q, seqs.long(), cu), {}), ((0, q, seqs, cu.float()), {}),
                     ((0, q, seqs, cu), dict(out=q[:2])), ((0, q, seqs, cu), dict(out=q[:, :2])), ((0, q, seqs, cu), dict(out=q.float()))):
        with pytest.raises(ValueError):
            c.attention(*args, **kw)
    with pytest.raises(AhaError, match="multiple of the cache"):
        c.attention(0, q[:, :3].contiguous(), seqs, cu)
    for kw in (dict(max_q=-1), dict(max_len=-1)):
        with pytest.raises(AhaError, match="negative"):
            c.attention(0, q, seqs, cu, **kw)
    p, b = q.data_ptr(), C.c_size_t()
    call = c.lib.aha_paged_attention

    def attend(layer=0, q=p, ldq=128, heads=4, seqs=p, cu=p, n=2, N=3, window=0, scale=0.1, out=p, ldo=128, ws=None, size=0):
        return call(c.handle, layer, q, ldq, heads, seqs, cu, n, N, 1, 16, window, scale, out, ldo, ws, size, None)

    assert call(None, 0, p, 128, 4, p, p, 2, 3, 1, 16, 0, 0.1, p, 128, None, 0, None) == -22
    assert attend(layer=1) == -34 and attend(layer=-1) == -34
    assert attend(window=-1) == -22
    for s in (0.0, -1.0, float("inf"), float("nan")):
        assert attend(scale=s) == -22
    assert attend(heads=0) == -34 and attend(heads=6, ldq=192, ldo=192, N=1 << 24) == -34
    assert c.lib.aha_paged_attention_workspace(c.handle, 4, 3, -1, 1, 1, C.byref(b)) == -22
    assert c.lib.aha_paged_attention_workspace(c.handle, 4, 3, 2, 1, 1, None) == -22


def test_outputs_that_overlap_inputs_are_refused(monkeypatch):
    """In place is fine, and so are columns of one buffer; anything else that shares an element is not."""
    monkeypatch.setattr(PagedKVCache, "_stream", lambda self: 0)
    c = make()
    buf = torch.zeros((8, 256), dtype=torch.bfloat16)
    q, k, v, s = buf[:3, :128], buf[:3, 128:192], buf[:3, 192:], torch.zeros(3, dtype=I)
    call, lib, p = c.lib.aha_paged_attention, c.lib, s.data_ptr()

    def attend(out):
        return call(c.handle, 0, q.data_ptr(), 256, 4, p, p, 1, 3, 1, 16, 0, 0.1, out.data_ptr(), out.stride(0), p, 0, None)

    flat = buf.view(-1)
    for out in (buf[1:4, :128], buf[:3, 64:192], buf[:3, 8:136], flat[:3 * 128].view(3, 128), flat[256:256 + 3 * 128].view(3, 128)):
        with pytest.raises(AhaError, match="overlaps"):
            c.append(0, q, k, v, s, q_out=out)
        assert attend(out) == -22 and b"out overlaps q" in lib.aha_paged_last_error()
    with pytest.raises(AhaError, match="overlaps k or v"):
        c.append(0, torch.zeros((3, 128), dtype=torch.bfloat16), k, v, s, q_out=buf[:3, 96:224])


def test_no_cpu_fallback_and_no_gradient():
    c = make()
    seqs, counts = torch.zeros(2, dtype=I), torch.ones(2, dtype=I)
    with pytest.raises(AhaError, match="GPU"):
        c.reserve(seqs, counts, 4)
    q = torch.zeros((3, 4, 32), dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        c.attention(0, q, seqs, torch.zeros(3, dtype=I))
    with torch.no_grad(), pytest.raises(AhaError, match="GPU"):
        c.append(0, q, q[:, :2], q[:, :2], torch.zeros(3, dtype=I))

"""Keys and values of many sequences in one pool of pages (include/aha_amd.h, "paged key-value cache").

Next to the ring caches of `aha_amd.cache` (one buffer per stream, at its full capacity) this one serves requests that come and go and grow to
unknown lengths: a sequence owns only the pages it fills, ragged requests run in one call, and lengths and block tables live on the device, so
that a step makes no host round trip and can be captured into a graph.

    cache = rt.open_paged(n_pages=4096, max_seqs=64)                       # or PagedKVCache(...) without a Runtime
    slots, positions, cu, status = cache.reserve(seqs, counts, n_tokens)   # pages, slots and positions of the step's new tokens
    for layer in range(layers):
        q = cache.append(layer, q, k, v, slots, positions)                 # rotates q and k, stores k and v
        o = cache.attention(layer, q, seqs, cu, max_q=..., max_len=...)
    cache.truncate(seqs, lens)                                             # rejected drafts, finished requests

`seqs`, `counts` and `lens` are int32 device tensors; a negative sequence is padding.  Inference only: nothing here has a gradient."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import lib as _l
from .runtime import AhaError

_ERRORS = ((1, "the free list is too short"), (2, "more new tokens than n_tokens"), (4, "a sequence out of range or a corrupt length"),
           (8, "a sequence is listed twice"), (16, "a sequence outgrows its block table"), (32, "a negative count or a length out of range"),
           (64, "a new token's page, from the free list or the block table, is none"))
_TYPES = {torch.bfloat16: _l.KV_BF16, torch.float8_e4m3fn: _l.KV_E4M3}
_MAX = 0x7fffffff


def _c_ints(*x):
    """As the library's 32-bit arguments: what lies beyond them at their nearer end, where it means or is refused as the same (ctypes would cut the bits off)."""
    return [max(-_MAX - 1, min(int(i), _MAX)) for i in x]


class PagedKVCache:
    """One pool.  `rope`: (cos, sin), bf16 [positions, head_dim], what `append` rotates with
    (positions behind its last as the last); without it keys and queries come rotated.
    `k_scale` / `v_scale`: fp32 [layers, kv_heads] of an e4m3 pool (default 1), finite and not negative (0: that head's values are 0).
    The tensors (`k_pages`, `v_pages`: [layers, n_pages, kv_heads, page_size, head_dim]; `block_table` [max_seqs, max_blocks],
    `lens` [max_seqs], `free_pages` [n_pages], `n_free` [1], all int32) are made here unless given, and are the caller's to look at; pages may hold anything.  `precise`: the attention of drafts, frames and prompts keeps its
    probabilities to 2^-17 (a token's always are) instead of rounding them to bf16, as the ring caches' attention does; up to half as slow again."""

    def __init__(self, n_pages: int, page_size: int, kv_heads: int, head_dim: int, max_seqs: int, max_blocks: int, *, layers: int = 1,
                 dtype: torch.dtype = torch.bfloat16, device="cuda:0", rope: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                 k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None, k_pages: Optional[torch.Tensor] = None,
                 v_pages: Optional[torch.Tensor] = None, block_table: Optional[torch.Tensor] = None, lens: Optional[torch.Tensor] = None,
                 free_pages: Optional[torch.Tensor] = None, n_free: Optional[torch.Tensor] = None, precise: bool = False):
        self.handle = None
        self.lib = _l.get()
        dev = torch.device(device)
        self.device = torch.device(dev.type, torch.cuda.current_device()) if dev.type == "cuda" and dev.index is None else dev
        if dtype not in _TYPES:
            raise ValueError(f"dtype must be torch.bfloat16 or torch.float8_e4m3fn, not {dtype}")
        self.dtype, self.layers, self.n_pages, self.page_size = dtype, int(layers), int(n_pages), int(page_size)
        self.kv_heads, self.head_dim, self.max_seqs, self.max_blocks = int(kv_heads), int(head_dim), int(max_seqs), int(max_blocks)
        shape = (self.layers, self.n_pages, self.kv_heads, self.page_size, self.head_dim)
        if min(shape + (self.max_seqs, self.max_blocks)) < 1:
            raise ValueError("sizes must be positive")
        if max(shape + (self.max_seqs, self.max_blocks)) > _MAX:
            raise ValueError("sizes must be below 2^31")
        if free_pages is not None and n_free is None:
            raise ValueError("free_pages needs n_free")
        self.k_pages = self._own("k_pages", k_pages, shape, dtype)
        self.v_pages = self._own("v_pages", v_pages, shape, dtype)
        self.block_table = self._own("block_table", block_table, (self.max_seqs, self.max_blocks), torch.int32, -1)
        self.lens = self._own("lens", lens, (self.max_seqs,), torch.int32, 0)
        self.n_free = self._own("n_free", n_free, (1,), torch.int32, self.n_pages)
        self.free_pages = self._own("free_pages", free_pages, (self.n_pages,), torch.int32)
        if free_pages is None:                                     # page 0 is taken first
            self.free_pages.copy_(torch.arange(self.n_pages - 1, -1, -1, dtype=torch.int32))
        self.k_scale = None if k_scale is None else self._own("k_scale", k_scale, (self.layers, self.kv_heads), torch.float32)
        self.v_scale = None if v_scale is None else self._own("v_scale", v_scale, (self.layers, self.kv_heads), torch.float32)
        self.cos = self.sin = None
        self._rope = (None, None, 0)
        if rope is not None:
            self.cos, self.sin = rope
            rows = self.cos.shape[0] if self.cos.dim() == 2 else 0
            for name, t in (("cos", self.cos), ("sin", self.sin)):
                self._own(name, t, (rows, self.head_dim), torch.bfloat16)
            if rows < 1:
                raise ValueError("rope: cos and sin must be [positions, head_dim]")
            self._rope = (self.cos.data_ptr(), self.sin.data_ptr(), min(rows, _MAX))
        d = _l.PagedDesc(k_pages=self.k_pages.data_ptr(), v_pages=self.v_pages.data_ptr(), block_table=self.block_table.data_ptr(),
                         lens=self.lens.data_ptr(), free_pages=self.free_pages.data_ptr(), n_free=self.n_free.data_ptr(),
                         k_scale=self.k_scale.data_ptr() if self.k_scale is not None else None,
                         v_scale=self.v_scale.data_ptr() if self.v_scale is not None else None, layers=self.layers, n_pages=self.n_pages,
                         page_size=self.page_size, kv_heads=self.kv_heads, head_dim=self.head_dim, kv_type=_TYPES[dtype],
                         max_seqs=self.max_seqs, max_blocks=self.max_blocks)
        h = C.c_void_p()
        self._chk(self.lib.aha_paged_create(C.byref(d), self.device.index or 0, C.byref(h)))
        self.handle = h
        if precise:
            self._chk(self.lib.aha_paged_set_precise(h, 1))
        self._workspace = {}                                       # sizes of a call -> bytes of its workspace

    # -- plumbing -----------------------------------------------------------------------------------------------------------
    def _own(self, name, t, shape, dtype, fill=None):
        if t is None:
            return torch.empty(shape, dtype=dtype, device=self.device) if fill is None else torch.full(shape, fill, dtype=dtype, device=self.device)
        if tuple(t.shape) != tuple(shape) or t.dtype != dtype or t.device != self.device or not t.is_contiguous():
            raise ValueError(f"{name}: a contiguous {dtype} tensor {list(shape)} on {self.device} is needed, not {t.dtype} {list(t.shape)} on {t.device}")
        return t

    # (these run on every call of a layer: one test of what is right, the reasons only where it is not)
    def _ints(self, name, t, n=None):
        if t.dtype is torch.int32 and t.device == self.device and t.dim() == 1 and (n is None or t.shape[0] == n) and t.is_contiguous():
            return t.data_ptr()
        raise ValueError(f"{name}: a contiguous int32 tensor{'' if n is None else f' of {n} elements'} on {self.device} is needed, not {t.dtype} {list(t.shape)} on {t.device}")

    def _rows(self, name, x, heads=None, out=False):
        """[N, heads, head_dim] or [N, heads * head_dim] -> (tensor, heads, row stride); rows may be strided, their elements not."""
        D, shape, stride = self.head_dim, x.shape, x.stride()
        if x.dtype is not torch.bfloat16 or x.device != self.device or len(shape) not in (2, 3) or (shape[2] != D if len(shape) == 3 else shape[1] % D):
            raise ValueError(f"{name}: a bfloat16 tensor [N, heads, {D}] or [N, heads * {D}] on {self.device} is needed, not {x.dtype} {list(x.shape)} on {x.device}")
        h = shape[1] if len(shape) == 3 else shape[1] // D
        if heads is not None and h != heads:
            raise ValueError(f"{name}: {heads} heads are needed, not {h}")
        if x.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires a gradient and nothing here has one: detach it, or call under torch.no_grad()")
        many = shape[0] > 1
        if stride[-1] != 1 or (len(shape) == 3 and h > 1 and stride[1] != D) or (many and stride[0] < h * D):
            if out:
                raise ValueError(f"{name}: the heads of a row must be contiguous and rows must not overlap")
            return x.contiguous(), h, h * D
        return x, h, stride[0] if many else h * D

    def _stream(self) -> int:
        if self.device.type != "cuda":
            raise AhaError("aha_amd needs a GPU: the product path has no CPU fallback")
        return torch._C._cuda_getCurrentRawStream(self.device.index)

    def _chk(self, rc: int):
        if rc != 0:
            raise AhaError(f"aha_amd error {rc}: {self.lib.aha_paged_last_error().decode()}")

    def check(self, status: torch.Tensor):
        """Raises if the call that returned `status` could not be done (it then changed nothing).  Reads the device: a host round trip."""
        code, missing = status.tolist()
        if code:
            why = "; ".join(text for bit, text in _ERRORS if code & bit)
            raise AhaError(f"paged cache: {why}" + (f" ({missing} pages missing)" if missing else ""))

    def close(self):
        if self.handle is not None:
            self.lib.aha_paged_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # -- the operators ------------------------------------------------------------------------------------------------------
    def reserve(self, seqs: torch.Tensor, counts: torch.Tensor, n_tokens: int):
        """Sequences grow by `counts` tokens, at most `n_tokens` in all -> (slots [n_tokens], positions [n_tokens], cu [n + 1], status [2])."""
        n = seqs.shape[0]
        if not 0 <= n_tokens <= _MAX - 4096:
            raise ValueError(f"n_tokens must be 0 .. {_MAX - 4096}")
        sp, cp = self._ints("seqs", seqs), self._ints("counts", counts, n)
        out = torch.empty(2 * n_tokens + n + 3, dtype=torch.int32, device=self.device)
        p = out.data_ptr()
        self._chk(self.lib.aha_paged_reserve(self.handle, sp, cp, min(n, _MAX), p, p + 4 * n_tokens, n_tokens, p + 8 * n_tokens, p + 8 * n_tokens + 4 * (n + 1), self._stream()))
        return out.split_with_sizes((n_tokens, n_tokens, n + 1, 2))

    def truncate(self, seqs: torch.Tensor, lens: torch.Tensor) -> torch.Tensor:
        """Sequences are cut to `lens` tokens (0 releases them) -> status [2].  Table entries that are no page give nothing back."""
        n = seqs.shape[0]
        sp, lp = self._ints("seqs", seqs), self._ints("lens", lens, n)
        status = torch.empty(2, dtype=torch.int32, device=self.device)
        self._chk(self.lib.aha_paged_truncate(self.handle, sp, lp, min(n, _MAX), status.data_ptr(), self._stream()))
        return status

    def append(self, layer: int, q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, positions: Optional[torch.Tensor] = None,
               q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Rotates q and k (with a `rope` table), stores k and v in their slots and returns the rotated q, [N, heads, head_dim] (`q_out`: where
        to, q itself included).  q, k, v: bf16 [N, heads, head_dim] or [N, heads * head_dim], rows strided as they come from a fused projection."""
        k, _, ldk = self._rows("k", k, self.kv_heads)
        v, _, ldv = self._rows("v", v, self.kv_heads)
        n = k.shape[0]
        if v.shape[0] != n or (q is not None and q.shape[0] != n):
            raise ValueError("q, k and v need the same number of tokens")
        sp = self._ints("slots", slots, n)
        cos, sin, rows = self._rope
        if cos is not None and positions is None:
            raise ValueError("positions are needed to rotate")
        pp = self._ints("positions", positions, n) if cos is not None else None
        heads, ldq, ldo, qp, op = 0, 0, 0, None, None
        if q is not None:
            q, heads, ldq = self._rows("q", q)
            if q_out is None:
                q_out = torch.empty(n, heads, self.head_dim, dtype=torch.bfloat16, device=self.device)
                ldo = heads * self.head_dim
            else:
                q_out, _, ldo = self._rows("q_out", q_out, heads, out=True)
                if q_out.shape[0] != n:
                    raise ValueError("q_out needs as many tokens as q")
            qp, op = q.data_ptr(), q_out.data_ptr()
        if (layer | n | heads) >> 31:
            layer, n, heads = _c_ints(layer, n, heads)
        self._chk(self.lib.aha_paged_append(self.handle, layer, qp, ldq, heads, op, ldo, k.data_ptr(), ldk, v.data_ptr(), ldv, sp, pp, n, cos, sin, rows, self._stream()))
        return q_out

    def attention(self, layer: int, q: torch.Tensor, seqs: torch.Tensor, cu: torch.Tensor, *, max_q: int = 0, max_len: int = 0, window: int = 0,
                  scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal attention of the sequences' last tokens (rows cu[i] .. cu[i+1] of q are those of seqs[i]) over their pages -> bf16 [N, heads,
        head_dim].  `window`: the nearest keys only; `scale`: head_dim ** -0.5 by default; `max_q` / `max_len`: the most new tokens and keys of
        a request where the caller knows them (they choose kernel and split, never the result's meaning).  Rows of no request are left alone:
        pass `out` where they matter (it may be q itself)."""
        q, heads, ldq = self._rows("q", q)
        n, N = seqs.shape[0], q.shape[0]
        sp, cp = self._ints("seqs", seqs), self._ints("cu", cu, n + 1)
        if out is None:
            out, ldo = torch.empty(N, heads, self.head_dim, dtype=torch.bfloat16, device=self.device), heads * self.head_dim
        else:
            out, _, ldo = self._rows("out", out, heads, out=True)
            if out.shape[0] != N:
                raise ValueError("out needs as many tokens as q")
        if window > _MAX:                                          # (more than a sequence can hold: all keys)
            window = 0
        if (layer | N | n | heads | max_q | max_len | window) >> 31:
            layer, N, n, heads, max_q, max_len, window = _c_ints(layer, N, n, heads, max_q, max_len, window)
        key = (heads, N, n, max_q, max_len)
        need = self._workspace.get(key)
        if need is None:                                           # (a function of the sizes alone, asked for once)
            b = C.c_size_t()
            self._chk(self.lib.aha_paged_attention_workspace(self.handle, heads, N, n, max_q, max_len, C.byref(b)))
            if len(self._workspace) >= 4096:
                self._workspace.clear()
            need = self._workspace[key] = b.value
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        self._chk(self.lib.aha_paged_attention(self.handle, layer, q.data_ptr(), ldq, heads, sp, cp, n, N, max_q, max_len, window,
                                               self.head_dim ** -0.5 if scale is None else scale, out.data_ptr(), ldo, ws.data_ptr() if need else None, need, self._stream()))
        return out

    # -- a look at a sequence -----------------------------------------------------------------------------------------------
    def export_kv(self, layer: int, seq: int, want_v: bool = False) -> torch.Tensor:
        """The keys (or values) of a sequence, [kv_heads, length, head_dim], scaled back to fp32 where the pool is e4m3; zeros where a table entry
        is no page, whose keys attention hides.  A host round trip."""
        if not (0 <= layer < self.layers and 0 <= seq < self.max_seqs):
            raise ValueError(f"layer {layer} of {self.layers} or sequence {seq} of {self.max_seqs} is out of range")
        n = int(self.lens[seq])
        if not 0 <= n <= self.max_blocks * self.page_size:
            raise AhaError(f"paged cache: sequence {seq} has a corrupt length, {n}")
        pages = self.block_table[seq, :-(-n // self.page_size)].long()
        raw = (self.v_pages if want_v else self.k_pages)[layer].view(torch.uint8)[pages.clamp(0, self.n_pages - 1)]
        raw[(pages < 0) | (pages >= self.n_pages)] = 0
        x = raw.view(self.dtype)
        x = x.transpose(0, 1).reshape(self.kv_heads, -1, self.head_dim)[:, :n]
        if self.dtype == torch.float8_e4m3fn:
            s = self.v_scale if want_v else self.k_scale
            x = x.float() * (1.0 if s is None else s[layer][:, None, None])
        return x

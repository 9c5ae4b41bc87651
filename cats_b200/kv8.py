"""Paged key/value cache in 8 bits (``cats_kv8_*`` of include/cats_b200.h).

A pool of pages holds the keys and values of all layers as e4m3 codes with one power-of-two scale
per (layer, page, keys or values, head): half the memory and half the bytes per decoded token of the
16-bit cache.  Every sequence has a row in a page table; sequences that continue the same beginning
share its full pages.  Table, lengths and counts are device tensors and every method only launches
kernels on the current stream (``fork``, ``free`` and ``check``, which take or give host values,
excepted), so a decode step over the cache can sit in a CUDA graph::

    cache = KVCache8(n_layers=32, n_pages=2048, n_seqs=16, max_len=4096, n_kv_heads=8, head_dim=128)
    cache.grow(1)                                   # one more token for every sequence
    for l in range(32):
        q = cache.append(l, qkv, n_heads, cos, sin) # rotary embedding, keys and values into the cache
        o = cache.attend(l, q)                      # causal attention over it
    cache.reorder(parents)                          # sequence i continues sequence parents[i]

Lengths, ids and counts are checked on the device, where they live: what does not fit is left out and recorded
(``check``), and what was cached stays as it was.  A page's scale serves all of its rows and channels of a head, so one
very large value costs its page's others their codes, but no other page anything.

The calls on one cache have to be ordered, those that only read it too (they share scratch): one
stream, or events between streams; so do the replays of graphs that hold them.  Its tensors keep their
addresses; they may be read and filled in place (after ``reset`` where the cache has been used: it forgets
which sequences ``grow`` refused).
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from .ops import _DTYPES, _raw_stream, dtype_code

_current_device = torch._C._cuda_getDevice

PAGES, HEAD_DIMS, MAX_SEQS, STATUS_INTS = (16, 32, 64, 128), (32, 64, 96, 128), 1024, 256
_STATUS = {1: "the pool has no free page left", 2: "a page id is out of range, or a shared page would have been written",
           4: "a sequence is longer than the page table allows, or a length or position is negative",
           8: "a parent is out of range", 16: "cu does not fit the number of tokens",
           32: "a wait inside a kernel ran out", 64: "tokens of a sequence that grow had not lengthened were left out"}


def _bad(msg: str) -> RuntimeError:
    return RuntimeError("cats_b200.kv8: " + msg)


class KVCache8:
    """See the module docstring.  ``max_len``: tokens a sequence can have (rounded up to whole pages)."""

    def __init__(self, n_layers: int, n_pages: int, n_seqs: int, max_len: int, n_kv_heads: int,
                 head_dim: int, page: int = 64, device="cuda"):
        dev = torch.device(device)
        if dev.type != "cuda":
            raise _bad("the cache needs a CUDA device (no CPU path)")
        if min(n_layers, n_pages, n_seqs, max_len, n_kv_heads) < 1:
            raise _bad("sizes must be positive")
        if page not in PAGES or head_dim not in HEAD_DIMS or n_seqs > MAX_SEQS:
            raise _bad(f"page must be one of {PAGES}, head_dim one of {HEAD_DIMS}, n_seqs at most {MAX_SEQS}")
        z = lambda *s, dt: torch.zeros(s, dtype=dt, device=dev)  # noqa: E731
        self._adopt(z(n_layers, n_pages, 2, n_kv_heads, page, head_dim, dt=torch.uint8).view(torch.float8_e4m3fn),
                    z(n_layers, n_pages, 2, n_kv_heads, dt=torch.float32),
                    torch.full((n_seqs, (max_len + page - 1) // page), -1, dtype=torch.int32, device=dev),
                    z(n_seqs, dt=torch.int32), z(n_pages, dt=torch.int32))

    @classmethod
    def from_tensors(cls, codes: torch.Tensor, scales: torch.Tensor, table: torch.Tensor,
                     lens: torch.Tensor, refs: torch.Tensor) -> "KVCache8":
        """A cache over existing device tensors: codes [layers, pages, 2, kv_heads, page, head_dim]
        (float8_e4m3fn or uint8), scales [layers, pages, 2, kv_heads] float32 powers of two, table
        [seqs, max_pages], lens [seqs], refs [pages] int32.  They are used in place."""
        self = cls.__new__(cls)
        self._adopt(codes, scales, table, lens, refs)
        return self

    def _adopt(self, codes, scales, table, lens, refs) -> None:
        for t, name, dts, dim in ((codes, "codes", (torch.float8_e4m3fn, torch.uint8), 6),
                                  (scales, "scales", (torch.float32,), 4), (table, "table", (torch.int32,), 2),
                                  (lens, "lens", (torch.int32,), 1), (refs, "refs", (torch.int32,), 1)):
            if not isinstance(t, torch.Tensor) or t.dtype not in dts or t.dim() != dim:
                raise _bad(f"{name} must be a {dim}-D tensor of {' or '.join(map(str, dts))}")
            if not t.is_cuda or t.device != codes.device or not t.is_contiguous():
                raise _bad(f"{name} must be contiguous and on the codes' CUDA device (there is no CPU path)")
        L, P, two, nkv, page, hd = codes.shape
        if two != 2 or tuple(scales.shape) != (L, P, 2, nkv) or lens.shape[0] != table.shape[0] or refs.shape[0] != P:
            raise _bad("the shapes of codes, scales, table, lens and refs do not fit together")
        if page not in PAGES or hd not in HEAD_DIMS or table.shape[0] > MAX_SEQS or min(*codes.shape, *table.shape) < 1:
            raise _bad(f"page must be one of {PAGES}, head_dim one of {HEAD_DIMS}, sequences 1 .. {MAX_SEQS}")
        self.codes, self.scales, self.table, self.lens, self.refs = codes, scales, table, lens, refs
        self._state = torch.zeros(STATUS_INTS, dtype=torch.int32, device=codes.device)
        self.status = self._state[:1]
        self.device = codes.device
        self.n_layers, self.n_pages, self.n_kv_heads, self.page, self.head_dim = L, P, nkv, page, hd
        self.n_seqs, self.max_pages = table.shape
        self.max_len = self.max_pages * page
        self._c = _lib.Kv8(codes.data_ptr(), scales.data_ptr(), table.data_ptr(), lens.data_ptr(), refs.data_ptr(),
                           self.status.data_ptr(), L, P, self.n_seqs, self.max_pages, nkv, page, hd)
        self._p = ctypes.byref(self._c)
        self._index = codes.device.index
        lib = _lib.lib()
        # Scratch of the calls, which are ordered anyway (see the module docstring), for the cache's life.
        # Only attention of many rows per key head (new tokens x heads) needs more: a buffer of its own.
        with torch.cuda.device(self._index):
            small = int(lib.cats_kv8_attend_bytes(self._p, self.n_seqs, nkv))
        self._attend_nbytes = {(self.n_seqs, nkv): small}     # by (tokens, heads)
        self._ws = torch.empty(max(small, int(lib.cats_kv8_reorder_bytes(self._p)), int(lib.cats_kv8_compact_bytes(self._p))),
                               dtype=torch.uint8, device=codes.device)
        self._ws_ptr, self._ws_nbytes = self._ws.data_ptr(), self._ws.numel()

    def _call(self, what: str, *args) -> None:
        """One C call on the current stream of the cache's device."""
        i = self._index
        if _current_device() == i:
            st = getattr(_lib.lib(), what)(self._p, *args, _raw_stream(i))
        else:
            with torch.cuda.device(i):
                st = getattr(_lib.lib(), what)(self._p, *args, _raw_stream(i))
        if st:
            _lib.check(st, what)

    # ---- argument checks ----------------------------------------------------------------------------
    def _cu(self, cu: Optional[torch.Tensor]) -> Optional[int]:
        if cu is None:
            return None
        if not isinstance(cu, torch.Tensor) or cu.dtype != torch.int32 or cu.device != self.device \
                or not cu.is_contiguous() or cu.numel() != self.n_seqs + 1:
            raise _bad(f"cu must be a contiguous int32 tensor of {self.n_seqs + 1} elements on {self.device}")
        return cu.data_ptr()

    def _tokens(self, t: torch.Tensor, name: str, cu) -> int:
        if not isinstance(t, torch.Tensor) or t.device != self.device or t.dim() < 1:
            raise _bad(f"{name} must be a tensor of rows on {self.device}")
        n = t.shape[0]
        if cu is None and n % self.n_seqs:
            raise _bad(f"{name} has {n} rows, not a multiple of the {self.n_seqs} sequences: pass cu")
        return n

    def _layer(self, layer: int) -> None:
        if not 0 <= layer < self.n_layers:
            raise _bad(f"layer {layer} is out of range (0 .. {self.n_layers - 1})")

    # ---- steps ------------------------------------------------------------------------------------------
    def grow(self, n_new: int = 1, cu: Optional[torch.Tensor] = None) -> None:
        """``lens += n_new`` (or the counts of ``cu``), taking the pages that needs (``cats_kv8_grow``).  A
        sequence that cannot have its pages keeps its length (see ``check``), and ``append`` leaves its tokens
        out until it grows."""
        if cu is None and n_new < 1:
            raise _bad("n_new must be positive")
        self._call("cats_kv8_grow", self._cu(cu), n_new)

    def append(self, layer: int, qkv: torch.Tensor, n_heads: int, cos: Optional[torch.Tensor] = None,
               sin: Optional[torch.Tensor] = None, cu: Optional[torch.Tensor] = None,
               q_out: Optional[torch.Tensor] = None, queries: bool = True) -> Optional[torch.Tensor]:
        """Rotary embedding of the newest tokens' queries and keys and the quantising cache write
        (``cats_kv8_append``).  qkv (tokens, (n_heads + 2 kv_heads) head_dim), rows may be strided;
        cos, sin (>= max_len, head_dim), or None for no rotation; ``cu`` int32 (seqs + 1): first row of
        every sequence, or None for the same number of rows each.  Returns the queries (tokens,
        n_heads, head_dim); with ``queries=False`` only keys and values are dealt with."""
        n = self._tokens(qkv, "qkv", cu)
        hd, dt = self.head_dim, qkv.dtype
        code = _DTYPES[dt] if dt in _DTYPES else dtype_code(dt)
        if qkv.dim() != 2 or qkv.shape[1] != (n_heads + 2 * self.n_kv_heads) * hd or n_heads < 1 \
                or n_heads % self.n_kv_heads:
            raise _bad(f"qkv must be (tokens, (n_heads + 2 * {self.n_kv_heads}) * {hd}) with n_heads a multiple of "
                       f"{self.n_kv_heads}, got {tuple(qkv.shape)} and {n_heads} heads")
        if qkv.stride(1) != 1:
            raise _bad("the rows of qkv must be contiguous")
        self._layer(layer)
        pc = ps = None
        rope = 0
        if cos is not None or sin is not None:
            for t in (cos, sin):
                if not isinstance(t, torch.Tensor) or t.dtype != dt or t.device != self.device or t.dim() != 2 \
                        or not t.is_contiguous() or t.shape[1] != hd or t.shape != cos.shape:
                    raise _bad(f"cos and sin must be contiguous (positions, {hd}) tables of {dt} on {self.device}")
            rope = cos.shape[0]
            if rope < self.max_len:
                raise _bad(f"cos and sin hold {rope} positions, the cache up to {self.max_len}")
            pc, ps = cos.data_ptr(), sin.data_ptr()
        if not queries:
            q_out = None
        elif q_out is None:
            q_out = torch.empty_strided((n, n_heads, hd), (n_heads * hd, hd, 1), dtype=dt, device=self.device)
        elif not isinstance(q_out, torch.Tensor) or q_out.dtype != dt or q_out.device != self.device \
                or not q_out.is_contiguous() or q_out.numel() != n * n_heads * hd:
            raise _bad("q_out must be contiguous with tokens * n_heads * head_dim elements of qkv's type")
        if n == 0:
            return q_out
        self._call("cats_kv8_append", layer, qkv.data_ptr(), qkv.stride(0) if n > 1 else qkv.shape[1], self._cu(cu), n,
                   pc, ps, rope, None if q_out is None else q_out.data_ptr(), n_heads, code)
        return q_out

    def attend(self, layer: int, q: torch.Tensor, cu: Optional[torch.Tensor] = None,
               scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal attention of the newest tokens over the cache (``cats_kv8_attend``).  q (tokens,
        n_heads, head_dim), tokens as in ``append``; ``scale`` defaults to head_dim ** -0.5.  Returns a
        tensor like q.  Every token sees the positions of its sequence up to its own."""
        n = self._tokens(q, "q", cu)
        hd, dt = self.head_dim, q.dtype
        code = _DTYPES[dt] if dt in _DTYPES else dtype_code(dt)
        if q.dim() != 3 or q.shape[2] != hd or q.shape[1] % self.n_kv_heads or q.shape[1] < 1:
            raise _bad(f"q must be (tokens, heads, {hd}) with heads a multiple of {self.n_kv_heads}, got {tuple(q.shape)}")
        nh = q.shape[1]
        if q.stride(2) != 1 or (q.stride(1) != hd and nh > 1):
            raise _bad("the heads of a token must be contiguous in q")
        self._layer(layer)
        if out is None:
            out = torch.empty_strided((n, nh, hd), (nh * hd, hd, 1), dtype=dt, device=self.device)
        elif not isinstance(out, torch.Tensor) or out.dtype != dt or out.device != self.device \
                or not out.is_contiguous() or out.numel() != n * nh * hd:
            raise _bad("out must be contiguous with as many elements as q, of q's type")
        if n == 0:
            return out
        nbytes = self._attend_nbytes.get((n, nh))
        if nbytes is None:
            with torch.cuda.device(self._index):
                nbytes = int(_lib.lib().cats_kv8_attend_bytes(self._p, n, nh))
            if len(self._attend_nbytes) >= 4096:
                self._attend_nbytes.clear()
            self._attend_nbytes[(n, nh)] = nbytes
        ws = self._ws_ptr
        if nbytes > self._ws_nbytes:
            large = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            ws = large.data_ptr()
        self._call("cats_kv8_attend", layer, q.data_ptr(), q.stride(0) if n > 1 else nh * hd, self._cu(cu), n, nh,
                   hd ** -0.5 if scale is None else scale, out.data_ptr(), ws, nbytes, code)
        return out

    # ---- pages --------------------------------------------------------------------------------------------
    def reorder(self, parents: torch.Tensor) -> None:
        """Sequence i continues what sequence ``parents[i]`` (int32, on the device) was before the call,
        -1: it becomes empty (``cats_kv8_reorder``).  Full pages are shared, the page that is still being
        filled is copied for every child but the first."""
        if not isinstance(parents, torch.Tensor) or parents.dtype != torch.int32 or parents.device != self.device \
                or not parents.is_contiguous() or parents.numel() != self.n_seqs:
            raise _bad(f"parents must be a contiguous int32 tensor of {self.n_seqs} elements on {self.device}")
        self._call("cats_kv8_reorder", parents.data_ptr(), self._ws_ptr, self._ws_nbytes)

    def _host_parents(self, changes) -> torch.Tensor:
        parents = list(range(self.n_seqs))
        for dst, src in changes:
            if not 0 <= dst < self.n_seqs or not -1 <= src < self.n_seqs:
                raise _bad(f"sequence {dst if not 0 <= dst < self.n_seqs else src} is out of range (0 .. {self.n_seqs - 1})")
            parents[dst] = src
        return torch.tensor(parents, dtype=torch.int32).to(self.device)

    def fork(self, src: Sequence[int], dst: Sequence[int]) -> None:
        """Sequence dst[i] becomes a continuation of src[i] (what dst[i] held is freed)."""
        src, dst = [int(i) for i in src], [int(i) for i in dst]
        if len(src) != len(dst) or len(set(dst)) != len(dst):
            raise _bad("fork needs as many sources as targets, every target once")
        if any(i < 0 for i in src):
            raise _bad("fork sources must be sequences")
        self.reorder(self._host_parents(zip(dst, src)))

    def free(self, seqs: Sequence[int]) -> None:
        """The sequences become empty; pages that nobody else holds are free again."""
        self.reorder(self._host_parents((int(i), -1) for i in seqs))

    def compact(self) -> torch.Tensor:
        """Move the live pages to the front of the pool (``cats_kv8_compact``).  Returns their number
        as a 0-dim int32 device tensor; the page ids from there on are free."""
        n = torch.empty((), dtype=torch.int32, device=self.device)
        self._call("cats_kv8_compact", n.data_ptr(), self._ws_ptr, self._ws_nbytes)
        return n

    def reset(self) -> None:
        """All sequences empty, all pages free, nothing recorded (see ``check``)."""
        self.table.fill_(-1)
        self.lens.zero_()
        self.refs.zero_()
        self._state.zero_()

    # ---- host side ---------------------------------------------------------------------------------------------
    def check(self) -> None:
        """Raise if a kernel found device data that does not fit (synchronises).  The status word
        stays set until ``status.zero_()`` or ``reset()``."""
        bits = int(self.status.item())
        if bits:
            raise _bad("; ".join(text for b, text in _STATUS.items() if bits & b) + f" (status {bits})")

    def read(self, layer: int, seq: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """(keys, values) of one sequence, fp32 [kv_heads, len, head_dim] (synchronises).  Raises if not
        all of its pages are there."""
        self._layer(layer)
        if not 0 <= seq < self.n_seqs:
            raise _bad(f"sequence {seq} is out of range (0 .. {self.n_seqs - 1})")
        n = int(self.lens[seq])
        if not 0 <= n <= self.max_len:
            raise _bad(f"sequence {seq} is {n} tokens long, the table holds up to {self.max_len}")
        ids = self.table[seq, :(n + self.page - 1) // self.page].long()
        if ids.numel() and not (0 <= int(ids.min()) and int(ids.max()) < self.n_pages):
            raise _bad(f"sequence {seq} lacks a page, or a page id is out of range")
        kv = self.codes.view(torch.float8_e4m3fn)[layer].view(torch.uint8)[ids].view(torch.float8_e4m3fn).float()
        kv = (kv * self.scales[layer][ids][..., None, None]).permute(1, 2, 0, 3, 4)
        kv = kv.reshape(2, self.n_kv_heads, ids.numel() * self.page, self.head_dim)[:, :, :n]
        return kv[0], kv[1]

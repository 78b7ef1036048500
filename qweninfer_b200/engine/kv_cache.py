"""Preallocated packed KV cache (QwenInfer's KVCache, qweninfer/engine/kv_cache.py:24-76).

Same layout and interface: K and V are each one allocation of shape
(layers, max_batch rows, kv_heads=2, max_len, head_dim=64), slot j of a row holds the
token at absolute position j, and `row_start` / `window` are set by the caller. One
head of one row is a contiguous run of max_len x 128 bytes, which is what the
attention kernel streams and what `move_row` copies.

On this path the append happens inside the QKV kernel's epilogue (qi_qkv_rope_append),
so `update` exists for API compatibility only; `move_row` runs the qi_move_rows kernel.

`PagedKVCache` (no reference counterpart: the reference kept packed rows, README.md:261-266)
stores positions in pages of 128 slots taken from a pool on demand, so the cache holds
the live tokens rather than rows x max_len, and a retired row's hole is filled by moving
page-table entries instead of copying K/V.

`Kv8Cache` (no reference counterpart either) holds 8-bit codes with a scale for each block
of positions and KV head: half the bytes to keep and to read. Every cache answers
`attend`, grouped-query attention of query tokens over one of its layers, with an optional
sliding window and first tokens that stay visible.
"""

from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

from qweninfer_b200 import _lib
from qweninfer_b200.models.config import Qwen2Config


def _require(t: torch.Tensor, name: str, device: torch.device) -> None:
    if device.type != "cuda" or t.device != device:
        raise _lib.QiError(f"{name}: qweninfer_b200 computes on CUDA (sm_100) tensors of one device only, "
                           f"got {t.device} and a cache on {device}")
    if t.dtype not in _lib.DTYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")


def _window(attn_window: int, attn_sinks: int) -> tuple[int, int]:
    if attn_window < 0 or attn_sinks < 0:
        raise ValueError(f"attn_window and attn_sinks must not be negative; got {attn_window} and {attn_sinks}")
    return attn_window, attn_sinks


class KVCache:
    # what the model's attention sees of a row: the last `attn_window` positions (0: all) and
    # the first `attn_sinks`
    attn_window = attn_sinks = 0

    def __init__(self, cfg: Qwen2Config, max_batch: int, max_len: int,
                 dtype: torch.dtype = torch.float16, device: str | torch.device = "cuda",
                 attn_window: int = 0, attn_sinks: int = 0) -> None:
        # The kernels read and write a bfloat16 cache (the reference's cache dtype for a
        # bf16 model). A float16 or float32 request (the reference's default is float16)
        # gets the same bfloat16 storage: `dtype` is accepted for API compatibility.
        if dtype not in (torch.bfloat16, torch.float16, torch.float32):
            raise ValueError(f"KV cache dtype must be bfloat16, float16 or float32; got {dtype}")
        shape = (cfg.num_hidden_layers, max_batch, cfg.num_key_value_heads, max_len, cfg.head_dim)
        self.k = torch.zeros(shape, dtype=torch.bfloat16, device=device)
        self.v = torch.zeros(shape, dtype=torch.bfloat16, device=device)
        self.max_batch = max_batch
        self.max_len = max_len
        self.window = 0
        self.row_start = 0
        self.attn_window, self.attn_sinks = _window(attn_window, attn_sinks)
        self._err = torch.zeros(1, dtype=torch.int32, device=device)
        self._native: _lib.QiCache | None = None

    def native(self) -> _lib.QiCache:
        if self._native is None:
            self._native = _lib.QiCache(self.k.data_ptr(), self.v.data_ptr(), self.max_batch, self.max_len,
                                        None, 0, 0, 0, _lib.QI_KV_BF16, 0, None, None, self.attn_window,
                                        self.attn_sinks)
        return self._native

    # ---------------------------------------------------------- operators of a layer

    def layer(self, layer: int) -> _lib.QiKvLayer:
        """The qi_kv_layer descriptor of one layer (kept for further calls)."""
        layers = self.__dict__.setdefault("_layers", {})
        if layer not in layers:
            if not 0 <= layer < self.k.shape[0]:
                raise IndexError(f"layer {layer} outside 0..{self.k.shape[0] - 1}")
            layers[layer] = self._layer(layer)
        return layers[layer]

    def _layer(self, i: int) -> _lib.QiKvLayer:
        return _lib.QiKvLayer(self.k[i].data_ptr(), self.v[i].data_ptr(), None, None, _lib.QI_KV_BF16, 0,
                              self.max_batch, self.k.shape[2], self.max_len, self.k.shape[-1], None, 0, 0, 0)

    def _errors(self) -> torch.Tensor:
        """The error word of `attend` and `append`. It is made with the cache: made by a call that
        is being captured, it would lie in the graph's memory and be zeroed by each replay."""
        return self._err

    def check(self) -> None:
        """Raise if an `attend` or `append` of this cache met a position, cache row or page
        outside it (synchronises)."""
        e = int(self._errors().item())
        if e:
            raise _lib.QiError(f"device error word = {e} (a position, cache row or page outside the cache)")

    def _tokens(self, M: int, rows: torch.Tensor, pos: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """Rows and positions of M tokens as int32 on the device; those given on the host are
        checked there."""
        dev = self.k.device
        if (rows.dtype is torch.int32 and pos.dtype is torch.int32 and rows.shape == pos.shape == (M,)
                and rows.device == dev and pos.device == dev and rows.is_contiguous() and pos.is_contiguous()
                and dev.type == "cuda"):
            return rows, pos
        out = []
        for name, t, lo, hi in (("rows", rows, 0, self.max_batch), ("pos", pos, -1, self.max_len)):
            if t.dim() != 1 or t.shape[0] != M:
                raise ValueError(f"{name} must have shape ({M},), got {tuple(t.shape)}")
            if t.device.type == "cpu":
                if t.dtype not in (torch.int32, torch.int64):
                    raise ValueError(f"{name} must be int32 or int64, got {t.dtype}")
                if M and (int(t.min()) < lo or int(t.max()) >= hi):
                    raise IndexError(f"{name} [{int(t.min())}, {int(t.max())}] outside {lo}..{hi - 1}")
                t = t.to(torch.int32).to(self.k.device)
            elif t.dtype != torch.int32 or t.device != self.k.device:
                raise ValueError(f"{name} on a device must be int32 on {self.k.device}, got {t.dtype} on {t.device}")
            out.append(t if t.is_contiguous() else t.contiguous())
        return out[0], out[1]

    def _operand(self, name: str, t: torch.Tensor, heads: int | None) -> None:
        _require(t, name, self.k.device)
        if t.dim() != 3 or t.shape[2] != self.k.shape[-1] or (heads is not None and t.shape[1] != heads):
            raise ValueError(f"{name} must be (tokens, {'heads' if heads is None else heads}, {self.k.shape[-1]}), "
                             f"got {tuple(t.shape)}")
        if t.stride(2) != 1:
            raise ValueError(f"the last dimension of {name} must be contiguous")

    def attend(self, layer: int, q: torch.Tensor, rows: torch.Tensor, pos: torch.Tensor, window: int = 0,
               sinks: int = 0, query_run: int = 0, out: torch.Tensor | None = None,
               tiles: bool = False) -> torch.Tensor:
        """Grouped-query attention of M query tokens over layer `layer` (qi_cache_attention).

        q: (M, heads, head_dim) float32, bfloat16 or float16, any strides of the first two
        dimensions; heads is 1 to 8 times the cache's KV heads and head_dim 64 or 128. Token
        t, at position pos[t] of cache row rows[t], sees key j if 0 <= j <= pos[t] and, with
        a `window` (> 0), j > pos[t] - window or j < sinks. pos[t] = -1 marks an idle slot:
        its output is zero. rows and pos: (M,) int32 on the cache's device, or integers on
        the host, which are checked (on the device, one outside the cache is recorded for
        `check()` and gives a zero output). `query_run`: the longest run of consecutive
        tokens of one row (a prompt's length), 1 for a decode step, 0 if unknown; it only
        picks the kernel: long runs share their keys in tiles where that pays if the rows
        are as long as max_len allows. `tiles`: whatever the size. Returns (M, heads, head_dim) of q's dtype (`out`, if given:
        contiguous, 16-byte aligned and apart from q), enqueued on the current stream.

        Scores, softmax and sums are fp32. q and the probabilities keep 22 bits over an 8-bit
        cache and 24 (16 for 16-bit q) over a bf16 one where each token reads its own keys; in
        tiles 22 bits over both, and 11 of the probabilities for bfloat16 q, whose outputs have 8."""
        # what the shapes alone decide is checked once for each kind of call
        key = (layer, q.shape, q.stride(), q.dtype, window, sinks, query_run, tiles)
        try:
            plan = self._plans.get(key)
        except AttributeError:
            self._plans, plan = {}, None
        if plan is None:
            plan = self._attend_plan(*key[:1], q, *key[4:])
            if len(self._plans) >= 4096:
                self._plans.clear()
            self._plans[key] = plan
        dev = self.k.device
        if q.device != dev:
            _require(q, "q", dev)
        M = q.shape[0]
        rows, pos = self._tokens(M, rows, pos)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)  # 1 us less than new_empty
        elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous {tuple(q.shape)} {q.dtype} tensor on {q.device}")
        elif out.data_ptr() % 16:
            raise ValueError("out must be 16-byte aligned")
        elif out.untyped_storage().data_ptr() == q.untyped_storage().data_ptr():
            raise ValueError("out must not share q's storage")
        if M == 0:
            return out
        if _lib.ready(dev.index):
            code = self._attend(plan, q, rows, pos, out)
        else:
            with _lib.on_device(dev):
                code = self._attend(plan, q, rows, pos, out)
        if code:
            _lib.check(code, "qi_cache_attention")
        return out

    def _attend(self, plan: tuple, q: torch.Tensor, rows: torch.Tensor, pos: torch.Tensor, out: torch.Tensor) -> int:
        d, st, sh, dtype, heads, window, sinks, query_run, part_floats, n_counters = plan
        dev = q.device
        stream = torch._C._cuda_getCurrentRawStream(dev.index)
        part = counters = 0
        if n_counters:
            part, counters, _keep = _lib.scratch(dev, stream, 4 * part_floats, n_counters)
        return _lib.lib().qi_cache_attention(
            d, q.data_ptr(), st, sh, dtype, heads, rows.data_ptr(), pos.data_ptr(), q.shape[0], window, sinks,
            query_run, out.data_ptr(), part, part_floats, counters, n_counters, self._errors().data_ptr(), stream)

    def _attend_plan(self, layer: int, q: torch.Tensor, window: int, sinks: int, query_run: int,
                     tiles: bool) -> tuple:
        """The arguments of an `attend` call that its shapes decide, checked, and its scratch."""
        d = self.layer(layer)
        self._operand("q", q, None)
        M, heads, D = q.shape
        if D not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {D}")
        if heads == 0 or heads % d.kv_heads or heads // d.kv_heads > 8:
            raise ValueError(f"{heads} query heads are not 1 to 8 for each of {d.kv_heads} KV heads")
        if window < 0 or sinks < 0 or query_run < 0:
            raise ValueError("window, sinks and query_run must not be negative")
        lim = 2**31 - 1
        window, sinks = min(window, lim), min(sinks, lim)
        query_run = min(query_run, _lib.QI_RUN_TILES - 1) | (_lib.QI_RUN_TILES if tiles else 0)
        a, b = C.c_longlong(), C.c_longlong()
        if M:
            with _lib.on_device(self.k.device):
                _lib.check(_lib.lib().qi_cache_attention_scratch(C.byref(d), heads, M, window, sinks, query_run,
                                                                 C.byref(a), C.byref(b)), "qi_cache_attention_scratch")
        return (C.byref(d), q.stride(0), q.stride(1), _lib.DTYPES[q.dtype], heads, window, sinks, query_run, a.value,
                b.value)

    # storage management hooks of the paged cache (every slot of a packed row exists)
    def reserve(self, row: int, length: int, start: int = 0) -> None:
        """Make positions [start, length) of `row` writable (no-op for packed rows)."""

    def release(self, row: int) -> None:
        """The row's request is gone (no-op for packed rows)."""

    def trim(self, row: int, length: int) -> None:
        """Give back what no query at position `length` or later sees (no-op for packed rows)."""

    def sync(self) -> None:
        """Publish storage changes to the device before a forward (no-op)."""

    def update(self, layer: int, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor):
        """kv_cache.py:48-63: scatter k/v (B, Hkv, S, hd) at positions (B, S) into rows
        [row_start, row_start + B), return the (B, Hkv, window, hd) history views."""
        B = k.shape[0]
        r = slice(self.row_start, self.row_start + B)
        rows = torch.arange(B, device=k.device).unsqueeze(1)
        self.k[layer, r][rows, :, positions] = k.transpose(1, 2).to(self.k.dtype)
        self.v[layer, r][rows, :, positions] = v.transpose(1, 2).to(self.v.dtype)
        return self.k[layer, r, :, : self.window], self.v[layer, r, :, : self.window]

    def move_row(self, src: int, dst: int, length: int) -> None:
        """kv_cache.py:65-73: copy positions [0, length) of row src to row dst, all layers."""
        self.move_rows([(src, dst, length)])

    def move_rows(self, moves: list[tuple[int, int, int]]) -> None:
        """Apply (src, dst, length) row copies in order, enqueued on the current stream."""
        if not moves:
            return
        _lib.ensure_device(self.k.device)
        flat = (C.c_int * (3 * len(moves)))(*[int(x) for m in moves for x in m])
        _lib.check(_lib.lib().qi_move_rows(self.k.data_ptr(), self.v.data_ptr(), self.k.shape[0],
                                           self.max_batch, self.max_len, flat, len(moves),
                                           _lib.stream_ptr(self.k.device)), "qi_move_rows")

    def memory_bytes(self) -> int:
        return 2 * self.k.numel() * self.k.element_size()


class PagedKVCache(KVCache):
    """K and V in pages of `page_size` positions (a multiple of 128) from a pool of
    `n_pages` pages per layer: `k`, `v` of shape (layers, n_pages, kv_heads, page_size,
    head_dim) and a page table (max_batch, pages_per_row) int32, -1 for unmapped, on the
    device with a host copy. Pages are taken from the pool as rows grow (`reserve`),
    returned when a row's request ends (`release`), and `move_row` moves page-table
    entries. The default pool (max_batch x pages_per_row pages) never runs out; a smaller
    one raises when it does. Only the forward's tensor-core path reads this layout."""

    def __init__(self, cfg: Qwen2Config, max_batch: int, max_len: int,
                 dtype: torch.dtype = torch.float16, device: str | torch.device = "cuda",
                 page_size: int = 128, n_pages: int | None = None,
                 attn_window: int = 0, attn_sinks: int = 0) -> None:
        if dtype not in (torch.bfloat16, torch.float16, torch.float32):
            raise ValueError(f"KV cache dtype must be bfloat16, float16 or float32; got {dtype}")
        if page_size < 128 or page_size % 128:
            raise ValueError(f"page_size must be a positive multiple of 128; got {page_size}")
        self.page_size = page_size
        self.pages_per_row = -(-max_len // page_size)
        self.n_pages = n_pages if n_pages is not None else max_batch * self.pages_per_row
        if self.n_pages < 1:
            raise ValueError("the pool needs at least one page")
        self._allocate((cfg.num_hidden_layers, self.n_pages, cfg.num_key_value_heads, page_size, cfg.head_dim), device)
        self.max_batch = max_batch
        self.max_len = max_len
        self.window = 0
        self.row_start = 0
        self.attn_window, self.attn_sinks = _window(attn_window, attn_sinks)
        self._err = torch.zeros(1, dtype=torch.int32, device=device)
        dev = torch.device(device)
        self.table_host = torch.full((max_batch, self.pages_per_row), -1, dtype=torch.int32)
        self.table = self.table_host.to(dev)
        self._published: torch.cuda.Event | None = None  # the last copy to the device
        self._ordered: set[int] = set()                  # streams whose work comes behind it
        self._t = self.table_host.numpy()
        # by row: pages mapped (a prefix, less what `trim` gave back), of them those that `trim` has
        # looked at, and the furthest position that it was told of
        self.mapped, self.trimmed, self.trim_at = (np.zeros(max_batch, dtype=np.int64) for _ in range(3))
        self.free = list(range(self.n_pages - 1, -1, -1))   # stack of free page ids
        self.dirty = False
        self._native = None

    def _allocate(self, shape: tuple, device: str | torch.device) -> None:
        self.k = torch.zeros(shape, dtype=torch.bfloat16, device=device)
        self.v = torch.zeros(shape, dtype=torch.bfloat16, device=device)

    def native(self) -> _lib.QiCache:
        if self._native is None:
            self._native = _lib.QiCache(self.k.data_ptr(), self.v.data_ptr(), self.max_batch, self.max_len,
                                        self.table.data_ptr(), self.page_size, self.pages_per_row, self.n_pages,
                                        _lib.QI_KV_BF16, 0, None, None, self.attn_window, self.attn_sinks)
        return self._native

    def _layer(self, i: int) -> _lib.QiKvLayer:
        return _lib.QiKvLayer(self.k[i].data_ptr(), self.v[i].data_ptr(), None, None, _lib.QI_KV_BF16, 0,
                              self.max_batch, self.k.shape[2], self.max_len, self.k.shape[-1],
                              self.table.data_ptr(), self.page_size, self.pages_per_row, self.n_pages)

    def attend(self, layer: int, q: torch.Tensor, rows: torch.Tensor, pos: torch.Tensor, window: int = 0,
               sinks: int = 0, query_run: int = 0, out: torch.Tensor | None = None,
               tiles: bool = False) -> torch.Tensor:
        """KVCache.attend; page-table changes are published first (`sync`). A page that a
        token sees but the table does not map is recorded for `check()` and counts as
        zeros."""
        self.sync()
        return super().attend(layer, q, rows, pos, window, sinks, query_run, out, tiles)

    def reserve(self, row: int, length: int, start: int = 0) -> None:
        """Map the pages of positions [start, length), `start` being the first position about
        to be written: 0 for a text that begins, the row's length for one that goes on. Pages
        that `trim` has given back are mapped again from `start` on (a text that begins gives
        back the others of such a row too); raises if a query at `start` would see positions
        that went back."""
        if not 0 <= row < self.max_batch or not 0 <= start <= length <= self.max_len:
            raise IndexError(f"row {row} / positions [{start}, {length}) outside the cache")
        size, need = self.page_size, -(-length // self.page_size)
        went_back = start < self.trim_at[row]  # pages from `start` on, or seen from there, may be gone
        if not went_back and need <= self.mapped[row]:
            return
        if went_back and start == 0:
            self.release(row)
        mapped, first = int(self.mapped[row]), start // size
        if went_back and start:
            seen = ((0, -(-min(self.attn_sinks, start) // size)),
                    (max(0, start - self.attn_window + 1) // size, -(-start // size)))
            if any((self._t[row, a:min(b, mapped)] < 0).any() for a, b in seen):
                raise RuntimeError(f"row {row} cannot go on at position {start}: positions before it that are seen "
                                   f"from there went back behind the window")
            self.trimmed[row] = min(int(self.trimmed[row]), first)
        for j in range(min(first, mapped), need):
            if self._t[row, j] < 0:
                if not self.free:
                    raise RuntimeError(f"KV page pool of {self.n_pages} pages exhausted")
                self._t[row, j] = self.free.pop()
                self.dirty = True
            self.mapped[row] = max(int(self.mapped[row]), j + 1)

    def release(self, row: int) -> None:
        for j in range(int(self.mapped[row]) - 1, -1, -1):
            if self._t[row, j] >= 0:
                self.free.append(int(self._t[row, j]))
            self._t[row, j] = -1
        if self.mapped[row]:
            self.dirty = True
        self.mapped[row] = self.trimmed[row] = self.trim_at[row] = 0

    def trim(self, row: int, length: int) -> None:
        """With a window, return the pages that no query at position `length` or later sees:
        those that end before its window and hold no first tokens. (`reserve` maps them again
        for a text that begins anew.)"""
        if not self.attn_window:
            return
        self.trim_at[row] = max(int(self.trim_at[row]), length)
        end = min(max(0, length - self.attn_window + 1) // self.page_size, int(self.mapped[row]))
        for j in range(int(self.trimmed[row]), end):
            if j * self.page_size >= self.attn_sinks and self._t[row, j] >= 0:
                self.free.append(int(self._t[row, j]))
                self._t[row, j] = -1
                self.dirty = True
        self.trimmed[row] = max(int(self.trimmed[row]), end)

    def move_row(self, src: int, dst: int, length: int) -> None:
        """Row dst takes over row src's pages (positions [0, length) and any beyond);
        dst's own pages return to the pool and src is left without pages."""
        if src == dst:
            return
        self.release(dst)
        self._t[dst] = self._t[src]
        self._t[src] = -1
        for n in (self.mapped, self.trimmed, self.trim_at):
            n[dst], n[src] = n[src], 0
        self.dirty = True

    def move_rows(self, moves: list[tuple[int, int, int]]) -> None:
        for src, dst, length in moves:
            self.move_row(src, dst, length)

    def sync(self) -> None:
        """Publish page-table changes to the device, before the call that reads them. The copy is
        enqueued on the current stream, out of memory of its own (the host goes on changing
        the table), and calls on other streams wait for it. A call that is being captured
        cannot publish: `sync` is called before the capture, and before a replay that
        follows changes."""
        dev = self.table.device
        if dev.type != "cuda":
            if self.dirty:
                self.table.copy_(self.table_host)
                self.dirty = False
            return
        stream = torch._C._cuda_getCurrentRawStream(dev.index)
        if not self.dirty and (self._published is None or stream in self._ordered):
            return
        with torch.cuda.device(dev):
            if torch.cuda.is_current_stream_capturing():
                if self.dirty:
                    raise _lib.QiError("page-table changes cannot be published while a graph is being captured: "
                                       "call sync() before")
                return  # (what is captured runs when it is replayed)
            if self.dirty:
                if self._published is not None and stream not in self._ordered:
                    torch.cuda.current_stream().wait_event(self._published)  # copies arrive in their order
                self.table.copy_(self.table_host.pin_memory(), non_blocking=True)
                self.dirty = False
                self._published = torch.cuda.Event()
                self._published.record()
                self._ordered = {stream}
            else:
                torch.cuda.current_stream().wait_event(self._published)
                self._ordered.add(stream)

    def pages_in_use(self) -> int:
        return self.n_pages - len(self.free)

    def update(self, layer: int, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor):
        raise NotImplementedError("the paged cache is written by the forward's kernels only")


class _Codes:
    """K and V as 8-bit codes with block scales: what Kv8Cache and PagedKv8Cache share."""

    FORMATS = {"int8": (_lib.QI_KV_INT8, torch.int8), "e4m3": (_lib.QI_KV_E4M3, torch.float8_e4m3fn)}

    def _format(self, format: str, block_tokens: int) -> None:
        if format not in self.FORMATS:
            raise ValueError(f"format must be one of {sorted(self.FORMATS)}; got {format!r}")
        if block_tokens not in (16, 32, 64, 128):
            raise ValueError(f"block_tokens must be 16, 32, 64 or 128; got {block_tokens}")
        self.format, self.block_tokens = format, block_tokens

    def _allocate(self, shape: tuple, device: str | torch.device) -> None:
        blocks = shape[:3] + (-(-shape[3] // self.block_tokens),)
        code = self.FORMATS[self.format][1]
        self.k = torch.zeros(shape, dtype=torch.int8, device=device).view(code)
        self.v = torch.zeros(shape, dtype=torch.int8, device=device).view(code)
        self.k_scale = torch.zeros(blocks, dtype=torch.float32, device=device)
        self.v_scale = torch.zeros(blocks, dtype=torch.float32, device=device)

    def native(self) -> _lib.QiCache:
        if self._native is None:
            n = super().native()
            n.format, n.block = self.FORMATS[self.format][0], self.block_tokens
            n.k_scale, n.v_scale = self.k_scale.data_ptr(), self.v_scale.data_ptr()
        return self._native

    def _layer(self, i: int) -> _lib.QiKvLayer:
        d = super()._layer(i)
        d.format, d.block = self.FORMATS[self.format][0], self.block_tokens
        d.k_scale, d.v_scale = self.k_scale[i].data_ptr(), self.v_scale[i].data_ptr()
        return d

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, rows: torch.Tensor, pos: torch.Tensor) -> None:
        """Write M tokens' keys and values into layer `layer` (qi_kv8_append): token t at
        position pos[t] of cache row rows[t]; pos[t] = -1 skips it.

        k, v: (M, kv_heads, head_dim) of one dtype (float32, bfloat16 or float16), any
        strides of the first two dimensions (slices of a fused projection's output will
        do). A row grows from its end: the positions before the first appended one keep
        their values (rounded again where their block's scale grows, at most one step of the
        final scale in all), those after the last one of its block are dead, and a block whose
        first position is appended starts over. The tokens may come in any order; of two with
        the same row and position the later one is kept. A value that is not finite makes
        its block's scale NaN, and so the outputs that read the block. rows and pos as in
        `attend`."""
        key = (layer, k.shape, k.stride(), v.shape, v.stride(), k.dtype, v.dtype)
        try:
            d = self._append_plans.get(key)
        except AttributeError:
            self._append_plans, d = {}, None
        if d is None:
            layer_ = self.layer(layer)
            self._operand("k", k, layer_.kv_heads)
            self._operand("v", v, layer_.kv_heads)
            if v.dtype != k.dtype or v.shape != k.shape:
                raise ValueError(f"k and v must have one shape and dtype, got {tuple(k.shape)} {k.dtype} and "
                                 f"{tuple(v.shape)} {v.dtype}")
            if layer_.head_dim not in (64, 128):
                raise ValueError(f"head_dim must be 64 or 128, got {layer_.head_dim}")
            if len(self._append_plans) >= 4096:
                self._append_plans.clear()
            d = self._append_plans[key] = C.byref(layer_)
        dev = self.k.device
        if k.device != dev or v.device != dev:
            _require(k, "k", dev)
            _require(v, "v", dev)
        M = k.shape[0]
        rows, pos = self._tokens(M, rows, pos)
        if M == 0:
            return
        args = (d, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                _lib.DTYPES[k.dtype], rows.data_ptr(), pos.data_ptr(), M, self._errors().data_ptr())
        if _lib.ready(dev.index):
            code = _lib.lib().qi_kv8_append(*args, torch._C._cuda_getCurrentRawStream(dev.index))
        else:
            with _lib.on_device(dev):
                code = _lib.lib().qi_kv8_append(*args, torch._C._cuda_getCurrentRawStream(dev.index))
        if code:
            _lib.check(code, "qi_kv8_append")

    def values(self, layer: int) -> tuple[torch.Tensor, torch.Tensor]:
        """What layer `layer` stands for: K and V (max_batch, kv_heads, max_len, head_dim)
        fp32 (qi_kv8_values). Dead positions give whatever their codes say."""
        try:
            plan = self._value_plans.get(layer)
        except AttributeError:
            self._value_plans, plan = {}, None
        if plan is None:
            d = self.layer(layer)
            dev = self.k.device
            if dev.type != "cuda":
                _require(self.k_scale, "values", dev)
            if d.head_dim not in (64, 128):
                raise ValueError(f"head_dim must be 64 or 128, got {d.head_dim}")
            shape = (self.max_batch, d.kv_heads, self.max_len, d.head_dim)
            strides = tuple(math.prod(shape[i + 1:]) for i in range(4))
            plan = self._value_plans[layer] = C.byref(d), dev, shape, strides
        d, dev, shape, strides = plan
        k, v = (torch.empty_strided(shape, strides, dtype=torch.float32, device=dev) for _ in range(2))
        if _lib.ready(dev.index):
            code = _lib.lib().qi_kv8_values(d, k.data_ptr(), v.data_ptr(), torch._C._cuda_getCurrentRawStream(dev.index))
        else:
            with _lib.on_device(dev):
                code = _lib.lib().qi_kv8_values(d, k.data_ptr(), v.data_ptr(), _lib.stream_ptr(dev))
        if code:
            _lib.check(code, "qi_kv8_values")
        return k, v

    def update(self, layer: int, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor):
        raise NotImplementedError("an 8-bit cache is written by append and by the model's forward")

    def memory_bytes(self) -> int:
        return 2 * (self.k.numel() + 4 * self.k_scale.numel())


class Kv8Cache(_Codes, KVCache):
    """K and V as 8-bit codes with block scales: `k`, `v` (layers, max_batch, kv_heads,
    max_len, head_dim) int8 or float8_e4m3fn and `k_scale`, `v_scale` (layers, max_batch,
    kv_heads, ceil(max_len / block_tokens)) fp32. The scale of a block of `block_tokens`
    (16, 32, 64 or 128) positions of one row and head is the least power of two s with
    127 s (int8) or 448 s (e4m3) >= all its values; the codes stand for code * s. `int8`
    is the more exact on even-sized values (a step of at most amax / 63.5), `e4m3` keeps
    small values next to large ones (relative steps of 2^-3).

    `append` writes new tokens, `attend` reads them (KVCache.attend), `values` gives back
    what the codes stand for; the model's forward, `generate` and `Engine(kv_format=...)`
    use it like a bf16 cache."""

    def __init__(self, cfg: Qwen2Config, max_batch: int, max_len: int,
                 dtype: torch.dtype = torch.float16, device: str | torch.device = "cuda",
                 format: str = "int8", block_tokens: int = 32,
                 attn_window: int = 0, attn_sinks: int = 0) -> None:
        if dtype not in (torch.bfloat16, torch.float16, torch.float32):
            raise ValueError(f"KV cache dtype must be bfloat16, float16 or float32; got {dtype}")
        self._format(format, block_tokens)
        self._allocate((cfg.num_hidden_layers, max_batch, cfg.num_key_value_heads, max_len, cfg.head_dim), device)
        self.max_batch = max_batch
        self.max_len = max_len
        self.window = 0
        self.row_start = 0
        self.attn_window, self.attn_sinks = _window(attn_window, attn_sinks)
        self._err = torch.zeros(1, dtype=torch.int32, device=device)
        self._native = None

    def move_rows(self, moves: list[tuple[int, int, int]]) -> None:
        """KVCache.move_rows: codes of positions [0, length) and the scales of their blocks."""
        for src, dst, length in moves:
            if not (0 <= src < self.max_batch and 0 <= dst < self.max_batch and 0 <= length <= self.max_len):
                raise IndexError(f"row move {(src, dst, length)} outside the cache")
            if src == dst or length == 0:
                continue
            blocks = -(-length // self.block_tokens)
            for t, n in ((self.k, length), (self.v, length), (self.k_scale, blocks), (self.v_scale, blocks)):
                t[:, dst, :, :n] = t[:, src, :, :n]


class PagedKv8Cache(_Codes, PagedKVCache):
    """Kv8Cache in pages: pools of codes (layers, n_pages, kv_heads, page_size, head_dim) and
    of scales (layers, n_pages, kv_heads, page_size / block_tokens), with PagedKVCache's
    page table and storage management."""

    def __init__(self, cfg: Qwen2Config, max_batch: int, max_len: int,
                 dtype: torch.dtype = torch.float16, device: str | torch.device = "cuda",
                 page_size: int = 128, n_pages: int | None = None, format: str = "int8", block_tokens: int = 32,
                 attn_window: int = 0, attn_sinks: int = 0) -> None:
        self._format(format, block_tokens)
        super().__init__(cfg, max_batch, max_len, dtype, device, page_size, n_pages, attn_window, attn_sinks)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, rows: torch.Tensor, pos: torch.Tensor) -> None:
        """Kv8Cache.append; the pages of the positions are mapped (`reserve`) by the caller and
        table changes published first. A token without a page is recorded for `check()`."""
        self.sync()
        super().append(layer, k, v, rows, pos)

    def values(self, layer: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Kv8Cache.values by cache row and position; zeros where no page is mapped."""
        self.sync()
        return super().values(layer)


def _single_layer_view(cache: KVCache, layer: int) -> tuple[torch.Tensor, torch.Tensor]:
    return cache.k[layer], cache.v[layer]

"""The reference engine's host-side API for the attention path, over the C ABI.

Mirrors, with the same names, argument meaning and error behaviour:

* ``RopeCache``            -- src/layers/rope.rs:5-40
* ``KVCache``              -- src/layers/kv_cache.rs:12-173 (pools, block table,
                              LIFO free list, prepare_for_step, update)
* ``apply_rope``           -- CudaFunctions::apply_rope, src/kernels.rs:203-246
* ``apply_flash_decoding`` -- CudaFunctions::apply_flash_decoding,
                              src/kernels.rs:248-320

and adds the batched forms the kernels are built for (``decode_step``), page
tables that live on the GPU (``DeviceBlocks``) and caches of 8 and 4 bits over
them (``Kv8Cache``, ``Kv4Cache``).
Device memory comes from torch; every launch goes through liblucattn.so.
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch

from . import library

BLOCK_SIZE = 16  # src/layers/kv_cache.rs:35


def _lib(lib):
    return lib if lib is not None else library.default(torch.cuda.current_device())


def sm_scale(head_dim: int) -> float:
    """1/sqrt(head_dim) rounded to f32, as src/kernels.rs:264."""
    return float(np.float32(1.0) / np.sqrt(np.float32(head_dim)))


class RopeCache:
    """cos/sin tables [max_pos][head_dim/2] (f32), built on the host and copied
    to the device -- RopeCache::new, src/layers/rope.rs:11-40."""

    def __init__(self, max_position_embeddings, head_dim, base=1e6, scale_factor=None,
                 device="cuda", lib=None):
        cos, sin = _lib(lib).rope_table(max_position_embeddings, head_dim, base, scale_factor)
        self.cos = cos.to(device)
        self.sin = sin.to(device)


def pool_blocks(free: int, total: int, memory_fraction: float, num_layers: int,
                num_kv_heads: int, head_dim: int, max_position_embeddings: int) -> int:
    """Pages of a KV pool sized from a VRAM budget, as KVCache::new does
    (src/layers/kv_cache.rs:37-59): the budget is total * memory_fraction (an
    f32 product, truncated) less the memory already used (total - free); a
    page holds K and V of 16 tokens for every layer and kv head in bf16; the
    pool holds at most the pages of max_position_embeddings.  Raises
    RuntimeError with the reference's message when the budget is below the
    memory already used (kv_cache.rs:40-48)."""
    used = total - free
    available_total = int(np.float32(total) * np.float32(memory_fraction))
    allocatable = available_total - used
    gb = 1024.0 ** 3
    if allocatable < 0:
        raise RuntimeError(
            "Not enough available GPU memory for KV Cache allocation, "
            f"free: {free / gb} GB, used: {used / gb} GB, total: {total / gb} GB, "
            f"requested fraction: {memory_fraction}")
    bytes_per_block = 2 * num_layers * num_kv_heads * BLOCK_SIZE * head_dim * 2
    return min(allocatable // bytes_per_block, (max_position_embeddings + BLOCK_SIZE - 1) // BLOCK_SIZE)


class KVCache:
    """Paged K/V pools [num_blocks][num_layers][Hkv][16][head_dim] and one block
    table -- src/layers/kv_cache.rs:12-104.  The pool size is given directly,
    or by `from_budget` from the free VRAM as the reference does
    (kv_cache.rs:37-59)."""

    @classmethod
    def from_budget(cls, num_layers, num_kv_heads, head_dim, max_position_embeddings,
                    memory_fraction, dtype=torch.bfloat16, device="cuda", lib=None,
                    mem_info=None):
        """KVCache::new: the pool sized by pool_blocks from (free, total) of the
        device (torch.cuda.mem_get_info) or `mem_info`."""
        free, total = mem_info if mem_info is not None else torch.cuda.mem_get_info(device)
        blocks = pool_blocks(free, total, memory_fraction, num_layers, num_kv_heads, head_dim,
                             max_position_embeddings)
        return cls(num_layers, num_kv_heads, head_dim, blocks, max_position_embeddings, dtype,
                   device, lib)

    def __init__(self, num_layers, num_kv_heads, head_dim, num_physical_blocks,
                 max_position_embeddings, dtype=torch.bfloat16, device="cuda", lib=None):
        self.lib = _lib(lib)
        self.block_size = BLOCK_SIZE
        self.num_layers = num_layers
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.num_physical_blocks = num_physical_blocks
        self.max_seq_len = max_position_embeddings
        shape = (num_physical_blocks, num_layers, num_kv_heads, BLOCK_SIZE, head_dim)
        self.k_pool = torch.zeros(shape, dtype=dtype, device=device)
        self.v_pool = torch.zeros(shape, dtype=dtype, device=device)
        max_logical = (max_position_embeddings + BLOCK_SIZE - 1) // BLOCK_SIZE
        self.block_table = torch.zeros(max_logical, dtype=torch.int32, device=device)
        self.block_table_cpu: list[int] = []
        # LIFO filled in reverse, so pops hand out 0, 1, 2, ... (kv_cache.rs:73-76)
        self.free_blocks = list(range(num_physical_blocks - 1, -1, -1))
        self._workspace = None

    def prepare_for_step(self, pos: int) -> None:
        """Append one page when `pos` enters a new logical block and copy the
        table to the device -- kv_cache.rs:106-122 (panics there when the free
        list is empty; raises here)."""
        logical = pos // self.block_size
        if logical >= len(self.block_table_cpu):
            if not self.free_blocks:
                raise RuntimeError("KVCache: Out of memory blocks")
            self.block_table_cpu.append(self.free_blocks.pop())
            n = len(self.block_table_cpu)
            self.block_table[:n].copy_(torch.tensor(self.block_table_cpu, dtype=torch.int32),
                                       non_blocking=False)

    def update(self, layer_idx, pos, pos_ptr, k_input, v_input, v_bias, stream=None):
        """Write one token's K (bit copy) and V + v_bias at slot `pos` of layer
        `layer_idx` -- KVCache::update, kv_cache.rs:124-173."""
        self.prepare_for_step(pos)
        row = self.num_kv_heads * self.head_dim
        self.lib.kv_cache_update(self.k_pool, self.v_pool, k_input, v_input, v_bias, row,
                                 self.block_table.view(1, -1), pos_ptr, 1, layer_idx,
                                 self.num_layers, self.num_kv_heads, self.head_dim,
                                 self.block_size, stream)

    def workspace(self, num_q_heads, max_ctx):
        """Zero-filled split-K workspace for one sequence, grown on demand."""
        need = self.lib.workspace_size(1, num_q_heads, self.num_kv_heads, self.head_dim, max_ctx)
        if need == 0:
            return None
        if self._workspace is None or self._workspace.numel() * 4 < need:
            self._workspace = torch.zeros(need // 4, dtype=torch.float32,
                                          device=self.k_pool.device)
        return self._workspace


class BlockManager:
    """Pages of one pool for many sequences, through the native allocator
    (luc_blocks_*): the reference's free list and prepare_for_step
    (kv_cache.rs:73-76, 106-122) per table row, with multi-page growth, batch
    admission (all or nothing) and release.  Host only; no GPU call."""

    def __init__(self, num_blocks: int, max_seqs: int, max_blocks_per_seq: int):
        self.cdll = library.load_cdll()
        self.max_seqs, self.max_pages = max_seqs, max_blocks_per_seq
        self.handle = ctypes.c_void_p()
        self._check(self.cdll.luc_blocks_create(num_blocks, max_seqs, max_blocks_per_seq,
                                                ctypes.byref(self.handle)))

    def _check(self, rc):
        if rc < 0:
            raise library.LucError(rc, self.cdll.luc_last_error().decode())
        return rc

    def close(self):
        if self.handle:
            self.cdll.luc_blocks_destroy(self.handle)
            self.handle = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def reserve(self, seq: int, num_tokens: int) -> None:
        self._check(self.cdll.luc_blocks_reserve(self.handle, seq, num_tokens))

    def reserve_batch(self, seqs, num_tokens) -> None:
        s = np.ascontiguousarray(seqs, dtype=np.int32)
        t = np.ascontiguousarray(num_tokens, dtype=np.int32)
        if s.shape != t.shape:
            raise ValueError("seqs and num_tokens differ in length")
        self._check(self.cdll.luc_blocks_reserve_batch(self.handle, s.size, s.ctypes.data,
                                                       t.ctypes.data))

    def release(self, seq: int) -> None:
        self._check(self.cdll.luc_blocks_release(self.handle, seq))

    @property
    def num_free(self) -> int:
        return self._check(self.cdll.luc_blocks_num_free(self.handle))

    def num_pages(self, seq: int) -> int:
        return self._check(self.cdll.luc_blocks_num_pages(self.handle, seq))

    def table(self, first_seq: int = 0, n: int | None = None) -> np.ndarray:
        n = self.max_seqs - first_seq if n is None else n
        out = np.empty((n, self.max_pages), np.int32)
        self._check(self.cdll.luc_blocks_table(self.handle, first_seq, n, out.ctypes.data,
                                               self.max_pages))
        return out


class PagedKVCache:
    """K/V pools shared by up to `max_seqs` sequences, their device block table
    [max_seqs, max_blocks_per_seq] and the native allocator behind it -- the
    batched form of KVCache.  `reserve` / `reserve_batch` / `release` change
    the allocation; `sync()` copies the table to the device before a launch."""

    def __init__(self, num_layers, num_kv_heads, head_dim, num_physical_blocks, max_seqs,
                 max_position_embeddings, dtype=torch.bfloat16, device="cuda"):
        self.num_layers, self.num_kv_heads, self.head_dim = num_layers, num_kv_heads, head_dim
        self.block_size = BLOCK_SIZE
        max_pages = (max_position_embeddings + BLOCK_SIZE - 1) // BLOCK_SIZE
        self.blocks = BlockManager(num_physical_blocks, max_seqs, max_pages)
        shape = (num_physical_blocks, num_layers, num_kv_heads, BLOCK_SIZE, head_dim)
        self.k_pool = torch.zeros(shape, dtype=dtype, device=device)
        self.v_pool = torch.zeros(shape, dtype=dtype, device=device)
        self.block_tables = torch.zeros((max_seqs, max_pages), dtype=torch.int32, device=device)

    def reserve(self, seq, num_tokens):
        self.blocks.reserve(seq, num_tokens)

    def reserve_batch(self, seqs, num_tokens):
        self.blocks.reserve_batch(seqs, num_tokens)

    def release(self, seq):
        self.blocks.release(seq)

    def sync(self):
        self.block_tables.copy_(torch.from_numpy(self.blocks.table()))


class DeviceBlocks:
    """Lengths, block tables and free list of up to `max_seqs` sequences over one
    pool of `num_blocks` pages, held on the GPU: BlockManager's counterpart for
    loops with no host work between steps, captured ones among them
    (luc_block_extend, luc_block_truncate).  A fresh one hands out pages 0, 1,
    2, ... as BlockManager does.

    After `extend`, the first `rows` of `slots` and `positions` are the step's
    packed new rows (behind them lies what an earlier step left: no step may
    have more), `cu_seqlens` and `start_pos` each sequence's rows among them.  Neither call
    waits for the GPU, so neither can raise for a step that could not be met;
    such a step takes nothing and has no rows, and `check()` raises for it.
    Calls must be in one stream's order."""

    def __init__(self, num_blocks: int, max_seqs: int, max_blocks_per_seq: int, max_rows: int,
                 device="cuda", lib=None):
        if min(num_blocks, max_seqs, max_blocks_per_seq, max_rows) < 1:
            raise ValueError(f"num_blocks {num_blocks}, max_seqs {max_seqs}, max_blocks_per_seq "
                             f"{max_blocks_per_seq} and max_rows {max_rows} must be positive")
        self.lib = _lib(lib)
        self.num_blocks, self.max_seqs, self.max_rows = num_blocks, max_seqs, max_rows
        kw = {"dtype": torch.int32, "device": device}
        self.lens = torch.zeros(max_seqs, **kw)
        self.block_tables = torch.zeros((max_seqs, max_blocks_per_seq), **kw)
        self.free_list = torch.arange(num_blocks - 1, -1, -1, **kw)
        self.state = torch.tensor([num_blocks, 0, 0, 0], **kw)
        self.slots = torch.full((max_rows,), -1, dtype=torch.int64, device=device)
        self.positions = torch.full((max_rows,), -1, **kw)
        self.cu_seqlens = torch.zeros(max_seqs + 1, **kw)
        self.start_pos = torch.zeros(max_seqs, **kw)
        self.rows = max_rows  # of the last extend

    def extend(self, new_tokens, rows: int | None = None, stream=None) -> None:
        """Pages, slots and positions for new_tokens (device int32 [max_seqs]) more
        tokens of every sequence, `rows` (default max_rows) of them at most."""
        rows = self.max_rows if rows is None else rows
        if not 0 <= rows <= self.max_rows:
            raise ValueError(f"rows {rows} outside [0, {self.max_rows}]")
        self.lib.block_extend(new_tokens, self.lens, self.block_tables, self.free_list, self.state,
                              self.slots[:rows], self.positions[:rows], self.cu_seqlens,
                              self.start_pos, stream=stream)
        self.rows = rows

    def truncate(self, keep, stream=None) -> None:
        """Every sequence back to at most keep (device int32 [max_seqs]) tokens, the pages
        behind those to the free list; the exact inverse of `extend`."""
        self.lib.block_truncate(keep, self.lens, self.block_tables, self.free_list, self.state,
                                stream=stream)

    def check(self) -> None:
        """Waits for the current stream; raises LucError (and forgets the fault) if a step since
        the last call could not be met."""
        status = int(self.state[1].item())
        if status == 0:
            return
        self.state[1].zero_()
        what = [text for bit, text in ((1, "free pages are short"), (2, "a block table row is"),
                                       (4, "a length, count or the state is out of range"),
                                       (8, "there are more rows than the step allows")) if status & bit]
        raise library.LucError(-6 if status == 1 else -1, "page maps: " + "; ".join(what))

    @property
    def num_free(self) -> int:
        """Free pages (waits for the current stream)."""
        return int(self.state[0].item())


class _QuantCache:
    """Pools of a quantised cache of up to `max_seqs` sequences, the DeviceBlocks behind them and the
    workspace of their attention.  `slab`: bytes of a page's K or V of one head, by dimension."""

    def __init__(self, slab, num_layers, num_q_heads, num_kv_heads, head_dim, num_physical_blocks,
                 max_seqs, max_position_embeddings, max_rows, device, lib):
        self.lib = _lib(lib)
        if head_dim not in (64, 128):
            raise library.LucError(-2, f"Unsupported head dimension for attention kernel: {head_dim}")
        self.num_layers, self.num_q_heads = num_layers, num_q_heads
        self.num_kv_heads, self.head_dim = num_kv_heads, head_dim
        self.block_size = BLOCK_SIZE
        self.max_seq_len = max_position_embeddings
        self.blocks = DeviceBlocks(num_physical_blocks, max_seqs, ceil_div(max_position_embeddings, BLOCK_SIZE),
                                   max_rows or max_seqs, device, self.lib)
        shape = (num_physical_blocks, num_layers, num_kv_heads, slab * head_dim)
        self.k_pool = torch.zeros(shape, dtype=torch.uint8, device=device)
        self.v_pool = torch.zeros(shape, dtype=torch.uint8, device=device)
        self._workspace = None
        self._captured = []  # workspaces that captured graphs hold

    def extend(self, new_tokens, rows=None, stream=None):
        self.blocks.extend(new_tokens, rows, stream)

    def truncate(self, keep, stream=None):
        self.blocks.truncate(keep, stream)

    def _step_rows(self, q):
        if q.shape[0] > self.blocks.rows:
            raise ValueError(f"{q.shape[0]} rows to append: the step has {self.blocks.rows}")

    @staticmethod
    def _capturing(stream):
        if stream is None:
            return torch.cuda.is_current_stream_capturing()
        with torch.cuda.stream(stream):
            return torch.cuda.is_current_stream_capturing()

    def _grown(self, need, stream):
        """The workspace, of at least `need` bytes; None for 0."""
        if need == 0:
            return None
        capturing = self._capturing(stream)
        old = self._workspace
        if old is None or old.numel() * 4 < need:
            if capturing:
                raise RuntimeError(f"{type(self).__name__}: a workspace of {need} bytes must be made before the "
                                   "capture")
            size = need // 4 if old is None else max(need // 4, old.numel() * 3 // 2)
            with torch.cuda.stream(stream):  # (None: the current one) filled in the launch's order
                self._workspace = torch.zeros(size, dtype=torch.float32, device=self.k_pool.device)
            if old is not None:  # launches before this one may still use it
                old.record_stream(torch.cuda.current_stream() if stream is None else stream)
        if capturing and not any(w is self._workspace for w in self._captured):
            self._captured.append(self._workspace)
        return self._workspace

    def _scale(self, scale):
        return sm_scale(self.head_dim) if scale is None else scale


class Kv4Cache(_QuantCache):
    """A 4-bit paged cache of up to `max_seqs` sequences (pools of luc_kv4_append, 0.31 of the
    bytes of 16 bits) and the DeviceBlocks behind it.  A step: `extend`, then `append` and
    `attend` for every layer; all of it may be captured in a HIP graph, and so may `truncate`.
    Calls, and replays of captured ones, must be in one stream's order: they share a workspace."""

    def __init__(self, num_layers, num_q_heads, num_kv_heads, head_dim, num_physical_blocks,
                 max_seqs, max_position_embeddings, max_rows=None, device="cuda", lib=None):
        super().__init__(10, num_layers, num_q_heads, num_kv_heads, head_dim, num_physical_blocks,
                         max_seqs, max_position_embeddings, max_rows, device, lib)

    def append(self, layer, q, k, v, rope, q_bias=None, k_bias=None, v_bias=None, q_norm=None, k_norm=None,
               eps=1e-6, q_out=None, k_out=None, v_out=None, stream=None):
        """Biases, head norms, RoPE and the cache write of the step's rows q [rows, Hq * d], k and v
        [rows, Hkv * d] in `layer` (luc_kv4_append); q_out (default: q itself) gets q.  At most the
        `rows` that the step's `extend` was given."""
        b = self.blocks
        self._step_rows(q)
        self.lib.kv4_append(q, k, v, rope.cos, rope.sin, b.positions, b.slots, self.k_pool, self.v_pool, layer,
                            self.num_layers, self.num_q_heads, self.num_kv_heads, self.head_dim, q_norm, k_norm,
                            eps, q_bias, k_bias, v_bias, q_out, k_out, v_out, stream=stream)

    def workspace(self, total_rows, max_rows, max_ctx, stream=None):
        """The zero-filled workspace of `attend`, grown on demand by half at least (None: none needed).  Ask
        for it before a capture that needs a larger one than there is.  A smaller one that it takes the
        place of is freed, unless it was handed out during a capture (by `attend`; a program that captures
        launches of its own on one holds it itself)."""
        return self._grown(self.lib.lib.luc_kv4_workspace_size(
            self.blocks.max_seqs, total_rows, max_rows, max_ctx, self.num_q_heads, self.num_kv_heads,
            self.head_dim), stream)

    def attend(self, layer, out, q, max_ctx, max_rows=None, scale=None, stream=None):
        """Attention of the step's rows (luc_kv4_attention): q and out [rows, Hq * d]; max_ctx and max_rows
        (default: all of q's rows) bound a sequence's context, its new rows among it, and its new
        rows; scale defaults to 1 / sqrt(d)."""
        b = self.blocks
        rows = q.shape[0]
        max_rows = rows if max_rows is None else max_rows
        self.lib.kv4_attention(out, q, self.k_pool, self.v_pool, b.block_tables, b.start_pos, b.max_seqs, rows,
                               max_rows, max_ctx, layer, self.num_layers, self.num_q_heads, self.num_kv_heads,
                               self.head_dim, self._scale(scale), cu_seqlens=b.cu_seqlens,
                               workspace=self.workspace(rows, max_rows, max_ctx, stream), stream=stream)


class Kv8Cache(_QuantCache):
    """An 8-bit paged cache of up to `max_seqs` sequences (pools and scales of luc_kv8_append, half the
    bytes of 16 bits) and the DeviceBlocks behind it: a step as Kv4Cache has it.  With `bounds` (1/16 of the
    pools more) a step of at most one row a sequence may `attend_sparse`: to the pages of each context that
    score highest, instead of to all of it.  One that was made without cannot.  Tokens that `truncate` drops still
    count in the scale and the bounds of the page that goes on, until its next first token: the same tokens
    again may have coarser codes there, and be chosen by wider bounds."""

    def __init__(self, num_layers, num_q_heads, num_kv_heads, head_dim, num_physical_blocks,
                 max_seqs, max_position_embeddings, max_rows=None, bounds=False, device="cuda", lib=None):
        super().__init__(16, num_layers, num_q_heads, num_kv_heads, head_dim, num_physical_blocks,
                         max_seqs, max_position_embeddings, max_rows, device, lib)
        shape = (num_physical_blocks, num_layers, num_kv_heads, 2)
        self.scales = torch.zeros(shape, dtype=torch.float32, device=device)
        self.bounds = torch.zeros((*shape, head_dim), dtype=torch.uint8, device=device) if bounds else None

    def append(self, layer, q, k, v, rope, q_bias=None, k_bias=None, v_bias=None, q_norm=None, k_norm=None,
               eps=1e-6, q_out=None, stream=None):
        """Biases, head norms, RoPE and the cache write of the step's rows q [rows, Hq * d], k and v
        [rows, Hkv * d] in `layer` (luc_kv8_append); q_out (default: q itself) gets q.  At most the
        `rows` that the step's `extend` was given."""
        b = self.blocks
        self._step_rows(q)
        self.lib.kv8_append(q, k, v, rope.cos, rope.sin, b.positions, b.slots, self.k_pool, self.v_pool, self.scales,
                            layer, self.num_layers, self.num_q_heads, self.num_kv_heads, self.head_dim, self.bounds,
                            q_norm, k_norm, eps, q_bias, k_bias, v_bias, q_out, stream=stream)

    def read(self, layer, k_out, v_out, slots, stream=None):
        """K and V of the tokens at `slots` (int64 [rows]: page * 16 + offset) in `layer`, in 16 bits, to k_out
        and v_out [rows, Hkv * d] (luc_kv8_read)."""
        self.lib.kv8_read(k_out, v_out, slots, self.k_pool, self.v_pool, self.scales, layer, self.num_layers,
                          self.num_kv_heads, self.head_dim, stream=stream)

    def workspace(self, total_rows, max_rows, max_ctx, budget=None, stream=None):
        """The zero-filled workspace of `attend` or, with a budget, of `attend_sparse`, grown on demand by half
        at least (None: none needed); one serves both.  Ask for it before a capture that needs a larger one than
        there is, and as Kv4Cache.workspace otherwise."""
        c, n, h = self.lib.lib, self.blocks.max_seqs, (self.num_q_heads, self.num_kv_heads, self.head_dim)
        if budget is None:
            return self._grown(c.luc_kv8_workspace_size(n, total_rows, max_rows, max_ctx, *h), stream)
        return self._grown(c.luc_kv8_sparse_workspace_size(n, max_ctx, budget, *h), stream)

    def attend(self, layer, out, q, max_ctx, max_rows=None, scale=None, stream=None):
        """Attention of the step's rows (luc_kv8_attention): q and out [rows, Hq * d]; max_ctx and max_rows
        (default: all of q's rows) bound a sequence's context, its new rows among it, and its new
        rows; scale defaults to 1 / sqrt(d)."""
        b = self.blocks
        rows = q.shape[0]
        max_rows = rows if max_rows is None else max_rows
        self.lib.kv8_attention(out, q, self.k_pool, self.v_pool, self.scales, b.block_tables, b.start_pos, b.max_seqs,
                               rows, max_rows, max_ctx, layer, self.num_layers, self.num_q_heads, self.num_kv_heads,
                               self.head_dim, self._scale(scale), cu_seqlens=b.cu_seqlens,
                               workspace=self.workspace(rows, max_rows, max_ctx, stream=stream), stream=stream)

    def attend_sparse(self, layer, out, q, max_ctx, budget, first=1, recent=2, scale=None, pages=None, stream=None):
        """Attention of a step with at most one row a sequence over `budget` pages of each context, chosen for
        every kv head by score (luc_kv8_select, luc_kv8_sparse_attention), the first `first` and the
        last `recent` always among them; the pages go to `pages` (int32 [max_seqs, Hkv, budget], default: a new
        tensor) and are returned."""
        if self.bounds is None:
            raise ValueError("this cache keeps no key bounds: make it with bounds=True")
        b, h = self.blocks, (layer, self.num_layers, self.num_q_heads, self.num_kv_heads, self.head_dim)
        if pages is None:
            with torch.cuda.stream(stream):  # (None: the current one)
                pages = torch.empty((b.max_seqs, self.num_kv_heads, budget), dtype=torch.int32,
                                    device=self.k_pool.device)
        ws = self.workspace(q.shape[0], 1, max_ctx, budget, stream)
        self.lib.kv8_select(pages, q, self.bounds, self.scales, b.block_tables, b.start_pos, b.max_seqs, max_ctx,
                            first, recent, *h, cu_seqlens=b.cu_seqlens, workspace=ws, stream=stream)
        self.lib.kv8_sparse_attention(out, q, self.k_pool, self.v_pool, self.scales, b.block_tables, b.start_pos,
                                      pages, b.max_seqs, max_ctx, *h, self._scale(scale), cu_seqlens=b.cu_seqlens,
                                      workspace=ws, stream=stream)
        return pages


def apply_rope(rope, qkv, q_start_idx, k_start_idx, q_bias, k_bias, pos_ptr, head_dim,
               num_q_heads, num_k_heads, lib=None, stream=None):
    """q/k bias + RoPE in place on views of qkv (flat) at the position held in
    pos_ptr -- src/kernels.rs:203-246."""
    q = qkv[q_start_idx:]
    k = qkv[k_start_idx:]
    _lib(lib).rope(q, q_bias, k, k_bias, num_q_heads * head_dim, rope.cos, rope.sin, pos_ptr, 1,
                   num_q_heads, num_k_heads, head_dim, stream)


def apply_flash_decoding(output, out_offset, q, q_offset, cache, layer_idx, pos, pos_ptr,
                         head_dim, num_q_heads, num_kv_heads, lib=None, stream=None):
    """Attention of one query row over positions 0..pos of the cache --
    src/kernels.rs:248-320.  Only head_dim 64/128 (kernels.rs:37-46)."""
    if head_dim not in (64, 128):
        raise library.LucError(-2, f"Unsupported head dimension for attention kernel: {head_dim}")
    ws = cache.workspace(num_q_heads, pos + 1)
    _lib(lib).paged_decode(output[out_offset:], q[q_offset:], cache.k_pool, cache.v_pool,
                           cache.block_table.view(1, -1), pos_ptr, 1, pos + 1, layer_idx,
                           cache.num_layers, num_q_heads, num_kv_heads, head_dim,
                           sm_scale(head_dim), 0, ws, stream=stream)


def decode_step(qkv, q_bias, k_bias, v_bias, rope, k_pool, v_pool, block_tables, positions,
                max_ctx, layer, num_layers, num_q_heads, num_kv_heads, head_dim, out,
                workspace=None, split_tokens=0, lib=None, stream=None):
    """One batched decode step of the attention path for one layer, in one
    launch (luc_decode_step): RoPE(q, k) and cache append of one new token per
    sequence, then paged attention.

    qkv: [B, (Hq + 2*Hkv)*head_dim], rows as the engine's qkv_states
    (src/models.rs:467-503); out: [B, Hq*head_dim]; positions: int32 [B] on
    the device (position of the new token); block_tables: int32 [B, pages];
    workspace: from LucAttn.workspace (zero-filled once, reusable)."""
    lib = _lib(lib)
    batch, row = qkv.shape
    lib.decode_step(qkv, q_bias, k_bias, v_bias, rope.cos, rope.sin, k_pool, v_pool, block_tables,
                    positions, batch, max_ctx, layer, num_layers, num_q_heads, num_kv_heads,
                    head_dim, sm_scale(head_dim), out, workspace, split_tokens,
                    qkv_row_stride=row, out_row_stride=out.shape[-1], stream=stream)


def decode_step_unfused(qkv, q_bias, k_bias, v_bias, rope, k_pool, v_pool, block_tables,
                        positions, max_ctx, layer, num_layers, num_q_heads, num_kv_heads,
                        head_dim, out, workspace=None, split_tokens=0, lib=None, stream=None):
    """The same step as two launches: luc_rope_append, then luc_paged_decode."""
    lib = _lib(lib)
    batch, row = qkv.shape
    qd = num_q_heads * head_dim
    kd = num_kv_heads * head_dim
    lib.rope_append(qkv, q_bias, qkv[:, qd:], k_bias, qkv[:, qd + kd:], v_bias, row, rope.cos,
                    rope.sin, positions, block_tables, k_pool, v_pool, batch, layer, num_layers,
                    num_q_heads, num_kv_heads, head_dim, stream=stream)
    lib.paged_decode(out, qkv, k_pool, v_pool, block_tables, positions, batch, max_ctx, layer,
                     num_layers, num_q_heads, num_kv_heads, head_dim, sm_scale(head_dim),
                     split_tokens, workspace, out_row_stride=out.shape[-1], q_row_stride=row,
                     stream=stream)


def ceil_div(a, b):
    return -(-a // b)


__all__ = ["RopeCache", "KVCache", "DeviceBlocks", "Kv4Cache", "Kv8Cache", "apply_rope", "apply_flash_decoding",
           "decode_step", "decode_step_unfused",
           "sm_scale", "BLOCK_SIZE"]

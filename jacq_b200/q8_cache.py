"""Paged KV cache in 8 bits with one scale per page and kv head: write, attention, page masses, eviction.

Stands beside ``KiviCache`` (int4, ``jacq_b200/cache.py``) where twice its bytes buy an error that does not depend on
per-channel statistics: K and V of a page are int8 or e4m3 codes under ONE fp32 scale each, and the tokens of a
sequence's last, incomplete page stay in fp16 tail rows until the page fills up, so every value is rounded once. Layout
and semantics are those of ``include/jacq_kivi_b200.h`` (section q8).

``Q8Cache`` owns (or is laid over) one layer's tensors, block tables and sequence lengths, all on the device; each
method is one library call on the current stream (slot ids take one more to gather tables and lengths, and a write one to
advance the lengths) and nothing synchronises with the host. The reference has no 8-bit
cache, no window and, for its page-drop mechanism, no eviction policy.

torch is plumbing here (device memory, streams); all arithmetic is in libjacq_kivi_b200.so.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import NamedTuple

import torch

from jacq_b200 import _native

_FORMATS = {"int8": (0, torch.int8), "e4m3": (1, torch.float8_e4m3fn)}


@dataclass(frozen=True)
class Q8Layout:
    """Heads, head_dim (64, 128 or 256), tokens per page (16, 32, 64 or 128) and code format ("int8" or "e4m3")."""
    num_q_heads: int
    num_kv_heads: int
    head_dim: int
    block_size: int = 16
    fmt: str = "int8"

    def validate(self) -> None:
        if self.fmt not in _FORMATS:
            raise ValueError(f"format must be one of {tuple(_FORMATS)}, got {self.fmt!r}")
        if self.num_kv_heads <= 0 or self.num_q_heads <= 0 or self.num_q_heads % self.num_kv_heads:
            raise ValueError("num_q_heads must be a positive multiple of num_kv_heads")
        if self.head_dim not in (64, 128, 256):
            raise ValueError(f"head_dim must be 64, 128 or 256, got {self.head_dim}")
        if self.block_size not in (16, 32, 64, 128):
            raise ValueError(f"block_size must be 16, 32, 64 or 128, got {self.block_size}")

    @property
    def code_dtype(self) -> torch.dtype:
        return _FORMATS[self.fmt][1]

    def page_bytes(self) -> int:
        """Bytes of one page of all kv heads: K and V codes and their scales."""
        return self.num_kv_heads * (2 * self.block_size * self.head_dim + 8)

    def decode_algorithmic_bytes(self, seq_len: int, window: int = 0, sinks: int = 0) -> int:
        """Bytes one single-token attention of one sequence must move: what its token sees, q and the fp16 output."""
        low = max(0, seq_len - window) if window else 0
        seen = seq_len - low + min(sinks, low)
        tail = min(seq_len % self.block_size, seen)
        pages = -(-(seen - tail) // self.block_size)
        return (self.num_kv_heads * self.head_dim * (2 * (seen - tail) + 4 * tail) + pages * (8 * self.num_kv_heads + 4)
                + 4 * self.num_q_heads * self.head_dim)


class Q8CacheTensors(NamedTuple):
    K_PAGES: torch.Tensor    # codes [num_blocks, NKV, B, D]
    V_PAGES: torch.Tensor
    SCALES: torch.Tensor     # fp32 [num_blocks, NKV, 2]: K, V
    K_TAIL: torch.Tensor     # fp16 [num_slots, NKV, B, D]
    V_TAIL: torch.Tensor


class Q8Eviction(NamedTuple):
    """What ``evict`` leaves: closed-up tables, masses and lengths, and the ids of the pages that are free."""
    block_tables: torch.Tensor   # int32 [batch, width], 0 behind the kept pages
    seq_lens: torch.Tensor       # int32 [batch]
    page_mass: torch.Tensor      # fp32 [batch, NKV, mass width], 0 behind the kept pages' columns and the open block's
    freed: torch.Tensor          # int32 [batch, width], -1 behind the evicted pages
    freed_counts: torch.Tensor   # int32 [batch]


# The calls of a decode step are a few microseconds long on the device, so the host side is kept short: integers instead
# of device objects, the raw stream handle, no context manager where the device is the current one already.
_raw_stream = torch._C._cuda_getCurrentRawStream


def _int32(t: torch.Tensor, name: str, index: int) -> int:
    if t.dtype is not torch.int32 or not t.is_contiguous():
        raise TypeError(f"{name} must be a contiguous torch.int32 tensor")
    if t.get_device() != index:
        raise RuntimeError(f"{name} is on {t.device}, expected cuda:{index}")
    return t.data_ptr()


_current_device = torch._C._cuda_getDevice


def _elsewhere(index: int, where: str, fn, *args) -> None:
    """A library call on the current stream of device `index` where another device is the current one."""
    with torch.cuda.device(index):
        rc = fn(*args, _raw_stream(index))
    if rc:
        _native.check(rc, where)


def _indexed(device: torch.device | str) -> torch.device:
    device = torch.device(device)
    if device.type != "cuda":
        raise RuntimeError("the 8-bit cache needs a CUDA device; its kernels have no CPU path")
    return torch.device("cuda", torch.cuda.current_device()) if device.index is None else device


class Q8Cache:
    """One layer's 8-bit cache for up to ``num_slots`` live sequences."""

    def __init__(self, layout: Q8Layout, num_blocks: int, num_slots: int, max_blocks_per_seq: int,
                 device: torch.device | str = "cuda"):
        layout.validate()
        device = _indexed(device)
        nkv, b, d = layout.num_kv_heads, layout.block_size, layout.head_dim
        codes = [torch.zeros((num_blocks, nkv, b, d), dtype=torch.uint8, device=device).view(layout.code_dtype) for _ in range(2)]
        tails = [torch.zeros((num_slots, nkv, b, d), dtype=torch.float16, device=device) for _ in range(2)]
        tensors = Q8CacheTensors(*codes, torch.zeros((num_blocks, nkv, 2), dtype=torch.float32, device=device), *tails)
        self._bind(layout, tensors, torch.zeros((num_slots, max_blocks_per_seq), dtype=torch.int32, device=device),
                   torch.zeros((num_slots,), dtype=torch.int32, device=device))

    @classmethod
    def over(cls, layout: Q8Layout, tensors: Q8CacheTensors, block_tables: torch.Tensor, seq_lens: torch.Tensor) -> "Q8Cache":
        """A cache laid over tensors that the caller owns (nothing is copied)."""
        layout.validate()
        self = cls.__new__(cls)
        self._bind(layout, tensors, block_tables, seq_lens)
        return self

    def _bind(self, layout, tensors, block_tables, seq_lens) -> None:
        nkv, b, d = layout.num_kv_heads, layout.block_size, layout.head_dim
        device = _indexed(tensors.K_PAGES.device)
        blocks, slots = tensors.K_PAGES.shape[0], tensors.K_TAIL.shape[0]
        want = {"K_PAGES": (layout.code_dtype, (blocks, nkv, b, d)), "V_PAGES": (layout.code_dtype, (blocks, nkv, b, d)),
                "SCALES": (torch.float32, (blocks, nkv, 2)), "K_TAIL": (torch.float16, (slots, nkv, b, d)),
                "V_TAIL": (torch.float16, (slots, nkv, b, d))}
        for name, (dtype, shape) in want.items():
            t = getattr(tensors, name)
            if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous() or t.device != device:
                raise TypeError(f"{name} must be a contiguous {dtype} tensor {shape} on {device}")
        for name, t, dim in (("block_tables", block_tables, 2), ("seq_lens", seq_lens, 1)):
            _int32(t, name, device.index)
            if t.dim() != dim:
                raise TypeError(f"{name} must have {dim} dimension(s)")
        self.layout, self.tensors, self.device, self._index = layout, tensors, device, device.index
        self.block_tables, self.seq_lens = block_tables, seq_lens
        self.max_blocks_per_seq = block_tables.shape[1]
        self.num_blocks, self.num_slots = blocks, slots
        self._geom = _native.KiviQ8Geometry(layout.num_q_heads, nkv, d, b, _FORMATS[layout.fmt][0])
        self._struct = _native.KiviQ8CacheStruct(*[t.data_ptr() for t in tensors], blocks, slots)
        self._geom_ref, self._cache_ref = ctypes.byref(self._geom), ctypes.byref(self._struct)
        lib = _native.lib()
        self._write, self._read, self._attention = lib.kivi_b200_q8_cache_write, lib.kivi_b200_q8_cache_read, lib.kivi_b200_q8_attention
        self._gather, self._advance = lib.kivi_b200_q8_gather_slots, lib.kivi_b200_q8_advance_slots
        self._workspace_of = lib.kivi_b200_q8_attention_workspace_bytes
        self._workspace_bytes: dict[tuple, int] = {}   # by the sizes of a call

    def set_block_tables(self, tables: torch.Tensor) -> None:
        """Install block tables ``[<= num_slots, <= max_blocks_per_seq]`` (int32; host or device)."""
        tables = tables.to(device=self.device, dtype=torch.int32)
        self.block_tables.zero_()
        self.block_tables[: tables.shape[0], : tables.shape[1]] = tables

    def _call(self, where: str, fn, *args) -> None:
        if self._index == _current_device():
            rc = fn(*args, _raw_stream(self._index))
            if rc:
                _native.check(rc, where)
        else:
            _elsewhere(self._index, where, fn, *args)

    def _rows(self, batch: int, slot_ids, lens):
        """Pointers of the batch's block-table rows, lengths and slots, and the tensors to keep alive: tables and lengths
        are stored per slot, the library indexes them per batch row. The gather refuses slots that are not there."""
        tables, by_slot = self.block_tables, lens is None
        if by_slot:
            lens = self.seq_lens
        at = _int32(lens, "sequence lengths", self._index)
        if slot_ids is None:
            if tables.shape[0] < batch or lens.numel() < batch:
                raise RuntimeError(f"a batch of {batch} exceeds the {tables.shape[0]} block-table rows / {lens.numel()} lengths")
            return tables.data_ptr(), at, 0, (tables, lens)
        slots = _int32(slot_ids, "slot_ids", self._index)
        if slot_ids.numel() != batch:
            raise RuntimeError(f"slot_ids holds {slot_ids.numel()} entries for a batch of {batch}")
        rows = tables.shape[0]
        if by_slot:
            rows = min(rows, lens.numel())
        elif lens.numel() < batch:
            raise RuntimeError(f"a batch of {batch} exceeds the {lens.numel()} lengths")
        picked, lengths = tables.new_empty((batch, self.max_blocks_per_seq)), tables.new_empty((batch,))
        args = (tables.data_ptr(), self.max_blocks_per_seq, at, int(by_slot), rows, slots, batch, picked.data_ptr(), lengths.data_ptr())
        self._call("kivi_b200_q8_gather_slots", self._gather, *args)
        return picked.data_ptr(), lengths.data_ptr(), slots, (picked, lengths)

    def _token_rows(self, t: torch.Tensor, name: str, heads: int) -> tuple[int, int]:
        """Checks ``[tokens, heads, head_dim]`` fp16 rows that are contiguous within a token; tokens, stride in elements."""
        if t.dtype is not torch.float16:
            raise TypeError(f"{name} must be torch.float16")
        d = self.layout.head_dim
        if t.dim() != 3 or t.get_device() != self._index:
            raise RuntimeError(f"{name} must be [tokens, {heads}, {d}] on {self.device}")
        n, h, width = t.shape
        if h != heads or width != d:
            raise RuntimeError(f"{name} must be [tokens, {heads}, {d}] on {self.device}")
        step, head, one = t.stride()
        if one != 1 or (head != d and heads > 1):
            raise RuntimeError(f"{name} must be contiguous within a token")
        return n, step if n > 1 else heads * d

    def write(self, new_k: torch.Tensor, new_v: torch.Tensor, new_offsets: torch.Tensor, *, max_new_per_seq: int,
              max_start_seq_len: int, slot_ids: torch.Tensor | None = None, start_seq_lens: torch.Tensor | None = None,
              advance: bool = True) -> None:
        """Append rows ``new_offsets[i]:new_offsets[i+1]`` of ``new_k/new_v [total, NKV, D]`` (fp16; token rows may be
        strided, as slices of a fused projection are) to sequence i. Lengths are read from, and with ``advance``
        updated in, ``self.seq_lens``; with ``start_seq_lens`` they are the caller's and nothing is updated."""
        nkv = self.layout.num_kv_heads
        total, ks = self._token_rows(new_k, "new_k", nkv)
        other, vs = self._token_rows(new_v, "new_v", nkv)
        if total != other:
            raise RuntimeError("new_k and new_v must hold the same tokens")
        offsets = _int32(new_offsets, "new_offsets", self._index)
        n = new_offsets.numel() - 1
        tables, starts, slots, keep = self._rows(n, slot_ids, start_seq_lens)
        index, geom, cache = self._index, self._geom_ref, self._cache_ref
        if index == _current_device():
            rc = self._write(geom, cache, new_k.data_ptr(), new_v.data_ptr(), ks, vs, tables, self.max_blocks_per_seq, starts, offsets,
                             slots, n, total, max_new_per_seq, max_start_seq_len, _raw_stream(index))
            if rc:
                _native.check(rc, "kivi_b200_q8_cache_write")
        else:
            _elsewhere(index, "kivi_b200_q8_cache_write", self._write, geom, cache, new_k.data_ptr(), new_v.data_ptr(), ks, vs, tables,
                       self.max_blocks_per_seq, starts, offsets, slots, n, total, max_new_per_seq, max_start_seq_len)
        if advance and start_seq_lens is None:
            if slot_ids is None:
                self.seq_lens[:n] += new_offsets[1:] - new_offsets[:-1]
            else:
                rows = min(self.block_tables.shape[0], self.seq_lens.numel())
                self._call("kivi_b200_q8_advance_slots", self._advance, self.seq_lens.data_ptr(), rows, slots, offsets, n)

    def read(self, row_offsets: torch.Tensor, first_rows: torch.Tensor, seq_lens: torch.Tensor | None = None, *, total: int,
             max_rows_per_seq: int, slot_ids: torch.Tensor | None = None, k_out: torch.Tensor | None = None,
             v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """What the cache holds, as fp16 ``[total, NKV, D]`` tensors: rows ``row_offsets[i]:row_offsets[i+1]`` receive
        tokens ``first_rows[i]`` onwards of sequence i, zeros behind its last token."""
        shape = (total, self.layout.num_kv_heads, self.layout.head_dim)
        if k_out is None:
            k_out = self.tensors.K_TAIL.new_empty(shape)
        elif k_out.dtype is not torch.float16 or k_out.shape != shape or not k_out.is_contiguous() or k_out.get_device() != self._index:
            raise TypeError(f"k_out must be a contiguous torch.float16 tensor {shape} on {self.device}")
        if v_out is None:
            v_out = self.tensors.K_TAIL.new_empty(shape)
        elif v_out.dtype is not torch.float16 or v_out.shape != shape or not v_out.is_contiguous() or v_out.get_device() != self._index:
            raise TypeError(f"v_out must be a contiguous torch.float16 tensor {shape} on {self.device}")
        offsets, first = _int32(row_offsets, "row_offsets", self._index), _int32(first_rows, "first_rows", self._index)
        n = row_offsets.numel() - 1
        if first_rows.numel() < n:
            raise RuntimeError(f"first_rows holds {first_rows.numel()} entries for a batch of {n}")
        tables, lens, slots, keep = self._rows(n, slot_ids, seq_lens)
        index, geom, cache = self._index, self._geom_ref, self._cache_ref
        if index == _current_device():
            rc = self._read(geom, cache, tables, self.max_blocks_per_seq, lens, slots, offsets, first, n, total, max_rows_per_seq,
                            k_out.data_ptr(), v_out.data_ptr(), _raw_stream(index))
            if rc:
                _native.check(rc, "kivi_b200_q8_cache_read")
        else:
            _elsewhere(index, "kivi_b200_q8_cache_read", self._read, geom, cache, tables, self.max_blocks_per_seq, lens, slots, offsets,
                       first, n, total, max_rows_per_seq, k_out.data_ptr(), v_out.data_ptr())
        return k_out, v_out

    def _ask_workspace(self, sizes: tuple) -> int:
        """Bytes for a call of these sizes, by the plan for this cache's device; the last sizes asked for are kept."""
        with torch.cuda.device(self._index):
            size = self._workspace_of(self._geom_ref, *sizes)
        if len(self._workspace_bytes) >= 64:   # a batch that grows by a token a step never asks for the same sizes again
            self._workspace_bytes.clear()
        self._workspace_bytes[sizes] = size
        return size

    def attend(self, q: torch.Tensor, out: torch.Tensor | None = None, *, max_seq_len: int, window: int = 0, sinks: int = 0,
               scale: float | None = None, q_offsets: torch.Tensor | None = None, max_q_per_seq: int = 1,
               page_mass: torch.Tensor | None = None, slot_ids: torch.Tensor | None = None,
               seq_lens: torch.Tensor | None = None) -> torch.Tensor:
        """Softmax attention of every sequence's last tokens over its cache (which holds them already).

        ``q [tokens, NH, D]`` (fp16, token rows may be strided): one token per sequence, or with ``q_offsets`` rows
        ``q_offsets[i]:q_offsets[i+1]``, at most ``max_q_per_seq``, the last ones of sequence i. Token i sees token
        j <= i if ``j < sinks`` or ``j > i - window``; ``window=0`` is no window. ``out`` is fp32, or fp16 when an fp16
        tensor is passed; rows that belong to no sequence, or to one that is refused, are left as they are (zeros without
        ``out``). ``page_mass`` (fp32 ``[batch, NKV, width]``, single tokens only; row i belongs to row i of the
        batch, whatever its slot) grows by the weight every page got. ``scale`` defaults to 1 / sqrt(D). A length above
        ``max_seq_len`` is taken as ``max_seq_len``, a negative one as 0; both are counted (``rejected_indices``)."""
        total, stride = self._token_rows(q, "q", self.layout.num_q_heads)
        if out is None:   # with offsets, rows of no sequence and of one that the device refuses are not written: zeros
            make = torch.empty if q_offsets is None else torch.zeros
            out = make(q.shape, dtype=torch.float32, device=self.device)
        half = out.dtype is torch.float16
        if not (half or out.dtype is torch.float32) or out.shape != q.shape or not out.is_contiguous() or out.get_device() != self._index:
            raise TypeError("out must be a contiguous torch.float32 or float16 tensor shaped like q")
        if scale is None:
            scale = 0.0
        elif not 0.0 < scale < 1e30:
            raise ValueError("scale must be positive and finite")
        if q_offsets is None:
            batch, offsets = total, 0
        else:
            batch, offsets = q_offsets.numel() - 1, _int32(q_offsets, "q_offsets", self._index)
        tables, lens, slots, keep = self._rows(batch, slot_ids, seq_lens)
        mass = mass_width = 0
        if page_mass is not None:
            if q_offsets is not None:
                raise RuntimeError("page_mass goes with one token per sequence")
            _check_mass(page_mass, batch, self.layout.num_kv_heads, self._index)
            mass, mass_width = page_mass.data_ptr(), page_mass.shape[2]
        sizes = (batch, max_q_per_seq, max_seq_len, window, sinks, page_mass is not None)
        size = self._workspace_bytes.get(sizes)
        if size is None:
            size = self._ask_workspace(sizes)
        workspace, at = None, 0
        if size:   # of this call alone: the allocator hands it on in stream order, or keeps it for a graph under capture
            workspace = torch.empty(size, dtype=torch.uint8, device=self.device)
            at = workspace.data_ptr()
        if half:
            out32, out16 = 0, out.data_ptr()
        else:
            out32, out16 = out.data_ptr(), 0
        index, geom, cache = self._index, self._geom_ref, self._cache_ref
        if index == _current_device():
            rc = self._attention(geom, cache, q.data_ptr(), stride, offsets, total, tables, self.max_blocks_per_seq, lens, slots, batch,
                                 max_q_per_seq, max_seq_len, window, sinks, scale, mass, mass_width, out32, out16, at, size,
                                 _raw_stream(index))
            if rc:
                _native.check(rc, "kivi_b200_q8_attention")
        else:
            _elsewhere(index, "kivi_b200_q8_attention", self._attention, geom, cache, q.data_ptr(), stride, offsets, total, tables,
                       self.max_blocks_per_seq, lens, slots, batch, max_q_per_seq, max_seq_len, window, sinks, scale, mass, mass_width,
                       out32, out16, at, size)
        return out

    def evict(self, page_mass: torch.Tensor, *, budget: int, first: int = 0, recent: int = 0, max_seq_len: int,
              install: bool = True) -> Q8Eviction:
        """``evict_pages`` on this cache's tables and lengths (one row per slot); with ``install`` the results replace
        them, and ``page_mass`` is updated in place. The pages named in ``freed`` belong to nobody afterwards.

        ``page_mass`` is ``[slots, NKV, width]``: where ``attend`` ran on some slots only, its rows go to their slots'.
        The installed tables keep the ids that were entered for the open block and for growth: they move up behind the
        kept pages. The columns that this empties hold -1, so a block that would complete there is refused and counted
        until the caller enters a page (``Q8Eviction.block_tables`` has 0 behind the kept pages)."""
        _check_mass(page_mass, self.block_tables.shape[0], self.layout.num_kv_heads, self._index)
        r = evict_pages(self.block_tables, self.seq_lens, page_mass, block_size=self.layout.block_size, budget=budget, first=first,
                        recent=recent, max_seq_len=max_seq_len)
        if install:
            block, width = self.layout.block_size, self.max_blocks_per_seq
            kept = (r.seq_lens // block)[:, None]
            column = torch.arange(width, dtype=torch.int32, device=self.device)
            source = column + (self.seq_lens // block)[:, None] - kept
            behind = self.block_tables.gather(1, source.clamp(0, max(width - 1, 0)).long()).masked_fill_(source >= width, -1)
            self.block_tables.copy_(torch.where(column < kept, r.block_tables, behind))
            self.seq_lens.copy_(r.seq_lens)
            page_mass.copy_(r.page_mass)
        return r


def _check_mass(mass: torch.Tensor, batch: int, nkv: int | None, index: int) -> None:
    if mass.dtype is not torch.float32 or mass.dim() != 3 or not mass.is_contiguous() or mass.get_device() != index:
        raise TypeError(f"page_mass must be a contiguous torch.float32 [batch, kv heads, width] tensor on cuda:{index}")
    if mass.shape[0] != batch or (nkv is not None and mass.shape[1] != nkv):
        raise RuntimeError(f"page_mass must be [{batch}, {'kv heads' if nkv is None else nkv}, width], got {tuple(mass.shape)}")


def evict_pages(block_tables: torch.Tensor, seq_lens: torch.Tensor, page_mass: torch.Tensor, *, block_size: int, budget: int,
                first: int = 0, recent: int = 0, max_seq_len: int) -> Q8Eviction:
    """Keep ``budget`` complete pages of every sequence that has more: its first ``first`` and last ``recent`` ones and, of
    the others, those with the largest ``page_mass [batch, NKV, width]`` over all kv heads (ties: the lowest page). A
    sequence whose length lies outside 0 .. ``max_seq_len`` goes through unchanged and is counted. The inputs stay as they are. Works on the tables of any paged cache whose pages are self-contained."""
    index = block_tables.get_device()
    if index < 0:
        raise RuntimeError("evict_pages needs CUDA tensors; its kernel has no CPU path")
    tables, lens = _int32(block_tables, "block_tables", index), _int32(seq_lens, "seq_lens", index)
    if block_tables.dim() != 2 or seq_lens.numel() != block_tables.shape[0]:
        raise TypeError("block_tables must be [batch, width] and seq_lens [batch]")
    batch, width = block_tables.shape
    _check_mass(page_mass, batch, None, index)
    _, nkv, mass_width = page_mass.shape
    mass = torch.empty_like(page_mass)
    new_tables, freed = torch.empty_like(block_tables), torch.empty_like(block_tables)
    new_lens, counts = torch.empty_like(seq_lens), torch.empty_like(seq_lens)
    args = (nkv, block_size, tables, width, lens, page_mass.data_ptr(), mass_width, batch, max_seq_len, budget, first, recent,
            new_tables.data_ptr(), new_lens.data_ptr(), mass.data_ptr(), freed.data_ptr(), counts.data_ptr())
    fn = _native.lib().kivi_b200_q8_evict
    if index == _current_device():
        rc = fn(*args, _raw_stream(index))
        if rc:
            _native.check(rc, "kivi_b200_q8_evict")
    else:
        _elsewhere(index, "kivi_b200_q8_evict", fn, *args)
    return Q8Eviction(new_tables, new_lens, mass, freed, counts)


def rejected_indices() -> int:
    """Sequences and ids the 8-bit cache's calls refused on the current device since the library was loaded."""
    out = ctypes.c_uint32(0)
    _native.check(_native.lib().kivi_b200_q8_rejected_indices(ctypes.byref(out)), "kivi_b200_q8_rejected_indices")
    return int(out.value)


def wait_failures() -> int:
    """CTAs of the attention kernel for many query rows that gave up a bounded wait on the current device since the library
    was loaded (their output is undefined); 0 in any healthy run."""
    out = ctypes.c_uint32(0)
    _native.check(_native.lib().kivi_b200_q8_wait_failures(ctypes.byref(out)), "kivi_b200_q8_wait_failures")
    return int(out.value)

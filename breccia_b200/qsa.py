"""Host-side mirror of the reference's `breccia-kernels::qsa` operator surface over libbreccia_kv.

Same names, argument meaning and error behaviour as the reference's `QsaState` / `QsaWorkspace` /
`Qsa` (crates/breccia-kernels/src/qsa/mod.rs:294-311, 606-650, 1107-1156, 1365-1580), so tests read
like the reference's own; the difference is that ONE pool per GPU is shared by all sequences and a
sequence is a block table into it.  `DecodeBatch` is the batched form the engine's decode loop uses.

torch is used for device buffers and streams only; every operator is a call through the C ABI.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

from . import _lib
from ._lib import BrcError, DTYPE_F16, DTYPE_F32

PAGE_CELLS = 16  # crates/breccia-kernels/src/qsa/mod.rs:114


def _ptr(t) -> C.c_void_p:
    return C.c_void_p(t.data_ptr()) if t is not None else C.c_void_p(0)


def _stream_ptr(stream=None) -> C.c_void_p:
    s = stream if stream is not None else torch.cuda.current_stream()
    return C.c_void_p(s.cuda_stream)


def _u32_array(a) -> np.ndarray:
    return np.ascontiguousarray(a, dtype=np.uint32)


class KvPool:
    """Paged f16 K/V pools of all layers on one GPU plus the page allocator (brc_pool).  v_q8: V page bodies
    as q8_0 blocks (the reference's VLayout::Q8_0, qsa/mod.rs:245-349): K stays binary16, append quantises
    from f32, and every operator reads the blocks.  kv8: K and V pages as 8-bit codes ("e4m3" or "int8") with one
    power-of-two scale per page, kv head and side, for kv8_append / kv8_read / kv8_attend (and DecodeBatch.append /
    attend)."""

    def __init__(self, device: int, n_layers: int, n_kv_head: int, head_dim: int, n_pages: int,
                 page_tokens: int = PAGE_CELLS, bookkeeping_only: bool = False, v_q8: bool = False,
                 kv8: str | None = None):
        self._h = C.c_void_p()
        self.v_q8, self.kv8 = v_q8, kv8
        if kv8 is not None:
            if v_q8 or bookkeeping_only or kv8 not in _lib.KV8_CODES:
                raise BrcError(_lib.ERR_INVALID, f"kv8={kv8!r}: \"e4m3\" or \"int8\", and neither v_q8 nor bookkeeping_only with it")
            _lib.call("brc_pool_create_kv8", device, n_layers, n_kv_head, head_dim, page_tokens, n_pages, _lib.KV8_CODES[kv8],
                      C.byref(self._h))
        elif v_q8:
            _lib.call("brc_pool_create_q8v", device, n_layers, n_kv_head, head_dim, page_tokens, n_pages, C.byref(self._h))
        elif bookkeeping_only:
            _lib.call("brc_pool_create_bookkeeping", n_layers, n_kv_head, head_dim, page_tokens, n_pages,
                      C.byref(self._h))
        else:
            _lib.call("brc_pool_create", device, n_layers, n_kv_head, head_dim, page_tokens, n_pages,
                      C.byref(self._h))
        self.device = device
        self.n_layers, self.n_kv_head, self.head_dim = n_layers, n_kv_head, head_dim
        self.n_pages, self.page_tokens = n_pages, page_tokens
        self.half_page_bytes = n_kv_head * page_tokens * head_dim * 2
        if kv8 is not None:   # one byte per value, then the heads' scales, to a multiple of 128 bytes
            self.half_page_bytes = (n_kv_head * (page_tokens * head_dim + 4) + 127) // 128 * 128

    # -- lifetime
    @property
    def handle(self) -> C.c_void_p:
        if not self._h:
            raise BrcError(_lib.ERR_INVALID, "pool already released")
        return self._h

    def release(self) -> None:
        if self._h:
            _lib.call("brc_pool_destroy", self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass

    def bytes(self) -> int:
        out = C.c_uint64()
        _lib.call("brc_pool_bytes", self.handle, C.byref(out))
        return out.value

    def zero(self, stream=None) -> None:
        _lib.call("brc_pool_zero", self.handle, _stream_ptr(stream))

    def poison_nan(self, stream=None) -> None:
        _lib.call("brc_pool_poison_nan", self.handle, _stream_ptr(stream))

    def check(self, stream=None) -> None:
        """Synchronise and raise if any kernel refused an index, gave up a wait or met an infinity or NaN in a quantising write."""
        _lib.call("brc_pool_check", self.handle, _stream_ptr(stream))

    def k_ptr(self, layer: int) -> int:
        out = C.c_void_p()
        _lib.call("brc_pool_k_ptr", self.handle, layer, C.byref(out))
        return out.value

    def v_ptr(self, layer: int) -> int:
        out = C.c_void_p()
        _lib.call("brc_pool_v_ptr", self.handle, layer, C.byref(out))
        return out.value

    def read(self, which: int, layer: int) -> np.ndarray:
        """Whole K (0) or V (1) pool of a layer as uint16 [n_pages, n_kv, page_tokens, head_dim]."""
        if which == 1 and self.v_q8:   # raw q8_0 rows: [n_pages * n_kv * page_tokens, head_dim / 32 * 36] bytes
            out = np.empty((self.n_pages * self.n_kv_head * self.page_tokens, self.head_dim // 32 * 36), np.uint8)
        elif self.kv8 is not None:             # whole half pages: codes, then scales
            out = np.empty((self.n_pages, self.half_page_bytes), np.uint8)
        else:
            out = np.empty((self.n_pages, self.n_kv_head, self.page_tokens, self.head_dim), np.uint16)
        _lib.call("brc_pool_read", self.handle, which, layer, 0, out.ctypes.data_as(C.c_void_p), out.nbytes,
                  _stream_ptr())
        return out

    def write(self, which: int, layer: int, data: np.ndarray, byte_offset: int = 0) -> None:
        data = np.ascontiguousarray(data)
        _lib.call("brc_pool_write", self.handle, which, layer, byte_offset, data.ctypes.data_as(C.c_void_p),
                  data.nbytes, _stream_ptr())

    def kv8_view(self, which: int, layer: int) -> tuple[torch.Tensor, torch.Tensor]:
        """The K (0) or V (1) pages of a layer of an 8-bit pool where they lie, as torch tensors: codes
        [n_pages, n_kv, page_tokens, head_dim] (float8_e4m3fn or int8) and scales [n_pages, n_kv] f32.  Views of the
        pool's own memory: valid until release(), written through at once."""
        if self.kv8 is None:
            raise BrcError(_lib.ERR_UNSUPPORTED, "kv8_view: the pool's pages are not 8-bit")
        if which not in (0, 1):
            raise BrcError(_lib.ERR_INVALID, f"kv8_view: which = {which} (0 = K, 1 = V)")
        ptr = self.v_ptr(layer) if which else self.k_ptr(layer)
        n, rows = self.n_pages * self.half_page_bytes, self.n_kv_head * self.page_tokens * self.head_dim

        class Memory:
            __cuda_array_interface__ = {"shape": (n,), "typestr": "|u1", "data": (ptr, False), "version": 3, "strides": None}

        raw = torch.as_tensor(Memory(), device=f"cuda:{self.device}")
        codes = raw.as_strided((self.n_pages, self.n_kv_head, self.page_tokens, self.head_dim),
                               (self.half_page_bytes, self.page_tokens * self.head_dim, self.head_dim, 1))
        scales = raw.view(torch.float32).as_strided((self.n_pages, self.n_kv_head), (self.half_page_bytes // 4, 1), rows // 4)
        return codes.view(torch.float8_e4m3fn if self.kv8 == "e4m3" else torch.int8), scales

    # -- allocator
    def alloc(self, n: int) -> np.ndarray:
        ids = np.empty(n, np.uint32)
        _lib.call("brc_pages_alloc", self.handle, n, ids.ctypes.data_as(C.POINTER(C.c_uint32)))
        return ids

    def retain(self, ids) -> None:
        ids = _u32_array(ids)
        _lib.call("brc_pages_retain", self.handle, ids.ctypes.data_as(C.POINTER(C.c_uint32)), ids.size)

    def release_pages(self, ids) -> None:
        ids = _u32_array(ids)
        _lib.call("brc_pages_release", self.handle, ids.ctypes.data_as(C.POINTER(C.c_uint32)), ids.size)

    def refcount(self, page: int) -> int:
        out = C.c_uint32()
        _lib.call("brc_page_refcount", self.handle, page, C.byref(out))
        return out.value

    def free_count(self) -> int:
        out = C.c_uint32()
        _lib.call("brc_pages_free_count", self.handle, C.byref(out))
        return out.value

    # -- page movers
    def copy_pages(self, src_ids, dst_ids, stream=None) -> None:
        src = torch.as_tensor(_u32_array(src_ids).astype(np.int32), device=f"cuda:{self.device}")
        dst = torch.as_tensor(_u32_array(dst_ids).astype(np.int32), device=f"cuda:{self.device}")
        _lib.call("brc_page_copy", self.handle, _ptr(src), _ptr(dst), src.numel(), _stream_ptr(stream))
        torch.cuda.current_stream().synchronize()  # src/dst tensors die with this frame

    def fork(self, parent_table, n_tokens: int, stream=None):
        """Copy-on-write fork -> (child table, id of the private last page or None)."""
        parent = _u32_array(parent_table)
        n_pages = (n_tokens + self.page_tokens - 1) // self.page_tokens
        child = np.zeros(max(n_pages, 1), np.uint32)
        fresh = C.c_uint32()
        _lib.call("brc_seq_fork", self.handle, parent.ctypes.data_as(C.POINTER(C.c_uint32)), n_tokens,
                  child.ctypes.data_as(C.POINTER(C.c_uint32)), C.byref(fresh), _stream_ptr(stream))
        return child[:n_pages], (None if fresh.value == 0xFFFFFFFF else fresh.value)

    def gather(self, layer: int, block_table_dev: torch.Tensor, n_tokens: int, stream=None):
        """Cells 0..n_tokens-1 of one sequence -> (K, V) tensors [n_tokens, n_kv, head_dim] holding binary16
        bits; on a q8_0 V pool V is the stored rows, uint8 [n_tokens, n_kv, head_dim / 32 * 36]."""
        dev = f"cuda:{self.device}"
        k = torch.empty((n_tokens, self.n_kv_head, self.head_dim), dtype=torch.float16, device=dev)
        v = torch.empty((n_tokens, self.n_kv_head, self.head_dim // 32 * 36), dtype=torch.uint8, device=dev) if self.v_q8 else torch.empty_like(k)
        _lib.call("brc_page_gather", self.handle, layer, _ptr(block_table_dev), block_table_dev.numel(), n_tokens,
                  _ptr(k), _ptr(v), _stream_ptr(stream))
        return k, v


class QsaState:
    """One sequence's view of one layer: a block table into the shared pool
    (reference: per-layer, per-sequence pools behind an identity page table, qsa/mod.rs:294-311)."""

    def __init__(self, pool: KvPool, capacity_cells: int, layer: int = 0, block_table=None):
        self.pool = pool
        self.layer = layer
        n_pages = (capacity_cells + PAGE_CELLS - 1) // PAGE_CELLS
        self.capacity_cells = n_pages * PAGE_CELLS  # rounded up to whole pages like the reference
        self._owned = block_table is None
        self.page_table = pool.alloc(n_pages) if block_table is None else _u32_array(block_table)[:n_pages].copy()
        if self.page_table.size != n_pages:
            raise BrcError(_lib.ERR_INVALID, f"block table of {self.page_table.size} pages for {n_pages} needed")
        self.page_table_dev = torch.as_tensor(self.page_table.astype(np.int32), device=f"cuda:{pool.device}")

    def bytes(self) -> int:
        return self.page_table.size * 2 * self.pool.half_page_bytes

    def release(self) -> None:
        if self._owned and self.page_table is not None:
            self.pool.release_pages(self.page_table)
        self.page_table = None


class QsaWorkspace:
    """Device buffers of one call (reference: qsa/mod.rs:606-650): k_cur / v_cur [T, n_kv*hd] f32,
    q [T, n_head, hd] (f32, or f16 when q_dtype says so), q_full [T, n_head*2*hd] f32 whose second
    half per head is the gate, attn_out [T, n_head, hd] f32."""

    def __init__(self, pool: KvPool, tokens: int, n_head: int, q_dtype: int = DTYPE_F32):
        dev = f"cuda:{pool.device}"
        hd, nkv = pool.head_dim, pool.n_kv_head
        self.tokens, self.n_head, self.q_dtype = tokens, n_head, q_dtype
        self.k_cur = torch.zeros((tokens, nkv * hd), dtype=torch.float32, device=dev)
        self.v_cur = torch.zeros_like(self.k_cur)
        self.q = torch.zeros((tokens, n_head, hd), dtype=torch.float32 if q_dtype == DTYPE_F32 else torch.float16,
                             device=dev)
        self.q_full = None  # set to a [T, n_head*2*hd] f32 tensor to enable the gate
        self.attn_out = torch.zeros((tokens, n_head, hd), dtype=torch.float32, device=dev)
        self.seq_lens = torch.zeros(tokens, dtype=torch.int32, device=dev)
        self.pos0 = torch.zeros(1, dtype=torch.int32, device=dev)
        ws_bytes = C.c_uint64()
        _lib.call("brc_decode_workspace_bytes", pool.handle, tokens, n_head, C.byref(ws_bytes))
        self.scratch = torch.empty(ws_bytes.value, dtype=torch.uint8, device=dev)
        self.tables = None


class Qsa:
    """Operator object (reference: `Qsa`, qsa/mod.rs:746-1580) — stateless here."""

    def __init__(self, pool: KvPool, n_head: int):
        self.pool, self.n_head = pool, n_head
        self.scale = 1.0 / math.sqrt(pool.head_dim)

    def workspace(self, tokens: int, q_dtype: int = DTYPE_F32) -> QsaWorkspace:
        return QsaWorkspace(self.pool, tokens, self.n_head, q_dtype)

    def kv_append(self, state: QsaState, ws: QsaWorkspace, pos0: int) -> None:
        """Append ws.tokens cells at pos0.. (reference: Qsa::kv_append, qsa/mod.rs:1107-1156)."""
        if pos0 + ws.tokens > state.capacity_cells:
            raise BrcError(_lib.ERR_CAPACITY,
                           f"kv_append would write cells {pos0}..{pos0 + ws.tokens} but the cache holds "
                           f"{state.capacity_cells} (a write past the page table reads an unmapped page index "
                           "and can scribble over live cells)")
        ws.pos0.fill_(pos0)
        _lib.call("brc_kv_append", self.pool.handle, state.layer, _ptr(state.page_table_dev),
                  state.page_table_dev.numel(), _ptr(ws.pos0), 1, ws.tokens, None, ws.tokens, pos0 + ws.tokens,
                  _ptr(ws.k_cur), _ptr(ws.v_cur), DTYPE_F32, _stream_ptr())

    def topk_dense(self, ws: QsaWorkspace, pos0: int) -> None:
        """Dense selection: every cell 0..=pos0+t for row t (reference: qsa/mod.rs:1365-1376).  The
        selection is carried as per-row lengths instead of an id list."""
        ws.seq_lens.copy_(torch.arange(pos0 + 1, pos0 + 1 + ws.tokens, dtype=torch.int32))

    def attend_apply(self, state: QsaState, ws: QsaWorkspace, pos0: int) -> None:
        """Scores, softmax, probability-weighted V and gate in one pass (reference: Qsa::attend then
        Qsa::apply, qsa/mod.rs:1382-1580).  Row t sees cells <= pos0 + t."""
        if pos0 + ws.tokens > state.capacity_cells:
            raise BrcError(_lib.ERR_CAPACITY, f"attend at cells {pos0}..{pos0 + ws.tokens} but the cache holds "
                                              f"{state.capacity_cells}")
        hd = self.pool.head_dim
        if ws.tables is None or ws.tables.shape[1] != state.page_table_dev.numel():
            ws.tables = state.page_table_dev.unsqueeze(0).repeat(ws.tokens, 1).contiguous()
        else:
            ws.tables.copy_(state.page_table_dev.unsqueeze(0).expand_as(ws.tables))
        gate, stride = None, 0
        if ws.q_full is not None:
            gate, stride = ws.q_full.view(-1)[hd:], 2 * hd
        _lib.call("brc_paged_decode_attn", self.pool.handle, state.layer, _ptr(ws.q), ws.q_dtype, self.n_head,
                  _ptr(gate), stride, _ptr(ws.tables), ws.tables.shape[1], _ptr(ws.seq_lens), ws.tokens,
                  pos0 + ws.tokens, self.scale, _ptr(ws.attn_out), _ptr(ws.scratch), ws.scratch.numel(),
                  _stream_ptr())

    # The reference splits the work into `attend` (scores + softmax) and `apply` (weighted V + gate);
    # the fused kernel does both, so `attend` runs it and `apply` is the completed second half.
    def attend(self, state: QsaState, ws: QsaWorkspace, pos0: int) -> None:
        self.attend_apply(state, ws, pos0)

    def apply(self, state: QsaState, ws: QsaWorkspace, pos0: int) -> None:
        return None


class DecodeBatch:
    """A batch of sequences decoding together from one shared pool: block tables [n_seqs, stride],
    lengths, and the workspace of the split-KV kernel.  One `append` + `attend` per layer per step."""

    def __init__(self, pool: KvPool, n_head: int, block_tables: np.ndarray, seq_lens: np.ndarray,
                 q_dtype: int = DTYPE_F16):
        dev = f"cuda:{pool.device}"
        self.pool, self.n_head, self.q_dtype = pool, n_head, q_dtype
        bt = _u32_array(block_tables)
        self.n_seqs, self.table_stride = bt.shape
        self.capacity = self.table_stride * pool.page_tokens
        self.seq_lens_host = np.asarray(seq_lens, np.int64).copy()
        self.block_tables = torch.as_tensor(bt.astype(np.int32), device=dev)
        self.seq_lens = torch.as_tensor(self.seq_lens_host.astype(np.int32), device=dev)
        self.pos0 = torch.empty_like(self.seq_lens)
        ws_bytes = C.c_uint64()
        _lib.call("brc_decode_workspace_bytes", pool.handle, self.n_seqs, n_head, C.byref(ws_bytes))
        # partial slots for every layer: brc_decode_step covers all layers of a step in one launch
        self.scratch = torch.empty(pool.n_layers * ws_bytes.value, dtype=torch.uint8, device=dev)
        self.scale = 1.0 / math.sqrt(pool.head_dim)

    def begin_step(self) -> None:
        """One new token per sequence: cells seq_len .. are about to be appended in every layer."""
        if int(self.seq_lens_host.max()) + 1 > self.capacity:
            raise BrcError(_lib.ERR_CAPACITY, f"kv_append would write cell {int(self.seq_lens_host.max())} but each "
                                              f"block table holds {self.capacity}")
        self.pos0.copy_(self.seq_lens)
        self.seq_lens_host += 1
        self.seq_lens.add_(1)

    def append(self, layer: int, k_new: torch.Tensor, v_new: torch.Tensor, src_dtype: int = DTYPE_F32) -> None:
        """k_new / v_new: [n_seqs, n_kv*hd] at cell pos0[s] of each sequence."""
        _lib.call("brc_kv_append", self.pool.handle, layer, _ptr(self.block_tables), self.table_stride,
                  _ptr(self.pos0), self.n_seqs, 1, None, self.n_seqs, int(self.seq_lens_host.max()), _ptr(k_new),
                  _ptr(v_new), src_dtype, _stream_ptr())

    def attend(self, layer: int, q: torch.Tensor, out: torch.Tensor, gate: torch.Tensor | None = None,
               gate_head_stride: int = 0) -> None:
        _lib.call("brc_paged_decode_attn", self.pool.handle, layer, _ptr(q), self.q_dtype, self.n_head, _ptr(gate),
                  gate_head_stride, _ptr(self.block_tables), self.table_stride, _ptr(self.seq_lens), self.n_seqs,
                  int(self.seq_lens_host.max()), self.scale, _ptr(out), _ptr(self.scratch), self.scratch.numel(),
                  _stream_ptr())

    def step(self, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, out: torch.Tensor, layer0: int = 0,
             kv_dtype: int = DTYPE_F32) -> None:
        """One decode step over the layers q carries: q [L, n_seqs, n_head, hd], k_new / v_new
        [L, n_seqs, n_kv*hd], out [L, n_seqs, n_head, hd] f32.  Positions advance on the device; one
        call into the library (brc_decode_step), asynchronous on the current stream."""
        n_layers = q.shape[0]
        if int(self.seq_lens_host.max()) + 1 > self.capacity:
            raise BrcError(_lib.ERR_CAPACITY, f"decode step would write cell {int(self.seq_lens_host.max())} but each "
                                              f"block table holds {self.capacity}")
        self.seq_lens_host += 1
        _lib.call("brc_decode_step", self.pool.handle, layer0, n_layers, _ptr(self.block_tables), self.table_stride,
                  _ptr(self.seq_lens), _ptr(self.pos0), self.n_seqs, int(self.seq_lens_host.max()), _ptr(q),
                  self.q_dtype, q.stride(0) * q.element_size(), self.n_head, _ptr(k_new), _ptr(v_new), kv_dtype,
                  k_new.stride(0) * k_new.element_size(), None, 0, 0, self.scale, _ptr(out),
                  out.stride(0) * out.element_size(), _ptr(self.scratch), self.scratch.numel(), _stream_ptr())

    def step_part(self, first: int, count: int, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                  out: torch.Tensor, layer0: int = 0, kv_dtype: int = DTYPE_F32) -> None:
        """Layers [first, first + count) of the step `step` would run on the same tensors
        (brc_decode_step_part); the part with first == 0 advances the positions."""
        if first == 0:
            if int(self.seq_lens_host.max()) + 1 > self.capacity:
                raise BrcError(_lib.ERR_CAPACITY, f"decode step would write cell {int(self.seq_lens_host.max())} but "
                                                  f"each block table holds {self.capacity}")
            self.seq_lens_host += 1
        _lib.call("brc_decode_step_part", self.pool.handle, layer0, q.shape[0], first, count, _ptr(self.block_tables),
                  self.table_stride, _ptr(self.seq_lens), _ptr(self.pos0), self.n_seqs, int(self.seq_lens_host.max()),
                  _ptr(q), self.q_dtype, q.stride(0) * q.element_size(), self.n_head, _ptr(k_new), _ptr(v_new), kv_dtype,
                  k_new.stride(0) * k_new.element_size(), None, 0, 0, self.scale, _ptr(out),
                  out.stride(0) * out.element_size(), _ptr(self.scratch), self.scratch.numel(), _stream_ptr())

    def host_staging(self, n_layers: int, kv_dtype: int = DTYPE_F32) -> torch.Tensor:
        """The device buffer step_host needs for steps of n_layers layers."""
        need = C.c_uint64()
        _lib.call("brc_decode_step_host_staging_bytes", self.pool.handle, n_layers, self.n_seqs, self.n_head, self.q_dtype,
                  kv_dtype, C.byref(need))
        return torch.empty(need.value, dtype=torch.uint8, device=self.seq_lens.device)

    def step_host(self, q_host: torch.Tensor, k_host: torch.Tensor, v_host: torch.Tensor, out_host: torch.Tensor,
                  staging: torch.Tensor | None, layer0: int = 0, parts: int = 1, kv_dtype: int = DTYPE_F32,
                  download: bool = False, upload: bool = False) -> None:
        """The same step for a caller whose activations live in host memory, one call into the library
        (brc_decode_step_host).  Pinned q / k / v are read by the kernels where they lie and the attention
        output is stored straight into a pinned out_host; pageable buffers (or `upload` / `download`) go
        through `staging` (from host_staging()).  `parts` > 1 uploads the layers in groups on a second
        stream; on the machines measured the hand-over between the streams cost more than the hidden copy
        saved, so one part is the default.  Returns when out_host is complete."""
        for t in (q_host, k_host, v_host, out_host):
            if t.is_cuda or not t.is_contiguous():
                raise ValueError("step_host takes contiguous host tensors")
        if int(self.seq_lens_host.max()) + 1 > self.capacity:
            raise BrcError(_lib.ERR_CAPACITY, f"decode step would write cell {int(self.seq_lens_host.max())} but each "
                                              f"block table holds {self.capacity}")
        self.seq_lens_host += 1
        _lib.call("brc_decode_step_host", self.pool.handle, layer0, q_host.shape[0], parts,
                  (1 if download else 0) | (2 if upload else 0),
                  _ptr(self.block_tables),
                  self.table_stride, _ptr(self.seq_lens), _ptr(self.pos0), self.n_seqs, int(self.seq_lens_host.max()),
                  _ptr(q_host), self.q_dtype, self.n_head, _ptr(k_host), _ptr(v_host), kv_dtype, self.scale, _ptr(out_host),
                  _ptr(staging), staging.numel() if staging is not None else 0, _ptr(self.scratch), self.scratch.numel(),
                  _stream_ptr())

    def reset_lengths(self, seq_lens) -> None:
        self.seq_lens_host = np.asarray(seq_lens, np.int64).copy()
        self.seq_lens.copy_(torch.as_tensor(self.seq_lens_host.astype(np.int32)))

    def partial(self, layer: int, q: torch.Tensor, partial_out: torch.Tensor) -> None:
        _lib.call("brc_decode_partial", self.pool.handle, layer, _ptr(q), self.q_dtype, self.n_head,
                  _ptr(self.block_tables), self.table_stride, _ptr(self.seq_lens), self.n_seqs,
                  int(self.seq_lens_host.max()), self.scale, _ptr(partial_out), _ptr(self.scratch),
                  self.scratch.numel(), _stream_ptr())


def sparse_attend(pool: KvPool, layer: int, q: torch.Tensor, n_head: int, block_tables: torch.Tensor, pos0: torch.Tensor,
                  rows_per_seq: int, ids: torch.Tensor, counts: torch.Tensor, max_pos_end: int, out: torch.Tensor,
                  gate: torch.Tensor | None = None, gate_head_stride: int = 0) -> None:
    """Attention over selected 4-cell blocks (reference: Qsa::attend + Qsa::apply over the `ids` / `counts` lists of
    its top-k stage, qsa/mod.rs:620-625, 1382-1580).  q [rows, n_head, hd] f32 or f16; ids [rows, max_ids] int32;
    counts [rows]; block_tables [n_seqs, stride]; pos0 [n_seqs]; out [rows, n_head, hd] f32."""
    q_dtype = DTYPE_F32 if q.dtype == torch.float32 else DTYPE_F16
    _lib.call("brc_paged_sparse_attn", pool.handle, layer, _ptr(q), q_dtype, n_head, _ptr(gate), gate_head_stride,
              _ptr(block_tables), block_tables.shape[1], _ptr(pos0), block_tables.shape[0], rows_per_seq, _ptr(ids),
              ids.shape[1], _ptr(counts), max_pos_end, 1.0 / math.sqrt(pool.head_dim), _ptr(out), _stream_ptr())


def topk_blocks(pool: KvPool, scores: torch.Tensor, pos0: torch.Tensor, rows_per_seq: int, topk: int = 512,
                dense: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """The selection lists sparse_attend takes, from indexer scores [rows, n_blocks] f32 (reference: Qsa::topk,
    shaders/qsa_topk.comp): per row the `topk` best blocks in descending score order (ties towards the lower
    block, scores <= -1e29 never), then the row's own block.  Returns (ids [rows, min(n_blocks, topk) + 1] int32,
    counts [rows] int32)."""
    rows, n_blocks = scores.shape
    max_ids = min(n_blocks, topk) + 1
    ids = torch.empty((rows, max_ids), dtype=torch.int32, device=scores.device)
    counts = torch.empty((rows,), dtype=torch.int32, device=scores.device)
    _lib.call("brc_topk_blocks", pool.handle, _ptr(scores), pos0.numel(), rows_per_seq, n_blocks, topk, max_ids, _ptr(pos0),
              1 if dense else 0, _ptr(ids), _ptr(counts), _stream_ptr())
    return ids, counts


IDX_DIM, IDX_BLOCK, IDX_N_HEAD = 128, 4, 4   # crates/breccia-kernels/src/qsa/mod.rs:77-81


class IndexerState:
    """The indexer's key cache of a batch of sequences (reference: `QsaState::idx_pooled` / `idx_tail`, one per
    sequence, qsa/mod.rs:294-311, 353-386): one pooled key per completed 4-cell block and the raw keys of the
    block being filled."""

    def __init__(self, pool: KvPool, n_seqs: int, capacity_cells: int):
        dev = f"cuda:{pool.device}"
        self.pool, self.n_seqs = pool, n_seqs
        self.max_blocks = capacity_cells // IDX_BLOCK + 1          # sizes::max_blocks, qsa/mod.rs:384-387
        self.pooled = torch.zeros((n_seqs, self.max_blocks, IDX_DIM), dtype=torch.float32, device=dev)
        self.tail = torch.zeros((n_seqs, IDX_BLOCK - 1, IDX_DIM), dtype=torch.float32, device=dev)

    def append(self, raw: torch.Tensor, pos0: torch.Tensor, max_pos_end: int, gamma: torch.Tensor, rope_table: torch.Tensor,
               n_rot: int, eps: float = 1e-6) -> None:
        """raw [n_seqs, tokens, 128] f32: this call's raw indexer keys at positions pos0[s] ..: pools every block
        the call completes, then stores the new incomplete block's keys in the tail (Qsa::idx_pool then
        Qsa::idx_tail, the order of Qsa::forward)."""
        n_seqs, tokens = raw.shape[0], raw.shape[1]
        _lib.call("brc_idx_pool", self.pool.handle, _ptr(raw), _ptr(self.tail), _ptr(gamma), _ptr(rope_table), n_rot,
                  rope_table.shape[0], eps, _ptr(pos0), n_seqs, tokens, max_pos_end, IDX_DIM, IDX_BLOCK, _ptr(self.pooled),
                  self.max_blocks, _stream_ptr())
        _lib.call("brc_idx_tail", self.pool.handle, _ptr(raw), _ptr(pos0), n_seqs, tokens, IDX_DIM, IDX_BLOCK, _ptr(self.tail),
                  _stream_ptr())

    def score(self, q: torch.Tensor, pos0: torch.Tensor, rows_per_seq: int, n_blocks: int) -> torch.Tensor:
        """q [rows, idx_n_head, 128] f32 -> scores [rows, n_blocks] f32 (Qsa::idx_score), ready for topk_blocks."""
        rows = q.shape[0]
        scores = torch.empty((rows, n_blocks), dtype=torch.float32, device=q.device)
        _lib.call("brc_idx_score", self.pool.handle, _ptr(q), q.shape[1], _ptr(self.pooled), self.max_blocks, _ptr(pos0),
                  rows // rows_per_seq, rows_per_seq, n_blocks, IDX_DIM, IDX_BLOCK, 1.0 / math.sqrt(IDX_DIM), _ptr(scores),
                  _stream_ptr())
        return scores


_DTYPES = {torch.float32: DTYPE_F32, torch.float16: DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
_WORD_TYPES = (torch.int32, torch.uint32)


def _raw_stream(stream, device: int) -> int:
    """The stream a call goes to: the one given, else the current one of the pool's GPU (whichever GPU is current)."""
    return torch._C._cuda_getCurrentRawStream(device) if stream is None else stream.cuda_stream


def _new(stream, make):
    """make(), in memory of the stream that will write it (the current one's may still be in use by what runs there)."""
    if stream is None:
        return make()
    with torch.cuda.stream(stream):
        return make()


def _dtype(t: torch.dtype, who: str) -> int:
    code = _DTYPES.get(t)
    if code is None:
        raise BrcError(_lib.ERR_INVALID, f"{who}: dtype {t} (float32, float16 or bfloat16)")
    return code


def _token_rows(t: torch.Tensor, heads: int, head_dim: int, who: str) -> int:
    """Elements from one token's row [heads, head_dim] (or [heads * head_dim]) to the next; the row itself is contiguous."""
    row, shape = heads * head_dim, t.shape
    if t.is_contiguous() and len(shape) == 3 and shape[1] == heads and shape[2] == head_dim:
        return row
    ok = (t.dim() == 2 and t.shape[1] == row and t.stride(1) == 1) or \
         (t.dim() == 3 and t.shape[1:] == (heads, head_dim) and t.stride(2) == 1 and (heads == 1 or t.stride(1) == head_dim))
    if not ok:
        raise BrcError(_lib.ERR_INVALID, f"{who}: {tuple(t.shape)} with strides {t.stride()} is not rows of {heads} x {head_dim} values")
    if t.shape[0] <= 1:
        return row
    if t.stride(0) < row:   # one row for all tokens (stride 0, which the library takes for packed rows), or overlapping ones
        raise BrcError(_lib.ERR_INVALID, f"{who}: {tuple(t.shape)} with strides {t.stride()}: tokens share memory")
    return t.stride(0)


def _words(t: torch.Tensor, device: int, who: str, n: int | None = None) -> int:
    """The address of a contiguous array of 32-bit words on the pool's GPU (what positions, lengths, tables and prefixes are)."""
    if t.dtype not in _WORD_TYPES or not t.is_contiguous() or t.get_device() != device:
        raise BrcError(_lib.ERR_INVALID, f"{who}: {t.dtype} {tuple(t.shape)} on {t.device}: contiguous 32-bit words on cuda:{device} wanted")
    if n is not None and t.numel() != n:
        raise BrcError(_lib.ERR_INVALID, f"{who}: {t.numel()} words, {n} wanted")
    return t.data_ptr()


class Rope:
    """Rotary positions without a cos / sin table: the first `n_rot` values of a head, in pairs (j, j + n_rot/2)
    (layout "half") or (2j, 2j + 1) ("interleaved"), with frequencies theta^(-2j/n_rot) that `scaling` stretches for long
    contexts: "linear", "ntk", "yarn", "bands" (include/breccia_kv.h, brc_rope_freqs; the reference has the half layout from a
    host-built table, crates/breccia-kernels/src/qsa/mod.rs:1612-1614).  `turns_low` / `turns_high` bound yarn's and bands' transition,
    in full turns over `orig_ctx` positions."""

    def __init__(self, n_rot: int, theta: float = 10000.0, layout: str = "half", scaling: str = "none", factor: float = 1.0,
                 orig_ctx: int = 0, turns_low: float = 1.0, turns_high: float | None = None, mscale: float = 0.0, device: int = 0):
        if layout not in _lib.ROPE_LAYOUTS or scaling not in _lib.ROPE_SCALINGS:
            raise BrcError(_lib.ERR_INVALID, f"Rope: layout {layout!r} of {list(_lib.ROPE_LAYOUTS)}, scaling {scaling!r} of {list(_lib.ROPE_SCALINGS)}")
        if turns_high is None:
            turns_high = 32.0 if scaling == "yarn" else 4.0
        a = _lib.RopeParams(theta=theta, factor=factor, turns_low=turns_low, turns_high=turns_high, mscale=mscale, n_rot=n_rot,
                            orig_ctx=orig_ctx, scaling=_lib.ROPE_SCALINGS[scaling])
        self.turns_host = np.zeros(max(n_rot // 2, 1), np.uint64)   # fractions of a turn per position, times 2^64
        f = C.c_double()
        _lib.call("brc_rope_freqs", C.byref(a), self.turns_host.ctypes.data_as(C.POINTER(C.c_uint64)), C.byref(f))
        self.factor, self.n_rot, self.layout, self.device = f.value, n_rot, _lib.ROPE_LAYOUTS[layout], device
        self.turns = torch.from_numpy(self.turns_host.view(np.int64)).to(f"cuda:{device}") if torch.cuda.is_available() else None
        self._turns_ptr = self.turns.data_ptr() if self.turns is not None else None
        self._call = _lib.load().brc_rope_apply

    def _side(self, name: str, x: torch.Tensor, y: torch.Tensor | None, tokens: int, hd: int, dtype: torch.dtype, to):
        """(output, heads, token stride of x, of the output)"""
        if x.dim() != 3:
            raise BrcError(_lib.ERR_INVALID, f"Rope.apply: {name} {tuple(x.shape)}: [tokens, heads, head_dim] wanted")
        n, heads, d = x.shape
        if n != tokens or d != hd or x.dtype != dtype or x.get_device() != self.device:
            raise BrcError(_lib.ERR_INVALID, f"Rope.apply: {name} {tuple(x.shape)} {x.dtype} on {x.device} beside {tokens} tokens of heads of {hd}, {dtype}, the "
                                             f"frequencies on cuda:{self.device}")
        row = heads * hd
        whole = x.is_contiguous()
        stride = row if whole else _token_rows(x, heads, hd, "Rope.apply")
        if y is None:
            return _new(to, lambda: torch.empty_like(x) if whole else torch.empty(x.shape, dtype=dtype, device=x.device)), heads, stride, row
        if y.shape != x.shape or y.dtype != dtype or y.get_device() != self.device:
            raise BrcError(_lib.ERR_INVALID, f"Rope.apply: {name} {tuple(x.shape)} {x.dtype} -> {tuple(y.shape)} {y.dtype} on {y.device}")
        return y, heads, stride, _token_rows(y, heads, hd, "Rope.apply")

    def apply(self, q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, q_out: torch.Tensor | None = None,
              k_out: torch.Tensor | None = None, stream=None):
        """q [tokens, n_head, head_dim], k [tokens, n_kv, head_dim] or None, positions [tokens] int32 (a negative one turns
        backwards) or uint32 -> (q_out, k_out), new tensors unless given (q_out=q rotates in place).  Tokens may be strided
        (columns of one projection)."""
        tokens, hd, dtype = q.shape[0], q.shape[-1], q.dtype
        if tokens >= 1 << 32:
            raise BrcError(_lib.ERR_UNSUPPORTED, f"Rope.apply: {tokens} tokens in one call (below 2^32)")
        qo, qh, qs, qos = self._side("q", q, q_out, tokens, hd, dtype, stream)
        if k is None:
            ko, k_ptr, ko_ptr, kh, ks, kos = None, None, None, 0, 0, 0
        else:
            ko, kh, ks, kos = self._side("k", k, k_out, tokens, hd, dtype, stream)
            k_ptr, ko_ptr = k.data_ptr(), ko.data_ptr()
        at = _words(positions, self.device, "Rope.apply: positions", tokens)
        _lib.check(self._call(self.device, q.data_ptr(), qo.data_ptr(), qh, qs, qos, k_ptr, ko_ptr, kh, ks, kos, hd,
                              _dtype(dtype, "Rope.apply"), at, tokens, self._turns_ptr, self.n_rot,
                              self.layout if positions.dtype == torch.uint32 else self.layout | _lib.ROPE_SIGNED, self.factor,
                              _raw_stream(stream, self.device)))
        return qo, ko


def kv8_append(pool: KvPool, layer: int, k: torch.Tensor, v: torch.Tensor, block_tables: torch.Tensor, pos0: torch.Tensor,
               max_pos_end: int, tokens_per_seq: int = 1, cu_tokens: torch.Tensor | None = None, rope: Rope | None = None,
               stream=None) -> None:
    """The quantising write into an 8-bit pool (brc_kv8_append): k / v [total_tokens, n_kv, hd] (tokens may be strided) at cells
    pos0[s] .. of each sequence, tokens_per_seq each or ragged by cu_tokens [n_seqs + 1] int32; `rope` rotates K on the way."""
    device, n_kv, hd = pool.device, pool.n_kv_head, pool.head_dim
    n_seqs, stride = block_tables.shape
    total = k.shape[0]
    if k.dtype != v.dtype or total != v.shape[0] or k.get_device() != device or v.get_device() != device:
        raise BrcError(_lib.ERR_INVALID, f"kv8_append: k {tuple(k.shape)} {k.dtype} {k.device}, v {tuple(v.shape)} {v.dtype} {v.device}")
    if rope is None:
        turns, n_rot, layout, factor = None, 0, 0, 1.0
    else:
        if rope.device != device:
            raise BrcError(_lib.ERR_INVALID, f"kv8_append: the frequencies lie on cuda:{rope.device}, the pool on cuda:{device}")
        turns, n_rot, layout, factor = rope._turns_ptr, rope.n_rot, rope.layout, rope.factor
    _lib.check(_lib.load().brc_kv8_append(
        pool.handle, layer, _words(block_tables, device, "kv8_append: block_tables"), stride, _words(pos0, device, "kv8_append: pos0", n_seqs),
        n_seqs, tokens_per_seq, None if cu_tokens is None else _words(cu_tokens, device, "kv8_append: cu_tokens", n_seqs + 1), total, max_pos_end,
        k.data_ptr(), _token_rows(k, n_kv, hd, "kv8_append"), v.data_ptr(), _token_rows(v, n_kv, hd, "kv8_append"), _dtype(k.dtype, "kv8_append"),
        turns, n_rot, layout, factor, _raw_stream(stream, device)))


def kv8_read(pool: KvPool, layer: int, block_tables: torch.Tensor, pos0: torch.Tensor, max_pos_end: int, tokens_per_seq: int = 1,
             cu_tokens: torch.Tensor | None = None, total_tokens: int | None = None, dtype: torch.dtype = torch.float16,
             stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Cells pos0[s] .. of each sequence of an 8-bit pool as values (brc_kv8_read) -> K, V [total_tokens, n_kv, hd]."""
    device = pool.device
    n_seqs, stride = block_tables.shape
    if total_tokens is None:
        if cu_tokens is not None:
            raise BrcError(_lib.ERR_INVALID, "kv8_read: total_tokens is needed beside cu_tokens")
        total_tokens = n_seqs * tokens_per_seq
    tables, at = _words(block_tables, device, "kv8_read: block_tables"), _words(pos0, device, "kv8_read: pos0", n_seqs)
    cu = None if cu_tokens is None else _words(cu_tokens, device, "kv8_read: cu_tokens", n_seqs + 1)
    code = _dtype(dtype, "kv8_read")
    n_kv, hd = pool.n_kv_head, pool.head_dim
    # (two tensors by their strides take the host half as long as one and its two halves)
    k, v = _new(stream, lambda: [torch.empty_strided((total_tokens, n_kv, hd), (n_kv * hd, hd, 1), dtype=dtype, device=block_tables.device)
                                 for _ in range(2)])
    _lib.check(_lib.load().brc_kv8_read(pool.handle, layer, tables, stride, at, n_seqs, tokens_per_seq, cu, total_tokens, max_pos_end, k.data_ptr(),
                                        v.data_ptr(), code, _raw_stream(stream, device)))
    return k, v


def kv8_workspace(pool: KvPool, n_seqs: int, n_head: int, max_q: int = 1) -> torch.Tensor:
    """The scratch kv8_attend needs for calls of at most these sizes."""
    need = C.c_uint64()
    _lib.call("brc_kv8_attn_workspace_bytes", pool.handle, n_seqs, n_head, max_q, C.byref(need))
    return torch.empty(need.value, dtype=torch.uint8, device=f"cuda:{pool.device}")


def kv8_attend(pool: KvPool, layer: int, q: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor, max_seq_len: int,
               workspace: torch.Tensor, max_q: int = 1, cu_q: torch.Tensor | None = None, scale: float | None = None,
               out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None, gate: torch.Tensor | None = None,
               gate_head_stride: int = 0, stream=None) -> torch.Tensor:
    """Attention over an 8-bit pool for the last T tokens of each sequence (brc_kv8_attn): q [tokens, n_head, hd], T = max_q, or
    ragged by cu_q [n_seqs + 1] int32 with T <= max_q (rows past q's end are left out and reported by check(); rows that are no
    sequence's are left as they were); token i of T sees seq_lens[s] - (T - 1 - i) cells.  Sums and softmax in f32, probabilities
    to 22 bits, one rounding to `out_dtype` (q's type unless given).  `out` may be q.  `workspace` from kv8_workspace; calls that
    may run at the same time need one each."""
    device = pool.device
    n_seqs, stride = block_tables.shape
    if q.dim() != 3 or q.shape[2] != pool.head_dim or not q.is_contiguous() or q.get_device() != device:
        raise BrcError(_lib.ERR_INVALID, f"kv8_attend: q {tuple(q.shape)} on {q.device}: contiguous [tokens, n_head, {pool.head_dim}] wanted")
    tokens, n_head, hd = q.shape
    if cu_q is not None:
        cu = _words(cu_q, device, "kv8_attend: cu_q", n_seqs + 1)
    elif tokens != n_seqs * max_q:
        raise BrcError(_lib.ERR_INVALID, f"kv8_attend: {tokens} rows of q for {n_seqs} sequences of {max_q} tokens")
    else:
        cu = None
    if out is None:
        out = _new(stream, lambda: torch.empty_like(q, dtype=out_dtype))
    elif out.shape != q.shape or not out.is_contiguous() or out.get_device() != device:
        raise BrcError(_lib.ERR_INVALID, f"kv8_attend: out {tuple(out.shape)} on {out.device} beside q {tuple(q.shape)}")
    elif out.data_ptr() < q.data_ptr() + q.nbytes and q.data_ptr() < out.data_ptr() + out.nbytes and \
            not (out.data_ptr() == q.data_ptr() and out.dtype == q.dtype):
        raise BrcError(_lib.ERR_INVALID, "kv8_attend: out overlaps q without being the same rows")
    if gate is not None and tokens:
        has = 1 + sum((n - 1) * s for n, s in zip(gate.shape, gate.stride())) if gate.numel() else 0
        if gate_head_stride < hd or has < (tokens * n_head - 1) * gate_head_stride + hd:
            raise BrcError(_lib.ERR_INVALID, f"kv8_attend: gate {tuple(gate.shape)} with strides {gate.stride()} for {tokens * n_head} rows of {hd} every {gate_head_stride} values")
    if workspace.get_device() != device or not workspace.is_contiguous() or (gate is not None and (gate.get_device() != device or gate.dtype != torch.float32)):
        raise BrcError(_lib.ERR_INVALID, f"kv8_attend: workspace {tuple(workspace.shape)} with strides {workspace.stride()} on {workspace.device}, gate {None if gate is None else (gate.dtype, gate.device)}: "
                                         f"contiguous on cuda:{device}, and a gate in float32, wanted")
    L, rows = _lib.load(), () if cu is None else (tokens,)
    _lib.check((L.brc_kv8_attn if cu is None else L.brc_kv8_attn_ragged)(
        pool.handle, layer, q.data_ptr(), _dtype(q.dtype, "kv8_attend"), *rows, n_head, None if gate is None else gate.data_ptr(), gate_head_stride,
        _words(block_tables, device, "kv8_attend: block_tables"), stride, _words(seq_lens, device, "kv8_attend: seq_lens", n_seqs), cu, n_seqs, max_q,
        max_seq_len, 1.0 / math.sqrt(hd) if scale is None else scale, out.data_ptr(), _dtype(out.dtype, "kv8_attend"), workspace.data_ptr(),
        workspace.nbytes, _raw_stream(stream, device)))
    return out


def decode_partial_bytes(n_seqs: int, n_head: int, head_dim: int) -> int:
    out = C.c_uint64()
    _lib.call("brc_decode_partial_bytes", n_seqs, n_head, head_dim, C.byref(out))
    return out.value


def decode_combine(device: int, parts: torch.Tensor, n_parts: int, part_stride_bytes: int, n_seqs: int, n_head: int,
                   head_dim: int, out: torch.Tensor, gate: torch.Tensor | None = None,
                   gate_head_stride: int = 0) -> None:
    _lib.call("brc_decode_combine", device, _ptr(parts), n_parts, part_stride_bytes, n_seqs, n_head, head_dim,
              _ptr(gate), gate_head_stride, _ptr(out), _stream_ptr())

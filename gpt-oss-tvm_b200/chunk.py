"""Batched chunks of new tokens over the paged KV cache, and the 8-bit cache.

``attend_chunks``   attention of every sequence's new tokens over its pages
                    (bf16 or 8-bit), one launch for a ragged batch
``rope_append_f8``  QKV split + RoPE, keys and values quantised into the pages
``write_pages_f8`` / ``read_pages_f8``  bf16 rows into 8-bit pages and back

An 8-bit pool is a float8_e4m3fn tensor [pages * 16, kv heads, 64] and a
float8_e8m0fnu tensor [pages, kv heads, 16] with one power of two per row and
head (``f8_pool`` makes an empty one): the smallest that brings the row's
largest magnitude to 448 or less, so a value read back is exact in bf16.

Every call runs on the current stream of its tensors' device and raises on
arguments it cannot take; there is no CPU path.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

PAGE_SIZE = 16
HEAD_DIM = 64
MAX_CHUNKS = 1024  # of one attend_chunks call
_BF16, _F8, _E8 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu


class ChunkWorkspace:
    """Device memory of attend_chunks for partial results, zeroed once; used
    by one stream at a time (one for all layers of a model).  Made before a
    capture, not in one: its zeros would be a node of that graph."""

    def __init__(self, device="cuda"):
        self.device = torch.device(device)
        with torch.cuda.device(self.device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a ChunkWorkspace is made before a graph is captured (its zeros would be a node of "
                                   "the graph)")
        self._allocate()

    def _allocate(self):
        lib = _lib.load()
        with torch.cuda.device(self.device):
            self.nbytes = int(lib.gptoss_attn_chunk_workspace_bytes())
            self.buf = torch.empty(self.nbytes, dtype=torch.uint8, device=self.device)
            self.buf[:int(lib.gptoss_attn_chunk_workspace_zero_bytes())].zero_()
        self.ptr = self.buf.data_ptr()
        return self

    def error_word(self) -> torch.Tensor:
        """Device error bits so far, int32 [1] on the device."""
        return self.buf[:4].view(torch.int32)

    def error(self) -> int:
        """Device error bits so far (synchronises)."""
        return int(self.error_word().item())

    def reset(self) -> None:
        """After a device error: the counters may be anything, and the error bits stay otherwise."""
        self.buf.zero_()


_workspaces: dict = {}


def _workspace(index: int) -> ChunkWorkspace:
    """The workspace of a call on device `index` that brings none: the current
    stream's, or, while that is being captured, memory of this call alone, zeroed
    in the graph.  (Streams that capture are shared: a workspace kept by stream
    would come to graphs that replay side by side, or before the one that holds
    its zeros.)"""
    if torch._C._cuda_getDevice() == index:
        capturing = torch._C._cuda_isCurrentStreamCapturing()
    else:
        with torch.cuda.device(index):
            capturing = torch._C._cuda_isCurrentStreamCapturing()
    if capturing:
        ws = ChunkWorkspace.__new__(ChunkWorkspace)
        ws.device = torch.device("cuda", index)
        return ws._allocate()
    stream = torch._C._cuda_getCurrentRawStream(index)
    ws = _workspaces.get((index, stream))
    if ws is None:
        ws = _workspaces[index, stream] = ChunkWorkspace(torch.device("cuda", index))
    return ws


def _run(index: int, name: str, *args) -> None:
    """A library call with the current stream of device `index` as its last argument."""
    fn, stream = getattr(_lib.load(), name), torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc)


def _bad(what: str):
    raise ValueError(what)


def _i32(t, n, name, index):
    if (t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous()
            or t.get_device() != index):
        raise ValueError(f"{name} must be a dense int32 tensor of {n} entries on cuda:{index}")
    return t.data_ptr()


def _table(t, index):
    if t.dtype is not torch.int32 or t.dim() != 2 or not t.is_contiguous() or t.get_device() != index:
        raise ValueError(f"page_table must be a dense int32 tensor [sequences, pages] on cuda:{index}")
    return t.data_ptr()


def _pools(k_pages, v_pages, k_scale, v_scale, index):
    """Checks a pair of pools; (kv heads, pages, whether 8-bit)."""
    shape, dt = k_pages.shape, k_pages.dtype
    if len(shape) != 3 or shape[2] != HEAD_DIM or shape[0] % PAGE_SIZE:
        _bad(f"page pools are [pages * {PAGE_SIZE}, kv heads, {HEAD_DIM}], got {tuple(shape)}")
    if v_pages.shape != shape or v_pages.dtype is not dt:
        _bad("the two pools differ in shape or type")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous() and k_pages.get_device() == index
            and v_pages.get_device() == index):
        _bad(f"page pools must be dense and on cuda:{index}")
    hkv, pages = shape[1], shape[0] // PAGE_SIZE
    if dt is _F8:
        if k_scale is None or v_scale is None:
            _bad("8-bit pools need k_scale and v_scale")
        want = (pages, hkv, PAGE_SIZE)
        for t in (k_scale, v_scale):
            if t.dtype is not _E8 or t.shape != want or not t.is_contiguous() or t.get_device() != index:
                _bad(f"scales of this pool are dense float8_e8m0fnu {want} on cuda:{index}")
        return hkv, pages, True
    if dt is not _BF16:
        _bad(f"page pools are bfloat16 or float8_e4m3fn, got {dt}")
    if k_scale is not None or v_scale is not None:
        _bad("bf16 pools have no scales")
    return hkv, pages, False


def f8_pool(pages: int, kv_heads: int, device="cuda"):
    """An empty 8-bit pool: values (zero) and scales (one)."""
    v = torch.zeros(pages * PAGE_SIZE, kv_heads, HEAD_DIM, dtype=torch.uint8, device=device).view(_F8)
    s = torch.full((pages, kv_heads, PAGE_SIZE), 127, dtype=torch.uint8, device=device).view(_E8)
    return v, s


def attend_chunks(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                  seq_rows: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor, *, max_q: int, window: int = 0,
                  sm_scale: float | None = None, sinks: torch.Tensor | None = None,
                  k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None, return_lse: bool = False,
                  out: torch.Tensor | None = None, workspace: ChunkWorkspace | None = None):
    """Attention of chunk b, tokens q_start[b] .. q_start[b + 1] - 1 of q
    [T, heads, 64], over the kv_len[b] positions that end with it, in the pages
    of row seq_rows[b] of page_table.  The chunk's own keys and values are in
    the pages already.  Token i sees keys 0..pos_i, with ``window`` the last
    ``window`` of them; one that sees none gives zeros (lse -inf).

    q: bf16, heads and values dense, any multiple of 8 elements between tokens
    (a slice of a wider projection will do).  q_start [N + 1], kv_len,
    seq_rows [N]: int32 on the device, N at most MAX_CHUNKS (a slice of more of
    them leaves the other tokens' rows of out as they are).  max_q: the longest chunk.  sinks
    [heads] bf16.  workspace: a ChunkWorkspace of calls that run one after
    another; without one a call has its stream's, or in a captured graph its own
    (20 MB and a memset a call, so a graph of many calls brings one).  Returns o
    [T, heads, 64] bf16, with return_lse also lse [T, heads] fp32 (base 2,
    without the sink)."""
    if not q.is_cuda or q.dtype is not _BF16 or q.dim() != 3 or q.shape[2] != HEAD_DIM:
        _bad(f"q must be a CUDA bfloat16 tensor [tokens, heads, {HEAD_DIM}]")
    index = q.get_device()
    T, Hq, _ = q.shape
    st = q.stride()
    if T and (st[2] != 1 or st[1] != HEAD_DIM or (T > 1 and (st[0] < Hq * HEAD_DIM or st[0] % 8))):
        _bad("q: heads and values must be dense, tokens a multiple of 8 elements apart")
    hkv, pages, f8 = _pools(k_pages, v_pages, k_scale, v_scale, index)
    if Hq % hkv or Hq // hkv > 64:
        _bad(f"{Hq} query heads do not fit {hkv} kv heads (a multiple, at most 64 for each)")
    table_p = _table(page_table, index)
    n = seq_rows.shape[0]
    rows_p, start_p, len_p = (_i32(seq_rows, n, "seq_rows", index), _i32(q_start, n + 1, "q_start", index),
                              _i32(kv_len, n, "kv_len", index))
    if sinks is not None and (sinks.dtype is not _BF16 or sinks.dim() != 1 or sinks.shape[0] != Hq
                              or not sinks.is_contiguous() or sinks.get_device() != index):
        _bad(f"sinks must be a dense bfloat16 tensor [{Hq}] on cuda:{index}")
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((T, Hq, HEAD_DIM))
    elif out.dtype is not _BF16 or out.shape != q.shape or not out.is_contiguous() or out.get_device() != index:
        _bad("out must be a dense bfloat16 tensor of q's shape on its device")
    lse = q.new_empty((T, Hq), dtype=torch.float32) if return_lse else None
    if T and n:
        ws = workspace
        if ws is None:
            ws = _workspace(index)
        elif ws.buf.get_device() != index:
            _bad("the workspace is on another device")
        _run(index, "gptoss_attn_chunk", q.data_ptr(), st[0] if T > 1 else Hq * HEAD_DIM, k_pages.data_ptr(),
             v_pages.data_ptr(), k_scale.data_ptr() if f8 else None, v_scale.data_ptr() if f8 else None, f8, pages,
             table_p, page_table.shape[0], page_table.shape[1], rows_p, start_p, len_p, n, T, max_q, Hq, hkv,
             HEAD_DIM, window, HEAD_DIM ** -0.5 if sm_scale is None else sm_scale,
             sinks.data_ptr() if sinks is not None else None, ws.ptr, ws.nbytes, out.data_ptr(),
             lse.data_ptr() if return_lse else None)
    return (out, lse) if return_lse else out


def rope_append_f8(qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, num_heads: int, inv_freq,
                   concentration: float, k_pages: torch.Tensor, v_pages: torch.Tensor, k_scale: torch.Tensor,
                   v_scale: torch.Tensor, q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Splits qkv [T, (num_heads + 2 kv heads) * 64], rotates q and k by their
    positions [T], and quantises k and v into pool rows slots [T].  inv_freq:
    32 floats on the host (a CPU float32 tensor or a ctypes array).  Returns q
    [T, num_heads, 64] bf16, the bits that the bf16 cache's append gives."""
    if not qkv.is_cuda or qkv.dtype is not _BF16 or qkv.dim() != 2 or not qkv.is_contiguous():
        _bad("qkv must be a dense CUDA bfloat16 tensor [tokens, (heads + 2 kv heads) * 64]")
    index, T = qkv.get_device(), qkv.shape[0]
    hkv, pages, f8 = _pools(k_pages, v_pages, k_scale, v_scale, index)
    if not f8:
        _bad("rope_append_f8 writes 8-bit pools")
    if qkv.shape[1] != (num_heads + 2 * hkv) * HEAD_DIM:
        _bad(f"qkv must have {(num_heads + 2 * hkv) * HEAD_DIM} columns for {num_heads} heads and {hkv} kv heads")
    pos_p, slot_p = _i32(positions, T, "positions", index), _i32(slots, T, "slots", index)
    if isinstance(inv_freq, torch.Tensor):
        if (inv_freq.is_cuda or inv_freq.dtype is not torch.float32 or not inv_freq.is_contiguous()
                or inv_freq.numel() != HEAD_DIM // 2):
            _bad(f"inv_freq must be {HEAD_DIM // 2} float32 values on the CPU")
        inv_p = inv_freq.data_ptr()
    else:
        if len(inv_freq) != HEAD_DIM // 2:
            _bad(f"inv_freq must be {HEAD_DIM // 2} values")
        inv_p = ctypes.addressof(inv_freq)
    if q_out is None:
        q_out = qkv.new_empty((T, num_heads, HEAD_DIM))
    elif (q_out.dtype is not _BF16 or q_out.shape != (T, num_heads, HEAD_DIM) or not q_out.is_contiguous()
          or q_out.get_device() != index):
        _bad(f"q_out must be a dense bfloat16 tensor [{T}, {num_heads}, {HEAD_DIM}] on cuda:{index}")
    if T:
        _run(index, "gptoss_qkv_rope_append_f8", qkv.data_ptr(), pos_p, slot_p, T, pages, num_heads, hkv, HEAD_DIM,
             inv_p, concentration, q_out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), k_scale.data_ptr(),
             v_scale.data_ptr())
    return q_out


def _copy_f8(k_pages, v_pages, k_scale, v_scale, page_table, seq, pos0, n, k_rows, v_rows, to_pages):
    if not k_pages.is_cuda or k_pages.dtype is not _F8:
        _bad("the pools must be 8-bit CUDA pools")
    index = k_pages.get_device()
    hkv, pages, _ = _pools(k_pages, v_pages, k_scale, v_scale, index)
    table_p = _table(page_table, index)
    if not 0 <= seq < page_table.shape[0] or pos0 < 0 or n < 0:
        _bad(f"no rows {pos0}, {n} of sequence {seq}")
    want = (n, hkv, HEAD_DIM)
    for t in (k_rows, v_rows):
        if t.dtype is not _BF16 or t.shape != want or not t.is_contiguous() or t.get_device() != index:
            _bad(f"rows must be dense bfloat16 tensors {want} on cuda:{index}")
    if n:
        _run(index, "gptoss_kv_pages_copy_f8", k_pages.data_ptr(), v_pages.data_ptr(), k_scale.data_ptr(),
             v_scale.data_ptr(), pages, hkv, HEAD_DIM, table_p, page_table.shape[1], seq, pos0, n, k_rows.data_ptr(),
             v_rows.data_ptr(), to_pages)


def read_pages_f8(k_pages, v_pages, k_scale, v_scale, page_table, seq: int, pos0: int, n: int, k_out=None, v_out=None):
    """Keys and values of positions pos0 .. pos0 + n - 1 of sequence ``seq`` as
    bf16 rows [n, kv heads, 64] (exact)."""
    shape = (n, k_pages.shape[1], HEAD_DIM)
    k_out = k_pages.new_empty(shape, dtype=_BF16) if k_out is None else k_out
    v_out = torch.empty_like(k_out) if v_out is None else v_out
    _copy_f8(k_pages, v_pages, k_scale, v_scale, page_table, seq, pos0, n, k_out, v_out, False)
    return k_out, v_out


def write_pages_f8(k_rows, v_rows, k_pages, v_pages, k_scale, v_scale, page_table, seq: int, pos0: int):
    """bf16 rows [n, kv heads, 64] quantised into positions pos0 .. of sequence ``seq``."""
    _copy_f8(k_pages, v_pages, k_scale, v_scale, page_table, seq, pos0, k_rows.shape[0], k_rows, v_rows, True)

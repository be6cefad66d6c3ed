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
_BF16, _F8, _E8 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu


class ChunkWorkspace:
    """Device memory of attend_chunks for partial results, zeroed once; used
    by one stream at a time (one for all layers of a model)."""

    def __init__(self, device="cuda"):
        self.device = torch.device(device)
        with torch.cuda.device(self.device):
            self.nbytes = int(_lib.load().gptoss_attn_chunk_workspace_bytes())
        self.buf = torch.zeros(self.nbytes, dtype=torch.uint8, device=self.device)
        self.ptr = self.buf.data_ptr()

    def error(self) -> int:
        """Device error bits so far (synchronises)."""
        return int(self.buf[:4].view(torch.int32).item())


_workspaces: dict = {}


def _workspace(device: torch.device, stream: int) -> ChunkWorkspace:
    """The workspace of calls on this device and stream that bring none (a
    program's own, as long as it runs: captured graphs keep using it)."""
    key = (device.index, stream)
    ws = _workspaces.get(key)
    if ws is None:
        ws = _workspaces[key] = ChunkWorkspace(device)
    return ws


def _need(cond: bool, what: str):
    if not cond:
        raise ValueError(what)


def _i32(t, n, name, dev):
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous() or t.device != dev:
        raise ValueError(f"{name} must be a dense int32 tensor of {n} entries on {dev}")
    return t.data_ptr()


def _pools(k_pages, v_pages, k_scale, v_scale, dev):
    """Checks a pair of pools; (kv heads, pages, whether 8-bit)."""
    _need(k_pages.dim() == 3 and k_pages.shape[2] == HEAD_DIM and k_pages.shape[0] % PAGE_SIZE == 0,
          f"page pools are [pages * {PAGE_SIZE}, kv heads, {HEAD_DIM}], got {tuple(k_pages.shape)}")
    _need(k_pages.shape == v_pages.shape and k_pages.dtype == v_pages.dtype, "the two pools differ in shape or type")
    _need(k_pages.is_contiguous() and v_pages.is_contiguous() and k_pages.device == dev and v_pages.device == dev,
          f"page pools must be dense and on {dev}")
    hkv, pages = k_pages.shape[1], k_pages.shape[0] // PAGE_SIZE
    f8 = k_pages.dtype == _F8
    if f8:
        _need(k_scale is not None and v_scale is not None, "8-bit pools need k_scale and v_scale")
        for t in (k_scale, v_scale):
            _need(t.dtype == _E8 and tuple(t.shape) == (pages, hkv, PAGE_SIZE) and t.is_contiguous()
                  and t.device == dev, f"scales of this pool are dense float8_e8m0fnu [{pages}, {hkv}, {PAGE_SIZE}]")
    else:
        _need(k_pages.dtype == _BF16, f"page pools are bfloat16 or float8_e4m3fn, got {k_pages.dtype}")
        _need(k_scale is None and v_scale is None, "bf16 pools have no scales")
    return hkv, pages, f8


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
    seq_rows [N]: int32 on the device.  max_q: the longest chunk.  sinks
    [heads] bf16.  Returns o [T, heads, 64] bf16, with return_lse also lse
    [T, heads] fp32 (base 2, without the sink)."""
    dev = q.device
    _need(q.is_cuda and q.dtype == _BF16 and q.dim() == 3 and q.shape[2] == HEAD_DIM,
          f"q must be a CUDA bfloat16 tensor [tokens, heads, {HEAD_DIM}]")
    T, Hq, _ = q.shape
    st = q.stride()
    _need(T == 0 or (st[2] == 1 and st[1] == HEAD_DIM and (T == 1 or (st[0] >= Hq * HEAD_DIM and st[0] % 8 == 0))),
          "q: heads and values must be dense, tokens a multiple of 8 elements apart")
    hkv, pages, f8 = _pools(k_pages, v_pages, k_scale, v_scale, dev)
    _need(Hq % hkv == 0 and Hq // hkv <= 64, f"{Hq} query heads do not fit {hkv} kv heads (at most 64 for each)")
    _need(page_table.dtype == torch.int32 and page_table.dim() == 2 and page_table.is_contiguous()
          and page_table.device == dev, f"page_table must be a dense int32 tensor [sequences, pages] on {dev}")
    n = seq_rows.shape[0]
    rows_p, start_p, len_p = (_i32(seq_rows, n, "seq_rows", dev), _i32(q_start, n + 1, "q_start", dev),
                              _i32(kv_len, n, "kv_len", dev))
    _need(sinks is None or (sinks.dtype == _BF16 and tuple(sinks.shape) == (Hq,) and sinks.is_contiguous()
                            and sinks.device == dev), f"sinks must be a dense bfloat16 tensor [{Hq}] on {dev}")
    if out is None:
        out = torch.empty(T, Hq, HEAD_DIM, dtype=_BF16, device=dev)
    else:
        _need(out.dtype == _BF16 and out.shape == q.shape and out.is_contiguous() and out.device == dev,
              "out must be a dense bfloat16 tensor of q's shape")
    lse = torch.empty(T, Hq, dtype=torch.float32, device=dev) if return_lse else None
    if T and n:
        with torch.cuda.device(dev):
            stream = torch.cuda.current_stream().cuda_stream
            ws = workspace if workspace is not None else _workspace(dev, stream)
            _need(ws.device.index in (None, dev.index), "the workspace is on another device")
            _lib.call("gptoss_attn_chunk", q.data_ptr(), st[0] if T > 1 else Hq * HEAD_DIM, k_pages.data_ptr(),
                      v_pages.data_ptr(), k_scale.data_ptr() if f8 else None, v_scale.data_ptr() if f8 else None,
                      int(f8), pages, page_table.data_ptr(), page_table.shape[0], page_table.shape[1], rows_p,
                      start_p, len_p, n, T, int(max_q), Hq, hkv, HEAD_DIM, int(window),
                      sm_scale if sm_scale is not None else HEAD_DIM ** -0.5,
                      sinks.data_ptr() if sinks is not None else None, ws.ptr, ws.nbytes, out.data_ptr(),
                      lse.data_ptr() if return_lse else None, stream)
    return (out, lse) if return_lse else out


def rope_append_f8(qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, num_heads: int, inv_freq,
                   concentration: float, k_pages: torch.Tensor, v_pages: torch.Tensor, k_scale: torch.Tensor,
                   v_scale: torch.Tensor, q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Splits qkv [T, (num_heads + 2 kv heads) * 64], rotates q and k by their
    positions [T], and quantises k and v into pool rows slots [T].  inv_freq:
    32 floats on the host (a CPU float32 tensor or a ctypes array).  Returns q
    [T, num_heads, 64] bf16, the bits that the bf16 cache's append gives."""
    dev = qkv.device
    hkv, pages, f8 = _pools(k_pages, v_pages, k_scale, v_scale, dev)
    _need(f8, "rope_append_f8 writes 8-bit pools")
    T = qkv.shape[0]
    _need(qkv.is_cuda and qkv.dtype == _BF16 and qkv.is_contiguous()
          and tuple(qkv.shape) == (T, (num_heads + 2 * hkv) * HEAD_DIM),
          f"qkv must be a dense CUDA bfloat16 tensor [tokens, {(num_heads + 2 * hkv) * HEAD_DIM}]")
    pos_p, slot_p = _i32(positions, T, "positions", dev), _i32(slots, T, "slots", dev)
    if isinstance(inv_freq, torch.Tensor):
        _need(inv_freq.device.type == "cpu" and inv_freq.dtype == torch.float32 and inv_freq.is_contiguous()
              and inv_freq.numel() == HEAD_DIM // 2, f"inv_freq must be {HEAD_DIM // 2} float32 values on the CPU")
        inv_p = inv_freq.data_ptr()
    else:
        _need(len(inv_freq) == HEAD_DIM // 2, f"inv_freq must be {HEAD_DIM // 2} values")
        inv_p = ctypes.addressof(inv_freq)
    if q_out is None:
        q_out = torch.empty(T, num_heads, HEAD_DIM, dtype=_BF16, device=dev)
    else:
        _need(q_out.dtype == _BF16 and tuple(q_out.shape) == (T, num_heads, HEAD_DIM) and q_out.is_contiguous()
              and q_out.device == dev, f"q_out must be a dense bfloat16 tensor [{T}, {num_heads}, {HEAD_DIM}]")
    if T:
        with torch.cuda.device(dev):
            _lib.call("gptoss_qkv_rope_append_f8", qkv.data_ptr(), pos_p, slot_p, T, pages, num_heads, hkv, HEAD_DIM,
                      inv_p, concentration, q_out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                      k_scale.data_ptr(), v_scale.data_ptr(), torch.cuda.current_stream().cuda_stream)
    return q_out


def _copy_f8(k_pages, v_pages, k_scale, v_scale, page_table, seq, pos0, n, k_rows, v_rows, to_pages):
    dev = k_pages.device
    hkv, pages, f8 = _pools(k_pages, v_pages, k_scale, v_scale, dev)
    _need(f8 and k_pages.is_cuda, "the pools must be 8-bit CUDA pools")
    _need(page_table.dtype == torch.int32 and page_table.dim() == 2 and page_table.is_contiguous()
          and page_table.device == dev, f"page_table must be a dense int32 tensor [sequences, pages] on {dev}")
    _need(0 <= seq < page_table.shape[0] and pos0 >= 0 and n >= 0, f"no rows {pos0}, {n} of sequence {seq}")
    for t in (k_rows, v_rows):
        _need(t.dtype == _BF16 and tuple(t.shape) == (n, hkv, HEAD_DIM) and t.is_contiguous() and t.device == dev,
              f"rows must be dense bfloat16 tensors [{n}, {hkv}, {HEAD_DIM}] on {dev}")
    if n:
        with torch.cuda.device(dev):
            _lib.call("gptoss_kv_pages_copy_f8", k_pages.data_ptr(), v_pages.data_ptr(), k_scale.data_ptr(),
                      v_scale.data_ptr(), pages, hkv, HEAD_DIM, page_table.data_ptr(), page_table.shape[1], seq, pos0,
                      n, k_rows.data_ptr(), v_rows.data_ptr(), int(to_pages),
                      torch.cuda.current_stream().cuda_stream)


def read_pages_f8(k_pages, v_pages, k_scale, v_scale, page_table, seq: int, pos0: int, n: int, k_out=None, v_out=None):
    """Keys and values of positions pos0 .. pos0 + n - 1 of sequence ``seq`` as
    bf16 rows [n, kv heads, 64] (exact)."""
    shape = (n, k_pages.shape[1], HEAD_DIM)
    k_out = torch.empty(shape, dtype=_BF16, device=k_pages.device) if k_out is None else k_out
    v_out = torch.empty(shape, dtype=_BF16, device=k_pages.device) if v_out is None else v_out
    _copy_f8(k_pages, v_pages, k_scale, v_scale, page_table, seq, pos0, n, k_out, v_out, False)
    return k_out, v_out


def write_pages_f8(k_rows, v_rows, k_pages, v_pages, k_scale, v_scale, page_table, seq: int, pos0: int):
    """bf16 rows [n, kv heads, 64] quantised into positions pos0 .. of sequence ``seq``."""
    _copy_f8(k_pages, v_pages, k_scale, v_scale, page_table, seq, pos0, k_rows.shape[0], k_rows, v_rows, True)

"""Speculative decoding's test of drafted tokens against the target's logits.

The random numbers are arguments and every sum is over whole numbers, so the
same inputs give the same tokens on any split of the work.
"""
from __future__ import annotations

import torch

from . import _lib
from .chunk import _bad, _i32, _run


def _dense_rows(t: torch.Tensor) -> bool:
    """Whether the values of each row of t are one after another (what is a
    stride of one entry does not matter)."""
    rows, n = t.shape
    return rows == 0 or ((n <= 1 or t.stride(1) == 1) and (rows == 1 or t.stride(0) >= n))


def verify_drafts(logits: torch.Tensor, tokens: torch.Tensor, row_start: torch.Tensor,
                  accept_draws: torch.Tensor | None = None, next_draws: torch.Tensor | None = None, *,
                  temperature: float = 1.0, draft_probs: torch.Tensor | None = None):
    """Rows row_start[b] .. row_start[b + 1] - 1 of logits [T, V] (float32 or
    bfloat16) are sequence b's: row r is the target's for the token after
    tokens[r], and tokens[r + 1] is the draft checked against it.  The draft is
    accepted when accept_draws[r] * q < p at that token, p = softmax(logits /
    temperature), q = draft_probs[r] (the distribution it was drawn from; None:
    drafts that were looked up, q = 1).  Returns int32 tensors on the device:
    accepted [N], the drafts before the first that is not, and next_token [N],
    drawn with next_draws [N] from what is left of p there, or from the last
    row's p.  temperature < 1e-6: greedy, no draws needed.  (Both are views of
    one buffer that held the scratch, 8 bytes for each 256 logits: what is kept
    for long is cloned.)"""
    if not logits.is_cuda or logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16):
        _bad("logits must be a CUDA tensor [rows, vocabulary], float32 or bfloat16")
    index = logits.get_device()
    T, V = logits.shape
    if not _dense_rows(logits):
        _bad("the values of a row of logits must be dense")
    n = row_start.shape[0] - 1
    if n < 0:
        _bad("row_start needs at least one entry")
    tokens_p, start_p = _i32(tokens, T, "tokens", index), _i32(row_start, n + 1, "row_start", index)
    greedy = temperature < 1e-6
    if not greedy:
        for t, m, name in ((accept_draws, T, "accept_draws"), (next_draws, n, "next_draws")):
            if (t is None or t.dtype is not torch.float32 or t.dim() != 1 or t.shape[0] != m or not t.is_contiguous()
                    or t.get_device() != index):
                _bad(f"{name} must be a dense float32 tensor of {m} entries on cuda:{index}")
    if draft_probs is not None and (draft_probs.dtype is not torch.float32 or draft_probs.shape != (T, V)
                                    or draft_probs.get_device() != index or not _dense_rows(draft_probs)):
        _bad(f"draft_probs must be a float32 tensor [{T}, {V}] with dense rows on cuda:{index}")
    # one allocation: the two answers, then the library's scratch
    nbytes = _lib.load().gptoss_verify_drafts_scratch_bytes(T, V)
    buf = tokens.new_empty(2 * n + nbytes // 4 + 1)
    if n:
        p = buf.data_ptr()
        _run(index, "gptoss_verify_drafts", logits.data_ptr(), logits.dtype is torch.bfloat16,
             logits.stride(0) if T > 1 else V, tokens_p, start_p, T, n, V, temperature,
             None if greedy else accept_draws.data_ptr(), None if greedy else next_draws.data_ptr(),
             draft_probs.data_ptr() if draft_probs is not None else None,
             draft_probs.stride(0) if draft_probs is not None and T > 1 else V, p + 8 * n, nbytes, p, p + 4 * n)
    return buf[:n], buf[n:2 * n]

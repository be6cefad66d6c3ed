"""Speculative decoding's test of drafted tokens against the target's logits.

The random numbers are arguments and every sum is over whole numbers, so the
same inputs give the same tokens on any split of the work.
"""
from __future__ import annotations

import torch

from . import _lib


def _need(cond: bool, what: str):
    if not cond:
        raise ValueError(what)


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
    row's p.  temperature < 1e-6: greedy, no draws needed."""
    dev = logits.device
    _need(logits.is_cuda and logits.dim() == 2 and logits.dtype in (torch.float32, torch.bfloat16),
          "logits must be a CUDA tensor [rows, vocabulary], float32 or bfloat16")
    T, V = logits.shape
    _need(T <= 1 or (logits.stride(1) == 1 and logits.stride(0) >= V), "the values of a row of logits must be dense")
    n = row_start.shape[0] - 1
    for t, m, name in ((tokens, T, "tokens"), (row_start, n + 1, "row_start")):
        _need(t.dtype == torch.int32 and t.dim() == 1 and t.shape[0] == m and t.is_contiguous() and t.device == dev,
              f"{name} must be a dense int32 tensor of {m} entries on {dev}")
    _need(n >= 0, "row_start needs at least one entry")
    greedy = temperature < 1e-6
    if not greedy:
        for t, m, name in ((accept_draws, T, "accept_draws"), (next_draws, n, "next_draws")):
            _need(t is not None and t.dtype == torch.float32 and t.dim() == 1 and t.shape[0] == m
                  and t.is_contiguous() and t.device == dev,
                  f"{name} must be a dense float32 tensor of {m} entries on {dev}")
    if draft_probs is not None:
        _need(draft_probs.dtype == torch.float32 and tuple(draft_probs.shape) == (T, V) and draft_probs.device == dev
              and (T <= 1 or (draft_probs.stride(1) == 1 and draft_probs.stride(0) >= V)),
              f"draft_probs must be a float32 tensor [{T}, {V}] with dense rows on {dev}")
    out = torch.empty(2, n, dtype=torch.int32, device=dev)
    if n:
        lib = _lib.load()
        nbytes = lib.gptoss_verify_drafts_scratch_bytes(T)
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        with torch.cuda.device(dev):
            _lib.call("gptoss_verify_drafts", logits.data_ptr(), int(logits.dtype == torch.bfloat16),
                      logits.stride(0) if T > 1 else V, tokens.data_ptr(), row_start.data_ptr(), T, n, V,
                      float(temperature), None if greedy else accept_draws.data_ptr(),
                      None if greedy else next_draws.data_ptr(),
                      draft_probs.data_ptr() if draft_probs is not None else None,
                      draft_probs.stride(0) if draft_probs is not None and T > 1 else V, scratch.data_ptr(), nbytes,
                      out[0].data_ptr(), out[1].data_ptr(), torch.cuda.current_stream().cuda_stream)
    return out[0], out[1]

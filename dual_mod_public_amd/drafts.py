"""Drafted tokens against the target's probabilities, from given random numbers (dm_verify_drafts).

A speculative step gives the model a chunk of input tokens per sequence: its last token and the drafts after it. Row t of
the chunk's ``logits`` is the target's distribution after ``ids[t]``, and ``ids[t + 1]`` the draft that it answers. With
p = softmax(logits / T), q = softmax(draft_logits / T) (or 1 at the draft, where it was looked up rather than drawn), a draft d is accepted
where ``uniforms[t, 0] q(d) < p(d)``; the first row without an accepted draft gives a token drawn from max(p - q, 0)
(the last row: from p) by ``uniforms[t, 1]``. The tokens are then distributed as if drawn from p one by one. T = 0 is greedy.
"""

from typing import NamedTuple

import torch

from . import _lib as L
from .logprobs import _rows
from .paged import _no_graph


class Verified(NamedTuple):
    tokens: torch.Tensor     # [N] int64: accepted drafts and the new token, each at the row that predicts it; -1 behind them
    accepted: torch.Tensor   # [B] int32: drafts accepted; the sequence's new token is at row starts[b] + accepted[b]
    logp: torch.Tensor       # [N] fp32: the tokens' log probabilities under the target (at T = 1 where T is 0)


def _like(t, name, shape, dtype, device):
    if t.dtype != dtype or t.shape != shape or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name}: {t.dtype} {tuple(t.shape)} on {t.device}; contiguous {dtype} {shape} on cuda:{device} is needed")
    return t.data_ptr()


def verify_drafts(logits, ids, uniforms, starts, draft_logits=None, temperature=1.0):
    """logits [N, V] (bf16 or fp32, any row stride) of the chunks' input tokens ids [N] (int64); starts [B + 1] (int32, on
    the device): sequence b's rows are starts[b] .. starts[b + 1] - 1. uniforms [N, 2] fp32 in [0, 1). draft_logits [N, V]: the
    distribution that ids[t + 1] was drawn from in row t (a sequence's last row is not read); None: the drafts are certain.
    temperature: one number, or [B] fp32. Returns Verified; no gradients. A row without a distribution (a NaN, +inf, nothing
    but -inf; a temperature that is negative or not finite) ends its sequence with token -1."""
    for t in (logits, draft_logits, temperature if torch.is_tensor(temperature) else None):
        _no_graph(t, "verify_drafts")
    if not logits.is_cuda or logits.dim() != 2:
        raise ValueError(f"logits: shape {tuple(logits.shape)} on {logits.device}; rows [N, V] on a GPU are needed")
    dev = logits.get_device()
    dtype = L.dtype_code(logits.dtype)
    if starts.dim() != 1 or starts.shape[0] < 1:
        raise ValueError(f"starts: {tuple(starts.shape)}; [B + 1] is needed")
    (N, V), B = logits.shape, starts.shape[0] - 1
    if N > 65535 or B > 65535:
        raise ValueError(f"{N} rows of {B} sequences (at most 65535)")
    ld, draft, ld_draft = _rows(logits, "logits")[1], None, 0
    if draft_logits is not None:
        if draft_logits.shape != logits.shape or draft_logits.dtype != logits.dtype or draft_logits.get_device() != dev:
            raise ValueError(f"draft_logits: {draft_logits.dtype} {tuple(draft_logits.shape)} on {draft_logits.device} for logits "
                             f"{logits.dtype} {tuple(logits.shape)} on {logits.device}")
        draft, ld_draft = draft_logits.data_ptr(), _rows(draft_logits, "draft_logits")[1]
    if not torch.is_tensor(temperature):
        if not 0 <= temperature < float("inf"):
            raise ValueError(f"temperature={temperature}")
        temperature = torch.full((B,), float(temperature), device=logits.device)
    args = (_like(ids, "ids", (N,), torch.int64, dev), _like(uniforms, "uniforms", (N, 2), torch.float32, dev),
            _like(temperature, "temperature", (B,), torch.float32, dev), _like(starts, "starts", (B + 1,), torch.int32, dev))
    out = Verified(ids.new_empty((N,)), starts.new_empty((B,)), uniforms.new_empty((N,)))
    if N == 0 or B == 0:
        out.tokens.fill_(-1), out.accepted.zero_(), out.logp.zero_()
        return out
    a = L.dm_verify_args(dtype, N, V, B, logits.data_ptr(), ld, draft, ld_draft, *args, out.tokens.data_ptr(), out.accepted.data_ptr(),
                         out.logp.data_ptr())
    args = L.byref(a)
    ws = torch.empty(L.lib().dm_verify_workspace_bytes(args), dtype=torch.uint8, device=logits.device)
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    L.call_on(logits.device, L.lib().dm_verify_drafts, args)
    return out

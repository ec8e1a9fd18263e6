"""Log probabilities of given tokens, entropies and the most likely tokens of logit rows, with the logits' gradient
(dm_logprob_rows, dm_logprob_rows_bwd).

For rows x of ``logits`` [..., V] (bf16 or fp32; rows may be padded, a slice ``[..., :V]`` of wider ones) and a target
per row: lse = logsumexp(x), logp = x[target] - lse, entropy = -sum p log p with p = exp(x - lse), in fp32.

  row_logprobs       the values alone (scoring, evaluation, a decode step's tokens)
  row_logprobs_grad  the values and the gradient of sum(g_logp logp + g_entropy entropy) in one pass, for
                     coefficients known beforehand (weights, advantages): what HipTrunk's weighted head runs
  row_logprobs_bwd   the gradient after row_logprobs
  token_logprobs     (logp, entropy) under torch's autograd

A target < 0 is ignored (logp 0, no gradient from it), one >= V gives NaN. Columns of -inf have no probability; a row
of nothing else gives every token -inf, entropy 0 and a zero gradient. A NaN makes its row's values NaN.
"""

from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib as L


class RowLogprobs(NamedTuple):
    logp: Optional[torch.Tensor]      # [...] fp32; None without targets
    entropy: torch.Tensor             # [...] fp32
    lse: torch.Tensor                 # [...] fp32
    stats: torch.Tensor               # [..., 3] fp32: maximum, lse less it, entropy, for row_logprobs_bwd
    top_logp: Optional[torch.Tensor]  # [..., top] fp32, descending; None without top
    top_ids: Optional[torch.Tensor]   # [..., top] int64, the lower id first among equals


def _rows(t, what):
    """(rows, row stride) of [..., V] with unit stride along V and one stride over all rows."""
    V, n = t.shape[-1], t.numel()
    if V > L.DM_LOGPROB_COLS or n > V * 0x7fffffff:
        raise ValueError(f"{what}: rows of shape {tuple(t.shape)} (at most {L.DM_LOGPROB_COLS} columns and 2^31 - 1 rows)")
    if n == 0:
        if V == 0:
            raise ValueError(f"{what}: no columns")
        return 0, V
    if t.is_contiguous():
        return n // V, V
    try:
        t2 = t.view(-1, V)
    except RuntimeError:
        raise ValueError(f"{what}: rows of shape {tuple(t.shape)} and strides {t.stride()} have no single stride; pass "
                         "a contiguous tensor") from None
    rows, ld = t2.shape[0], t2.stride(0)
    if V > 1 and t2.stride(1) != 1:
        raise ValueError(f"{what}: stride {t2.stride(1)} along the columns (1)")
    if rows == 1:
        ld = V
    if ld < V:
        raise ValueError(f"{what}: row stride {ld} < {V} columns (expanded rows overlap; pass a contiguous tensor)")
    return rows, ld


def _per_row(t, logits, what, dtype):
    if t is None:
        return None
    if t.dtype != dtype or t.shape != logits.shape[:-1] or t.device != logits.device or not t.is_contiguous():
        raise ValueError(f"{what}: {t.dtype} {tuple(t.shape)} on {t.device}; contiguous {dtype} "
                         f"{tuple(logits.shape[:-1])} on {logits.device} is needed")
    return t.data_ptr()


def _logits(logits):
    if not logits.is_cuda or logits.dim() < 1:
        raise ValueError(f"logits: shape {tuple(logits.shape)} on {logits.device}; rows [..., V] on a GPU are needed")
    if logits.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("row_logprobs and its like keep no autograd graph: token_logprobs does, or call them under "
                                  "torch.no_grad() or on logits.detach()")
    if forward_ad.unpack_dual(logits).tangent is not None:
        raise NotImplementedError("row_logprobs and its like carry no tangent: call them on logits.detach()")
    return _rows(logits, "logits")


def _gradient(logits, targets, g_logp, g_entropy, dlogits):
    """(dlogits, the arguments that say where the gradient comes from and goes to)."""
    if g_logp is None and g_entropy is None:
        raise ValueError("a gradient needs g_logp or g_entropy")
    if g_logp is not None and targets is None:
        raise ValueError("g_logp needs targets")
    if dlogits is None:
        dlogits = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
    elif dlogits.shape != logits.shape or dlogits.dtype != logits.dtype or dlogits.device != logits.device:
        raise ValueError(f"dlogits: {dlogits.dtype} {tuple(dlogits.shape)} on {dlogits.device} for logits {logits.dtype} "
                         f"{tuple(logits.shape)} on {logits.device}")
    else:   # what torch saved of it is no longer there
        torch.autograd.graph.increment_version(dlogits)
    return dlogits, (_per_row(g_logp, logits, "g_logp", torch.float32), _per_row(g_entropy, logits, "g_entropy", torch.float32),
                     dlogits.data_ptr(), _rows(dlogits, "dlogits")[1])


def _outputs(logits, targets, top):
    lead, dev = logits.shape[:-1], logits.device
    return RowLogprobs(
        None if targets is None else torch.empty(lead, device=dev, dtype=torch.float32),
        torch.empty(lead, device=dev, dtype=torch.float32),
        torch.empty(lead, device=dev, dtype=torch.float32),
        torch.empty((*lead, 3), device=dev, dtype=torch.float32),
        torch.empty((*lead, top), device=dev, dtype=torch.float32) if top else None,
        torch.empty((*lead, top), device=dev, dtype=torch.int64) if top else None)


def _check_outputs(out, logits, targets, top):
    lead = tuple(logits.shape[:-1])
    if out.logp is not None and targets is None:
        raise ValueError("out.logp without targets")
    if (out.top_logp is None or out.top_ids is None) if top else (out.top_logp is not None or out.top_ids is not None):
        raise ValueError(f"out.top_logp and out.top_ids belong to top > 0, both of them (top={top})")
    for name, t, last in zip(RowLogprobs._fields, out, ((), (), (), (3,), (top,), (top,))):
        dtype = torch.int64 if name == "top_ids" else torch.float32
        if t is not None and (t.shape != lead + last or t.dtype != dtype or t.device != logits.device or not t.is_contiguous()):
            raise ValueError(f"out.{name}: {t.dtype} {tuple(t.shape)} on {t.device}; contiguous {dtype} {lead + last} on {logits.device}")


def _forward(logits, targets, top, out, rows, ld, gradient=(None, None, None, 0)):
    V = logits.shape[-1]
    if not 0 <= top <= min(L.DM_TOP_MAX, V):
        raise ValueError(f"top={top} of {V} columns (at most {L.DM_TOP_MAX})")
    t = _per_row(targets, logits, "targets", torch.int64)
    if out is None:
        out = _outputs(logits, targets, top)
    else:
        _check_outputs(out, logits, targets, top)
        torch.autograd.graph.increment_version([o for o in out if o is not None])
    logp, entropy, lse, stats, top_logp, top_ids = out
    a = L.dm_logprob_args(L.dtype_code(logits.dtype), rows, V, top, logits.data_ptr(), ld, t, L.ptr(logp), L.ptr(lse), L.ptr(entropy),
                          L.ptr(stats), L.ptr(top_logp), L.ptr(top_ids), *gradient)
    L.call_on(logits.device, L.lib().dm_logprob_rows, L.byref(a))
    return out


def row_logprobs(logits, targets=None, top=0, out=None):
    """The values of logits [..., V]: logp of ``targets`` (int64 [...], optional), entropy, lse and the ``top`` most
    likely tokens of each row (at most 32). No autograd graph: logits that would need one, or that hold a forward-mode
    tangent, are refused. out: a RowLogprobs of tensors to write into (static buffers of a decode loop), apart from each
    other and the inputs; a field that is None is left out."""
    return _forward(logits, targets, top, out, *_logits(logits))


def row_logprobs_grad(logits, targets, g_logp, g_entropy=None, top=0, dlogits=None, out=None):
    """row_logprobs, and the gradient of sum(g_logp logp + g_entropy entropy) to the logits (fp32 coefficients [...],
    either may be None) in the same pass: (RowLogprobs, dlogits). dlogits: a tensor for the gradient, the logits
    themselves too (in place); by default a new one."""
    rows, ld = _logits(logits)
    dlogits, gradient = _gradient(logits, targets, g_logp, g_entropy, dlogits)
    return _forward(logits, targets, top, out, rows, ld, gradient), dlogits


def row_logprobs_bwd(logits, targets, stats, g_logp, g_entropy=None, dlogits=None):
    """The gradient of row_logprobs_grad after row_logprobs, from the ``stats`` of its result."""
    rows, ld = _logits(logits)
    dlogits, gradient = _gradient(logits, targets, g_logp, g_entropy, dlogits)
    if (stats.shape != logits.shape[:-1] + (3,) or stats.dtype != torch.float32 or stats.device != logits.device
            or not stats.is_contiguous()):
        raise ValueError(f"stats: {stats.dtype} {tuple(stats.shape)} on {stats.device} for logits {tuple(logits.shape)} on {logits.device}")
    a = L.dm_logprob_args(L.dtype_code(logits.dtype), rows, logits.shape[-1], 0, logits.data_ptr(), ld,
                          _per_row(targets, logits, "targets", torch.int64), None, None, None, stats.data_ptr(), None, None,
                          *gradient)
    L.call_on(logits.device, L.lib().dm_logprob_rows_bwd, L.byref(a))
    return dlogits


class TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets):
        r = row_logprobs(logits, targets)
        ctx.save_for_backward(logits, targets)
        ctx.stats = r.stats
        ctx.set_materialize_grads(False)
        return r.logp, r.entropy

    @staticmethod
    def backward(ctx, g_logp, g_entropy):
        if torch.is_grad_enabled():
            raise NotImplementedError("token_logprobs is differentiable once (create_graph)")
        if g_logp is None and g_entropy is None:
            return None, None
        logits, targets = ctx.saved_tensors
        g_logp, g_entropy = (None if g is None else g.contiguous() for g in (g_logp, g_entropy))
        return row_logprobs_bwd(logits, targets, ctx.stats, g_logp, g_entropy), None


def token_logprobs(logits, targets):
    """(logp, entropy) of logits [..., V] and targets [...], differentiable in the logits."""
    rows_ok = logits.stride(-1) == 1 and (logits.dim() < 2 or logits.is_contiguous())
    return TokenLogprobsFn.apply(logits if rows_ok else logits.contiguous(), targets.contiguous())

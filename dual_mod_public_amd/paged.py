"""A paged cache of key / value rows, the attention that reads it, and eviction from it (dm_paged_write,
dm_paged_attention, dm_paged_evict).

``StaticTape`` holds one tape row per batch row and step, all at the same position. Here each sequence has its own length and
its rows lie in pages of a common pool, so requests come and go, and a pass takes any number of new tokens of each:

  K, V      pages [n_pages, h_kv, page, dh] (bf16 or fp32; ``new_pages``)
  table     [B, cols] int32: sequence b's row r lies in page ``table[b, r // page]``
  lengths   [B] int32: cached rows, the pass's new tokens among them
  starts    [B + 1] int32: sequence b's new tokens are ``starts[b] .. starts[b + 1] - 1`` (none is allowed); None: one each,
            none where the length is 0

All of them lie on the device and are read there: a captured pass is replayed with other lengths, tables and starts. The host
does not look at them. A sequence that its table does not hold, or one that reads a page outside the pool, gets NaN; the
results of tokens of no sequence (behind ``starts[B]``) are left as they are.

  paged_write       the new tokens' rows into the pages
  paged_attention   the new tokens' attention over their sequences' rows
  evict_rows        the rows with the largest accumulated attention weight, gathered into new pages
"""

import math
from typing import NamedTuple, Optional

import torch

from . import _lib as L


class PagedAttention(NamedTuple):
    o: torch.Tensor       # [N, h, dh] in q's dtype
    lse: torch.Tensor     # [N, h] fp32: the logarithm of the sum of the exponentials (with the self pair's)


class Evicted(NamedTuple):
    rows: torch.Tensor       # [B, h_kv, keep] int32: the rows kept, ascending; -1 behind them
    lengths: torch.Tensor    # [B] int32
    weights: torch.Tensor    # [B, h_kv, new cols * page] fp32: the kept rows' weights, 0 behind them


def new_pages(n_pages, h_kv, page, dh, device="cuda", dtype=torch.bfloat16):
    """(K, V): an empty pool of n_pages pages of ``page`` rows (a power of two, 16 .. 1024) per key head."""
    shape = (n_pages, h_kv, page, dh)
    return torch.zeros(shape, device=device, dtype=dtype), torch.zeros(shape, device=device, dtype=dtype)


def _forward_only(*tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise NotImplementedError("the paged cache keeps no autograd graph; call it under torch.no_grad() or on detached tensors")


def _pages(K, V):
    if not K.is_cuda or K.dim() != 4 or K.shape != V.shape or K.dtype != V.dtype or K.device != V.device:
        raise ValueError(f"pages: K {K.dtype} {tuple(K.shape)} on {K.device}, V {V.dtype} {tuple(V.shape)} on {V.device}; "
                         "[n_pages, h_kv, page, dh] on a GPU are needed")
    n, h, page, dh = K.shape
    for t in (K, V):
        if t.stride()[1:] != (page * dh, dh, 1) or (n > 1 and t.stride(0) < h * page * dh):
            raise ValueError(f"pages of strides {t.stride()}: each page's rows are contiguous, pages do not overlap")
    if dh not in (64, 128) or page & (page - 1) or not 16 <= page <= L.DM_PAGE_MAX:
        raise NotImplementedError(f"pages of {page} rows of {dh} (a power of two, 16..{L.DM_PAGE_MAX}, rows of 64 or 128)")
    return L.dtype_code(K.dtype), n, h, page, dh, max(K.stride(0), h * page * dh), max(V.stride(0), h * page * dh)


def _index(t, name, shape, device):
    if t.dtype != torch.int32 or t.device != device or not t.is_contiguous() or (shape is not None and tuple(t.shape) != shape):
        raise ValueError(f"{name}: {t.dtype} {tuple(t.shape)} on {t.device}; contiguous int32"
                         f"{'' if shape is None else f' {shape}'} on {device} is needed")
    return t.data_ptr()


def _tokens(t, name, shape, like):
    """(address, token stride, head stride) of rows [N, heads, dh]."""
    if t.dtype != like.dtype or tuple(t.shape) != shape or t.device != like.device or (t.numel() and t.stride(2) != 1):
        raise ValueError(f"{name}: {t.dtype} {tuple(t.shape)} of strides {t.stride()} on {t.device}; {like.dtype} {shape} with "
                         f"unit stride in a row on {like.device} is needed")
    return t.data_ptr(), t.stride(0), t.stride(1)


def _args(K, V, table, lengths, starts, n_tokens):
    dtype, n_pages, h_kv, page, dh, k_page, v_page = _pages(K, V)
    if table.dim() != 2:
        raise ValueError(f"table: {tuple(table.shape)}; [B, cols] is needed")
    B, dev = table.shape[0], K.device
    if starts is None and n_tokens != B:
        raise ValueError(f"{n_tokens} tokens of {B} sequences without starts")
    a = L.dm_paged_args(dtype=dtype, B=B, h_kv=h_kv, dh=dh, page=page, n_pages=n_pages, table_cols=table.shape[1],
                        n_tokens=n_tokens, K=K.data_ptr(), V=V.data_ptr(), k_page=k_page, v_page=v_page,
                        table=_index(table, "table", None, dev), lengths=_index(lengths, "lengths", (B,), dev),
                        starts=None if starts is None else _index(starts, "starts", (B + 1,), dev))
    return a


def paged_write(k, v, K, V, table, lengths, starts=None):
    """The rows k, v [N, h_kv, dh] of the new tokens (any strides of tokens and heads) into their places in the pages."""
    _forward_only(k, v, K, V)
    a = _args(K, V, table, lengths, starts, k.shape[0])
    shape = (k.shape[0], a.h_kv, a.dh)
    a.k_rows, a.k_token, a.k_head = _tokens(k, "k", shape, K)
    a.v_rows, a.v_token, a.v_head = _tokens(v, "v", shape, K)
    if a.B == 0 or a.n_tokens == 0:
        return
    torch.autograd.graph.increment_version([K, V])
    L.call_on(K.device, L.lib().dm_paged_write, L.byref(a))


def paged_attention(q, K, V, table, lengths, starts=None, k_self=None, v_self=None, window=0, scale=None, weights=None, out=None):
    """Attention of the new tokens' queries q [N, h, dh] (h a multiple of the pages' h_kv; any strides of tokens and heads)
    over their sequences' cached rows, each token over the rows up to its own.

    k_self, v_self [N, h_kv, dh]: a pair per token that takes its own row's place (the raw self pair of
    ``DualModAttention.attend_one``: the cache's row is the refined one, written later, and is not read). window W: the last W rows, the
    token's own counted. scale: by default 1 / sqrt(dh). weights [B, h_kv, cols * page] fp32: to each cached row its probabilities
    are added, summed over the pass's tokens and the heads that share the key head. out: a tensor [N, h, dh] for o.
    Returns PagedAttention(o, lse); a token that reads nothing has o = 0 and lse = -inf. No gradients."""
    _forward_only(q, K, V, k_self, v_self)
    if q.dim() != 3:
        raise ValueError(f"q: {tuple(q.shape)}; [N, h, dh] is needed")
    N, h, dev = q.shape[0], q.shape[1], K.device
    a = _args(K, V, table, lengths, starts, N)
    if h == 0 or h % a.h_kv:
        raise ValueError(f"{h} query heads for {a.h_kv} key heads")
    a.h = h
    a.q, a.q_token, a.q_head = _tokens(q, "q", (N, h, a.dh), K)
    if (k_self is None) != (v_self is None):
        raise ValueError("k_self and v_self belong together")
    if k_self is not None:
        a.k_rows, a.k_token, a.k_head = _tokens(k_self, "k_self", (N, a.h_kv, a.dh), K)
        a.v_rows, a.v_token, a.v_head = _tokens(v_self, "v_self", (N, a.h_kv, a.dh), K)
    if window < 0:
        raise ValueError(f"window={window}")
    a.window, a.scale = min(int(window), 0x7fffffff), 1.0 / math.sqrt(a.dh) if scale is None else float(scale)
    if weights is not None:
        shape = (a.B, a.h_kv, a.table_cols * a.page)
        if weights.dtype != torch.float32 or tuple(weights.shape) != shape or weights.device != dev or not weights.is_contiguous():
            raise ValueError(f"weights: {weights.dtype} {tuple(weights.shape)} on {weights.device}; contiguous fp32 {shape} on {dev}")
        a.weights = weights.data_ptr()
    if out is None:
        out = torch.empty(N, h, a.dh, device=dev, dtype=q.dtype)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError(f"out: {out.dtype} {tuple(out.shape)} on {out.device}; contiguous {q.dtype} {tuple(q.shape)} on {dev}")
    lse = torch.empty(N, h, device=dev)
    if N == 0 or a.B == 0:
        return PagedAttention(out, lse)
    a.o, a.lse = out.data_ptr(), lse.data_ptr()
    ws = torch.empty(L.lib().dm_paged_workspace_bytes(L.byref(a)), dtype=torch.uint8, device=dev)
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    written = [t for t in (out, weights) if t is not None]
    torch.autograd.graph.increment_version(written)
    L.call_on(dev, L.lib().dm_paged_attention, L.byref(a))
    return PagedAttention(out, lse)


def evict_rows(K, V, weights, table, lengths, keep, new_table, sinks=0, recent=0):
    """Shortens sequences to at most ``keep`` rows: of each key head the rows 0 .. sinks - 1, the last ``recent`` ones and those of
    the others with the largest ``weights`` [B, h_kv, cols * page] (of equal ones the lower row), copied in their order into
    the pages that new_table [B, new cols] names, which no table of the call names as sources. The old pages are left as they
    are (a prefix that sequences share stays whole). Positions are the caller's: keys are stored rotated. Returns Evicted; the sequences go
    on with new_table, its lengths and weights."""
    _forward_only(K, V)
    dtype, n_pages, h_kv, page, dh, k_page, v_page = _pages(K, V)
    if table.dim() != 2 or new_table.dim() != 2 or new_table.shape[0] != table.shape[0]:
        raise ValueError(f"tables: {tuple(table.shape)}, {tuple(new_table.shape)}; [B, cols] of the same sequences are needed")
    B, dev = table.shape[0], K.device
    cap, new_cap = table.shape[1] * page, new_table.shape[1] * page
    keep, sinks, recent = int(keep), int(sinks), int(recent)
    if keep < 1 or sinks < 0 or recent < 0 or sinks + recent > keep:
        raise ValueError(f"keep={keep} sinks={sinks} recent={recent}")
    if new_cap < min(keep, cap):
        raise ValueError(f"new_table holds {new_cap} rows; keep={keep}")
    if weights.dtype != torch.float32 or tuple(weights.shape) != (B, h_kv, cap) or weights.device != dev or not weights.is_contiguous():
        raise ValueError(f"weights: {weights.dtype} {tuple(weights.shape)} on {weights.device}; contiguous fp32 {(B, h_kv, cap)} on {dev}")
    out = Evicted(torch.empty(B, h_kv, keep, dtype=torch.int32, device=dev), torch.empty(B, dtype=torch.int32, device=dev),
                  torch.empty(B, h_kv, new_cap, device=dev))
    a = L.dm_evict_args(dtype, B, h_kv, dh, page, n_pages, table.shape[1], new_table.shape[1], keep, sinks, recent, 0, K.data_ptr(),
                        V.data_ptr(), k_page, v_page, _index(table, "table", None, dev), _index(lengths, "lengths", (B,), dev),
                        _index(new_table, "new_table", None, dev), weights.data_ptr(), out.weights.data_ptr(),
                        out.rows.data_ptr(), out.lengths.data_ptr())
    if B == 0:
        return out
    torch.autograd.graph.increment_version([K, V])
    L.call_on(dev, L.lib().dm_paged_evict, L.byref(a))
    return out

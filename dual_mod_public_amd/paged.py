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
does not look at them. A sequence that its table does not hold gets NaN, and so does a token that reads a row of a page outside the
pool (and others of its sequence may); the results of tokens of no sequence (behind ``starts[B]``) are left as they are.

  paged_write       the new tokens' rows into the pages
  paged_attention   the new tokens' attention over their sequences' rows
  evict_rows        the rows with the largest accumulated attention weight, gathered into new pages
"""

from typing import NamedTuple

import torch
from torch.autograd import forward_ad

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


def _no_graph(t, what="the paged cache"):
    if t is None:
        return
    if t.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"{what} keeps no autograd graph; call it under torch.no_grad() or on detached tensors")
    # (the level first: unpacking costs more than the rest of a check, and outside of one there are no tangents)
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise NotImplementedError(f"{what} carries no tangent; call it on detached tensors")


def _extent(t):
    """The addresses [from, to) that a tensor's elements lie in."""
    p = t.data_ptr()
    return p, p + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size() if t.numel() else p


def _apart(what, out, *others):
    lo, hi = _extent(out)
    for t in others:
        if t is not None:
            a, b = _extent(t)
            if a < hi and lo < b:
                raise ValueError(f"{what} overlaps a tensor that the call reads")


# The checks compare device numbers and whole tuples: small calls are bound by the host, and torch's device objects and
# generators over tensors cost more than the rest of a check.

def _pages(K, V):
    """(dtype, n_pages, h_kv, page, dh, strides of K's and V's pages)."""
    if not K.is_cuda or K.dim() != 4 or K.shape != V.shape or K.dtype != V.dtype or K.get_device() != V.get_device():
        raise ValueError(f"pages: K {K.dtype} {tuple(K.shape)} on {K.device}, V {V.dtype} {tuple(V.shape)} on {V.device}; "
                         "[n_pages, h_kv, page, dh] on a GPU are needed")
    _no_graph(K), _no_graph(V)
    n, h, page, dh = K.shape
    rows, ks, vs = h * page * dh, K.stride(), V.stride()
    if n == 1:
        ks, vs = (max(ks[0], rows), *ks[1:]), (max(vs[0], rows), *vs[1:])
    for s in (ks, vs):
        if s[3] != 1 or s[2] != dh or s[1] != page * dh or s[0] < rows:
            raise ValueError(f"pages of strides {s}: each page's rows are contiguous, pages do not overlap")
    if dh not in (64, 128) or page & (page - 1) or not 16 <= page <= L.DM_PAGE_MAX:
        raise NotImplementedError(f"pages of {page} rows of {dh} (a power of two, 16..{L.DM_PAGE_MAX}, rows of 64 or 128)")
    return L.dtype_code(K.dtype), n, h, page, dh, ks[0], vs[0]


def _index(t, name, shape, device):
    if t.dtype != torch.int32 or t.get_device() != device or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name}: {t.dtype} {tuple(t.shape)} on {t.device}; contiguous int32 {tuple(shape)} on cuda:{device} is needed")
    return t.data_ptr()


def _tokens(t, name, shape, like):
    """(address, token stride, head stride) of rows [N, heads, dh]."""
    _no_graph(t)
    if t.dtype != like.dtype or t.shape != shape or t.get_device() != like.get_device():
        raise ValueError(f"{name}: {t.dtype} {tuple(t.shape)} on {t.device}; {like.dtype} {shape} on {like.device} is needed")
    s = t.stride()
    if s[2] != 1 and t.numel():
        raise ValueError(f"{name}: strides {s}; unit stride in a row is needed")
    return t.data_ptr(), s[0], s[1]


def _weights(t, shape, device):
    _no_graph(t)
    if t.dtype != torch.float32 or t.shape != shape or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"weights: {t.dtype} {tuple(t.shape)} on {t.device}; contiguous fp32 {shape} on cuda:{device} is needed")
    return t.data_ptr()


def _sequences(table, lengths, starts, n_tokens, device):
    """(B, cols, addresses of table, lengths and starts)."""
    if table.dim() != 2:
        raise ValueError(f"table: {tuple(table.shape)}; [B, cols] is needed")
    B, cols = table.shape
    if n_tokens > 0x7fffffff or B > 0x7fffffff or cols > 0x7fffffff:     # (the library's counts; it refuses most of these too)
        raise ValueError(f"{n_tokens} tokens of sequences of a table {tuple(table.shape)}: too many")
    if starts is None and n_tokens != B:
        raise ValueError(f"{n_tokens} tokens of {B} sequences without starts")
    return (B, cols, _index(table, "table", table.shape, device), _index(lengths, "lengths", (B,), device),
            None if starts is None else _index(starts, "starts", (B + 1,), device))


def paged_write(k, v, K, V, table, lengths, starts=None):
    """The rows k, v [N, h_kv, dh] of the new tokens (any strides of tokens and heads; rows of the pool too, but none that the call
    writes) into their places in the pages."""
    dtype, n_pages, h_kv, page, dh, k_page, v_page = _pages(K, V)
    N = k.shape[0]
    B, cols, table_p, lengths_p, starts_p = _sequences(table, lengths, starts, N, K.get_device())
    k_rows, v_rows = _tokens(k, "k", (N, h_kv, dh), K), _tokens(v, "v", (N, h_kv, dh), K)
    if B == 0 or N == 0:
        return
    a = L.dm_paged_args(dtype, B, h_kv, h_kv, dh, page, n_pages, cols, N, 0, 1.0, 0, None, 0, 0, K.data_ptr(), V.data_ptr(), k_page, v_page,
                        table_p, lengths_p, starts_p, *k_rows, *v_rows)
    torch.autograd.graph.increment_version((K, V))
    L.call_on(K.device, L.lib().dm_paged_write, L.byref(a))


def paged_attention(q, K, V, table, lengths, starts=None, k_self=None, v_self=None, window=0, scale=None, weights=None, out=None):
    """Attention of the new tokens' queries q [N, h, dh] (h a multiple of the pages' h_kv; any strides of tokens and heads)
    over their sequences' cached rows, each token over the rows up to its own.

    k_self, v_self [N, h_kv, dh]: a pair per token that takes its own row's place (the raw self pair of
    ``DualModAttention.attend_one``: the cache's row is the refined one, written later, and is not read). window W: the last W rows, the
    token's own counted. scale: by default 1 / sqrt(dh). weights [B, h_kv, cols * page] fp32: to each cached row its probabilities
    are added, summed over the pass's tokens and the heads that share the key head. out: a tensor [N, h, dh] for o.
    Returns PagedAttention(o, lse); a token that reads nothing has o = 0 and lse = -inf. No gradients."""
    _no_graph(q)
    dtype, n_pages, h_kv, page, dh, k_page, v_page = _pages(K, V)
    if q.dim() != 3:
        raise ValueError(f"q: {tuple(q.shape)}; [N, h, dh] is needed")
    N, h, _ = q.shape
    if h == 0 or h % h_kv:
        raise ValueError(f"{h} query heads for {h_kv} key heads")
    dev = K.get_device()
    B, cols, table_p, lengths_p, starts_p = _sequences(table, lengths, starts, N, dev)
    if k_self is not None and v_self is not None:
        pair = (*_tokens(k_self, "k_self", (N, h_kv, dh), K), *_tokens(v_self, "v_self", (N, h_kv, dh), K))
    elif k_self is None and v_self is None:
        pair = (None, 0, 0, None, 0, 0)
    else:
        raise ValueError("k_self and v_self belong together")
    if window < 0:
        raise ValueError(f"window={window}")
    q_rows = _tokens(q, "q", (N, h, dh), K)
    weights_p = None if weights is None else _weights(weights, (B, h_kv, cols * page), dev)
    if out is None:
        out = q.new_empty((N, h, dh))
    elif out.shape != q.shape or out.dtype != q.dtype or out.get_device() != dev or not out.is_contiguous():
        raise ValueError(f"out: {out.dtype} {tuple(out.shape)} on {out.device}; contiguous {q.dtype} {tuple(q.shape)} on {K.device}")
    else:
        _no_graph(out)
        _apart("out", out, q, K, V, k_self, v_self, weights)
        torch.autograd.graph.increment_version(out)
    if weights is not None and K.dtype == torch.float32:
        _apart("weights", weights, q, K, V, k_self, v_self)
    lse = torch.empty((N, h), dtype=torch.float32, device=K.device)
    if N == 0 or B == 0:
        return PagedAttention(out, lse)
    a = L.dm_paged_args(dtype, B, h, h_kv, dh, page, n_pages, cols, N, min(int(window), 0x7fffffff),
                        dh ** -0.5 if scale is None else float(scale), 0, *q_rows, K.data_ptr(), V.data_ptr(), k_page, v_page, table_p,
                        lengths_p, starts_p, *pair, out.data_ptr(), lse.data_ptr(), weights_p)
    args = L.byref(a)
    nb = L.lib().dm_paged_workspace_bytes(args)
    if nb:
        ws = torch.empty(nb, dtype=torch.uint8, device=K.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), nb
    if weights is not None:
        torch.autograd.graph.increment_version(weights)
    L.call_on(K.device, L.lib().dm_paged_attention, args)
    return PagedAttention(out, lse)


def evict_rows(K, V, weights, table, lengths, keep, new_table, sinks=0, recent=0):
    """Shortens sequences to at most ``keep`` rows: of each key head the rows 0 .. sinks - 1, the last ``recent`` ones and those of
    the others with the largest ``weights`` [B, h_kv, cols * page] (of equal ones the lower row), copied in their order into
    the pages that new_table [B, new cols] names, which no table of the call names as sources. The old pages are left as they
    are (a prefix that sequences share stays whole). Positions are the caller's: keys are stored rotated. Returns Evicted; the sequences go
    on with new_table, its lengths and weights."""
    dtype, n_pages, h_kv, page, dh, k_page, v_page = _pages(K, V)
    if new_table.dim() != 2 or new_table.shape[0] != table.shape[0]:
        raise ValueError(f"tables: {tuple(table.shape)}, {tuple(new_table.shape)}; [B, cols] of the same sequences are needed")
    dev = K.get_device()
    B, cols, table_p, lengths_p, _ = _sequences(table, lengths, None, table.shape[0], dev)
    cap, new_cols = cols * page, new_table.shape[1]
    keep, sinks, recent = int(keep), int(sinks), int(recent)
    if not 1 <= keep <= 0x7fffffff or sinks < 0 or recent < 0 or sinks + recent > keep:
        raise ValueError(f"keep={keep} sinks={sinks} recent={recent} (at most 2^31 - 1)")
    if new_cols * page < min(keep, cap):
        raise ValueError(f"new_table holds {new_cols * page} rows; keep={keep}")
    weights_p = _weights(weights, (B, h_kv, cap), dev)
    out = Evicted(table.new_empty((B, h_kv, keep)), table.new_empty((B,)), weights.new_empty((B, h_kv, new_cols * page)))
    if B == 0:
        return out
    a = L.dm_evict_args(dtype, B, h_kv, dh, page, n_pages, cols, new_cols, keep, sinks, recent, 0, K.data_ptr(), V.data_ptr(), k_page,
                        v_page, table_p, lengths_p, _index(new_table, "new_table", new_table.shape, dev), weights_p,
                        out.weights.data_ptr(), out.rows.data_ptr(), out.lengths.data_ptr())
    torch.autograd.graph.increment_version((K, V))
    L.call_on(K.device, L.lib().dm_paged_evict, L.byref(a))
    return out

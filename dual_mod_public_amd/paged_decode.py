"""Dual-Mod layers and models over a paged cache: sequences of different lengths, any number of new tokens of each per pass
(continuous batching, prompt chunks, drafted tokens).

``StaticTape`` and ``GraphDecoder`` step a fixed batch, all rows at one position, a token at a time. Here a pass takes N new
tokens of B sequences (``paged``'s table, lengths and starts). One new token per sequence is the exact step. A chunk of c
tokens is the chunk cell's (engine.chunk_cell_forward): its raw pairs go into the pages, then each sweep reads the cache with the
tokens' own raw pairs (paged.paged_attention), refines every token's pair (dm_refine_kv) and writes it; c sweeps are the exact
scan (nilpotency, scan_cell_fwd.py:1-10), fewer the chunked Jacobi result. ``positions`` are the tokens' places in their texts
(for the rotation); a sequence's rows may be fewer, after an eviction.
"""

import ctypes

import torch
import torch.nn.functional as F

from . import _lib as L
from .engine import LayerBufs, PackedWeights, check_supported
from .paged import evict_rows, new_pages, paged_attention, paged_write


class PagedTape:
    """One layer's pages of refined keys (rotated) and values. attn: a DualModAttention."""

    def __init__(self, attn, n_pages, page=64, dtype=torch.bfloat16):
        cfg = attn.cfg
        check_supported(cfg)
        self.attn, self.cfg, self.dtype = attn, cfg, dtype
        self.device = attn.wq.weight.device
        self.K, self.V = new_pages(n_pages, cfg.n_heads, page, cfg.head_dim, self.device, dtype)
        self.w = PackedWeights(cfg, self.device, dtype, with_transposes=False)
        self.conf = L.make_config(cfg, 1, dtype)
        # attend_one's window: with W = 1 it reads the whole past (attention.py:292-293)
        W = int(getattr(cfg, "local_window", 0) or 0)
        self.window = W if W > 1 else 0
        self._ver = None
        self.refresh()

    def refresh(self):
        """Packs the attention's weights again where a parameter has changed (outside a capture)."""
        ver = self.attn._param_version()
        if ver != self._ver:
            self.w.pack(dict(self.attn.named_parameters()))
            self._ver = ver

    @torch.no_grad()
    def extend(self, xhat, positions, cos, sin, table, lengths, starts=None, n_sweeps=None, weights=None):
        """xhat [N, d] (pre-normed, the tape's dtype) of the new tokens at ``positions`` [N] (int64); cos, sin: RoPE tables.
        Their refined rows are in the pages afterwards. n_sweeps: 1 without starts; with starts the longest chunk's length gives
        the exact scan, fewer the chunk cell's Jacobi result. weights: see paged_attention (of the last sweep). Returns W_O o [N, d]; rows of
        tokens of no sequence hold anything (their positions are looked up all the same)."""
        if n_sweeps is None:
            if starts is not None:
                raise ValueError("chunks need n_sweeps (the longest one's length: the exact scan)")
            n_sweeps = 1
        if n_sweeps < 1:
            raise ValueError(f"n_sweeps={n_sweeps}")
        N, d = xhat.shape[0], self.cfg.d_model
        if xhat.dtype != self.dtype or xhat.shape != (N, d) or xhat.device != self.device:
            raise ValueError(f"xhat: {xhat.dtype} {tuple(xhat.shape)} on {xhat.device}; {self.dtype} [N, {d}] on {self.device} is needed")
        if positions.shape != (N,) or positions.dtype != torch.int64:
            raise ValueError(f"positions: {positions.dtype} {tuple(positions.shape)}; int64 [{N}] is needed")
        if N == 0:
            return xhat.new_empty(0, d)
        with torch.cuda.device(self.device):     # the launches below are the current device's
            return self._extend(xhat, positions, cos, sin, (self.K, self.V, table, lengths, starts), n_sweeps, weights)

    def _extend(self, xhat, positions, cos, sin, cache, n_sweeps, weights):
        cfg, N = self.cfg, xhat.shape[0]
        d, h, dh = cfg.d_model, cfg.n_heads, cfg.head_dim
        self.refresh()
        xhat = xhat.contiguous()
        cos, sin = (t.index_select(0, positions).float().contiguous() for t in (cos, sin))
        bufs = LayerBufs(cfg, 1, N, self.device, self.dtype)
        conf, w, b = ctypes.byref(self.conf), self.w.struct(with_attn_norm=False), bufs.struct()
        L.check(L.lib().dm_layer_proj(conf, ctypes.byref(w), L.ptr(xhat), L.ptr(cos), L.ptr(sin), ctypes.byref(b), L.stream_ptr()))
        q, k_self, v_self = (t[0].transpose(0, 1) for t in (bufs.qr, bufs.kself, bufs.vraw))      # [N, h, dh]
        K, V = (torch.empty(h, N, dh, device=self.device, dtype=self.dtype) for _ in range(2))
        nb = L.lib().dm_refine_kv_workspace_bytes(conf, N)
        ws = torch.empty(nb, device=self.device, dtype=torch.uint8)
        if cache[-1] is not None:     # chunks: the first sweep, which may be the only one, reads their raw rows
            paged_write(k_self, v_self, *cache)
        for i in range(n_sweeps):
            o = paged_attention(q, *cache, k_self=k_self, v_self=v_self, window=self.window,
                                weights=weights if i + 1 == n_sweeps else None).o
            L.check(L.lib().dm_refine_kv(conf, ctypes.byref(w), ctypes.byref(b), L.ptr(o), L.ptr(cos), L.ptr(sin), L.ptr(K), L.ptr(V),
                                         L.ptr(ws), nb, L.stream_ptr()))
            paged_write(K.transpose(0, 1), V.transpose(0, 1), *cache)
        return L.linear(o.view(N, d), self.w.wo)

    def evict(self, weights, table, lengths, keep, new_table, sinks=0, recent=0):
        """paged.evict_rows on this layer's pages."""
        if self.window:
            raise NotImplementedError("a local window counts cached rows: its rows are not evicted")
        return evict_rows(self.K, self.V, weights, table, lengths, keep, new_table, sinks=sinks, recent=recent)


class PagedDecoder:
    """A DualModLM over paged tapes, one per layer with the same table: ``extend`` gives the logits of every new token's row
    (the next token's distribution), for sampling or for drafts.verify_drafts."""

    def __init__(self, model, n_pages, page=64, dtype=None):
        self.m, self.dt = model, dtype or model.dtype
        self.tapes = [PagedTape(blk.attn, n_pages, page, self.dt) for blk in model.blocks]

    @torch.no_grad()
    def extend(self, ids, positions, table, lengths, starts=None, n_sweeps=None, weights=None):
        """ids [N] (int64) at ``positions`` [N]; weights: one tensor per layer (paged_attention's), or None. Returns logits [N, V]
        in the compute dtype."""
        m, dt = self.m, self.dt
        x = F.embedding(ids, m.tok_emb.weight).float().contiguous()          # the fp32 residual stream [N, d]
        if ids.numel() == 0:
            return x.new_empty(0, m.cfg.vocab_size, dtype=dt)
        h = L.residual_rmsnorm(x, None, m.blocks[0].attn_norm.weight, dt, eps=m.blocks[0].attn_norm.eps)
        for l, (blk, tape) in enumerate(zip(m.blocks, self.tapes)):
            y = tape.extend(h, positions, m.rope_cos, m.rope_sin, table, lengths, starts, n_sweeps, None if weights is None else weights[l])
            h = L.residual_rmsnorm(x, y, blk.mlp_norm.weight, dt, eps=blk.mlp_norm.eps)
            nrm = m.blocks[l + 1].attn_norm if l + 1 < len(m.blocks) else m.norm_f
            h = L.residual_rmsnorm(x, blk.mlp.decode(h), nrm.weight, dt, eps=nrm.eps)
        return F.linear(h, m.lm_head.weight.to(dt))

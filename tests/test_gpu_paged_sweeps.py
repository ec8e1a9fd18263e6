"""Chunks through PagedTape and PagedDecoder with any number of sweeps, in both types, on pages whose places hold NaN until
a call fills them."""

import math

import pytest
import torch

import oracle as O
from dual_mod_public_amd import _lib as L
from dual_mod_public_amd.attention import DualModAttention
from dual_mod_public_amd.paged_decode import PagedTape
from dual_mod_public_amd.synthetic import make_input, make_state_dict
from tests.hip_helpers import DEV, cfg_of, record, relerr

pytestmark = pytest.mark.gpu
# Relative errors in the 2-norm. fp32: sums of 256 and 512 products, whose roundings of 2^-24 each add like their squares' root (some
# 2e-6 through a layer). bf16: x^, q, k, v, o, the refined pair and y are rounded once each, up to 2^-8 and 2^-8 / sqrt(3) on
# average: sqrt(8) of those are 6e-3, and a refined row takes o's into its products again.
TOL = {torch.float32: 1e-5, torch.bfloat16: 2e-2}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    L.load()


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def attention(cfg, sd):
    attn = DualModAttention(cfg).to(DEV)
    attn.load_state_dict({k: v.float() for k, v in sd.items()}, strict=False)
    return attn


def filled(tape, table, pasts, seed):
    """NaN in all pages but for random rows of each sequence's past; (K, V) of those in 64 bits, [1, h, past, dh] each."""
    g = torch.Generator().manual_seed(seed)
    tape.K.fill_(math.nan), tape.V.fill_(math.nan)
    page, out = tape.K.shape[2], []
    for b, n in enumerate(pasts):
        r = torch.arange(n, device=DEV)
        at = table[b].long()[r // page]
        pair = []
        for pages in (tape.K, tape.V):
            rows = torch.randn(n, pages.shape[1], pages.shape[3], generator=g).to(tape.dtype)
            pages[at, :, r % page] = rows.to(DEV)
            pair.append(rows.double().transpose(0, 1)[None])
        out.append(pair)
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n_sweeps", [1, 2, 5, 6])
@pytest.mark.parametrize("knobs", [dict(ctx_mod="mult_res"), dict(ctx_mod="linear", local_window=4),
                                   dict(ctx_mod="mult", local_window=1)])
def test_chunks_with_any_number_of_sweeps(dtype, n_sweeps, knobs):
    """Chunks of 6, 1 and 3 tokens behind pasts of 19, 5 and no rows: n_sweeps Jacobi sweeps, of which the first reads the chunk's
    raw rows (the oracle's cell in 64 bits; sweeps beyond a chunk's length change nothing)."""
    cfg = cfg_of(d=256, h=4, T=64, **knobs)
    sd = make_state_dict(cfg, seed=31, with_attn_norm=False)
    sd = {k: (v.to(dtype) if v.dim() == 2 else v).double() for k, v in sd.items()}
    cos, sin = O.build_rope_cache(64, cfg.head_dim, cfg.rope_theta, dtype=torch.float64)
    pasts, counts, page = [19, 5, 0], [6, 1, 3], 16
    tape = PagedTape(attention(cfg, sd), 8, page, dtype)
    table = i32([7, 2], [0, -1], [4, -1])
    past = filled(tape, table, pasts, seed=5)
    x = make_input((1, sum(counts), 256), seed=6)[0].to(dtype)
    pos = torch.cat([torch.arange(p, p + c) for p, c in zip(pasts, counts)])
    y = tape.extend(x.to(DEV), pos.to(DEV), cos.to(DEV), sin.to(DEV), table, i32(*[p + c for p, c in zip(pasts, counts)]),
                    i32(0, 6, 7, 10), n_sweeps=n_sweeps)
    errs, t0 = {}, 0
    for b, (p, c) in enumerate(zip(pasts, counts)):
        o, K, V = O.chunk_cell_forward(cfg, sd, x[None, t0:t0 + c].double(), cos[p:p + c], sin[p:p + c], *past[b], n_sweeps)
        errs[f"y{b}"] = relerr(y[t0:t0 + c], o[0] @ sd["wo.weight"].t())
        r = torch.arange(p, p + c, device=DEV)
        at = table[b].long()[r // page]
        for name, pages, rows in (("K", tape.K, K), ("V", tape.V, V)):
            errs[f"{name}{b}"] = relerr(pages[at, :, r % page].transpose(0, 1), rows[0])
        t0 += c
    record(f"paged chunks {knobs} {dtype} sweeps {n_sweeps}", errs, TOL[dtype])
    assert all(e < TOL[dtype] for e in errs.values()), errs

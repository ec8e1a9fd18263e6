"""Chunks through PagedTape and PagedDecoder with any number of sweeps, in both types, on pages whose places hold NaN until
a call fills them."""

import math

import pytest
import torch

import oracle as O
from dual_mod_public_amd import _lib as L
from dual_mod_public_amd.attention import DualModAttention
from dual_mod_public_amd.config import DualModConfig
from dual_mod_public_amd.model import DualModLM
from dual_mod_public_amd.paged_decode import PagedDecoder, PagedTape
from dual_mod_public_amd.synthetic import make_input, make_lm_state_dict, make_state_dict
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


@pytest.mark.parametrize("with_starts", [False, True])
@pytest.mark.parametrize("knobs", [dict(ctx_mod="mult_res"), dict(ctx_mod="fusion", local_window=30)])
@pytest.mark.parametrize("d,h", [(256, 4), (256, 2)])
def test_single_tokens_in_bf16(with_starts, knobs, d, h):
    """Three steps of one token per sequence behind pasts of 100, 1 and 0 rows, against the oracle's step in 64 bits."""
    cfg = cfg_of(d=d, h=h, T=128, **knobs)
    sd = make_state_dict(cfg, seed=32, with_attn_norm=False)
    sd = {k: (v.bfloat16() if v.dim() == 2 else v).double() for k, v in sd.items()}
    cos, sin = O.build_rope_cache(128, cfg.head_dim, cfg.rope_theta, dtype=torch.float64)
    pasts, page = [100, 1, 0], 16
    tape = PagedTape(attention(cfg, sd), 12, page)
    table = i32([7, 2, 9, 4, 11, 0, 5], [1] + [-1] * 6, [8] + [-1] * 6)
    caches = [dict(zip("KV", kv)) for kv in filled(tape, table, pasts, seed=8)]
    x = make_input((3, 3, d), seed=9).bfloat16()
    errs = {}
    for t in range(3):
        lengths = [p + t + 1 for p in pasts]
        y = tape.extend(x[:, t].to(DEV), torch.tensor([n - 1 for n in lengths], device=DEV), cos.to(DEV), sin.to(DEV), table, i32(*lengths),
                        **(dict(starts=i32(0, 1, 2, 3), n_sweeps=1) if with_starts else {}))
        for b, n in enumerate(lengths):
            _, want = O.decode_step(cfg, sd, x[b:b + 1, t:t + 1].double(), n - 1, caches[b], cos, sin)
            errs[f"y{b}@{t}"] = relerr(y[b], want[0, 0])
            at = int(table[b, (n - 1) // page])
            for name, pages in (("K", tape.K), ("V", tape.V)):
                errs[f"{name}{b}@{t}"] = relerr(pages[at, :, (n - 1) % page], caches[b][name][0, :, n - 1])
    record(f"paged single tokens {knobs} h={h}", errs, TOL[torch.bfloat16])
    assert all(e < TOL[torch.bfloat16] for e in errs.values()), errs


def test_decoder_in_bf16():
    """Three texts through a bf16 model in chunks of 0 to 9 tokens, exact sweeps: the oracle's 64-bit model within bf16's tolerance,
    and the same token wherever its two largest logits lie further apart than twice the largest error."""
    cfg = DualModConfig(d_model=256, n_heads=4, n_layers=2, vocab_size=512, max_seq_len=64, mlp_hidden_override=512, checkpoint_chunk=0,
                        ctx_mod="mult_res")
    sd = make_lm_state_dict(cfg, seed=7, std=0.02)
    m = DualModLM(cfg, dtype=torch.bfloat16).to(DEV)
    m.load_state_dict({k: v.to(DEV) for k, v in sd.items()})
    dec = PagedDecoder(m, 10, 16)
    for tape in dec.tapes:
        assert tape.K.dtype == torch.bfloat16
        tape.K.fill_(math.nan), tape.V.fill_(math.nan)
    g = torch.Generator().manual_seed(3)
    texts = [torch.randint(0, 512, (n,), generator=g) for n in (48, 17, 31)]
    table = i32([9, 0, 4], [2, 7, -1], [5, 3, -1])
    done, rows = [0, 0, 0], [[], [], []]
    while done != [48, 17, 31]:
        n = [min(int(torch.randint(0, 10, (), generator=g)), len(t) - k) for t, k in zip(texts, done)]
        if not sum(n):
            continue
        ids = torch.cat([t[k:k + c] for t, k, c in zip(texts, done, n)]).to(DEV)
        pos = torch.cat([torch.arange(k, k + c) for k, c in zip(done, n)]).to(DEV)
        done = [k + c for k, c in zip(done, n)]
        logits = dec.extend(ids, pos, table, i32(*done), i32(0, n[0], n[0] + n[1], sum(n)), n_sweeps=max(n))
        for b, part in enumerate(logits.cpu().split(n)):
            rows[b].append(part)
    for b, text in enumerate(texts):
        got = torch.cat(rows[b]).double()
        cos, sin = O.build_rope_cache(len(text), cfg.head_dim, cfg.rope_theta, dtype=torch.float64)
        want = O.lm_forward(cfg, {k: v.double() for k, v in sd.items()}, text[None], cos, sin)[0]
        err, off = relerr(got, want), float((got - want).abs().max())
        record(f"paged decoder bf16 text {b}", {"logits": err}, TOL[torch.bfloat16])
        top = want.topk(2, -1).values
        decided = top[:, 0] - top[:, 1] > 2 * off
        assert err < TOL[torch.bfloat16] and torch.equal(got.argmax(-1)[decided], want.argmax(-1)[decided])

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


def decoder(dtype, n_pages, layers=2):
    cfg = DualModConfig(d_model=256, n_heads=4, n_layers=layers, vocab_size=512, max_seq_len=128, mlp_hidden_override=512,
                        checkpoint_chunk=0, ctx_mod="mult_res")
    m = DualModLM(cfg, dtype=dtype).to(DEV)
    m.load_state_dict({k: v.to(DEV) for k, v in make_lm_state_dict(cfg, seed=7, std=0.02).items()})
    return m, PagedDecoder(m, n_pages, 16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_decoder_with_other_sequences(dtype):
    """A decoder's pass over ragged chunks, captured once and replayed with other tokens, positions, tables, lengths and starts; eager
    work and synchronizations between the replays."""
    B, N, cols = 3, 12, 7
    m, dec = decoder(dtype, B * cols + 4)
    s = dict(ids=torch.zeros(N, dtype=torch.int64, device=DEV), pos=torch.zeros(N, dtype=torch.int64, device=DEV),
             table=torch.zeros(B, cols, dtype=torch.int32, device=DEV), lengths=i32(4, 4, 4), starts=i32(0, 4, 8, 12))
    w = [torch.zeros(B, 4, cols * 16, device=DEV) for _ in range(2)]
    before = [[torch.randn(t.K.shape, generator=torch.Generator().manual_seed(i)).to(dtype).to(DEV) for _ in "KV"] for i, t in enumerate(dec.tapes)]

    def fill(seed):
        c = torch.Generator().manual_seed(seed)
        s["ids"].copy_(torch.randint(0, 512, (N,), generator=c))
        s["table"].copy_(torch.randperm(B * cols + 4, generator=c)[:B * cols].view(B, cols))
        cuts = sorted(torch.randint(0, N + 1, (B - 1,), generator=c).tolist()) + [N]
        counts = [b - a for a, b in zip([0] + cuts, cuts)]
        past = [int(torch.randint(0, 100, (), generator=c)) for _ in range(B)]
        s["starts"].copy_(torch.tensor([0] + cuts))
        s["lengths"].copy_(torch.tensor([max(1, p + n) for p, n in zip(past, counts)]))
        s["pos"].copy_(torch.cat([torch.arange(p, p + n) for p, n in zip(past, counts)]))
        for t, (k, v), x in zip(dec.tapes, before, w):
            t.K.copy_(k), t.V.copy_(v), x.zero_()

    def run():
        return dec.extend(s["ids"], s["pos"], s["table"], s["lengths"], s["starts"], n_sweeps=3, weights=w)

    def everything(logits):
        return [logits.clone(), *(x.clone() for x in w), *(x.clone() for t in dec.tapes for x in (t.K, t.V))]

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for seed in range(1, 5):
        fill(seed)
        want = everything(run())
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(everything(held), want)), seed


def test_parameters_that_change():
    """A step of an optimizer between two passes: the second one has the new parameters, in every layer and the head."""
    m, dec = decoder(torch.float32, 4)
    table, ids, pos = i32([0, 1]), torch.tensor([3, 9, 4], device=DEV), torch.arange(3, device=DEV)
    dec.extend(ids, pos, table, i32(3), i32(0, 3), n_sweeps=3)
    g = torch.Generator().manual_seed(2)
    with torch.no_grad():
        for p in m.parameters():
            p.add_((0.01 * torch.randn(p.shape, generator=g)).to(DEV))
    got = dec.extend(ids, pos, table, i32(3), i32(0, 3), n_sweeps=3)
    assert torch.equal(got, PagedDecoder(m, 4, 16).extend(ids, pos, table, i32(3), i32(0, 3), n_sweeps=3))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_tokens_in_one_pass(dtype):
    """2500 tokens of 70 sequences in one pass, a layer of the larger width, against each sequence's own pass. The products may take
    other forms at other sizes, so their sums another order: within the tolerance of two computations."""
    cfg = cfg_of(d=1024, h=16, T=128, ctx_mod="mult_res")
    sd = {k: v.double() for k, v in make_state_dict(cfg, seed=33, with_attn_norm=False).items()}
    attn = attention(cfg, sd)
    cos, sin = (t.to(DEV) for t in O.build_rope_cache(128, cfg.head_dim, cfg.rope_theta, dtype=torch.float64))
    g = torch.Generator().manual_seed(4)
    counts = torch.randint(1, 72, (70,), generator=g).tolist()
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    x = torch.randn(starts[-1], 1024, generator=g).to(dtype).to(DEV)
    pos = torch.cat([torch.arange(n) for n in counts]).to(DEV)
    tape = PagedTape(attn, 70 * 5, 16, dtype)
    table = torch.arange(350, dtype=torch.int32, device=DEV).view(70, 5)
    y = tape.extend(x, pos, cos, sin, table, i32(*counts), i32(*starts), n_sweeps=2)
    own = PagedTape(attn, 70 * 5, 16, dtype)
    errs = {}
    for b in (0, 1, 33, 69):
        rows = slice(starts[b], starts[b + 1])
        want = own.extend(x[rows], pos[rows], cos, sin, table[b:b + 1], i32(counts[b]), i32(0, counts[b]), n_sweeps=2)
        at = torch.arange(counts[b], device=DEV)
        page = table[b].long()[at // 16]
        errs[f"y{b}"] = relerr(y[rows], want)
        errs[f"K{b}"] = relerr(tape.K[page, :, at % 16], own.K[page, :, at % 16])
        errs[f"V{b}"] = relerr(tape.V[page, :, at % 16], own.V[page, :, at % 16])
    record(f"paged pass of many tokens {dtype}", errs, TOL[dtype])
    assert all(e < TOL[dtype] for e in errs.values()), errs

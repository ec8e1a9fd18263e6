"""Dual-Mod layers and models over a paged cache: against the oracle's scan, the static tape and the graph decoder; the paged
operators used together, and in a captured graph."""

import pytest
import torch

import oracle as O
from dual_mod_public_amd import _lib as L
from dual_mod_public_amd import paged
from dual_mod_public_amd.attention import DualModAttention
from dual_mod_public_amd.config import DualModConfig
from dual_mod_public_amd.drafts import verify_drafts
from dual_mod_public_amd.graph_decode import GraphDecoder
from dual_mod_public_amd.model import DualModLM
from dual_mod_public_amd.paged_decode import PagedDecoder, PagedTape
from dual_mod_public_amd.synthetic import make_input, make_lm_state_dict, make_state_dict
from tests.hip_helpers import DEV, cfg_of, record, relerr

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    L.load()


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def attention(cfg, sd, dtype):
    attn = DualModAttention(cfg).to(DEV)
    attn.load_state_dict({k: v.float() for k, v in sd.items()}, strict=False)
    return attn


KNOBS = [dict(ctx_mod="mult_res"), dict(ctx_mod="linear", local_window=9), dict(ctx_mod="fusion"), dict(ctx_mod="mult", local_window=1),
         dict(ctx_mod="mult_res", v_norm="rms", k_ctx_norm="rms")]


@pytest.mark.parametrize("knobs", KNOBS)
@pytest.mark.parametrize("d,h", [(256, 4), (256, 2)])
def test_tape_in_chunks_is_the_sequential_scan(knobs, d, h):
    """Three sequences whose tokens come in chunks of 0 to 7, exact sweeps; fp32 against the oracle's scan in 64 bits."""
    cfg = cfg_of(d=d, h=h, T=64, **knobs)
    sd = {k: v.double() for k, v in make_state_dict(cfg, seed=3, with_attn_norm=False).items()}
    lens, page = [37, 20, 29], 16
    xs = [make_input((1, n, d), seed=20 + i, dtype=torch.float64) for i, n in enumerate(lens)]
    cos, sin = O.build_rope_cache(64, cfg.head_dim, cfg.rope_theta, dtype=torch.float64)
    want = [O.sequential_scan(cfg, sd, x, cos, sin, return_cache=True) for x in xs]
    tape = PagedTape(attention(cfg, sd, torch.float32), 9, page, torch.float32)
    table = i32([8, 0, 3], [1, 7, -1], [2, 6, -1])
    g = torch.Generator().manual_seed(4)
    done, outs = [0, 0, 0], [[], [], []]
    while done != lens:
        n = [min(int(torch.randint(0, 8, (), generator=g)), m - k) for m, k in zip(lens, done)]
        if not sum(n):
            continue
        rows = torch.cat([x[0, k:k + c] for x, k, c in zip(xs, done, n)]).float().to(DEV)
        pos = torch.cat([torch.arange(k, k + c) for k, c in zip(done, n)]).to(DEV)
        done = [k + c for k, c in zip(done, n)]
        starts = i32(0, n[0], n[0] + n[1], sum(n))
        y = tape.extend(rows, pos, cos.to(DEV), sin.to(DEV), table, i32(*done), starts, n_sweeps=max(n))
        for b, part in enumerate(y.cpu().split(n)):
            outs[b].append(part)
    errs = {}
    for b, n in enumerate(lens):
        o, K, V = want[b]
        errs[f"y{b}"] = relerr(torch.cat(outs[b]), (o[0] @ sd["wo.weight"].t()))
        r = torch.arange(n, device=DEV)
        at = table[b].long()[r // page]
        errs[f"K{b}"], errs[f"V{b}"] = relerr(tape.K[at, :, r % page].transpose(0, 1), K[0]), relerr(tape.V[at, :, r % page].transpose(0, 1), V[0])
    record(f"paged tape {knobs} h={h}", errs, 1e-5)
    assert max(errs.values()) < 1e-5, errs


def test_single_tokens_are_the_static_tape():
    """One token per sequence at a time, all at one position: the static tape's step within fp32 rounding."""
    from dual_mod_public_amd.decode import StaticTape
    cfg = cfg_of(d=256, h=4, T=64)
    sd = {k: v.double() for k, v in make_state_dict(cfg, seed=5, with_attn_norm=False).items()}
    attn = attention(cfg, sd, torch.float32)
    B, T = 3, 20
    x = make_input((B, T, 256), seed=6).to(DEV)
    cos, sin = (t.to(DEV) for t in O.build_rope_cache(64, 64, cfg.rope_theta))
    static, tape = StaticTape(attn, B, 64, DEV, torch.float32), PagedTape(attn, 6, 16, torch.float32)
    table = i32([5, 0], [2, 4], [1, 3])
    for t in range(T):
        _, want = static.step(x[:, t].contiguous(), t, cos, sin, with_wo=True)
        y = tape.extend(x[:, t], torch.full((B,), t, device=DEV), cos, sin, table, i32(*[t + 1] * B))
        assert relerr(y, want) < 1e-5, t


def lm(layers=2, vocab=97, T=128, seed=1, dtype=torch.float32, std=None):
    cfg = DualModConfig(d_model=256, n_heads=4, n_layers=layers, vocab_size=vocab, max_seq_len=T, mlp_hidden_override=384, ctx_mod="mult_res")
    m = DualModLM(cfg, dtype=dtype)
    m.load_state_dict(make_lm_state_dict(cfg, seed=seed), strict=True)
    return m.to(DEV)


class Pages:
    """The host's side of a pool: which pages a sequence has."""

    def __init__(self, n, page):
        self.free, self.page, self.has = list(range(n)), page, {}

    def table(self, lengths, cols):
        rows = []
        for b, n in enumerate(lengths):
            own = self.has.setdefault(b, [])
            while len(own) * self.page < n:
                own.append(self.free.pop())
            rows.append(own + [-1] * (cols - len(own)))
        return i32(*rows)


def test_drafts_decode_what_the_graph_decoder_does():
    """Greedy decoding by verified drafts (right and wrong ones) gives the graph decoder's tokens and log probabilities; two
    prompts of different lengths, chunks of ragged sizes, fp32."""
    m = lm()
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 97, (n,), generator=g) for n in (11, 4)]
    new, page = 24, 16
    want = []
    for p in prompts:
        dec = GraphDecoder(m, 1, 128, top=0)
        tokens, k = dec.generate(p[None].to(DEV), new)
        want.append((tokens[0].tolist(), dec.gen_logp[0]))
    dec, pool = PagedDecoder(m, 12, page), Pages(12, page)
    texts = [p.tolist() for p in prompts]
    cached = [0, 0]
    got, logps = [[], []], [[], []]
    step = 0
    while min(len(t) for t in got) < new:
        chunks, counts = [], []
        for b in range(2):
            drafts = []
            if cached[b]:       # drafts: the right continuation, sometimes with a wrong token in it
                k = len(got[b])
                drafts = want[b][0][k:k + (step + b) % 4]
                if drafts and (step + b) % 3 == 0:
                    drafts[-1] = (drafts[-1] + 1) % 97
            chunks.append(texts[b][cached[b]:] + drafts)
            counts.append(len(chunks[-1]))
        lengths = [c + n for c, n in zip(cached, counts)]
        ids = torch.tensor(chunks[0] + chunks[1], device=DEV)
        pos = torch.cat([torch.arange(c, c + n) for c, n in zip(cached, counts)]).to(DEV)
        starts = i32(0, counts[0], sum(counts))
        logits = dec.extend(ids, pos, pool.table(lengths, 6), i32(*lengths), starts, n_sweeps=max(counts))
        # verified from each text's last token on; the prompt's rows before it are of no sequence
        first = [len(t) - c - 1 for t, c in zip(texts, cached)]
        for b in range(2):
            lo, hi = (first[0], counts[0]) if b == 0 else (counts[0] + first[1], sum(counts))
            r = verify_drafts(logits[lo:hi], ids[lo:hi].contiguous(), torch.rand(hi - lo, 2, device=DEV), i32(0, hi - lo), temperature=0.0)
            n = int(r.accepted[0]) + 1
            fresh = r.tokens[:n].tolist()
            assert (r.tokens[n:] == -1).all()
            got[b] += fresh
            logps[b] += r.logp[:n].tolist()
            cached[b] = len(texts[b]) + n - 1       # the new token's row is not there yet
            texts[b] += fresh
        step += 1
    for b in range(2):
        assert got[b][:new] == want[b][0][:new]
        assert (torch.tensor(logps[b][:new]) - want[b][1][:new]).abs().max() < 1e-4


def test_serving_step_with_eviction():
    """Decode with weights, evict every layer to a budget, go on: each pass against attention over the rows that are left,
    gathered by hand from the pages (fp32)."""
    cfg = cfg_of(d=256, h=4, T=128)
    sd = {k: v.double() for k, v in make_state_dict(cfg, seed=8, with_attn_norm=False).items()}
    tape = PagedTape(attention(cfg, sd, torch.float32), 20, 16, torch.float32)
    cos, sin = (t.to(DEV) for t in O.build_rope_cache(128, 64, cfg.rope_theta))
    x = make_input((2, 70, 256), seed=9).to(DEV)
    lengths, pool = [50, 33], Pages(20, 16)
    table = pool.table(lengths, 5)
    w = torch.zeros(2, 4, 80, device=DEV)
    starts = i32(0, 50, 83)
    pos = torch.cat([torch.arange(50), torch.arange(33)]).to(DEV)
    tape.extend(torch.cat([x[0, :50], x[1, :33]]), pos, cos, sin, table, i32(*lengths), starts, n_sweeps=50, weights=w)
    # every token gives its probabilities to the rows before it; the rest is its own pair's
    assert (w.sum(2) < torch.tensor([[50.0], [33.0]], device=DEV)).all() and (w >= 0).all()
    assert (w[1, :, 33:] == 0).all() and (w[:, :, 32:].sum() > 0)
    new_pool = Pages(0, 16)
    new_pool.free = pool.free
    keep = 24
    e = tape.evict(w, table, i32(*lengths), keep, new_pool.table([24, 24], 2), sinks=2, recent=8)
    new_table = new_pool.table([24, 24], 2)
    assert e.lengths.tolist() == [24, 24]
    for b, n in enumerate(lengths):
        for c in range(4):
            r = e.rows[b, c].long()
            assert r[:2].tolist() == [0, 1] and r[-8:].tolist() == list(range(n - 8, n)) and (r[1:] > r[:-1]).all()
            i = torch.arange(24, device=DEV)
            assert torch.equal(tape.K[new_table[b].long()[i // 16], c, i % 16], tape.K[table[b].long()[r // 16], c, r % 16])
    # the next token reads what is left
    table3 = new_pool.table([25, 25], 3)
    K0, V0 = tape.K.clone(), tape.V.clone()
    w3 = torch.zeros(2, 4, 48, device=DEV)
    w3[:, :, :32] = e.weights
    y = tape.extend(x[:, 60], torch.tensor([50, 33], device=DEV), cos, sin, table3, i32(25, 25), weights=w3)
    attn = tape.attn
    sdf = {k: v.double().cpu() for k, v in attn.state_dict().items()}
    for b, p in enumerate((50, 33)):
        i = torch.arange(24)
        at = table3[b].long().cpu()[i // 16]
        cache = {"K": K0.cpu()[at, :, i % 16].transpose(0, 1)[None].double(), "V": V0.cpu()[at, :, i % 16].transpose(0, 1)[None].double()}
        o, want = O.decode_step(cfg, sdf, x[b:b + 1, 60:61].double().cpu(), p, cache, *(t.double().cpu() for t in (cos, sin)))
        assert relerr(y[b], want[0, 0]) < 1e-5
    assert ((w3[:, :, :24] - e.weights[:, :, :24]).sum(2) < 1).all() and (w3[:, :, 24:] == 0).all()


def test_captured_pass_with_other_lengths():
    """A captured pass (attention with weights, then verification) replayed with other lengths, tables, starts and inputs gives
    the eager results each time; eager work and synchronizations between the replays."""
    g = torch.Generator(device=DEV).manual_seed(11)
    B, N, h, h_kv, dh, page, cols, V = 3, 12, 4, 2, 64, 16, 20, 1000
    K, Vp = (torch.randn(70, h_kv, page, dh, generator=g, device=DEV) for _ in range(2))
    s = dict(q=torch.empty(N, h, dh, device=DEV), k=torch.empty(N, h_kv, dh, device=DEV), v=torch.empty(N, h_kv, dh, device=DEV),
             table=torch.zeros(B, cols, dtype=torch.int32, device=DEV), lengths=i32(4, 4, 4), starts=i32(0, 4, 8, 12),
             weights=torch.zeros(B, h_kv, cols * page, device=DEV), x=torch.empty(N, V, device=DEV), y=torch.empty(N, V, device=DEV),
             ids=torch.zeros(N, dtype=torch.int64, device=DEV), u=torch.empty(N, 2, device=DEV), T=torch.ones(B, device=DEV))

    def run(K, Vp):
        paged.paged_write(s["k"], s["v"], K, Vp, s["table"], s["lengths"], s["starts"])
        r = paged.paged_attention(s["q"], K, Vp, s["table"], s["lengths"], s["starts"], weights=s["weights"], out=out)
        return r.o, r.lse, verify_drafts(s["x"], s["ids"], s["u"], s["starts"], draft_logits=s["y"], temperature=s["T"])

    def fill(seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        c = torch.Generator().manual_seed(seed)
        for n in ("q", "k", "v", "x", "y"):
            s[n].normal_(generator=g)
        s["u"].uniform_(generator=g)
        s["ids"].copy_(torch.randint(0, V, (N,), generator=c))
        s["table"].copy_(torch.randperm(B * cols + 10, generator=c)[:B * cols].view(B, cols))
        cuts = sorted(torch.randint(0, N + 1, (B,), generator=c).tolist())
        s["starts"].copy_(torch.tensor([0] + cuts))
        s["lengths"].copy_(torch.tensor([max(1, b - a) + int(torch.randint(0, 250, (), generator=c)) for a, b in zip([0] + cuts, cuts)]))
        s["weights"].uniform_(generator=g)
        out.fill_(7.0)

    out = torch.empty(N, h, dh, device=DEV)
    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(K, Vp)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run(K, Vp)
    for seed in (1, 2, 3, 4):
        fill(seed)
        K2, V2 = K.clone(), Vp.clone()
        want = run(K2, V2)
        want = [t.clone() for t in (want[0], want[1], *want[2], s["weights"])]
        n = int(s["starts"][-1])
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [held[0], held[1], *held[2], s["weights"]]
        for i, (a, b) in enumerate(zip(got, want)):
            if i == 1:      # rows of no sequence are not written
                a, b = a[:n], b[:n]
            assert torch.equal(a, b), (seed, i)
        assert torch.equal(K, K2) and torch.equal(Vp, V2)


def test_other_stream():
    """On a stream of its own, beside work on the default one."""
    g = torch.Generator(device=DEV).manual_seed(12)
    K, V = (torch.randn(64, 2, 16, 64, generator=g, device=DEV).bfloat16() for _ in range(2))
    table = torch.randperm(64, generator=torch.Generator().manual_seed(1)).view(2, 32).int().to(DEV)
    q = torch.randn(2, 8, 64, generator=g, device=DEV).bfloat16()
    lengths = i32(511, 200)
    want = paged.paged_attention(q, K, V, table, lengths)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [paged.paged_attention(q, K, V, table, lengths) for _ in range(8)]
    for _ in range(8):
        paged.paged_attention(q * 2, K, V, table, lengths)
    torch.cuda.synchronize()
    assert all(torch.equal(r.o, want.o) and torch.equal(r.lse, want.lse) for r in got)


def test_python_refusals():
    K, V = paged.new_pages(4, 2, 16, 64, dtype=torch.float32)
    table, lengths = torch.zeros(2, 2, dtype=torch.int32, device=DEV), i32(3, 4)
    q = torch.zeros(2, 4, 64, device=DEV)
    ok = dict(q=q, K=K, V=V, table=table, lengths=lengths)
    paged.paged_attention(**ok)
    for bad in (dict(q=q.bfloat16()), dict(q=q[:1]), dict(q=torch.zeros(2, 3, 64, device=DEV)), dict(q=torch.zeros(2, 4, 128, device=DEV)),
                dict(q=torch.zeros(2, 4, 128, device=DEV)[..., ::2]), dict(K=K[:, :, ::2]), dict(K=K.transpose(0, 1)), dict(V=V[:2]),
                dict(table=table.long()), dict(table=table[0]), dict(lengths=lengths[:1]), dict(lengths=lengths.cpu()), dict(starts=i32(0, 2)),
                dict(starts=torch.zeros(3, dtype=torch.int64, device=DEV)), dict(k_self=torch.zeros(2, 2, 64, device=DEV)), dict(window=-1),
                dict(weights=torch.zeros(2, 2, 31, device=DEV)), dict(weights=torch.zeros(2, 2, 32, device=DEV).bfloat16()),
                dict(out=torch.zeros(2, 4, 64, device=DEV).bfloat16()), dict(out=torch.zeros(4, 2, 64, device=DEV).transpose(0, 1))):
        with pytest.raises(ValueError):
            paged.paged_attention(**dict(ok, **bad))
    with pytest.raises(NotImplementedError):
        paged.paged_attention(q[:, :, :32].contiguous(), K[..., :32].contiguous(), V[..., :32].contiguous(), table, lengths)
    with pytest.raises(NotImplementedError):
        paged.paged_attention(q.requires_grad_(), K, V, table, lengths)
    w = torch.zeros(2, 2, 32, device=DEV)
    for kw in (dict(keep=0), dict(keep=4, sinks=3, recent=2), dict(keep=32, new_table=table[:, :1]), dict(keep=4, weights=w[:1]),
               dict(keep=4, new_table=table[:1]), dict(keep=4, new_table=table.long())):
        with pytest.raises(ValueError):
            paged.evict_rows(**dict(dict(K=K, V=V, weights=w, table=table, lengths=lengths, new_table=table + 2), **kw))
    x, ids, u, st = torch.zeros(4, 9, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV), torch.zeros(4, 2, device=DEV), i32(0, 4)
    for kw in (dict(logits=x[0]), dict(ids=ids.int()), dict(uniforms=u[:, 0]), dict(starts=st.long()), dict(draft_logits=x.bfloat16()),
               dict(temperature=-1.0), dict(temperature=torch.ones(2, device=DEV)), dict(logits=x.t())):
        with pytest.raises(ValueError):
            verify_drafts(**dict(dict(logits=x, ids=ids, uniforms=u, starts=st), **kw))


def test_sizes_of_nothing():
    K, V = paged.new_pages(4, 2, 16, 64)
    none = torch.zeros(0, 4, 64, device=DEV, dtype=torch.bfloat16)
    r = paged.paged_attention(none, K, V, torch.zeros(2, 2, dtype=torch.int32, device=DEV), i32(3, 4), i32(0, 0, 0))
    assert r.o.shape == (0, 4, 64) and r.lse.shape == (0, 4)
    paged.paged_write(none[:, :2], none[:, :2], K, V, torch.zeros(2, 2, dtype=torch.int32, device=DEV), i32(3, 4), i32(0, 0, 0))
    r = paged.paged_attention(none, K, V, torch.zeros(0, 2, dtype=torch.int32, device=DEV), i32(), None)
    assert r.o.shape == (0, 4, 64)
    v = verify_drafts(torch.zeros(3, 9, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV), torch.zeros(3, 2, device=DEV), i32(0))
    assert v.tokens.tolist() == [-1] * 3 and v.accepted.numel() == 0


def test_outputs_in_the_place_of_inputs():
    K, V = paged.new_pages(4, 2, 16, 64, dtype=torch.float32)
    table, lengths = torch.zeros(2, 2, dtype=torch.int32, device=DEV), i32(3, 4)
    q = torch.zeros(4, 4, 64, device=DEV)
    pair = torch.zeros(2, 2, 64, device=DEV)
    for kw in (dict(out=q[:2]), dict(out=q[1:3]), dict(out=K[2].view(-1)[:512].view(2, 4, 64)), dict(weights=V[1].view(-1)[:128].view(2, 2, 32)),
               dict(weights=q[:2].view(-1)[:128].view(2, 2, 32))):
        with pytest.raises(ValueError, match="overlaps"):
            paged.paged_attention(q[:2], K, V, table, lengths, k_self=pair, v_self=pair, **kw)
    r = paged.paged_attention(q[:2], K, V, table, lengths, out=q[2:])       # beside it
    assert r.o.data_ptr() == q[2:].data_ptr()
    w = torch.zeros(2, 2, 32, device=DEV, requires_grad=True)
    with pytest.raises(NotImplementedError):
        paged.paged_attention(q[:2], K, V, table, lengths, weights=w)
    x = torch.zeros(4, 9, device=DEV)
    rest = (torch.zeros(4, dtype=torch.int64, device=DEV), torch.zeros(4, 2, device=DEV), i32(0, 4))
    y = x.clone().requires_grad_()
    for kw in (dict(logits=y), dict(logits=x, draft_logits=y)):
        with pytest.raises(NotImplementedError):
            verify_drafts(kw.pop("logits"), *rest, **kw)
    with torch.no_grad():
        verify_drafts(y, *rest)


@pytest.mark.parametrize("h", [4, 16])
def test_captured_prompts_lookups_and_eviction(h):
    """Tiles of 128 and of 256 query rows, drafts looked up and an eviction in one graph, replayed with other lengths and starts; two
    graphs of the same calls in turn, each with workspaces of its own."""
    B, N, h_kv, dh, page, cols, V, keep = 3, 210, 2, 64, 32, 24, 9000, 100
    K, Vp = (torch.randn(B * cols + 12 + 4, h_kv, page, dh, device=DEV).bfloat16() for _ in range(2))
    new_table = torch.arange(B * cols + 4, B * cols + 16, device=DEV, dtype=torch.int32).view(3, 4)
    s = dict(q=torch.randn(N, h, dh, device=DEV).bfloat16(), table=torch.zeros(B, cols, dtype=torch.int32, device=DEV),
             lengths=i32(70, 70, 70), starts=i32(0, 70, 140, 210), weights=torch.zeros(B, h_kv, cols * page, device=DEV),
             x=torch.randn(N, V, device=DEV).bfloat16(), ids=torch.zeros(N, dtype=torch.int64, device=DEV), u=torch.rand(N, 2, device=DEV))

    def run():
        r = paged.paged_attention(s["q"], K, Vp, s["table"], s["lengths"], s["starts"], window=0, weights=s["weights"], out=out)
        e = paged.evict_rows(K, Vp, s["weights"], s["table"], s["lengths"], keep, new_table, sinks=2, recent=9)
        v = verify_drafts(s["x"], s["ids"], s["u"], s["starts"], temperature=0.7)
        return r.o, r.lse, *e, *v

    def fill(seed):
        c = torch.Generator().manual_seed(seed)
        s["table"].copy_(torch.randperm(B * cols + 4, generator=c)[:B * cols].view(B, cols))
        cuts = sorted(torch.randint(0, N + 1, (B,), generator=c).tolist())
        s["starts"].copy_(torch.tensor([0] + cuts))
        s["lengths"].copy_(torch.tensor([max(1, b - a) + int(torch.randint(0, 500, (), generator=c)) for a, b in zip([0] + cuts, cuts)]))
        s["ids"].copy_(torch.randint(0, V, (N,), generator=c))
        s["u"].copy_(torch.rand(N, 2, generator=c) * torch.tensor([1e-4, 1.0]))
        s["weights"].copy_(torch.rand(B, h_kv, cols * page, generator=c))
        out.fill_(3.0)

    out = torch.empty(N, h, dh, device=DEV, dtype=torch.bfloat16)
    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = run()
        graphs.append((graph, held))
    for seed in range(1, 7):
        fill(seed)
        want = [t.clone() for t in (*run(), s["weights"], K[-12:], Vp[-12:])]
        n = int(s["starts"][-1])
        fill(seed)
        K[-12:], Vp[-12:] = 0, 0
        graph, held = graphs[seed % 2]
        graph.replay()
        torch.cuda.synchronize()
        rows = torch.arange(4 * page, device=DEV)
        for i, (a, b) in enumerate(zip((*held, s["weights"]), want)):
            if i == 1:
                a, b = a[:n], b[:n]
            assert torch.equal(a, b), (seed, i)
        for pool, w in zip((K[-12:], Vp[-12:]), want[-2:]):     # the kept rows; what lies behind them stays
            for b in range(B):
                left = int(held[3][b])
                got, exp = (t[4 * b:4 * b + 4].transpose(0, 1).reshape(h_kv, -1, dh)[:, rows < left] for t in (pool, w))
                assert torch.equal(got, exp)

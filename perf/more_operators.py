"""The operators of a server's step over a paged cache, with the sizes they are called at, for timing and for comparing
outputs.

Every case is a dict of plain values; ``kind`` names the public entry point it goes through:

  attend  ``paged.paged_attention``: new tokens of sequences of different lengths over their pages, one token each or a
          chunk, with or without a raw self pair per token, a local window, key heads shared by several query heads and
          the attention weight accumulated per cached row. With ``write`` the chunk's rows go into the pages first
          (``paged.paged_write``)
  evict   ``paged.evict_rows``: the rows of each key head with the largest accumulated weight (and the first and the last
          ones) gathered into new pages
  verify  ``drafts.verify_drafts``: drafted tokens against the target's probabilities from given random numbers

With ``own`` false ``run`` computes the same by elementary torch operations: attention in 32 bits over the whole
capacity of the table, verification in 64 bits (sums of many probabilities are compared with random numbers).
"""

import math
import random

import torch

own = False

DEV = "cuda"


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------

def listed():
    return [
        # one interactive request: a token's read of a paged tape, with its raw self pair
        dict(name="one_token", kind="attend", B=1, new=1, ragged=False, h=16, hkv=16, dh=64, page=64, short=1024, long=1024,
             window=0, self=True, write=False, weights=False, dtype="bf16", lens=0),
        # a serving batch of requests of very different lengths
        dict(name="tokens_64", kind="attend", B=64, new=1, ragged=False, h=16, hkv=16, dh=64, page=64, short=100, long=8192,
             window=0, self=True, write=False, weights=False, dtype="bf16", lens=1),
        # key heads shared by four query heads, small pages, weights kept for eviction
        dict(name="tokens_shared", kind="attend", B=32, new=1, ragged=False, h=32, hkv=8, dh=128, page=16, short=3000,
             long=16384, window=0, self=False, write=True, weights=True, dtype="bf16", lens=2),
        # drafted chunks of 0 to 8 tokens, rows written, read with self pairs, weights kept
        dict(name="drafted", kind="attend", B=24, new=8, ragged=True, h=16, hkv=16, dh=64, page=32, short=50, long=4001,
             window=0, self=True, write=True, weights=True, dtype="bf16", lens=3),
        # two prompts' next chunks over what they have already cached
        dict(name="prompt_chunk", kind="attend", B=2, new=2048, ragged=False, h=32, hkv=8, dh=128, page=256, short=15000,
             long=16384, window=0, self=False, write=True, weights=False, dtype="bf16", lens=4),
        # the small fp32 configuration: odd chunks in small pages, a local window
        dict(name="window_fp32", kind="attend", B=7, new=130, ragged=True, h=8, hkv=4, dh=64, page=16, short=1, long=1501,
             window=256, self=True, write=True, weights=True, dtype="fp32", lens=5),
        # one request over its budget
        dict(name="evict_one", kind="evict", B=1, h=16, dh=64, page=64, short=2304, long=2304, keep=2048, sinks=4, recent=256,
             grid=0, dtype="bf16", lens=6),
        # a batch, some of it not yet over the budget
        dict(name="evict_batch", kind="evict", B=32, h=8, dh=128, page=16, short=3000, long=16384, keep=4096, sinks=4,
             recent=512, grid=0, dtype="bf16", lens=7),
        # odd sizes with many equal weights
        dict(name="evict_ties", kind="evict", B=5, h=3, dh=64, page=32, short=1, long=5001, keep=999, sinks=0, recent=1,
             grid=16, dtype="fp32", lens=8),
        # one request, four drafted tokens
        dict(name="verify_one", kind="verify", B=1, drafts=4, ragged=False, V=32000, dtype="bf16", draft=True, greedy=0.0,
             mask=False, lens=9),
        # a batch over the default configuration's odd vocabulary, fp32, 0 to 7 drafts each
        dict(name="verify_64", kind="verify", B=64, drafts=7, ragged=True, V=50257, dtype="fp32", draft=True, greedy=0.2,
             mask=False, lens=10),
        # drafts looked up in the prompt (no draft distribution), a large odd vocabulary, some tokens forbidden
        dict(name="verify_lookup", kind="verify", B=48, drafts=5, ragged=True, V=100003, dtype="bf16", draft=False, greedy=0.3,
             mask=True, lens=11),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: the same entry points over the ranges that the listed ones stand for."""
    kind = rng.choice(["attend", "attend", "attend", "attend", "evict", "verify", "verify"])
    lens = rng.randrange(1 << 20)
    if kind == "verify":
        V, B, k = _log(rng, 300, 100003), _log(rng, 1, 64), rng.randint(1, 8)
        if rng.random() < 0.4:
            V += -V % 8
        while B * (k + 1) * V > 3 * 10 ** 7:
            B = max(1, B // 2)
        return dict(kind=kind, B=B, drafts=k, ragged=rng.random() < 0.6, V=V, dtype=rng.choice(["bf16", "bf16", "fp32"]),
                    draft=rng.random() < 0.6, greedy=rng.choice([0.0, 0.3, 1.0]), mask=rng.random() < 0.3, lens=lens)
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    page = rng.choice([16, 32, 64, 128, 256])
    dh = rng.choice([64, 128])
    long = _log(rng, 60, 16384)
    short = max(1, min(long, _log(rng, 1, 16384)))
    if kind == "evict":
        h = rng.choice([1, 3, 4, 8, 16])
        B = max(1, min(_log(rng, 1, 48), 2 ** 29 // (h * long * dh * (2 if dtype == "bf16" else 4))))
        keep = max(2, _log(rng, max(2, long // 8), long))
        sinks, recent = rng.randint(0, min(8, keep // 2)), rng.randint(0, keep // 2)
        return dict(kind=kind, B=B, h=h, dh=dh, page=page, short=short, long=long, keep=keep, sinks=sinks, recent=recent,
                    grid=rng.choice([0, 0, 16]), dtype=dtype, lens=lens)
    hkv = rng.choice([2, 4, 8, 16])
    h = hkv * rng.choice([1, 1, 2, 4, 8] if hkv < 16 else [1, 2])
    new = rng.choice([1, 1, rng.randint(2, 9), _log(rng, 10, 700)])
    size = hkv * long * dh * (2 if dtype == "bf16" else 4)
    B = max(1, min(_log(rng, 1, 64), 2 ** 30 // size, 2 ** 31 // (h * new * long)))
    new = min(new, long)
    return dict(kind=kind, B=B, new=new, ragged=new > 1 and rng.random() < 0.7, h=h, hkv=hkv, dh=dh, page=page, short=short,
                long=long, window=rng.choice([0, 0, 0, rng.randint(2, 2000)]), self=rng.random() < 0.5,
                write=rng.random() < 0.5, weights=rng.random() < 0.4, dtype=dtype, lens=lens)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------

def _dtype(name):
    return torch.float32 if name == "fp32" else torch.bfloat16


def _spread(rng, lo, hi):
    """A whole number of lo..hi, spread over its logarithm where the range is wide."""
    return min(hi, max(lo, _log(rng, lo, hi))) if hi > 10 * lo else rng.randint(lo, hi)


def _lengths(case):
    """(new tokens, cached rows with them) of each sequence: the case's own, the same for every seed."""
    rng = random.Random(case["lens"])
    lens = [_spread(rng, case["short"], case["long"]) for _ in range(case["B"])]
    lens[rng.randrange(case["B"])] = case["long"]
    if case["kind"] == "evict":
        return None, lens
    new = [rng.randint(0, case["new"]) if case["ragged"] else case["new"] for _ in lens]
    new[lens.index(case["long"])] = case["new"]
    return new, [max(n, t) for n, t in zip(new, lens)]


def _starts(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def _table(lens, page, g):
    """A block table for lens rows each, its pages in random order; -1 where a sequence has no page; the pool's size."""
    need = [-(-n // page) for n in lens]
    total = sum(need)
    at = torch.tensor(_starts(need)[:-1], device=DEV)[:, None]
    k = torch.arange(max(max(need), 1), device=DEV)[None, :]
    order = torch.randperm(total, generator=g, device=DEV)
    ids = order[(at + k).clamp(max=total - 1)]
    return torch.where(k < torch.tensor(need, device=DEV)[:, None], ids, -1).to(torch.int32), total


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(7919 * (seed + 1))
    if case["kind"] == "verify":
        return _prepare_verify(case, g)
    new, lens = _lengths(case)
    dt, dh, page, B = _dtype(case["dtype"]), case["dh"], case["page"], case["B"]
    table, total = _table(lens, page, g)
    s = dict(case=case, table=table, lengths=torch.tensor(lens, dtype=torch.int32, device=DEV))
    if case["kind"] == "evict":
        kept = [min(n, case["keep"]) for n in lens]
        s["new_table"], more = _table(kept, page, g)
        s["new_table"] = torch.where(s["new_table"] >= 0, s["new_table"] + total, -1)
        s["K"], s["V"] = (torch.randn(total + more, case["h"], page, dh, generator=g, device=DEV).to(dt) for _ in range(2))
        # what attention leaves behind: few rows with much of it, most with little, recent ones with none yet
        w = torch.exp(2.5 * torch.randn(B, case["h"], table.shape[1] * page, generator=g, device=DEV) - 3)
        if case["grid"]:
            w = (w * case["grid"]).floor() / case["grid"]
        s["weights"] = w
        return s
    h, hkv = case["h"], case["hkv"]
    starts = _starts(new)
    N = starts[-1]
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    s["K"], s["V"] = (torch.randn(total, hkv, page, dh, generator=g, device=DEV).to(dt) for _ in range(2))
    s["q"] = (2 * torch.randn(N, h, dh, generator=g, device=DEV)).to(dt)
    if case["self"]:
        s["k_self"], s["v_self"] = (torch.randn(N, hkv, dh, generator=g, device=DEV).to(dt) for _ in range(2))
    if case["write"]:
        s["k"], s["v"] = (torch.randn(N, hkv, dh, generator=g, device=DEV).to(dt) for _ in range(2))
    if case["weights"]:
        s["weights"] = torch.rand(B, hkv, table.shape[1] * page, generator=g, device=DEV)
    return s


def _prepare_verify(case, g):
    B, V = case["B"], case["V"]
    rng = random.Random(case["lens"])
    counts = [1 + (rng.randint(0, case["drafts"]) if case["ragged"] else case["drafts"]) for _ in range(B)]
    counts[rng.randrange(B)] = 1 + case["drafts"]
    starts = _starts(counts)
    N = starts[-1]
    # logits as a head makes them, and a smaller model's beside them
    x = torch.randn(N, V, generator=g, device=DEV)
    x *= 1.5 + 2.5 * torch.rand(N, 1, generator=g, device=DEV)
    y = x + 0.7 * torch.randn(N, V, generator=g, device=DEV)
    temperature = 0.6 + 0.8 * torch.rand(B, generator=g, device=DEV)
    seq = torch.repeat_interleave(torch.arange(B, device=DEV), torch.tensor(counts, device=DEV))
    if case["mask"]:
        x = x.masked_fill(torch.rand(N, V, generator=g, device=DEV) < 0.5, float("-inf"))
    x, y = x.to(_dtype(case["dtype"])), y.to(_dtype(case["dtype"]))
    # the drafts: drawn from the draft's distribution
    noise = -torch.log(-torch.log(torch.rand(N, V, generator=g, device=DEV).clamp(1e-7, 1 - 1e-7)))
    source = y if case["draft"] else x
    ids = torch.randint(0, V, (N,), generator=g, device=DEV)
    ids[1:] = (source.float() / temperature[seq, None] + noise).argmax(1)[:-1]
    temperature[torch.rand(B, generator=g, device=DEV) < case["greedy"]] = 0.0
    # greedy requests are drafted greedily, with one in four drafts off
    best = (temperature[seq] == 0) & (torch.rand(N, generator=g, device=DEV) < 0.75)
    ids[1:] = torch.where(best, x.float().argmax(1), ids.roll(-1))[:-1]
    return dict(case=case, x=x, y=y if case["draft"] else None, ids=ids, temperature=temperature,
                u=torch.rand(N, 2, generator=g, device=DEV), starts=torch.tensor(starts, dtype=torch.int32, device=DEV))


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if case["kind"] == "attend":
        return _own_attend(s) if own else _plain_attend(s)
    if case["kind"] == "evict":
        return _own_evict(s) if own else _plain_evict(s)
    return _own_verify(s) if own else _plain_verify(s)


def _own_attend(s):
    from dual_mod_public_amd import paged
    case = s["case"]
    # one new token per sequence: the table's order is the tokens'
    starts = s["starts"] if case["ragged"] or case["new"] > 1 else None
    if case["write"]:
        paged.paged_write(s["k"], s["v"], s["K"], s["V"], s["table"], s["lengths"], starts)
    r = paged.paged_attention(s["q"], s["K"], s["V"], s["table"], s["lengths"], starts, k_self=s.get("k_self"),
                              v_self=s.get("v_self"), window=case["window"], weights=s.get("weights"))
    return _attend_outputs(s, r.o, r.lse)


def _attend_outputs(s, o, lse):
    out = dict(o=o, lse=lse)
    if s["case"]["weights"]:
        out["weights"] = s["weights"]
    if s["case"]["write"]:
        out["K"], out["V"] = s["K"], s["V"]
    return out


def _rows_of(pages, table):
    """[B, hkv, rows, dh] in fp32 of the table's pages."""
    B, P = table.shape
    x = pages[table.clamp(min=0)].float()                       # [B, P, hkv, page, dh]
    return x.transpose(1, 2).reshape(B, x.shape[2], P * x.shape[3], x.shape[4])


def _plain_attend(s):
    case = s["case"]
    table, lengths, starts = s["table"].long(), s["lengths"].long(), s["starts"].long()
    B, new, page, dh, hkv = case["B"], case["new"], case["page"], case["dh"], case["hkv"]
    h, g = case["h"], case["h"] // case["hkv"]
    count = starts[1:] - starts[:-1]
    j = torch.arange(new, device=DEV)
    live = j < count[:, None]                                   # [B, new]
    token = (starts[:-1, None] + j).clamp(max=s["q"].shape[0] - 1)
    row = lengths[:, None] - count[:, None] + j                 # the token's row
    if case["write"]:
        b, i = live.nonzero(as_tuple=True)
        r, t = row[b, i], token[b, i]
        at = table[b, r // page]
        s["K"][at, :, r % page], s["V"][at, :, r % page] = s["k"][t], s["v"][t]
    K, V = _rows_of(s["K"], table), _rows_of(s["V"], table)

    def heads(x):                                               # [N, h, dh] -> [B, hkv, new * g, dh]
        return x[token].float().view(B, new, hkv, -1, dh).permute(0, 2, 1, 3, 4).reshape(B, hkv, -1, dh)

    scale = 1 / math.sqrt(dh)
    q = heads(s["q"])
    x = torch.matmul(q, K.transpose(2, 3)).mul_(scale).view(B, hkv, new, g, -1)
    r = torch.arange(K.shape[2], device=DEV)
    last = row if not case["self"] else row - 1
    seen = r <= last[:, :, None]
    if case["window"]:
        seen &= r > row[:, :, None] - case["window"]
    x.masked_fill_(~(seen & live[:, :, None])[:, None, :, None], float("-inf"))
    m = x.amax(-1, keepdim=True)
    if case["self"]:
        ks, vs = (heads(s[n])[:, :, :, None] for n in ("k_self", "v_self"))
        own_score = (q.view(B, hkv, new, g, dh) * ks).sum(-1, keepdim=True) * scale
        m = torch.maximum(m, own_score)
    m = torch.where(m == float("-inf"), 0.0, m)
    x = x.sub_(m).exp_()
    z = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(B, hkv, new * g, -1), V).view(B, hkv, new, g, dh)
    if case["self"]:
        e = torch.exp(own_score - m)
        z = z + e
        o = o + e * vs
    o = torch.where(z > 0, o / z, 0.0)
    lse = m + torch.log(z)
    if case["weights"]:
        s["weights"] += (x / torch.where(z > 0, z, 1.0)).sum((2, 3))
    b, i = live.nonzero(as_tuple=True)
    o = o.permute(0, 2, 1, 3, 4).reshape(B, new, h, dh)[b, i]
    lse = lse[..., 0].permute(0, 2, 1, 3).reshape(B, new, h)[b, i]
    return _attend_outputs(s, o.to(s["q"].dtype), lse)


def _own_evict(s):
    from dual_mod_public_amd import paged
    case = s["case"]
    r = paged.evict_rows(s["K"], s["V"], s["weights"], s["table"], s["lengths"], case["keep"], s["new_table"],
                         sinks=case["sinks"], recent=case["recent"])
    return dict(rows=r.rows, lengths=r.lengths, weights=r.weights, K=s["K"], V=s["V"])


def _plain_evict(s):
    case = s["case"]
    table, new_table, lengths = s["table"].long(), s["new_table"].long(), s["lengths"].long()
    B, H, page, keep = case["B"], case["h"], case["page"], case["keep"]
    w = s["weights"]
    r = torch.arange(w.shape[2], device=DEV)
    n = lengths[:, None, None]
    always = (r < case["sinks"]) | (r >= n - case["recent"])
    rank = torch.where(always, float("inf"), w)
    rank = torch.where(r < n, rank, float("-inf")).expand(B, H, -1)
    first = rank.sort(dim=2, descending=True, stable=True).indices[:, :, :keep]     # equal weights: the lower row first
    left = torch.minimum(lengths, torch.tensor(keep, device=DEV))
    slot = torch.arange(keep, device=DEV)
    # rows past the end come last; beyond the table's rows there are none
    first = torch.nn.functional.pad(first, (0, keep - first.shape[2]), value=w.shape[2])
    rows = torch.where(slot < left[:, None, None], first, w.shape[2]).sort(dim=2).values
    used = slot < left[:, None, None]
    b, c, i = used.expand(B, H, -1).nonzero(as_tuple=True)
    from_row = rows[b, c, i]
    src, dst = table[b, from_row // page], new_table[b, i // page]
    for t in (s["K"], s["V"]):
        t[dst, c, i % page] = t[src, c, from_row % page]
    weights = torch.zeros(B, H, new_table.shape[1] * page, device=DEV)
    weights[b, c, i] = w[b, c, from_row]
    return dict(rows=torch.where(used, rows, -1).to(torch.int32), lengths=left.to(torch.int32), weights=weights, K=s["K"],
                V=s["V"])


def _own_verify(s):
    from dual_mod_public_amd import drafts
    r = drafts.verify_drafts(s["x"], s["ids"], s["u"], s["starts"], draft_logits=s["y"], temperature=s["temperature"])
    return dict(tokens=r.tokens, accepted=r.accepted, logp=r.logp)


def _softmax64(x, divide):
    """Probabilities and log probabilities of rows in 64 bits."""
    d = x.double() / divide
    d = d - d.amax(1, keepdim=True)
    e = torch.exp(d)
    z = e.sum(1, keepdim=True)
    return e / z, d - torch.log(z)


def _plain_verify(s):
    x, ids, u, T = s["x"], s["ids"], s["u"].double(), s["temperature"].double()
    starts = s["starts"].long()
    N, V = x.shape
    B = starts.shape[0] - 1
    i = torch.arange(N, device=DEV)
    seq = torch.searchsorted(starts, i, right=True) - 1
    last = i == starts[seq + 1] - 1
    greedy = T[seq] == 0
    p, logp = _softmax64(x, torch.where(greedy, 1.0, T[seq])[:, None])
    drafted = ids.roll(-1)
    q = _softmax64(s["y"], torch.where(greedy, 1.0, T[seq])[:, None])[0] if s["y"] is not None else None
    best = (x == x.amax(1, keepdim=True)).to(torch.uint8).argmax(1)                  # the first of the largest
    pd = p.gather(1, drafted[:, None])[:, 0]
    qd = 1.0 if q is None else q.gather(1, drafted[:, None])[:, 0]
    ok = torch.where(greedy, drafted == best, u[:, 0] * qd < pd) & ~last
    # the row at which each sequence ends
    end = torch.full((B,), N, device=DEV).scatter_reduce(0, seq, torch.where(ok, N, i), "amin")
    c = end.clamp(max=N - 1)
    r = p[c]
    if q is None:
        r = torch.where(~last[c, None] & (torch.arange(V, device=DEV) == drafted[c, None]), 0.0, r)
    else:
        r = torch.where(last[c, None], r, (r - q[c]).clamp(min=0))
    r = torch.where(r.sum(1, keepdim=True) > 0, r, p[c])
    total = r.cumsum(1)
    v = (total <= u[c, 1:] * total[:, -1:]).sum(1)
    v = torch.where(greedy[c], best[c], v.clamp(max=V - 1))
    tokens = torch.where(i < end[seq], drafted, torch.where(i == end[seq], v[seq], -1))
    given = logp.gather(1, tokens.clamp(min=0)[:, None])[:, 0]
    return dict(tokens=tokens, accepted=(end - starts[:-1]).to(torch.int32), logp=torch.where(tokens < 0, 0.0, given).float())


# ---------------------------------------------------------------------------------------------
# what one pass cannot do without
# ---------------------------------------------------------------------------------------------

def work(case):
    es = 2 if case.get("dtype") == "bf16" else 4
    if case["kind"] == "verify":
        rng = random.Random(case["lens"])
        rows = sum(1 + (rng.randint(0, case["drafts"]) if case["ragged"] else case["drafts"]) for _ in range(case["B"]))
        n = rows + (rows - case["B"] if case["draft"] else 0)
        return dict(bytes=n * case["V"] * es + 36 * rows, flops=4 * n * case["V"])
    new, lens = _lengths(case)
    dh = case["dh"]
    if case["kind"] == "evict":
        kept = sum(min(n, case["keep"]) for n in lens) * case["h"]
        return dict(bytes=sum(lens) * case["h"] * 4 + kept * (4 * dh * es + 8), flops=sum(lens) * case["h"])
    h, hkv, W = case["h"], case["hkv"], case["window"]
    pairs = rows = 0
    for n, t in zip(new, lens):
        first = t - n
        if n and W:
            pairs += sum(min(W, first + j + 1) for j in range(n))
            rows += t - max(0, first - W + 1)
        elif n:
            pairs += n * first + n * (n + 1) // 2
            rows += t
    N = sum(new)
    nbytes = 2 * rows * hkv * dh * es + N * h * (2 * dh * es + 4)
    if case["self"]:
        nbytes += 2 * N * hkv * dh * es
    if case["write"]:
        nbytes += 4 * N * hkv * dh * es
    if case["weights"]:
        nbytes += 8 * rows * hkv
    return dict(bytes=nbytes, flops=4 * dh * h * pairs)


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "evict":
        return _exact_evict(s)
    if case["kind"] == "verify":
        return _exact_verify(s)
    new, lens = _lengths(case)
    page, dh, hkv = case["page"], case["dh"], case["hkv"]
    g = case["h"] // hkv
    starts = _starts(new)
    if case["write"]:
        for b, (n, t) in enumerate(zip(new, lens)):
            r = torch.arange(t - n, t, device=DEV)
            at = s["table"][b].long()[r // page]
            s["K"][at, :, r % page] = s["k"][starts[b]:starts[b + 1]]
            s["V"][at, :, r % page] = s["v"][starts[b]:starts[b + 1]]
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["q"].shape[:2], float("-inf"), dtype=torch.float64, device=DEV)
    weights = s["weights"].double() if case["weights"] else None
    for b, (n, t) in enumerate(zip(new, lens)):
        if not n:
            continue
        at = s["table"][b, :-(-t // page)].long()
        tokens = slice(starts[b], starts[b + 1])
        i = torch.arange(t - n, t, device=DEV)[:, None]
        r = torch.arange(t, device=DEV)
        hidden = r > i - (1 if case["self"] else 0)
        if case["window"]:
            hidden |= i - r >= case["window"]
        for c in range(hkv):
            K = s["K"][at, c].reshape(-1, dh)[:t].double()
            V = s["V"][at, c].reshape(-1, dh)[:t].double()
            for a in range(c * g, c * g + g):
                q = s["q"][tokens, a].double()
                x = (q @ K.t() / math.sqrt(dh)).masked_fill_(hidden, float("-inf"))
                if case["self"]:
                    mine = (q * s["k_self"][tokens, c].double()).sum(1, keepdim=True) / math.sqrt(dh)
                    total = torch.logsumexp(torch.cat([x, mine], 1), 1, keepdim=True)
                else:
                    total = torch.logsumexp(x, 1, keepdim=True)
                p = torch.exp(x - total)
                o[tokens, a] = p @ V
                if case["self"]:
                    o[tokens, a] += torch.exp(mine - total) * s["v_self"][tokens, c].double()
                lse[tokens, a] = total[:, 0]
                if case["weights"]:
                    weights[b, c, :t] += p.sum(0)
    out = dict(o=o, lse=lse)
    if case["weights"]:
        out["weights"] = weights
    if case["write"]:
        out["K"], out["V"] = None, None
    return out


def _exact_evict(s):
    """The pages and weights after each key head's kept rows were moved, sequence by sequence."""
    case, page, H = s["case"], s["case"]["page"], s["case"]["h"]
    K, V = s["K"].double(), s["V"].double()
    weights = torch.zeros(case["B"], H, s["new_table"].shape[1] * page, dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["lengths"].tolist()):
        left = min(n, case["keep"])
        at = s["new_table"][b].long()
        dst, slot = at[torch.arange(left, device=DEV) // page], torch.arange(left, device=DEV) % page
        for c in range(H):
            w = s["weights"][b, c, :n]
            kept = torch.zeros(n, dtype=torch.bool, device=DEV)
            kept[:case["sinks"]] = kept[max(0, n - case["recent"]):] = True
            if left == n:
                kept[:] = True
            elif left > case["sinks"] + case["recent"]:
                need = left - case["sinks"] - case["recent"]
                free = w[~kept]
                least = free.topk(need).values[-1]                  # all above it, and the first of those equal to it
                take = free > least
                take[(free == least).nonzero()[:need - int(take.sum()), 0]] = True
                kept[~kept] = take
            r = kept.nonzero()[:, 0]
            src = s["table"][b].long()[r // page]
            K[dst, c, slot], V[dst, c, slot] = K[src, c, r % page], V[src, c, r % page]
            weights[b, c, :left] = w[r].double()
    return dict(rows=None, lengths=None, weights=weights, K=K, V=V)


def _exact_verify(s):
    """The log probabilities of the tokens that the definition gives, sequence by sequence."""
    starts = s["starts"].tolist()
    logp = torch.zeros(s["x"].shape[0], dtype=torch.float64, device=DEV)
    for b, T in enumerate(s["temperature"].double().tolist()):
        for i in range(starts[b], starts[b + 1]):
            x = s["x"][i].double()
            lp = torch.log_softmax(x / (T or 1.0), 0)
            end = i == starts[b + 1] - 1
            d = None if end else int(s["ids"][i + 1])
            y = None if end or s["y"] is None else torch.log_softmax(s["y"][i].double() / (T or 1.0), 0).exp()
            if not end:
                taken = d == int((x == x.max()).nonzero()[0]) if T == 0 else \
                    float(s["u"][i, 0]) * (1.0 if y is None else float(y[d])) < float(lp[d].exp())
                if taken:
                    logp[i] = lp[d]
                    continue
            if T == 0:
                v = int((x == x.max()).nonzero()[0])
            else:
                r = lp.exp()
                if not end:
                    r = (r - y).clamp(min=0) if y is not None else r.index_fill(0, torch.tensor([d], device=DEV), 0.0)
                c = r.cumsum(0)
                v = int(torch.searchsorted(c, float(s["u"][i, 1]) * c[-1:], right=True))
            logp[i] = lp[v]
            break
    return dict(tokens=None, accepted=None, logp=logp)

"""The paged cache (paged_write, paged_attention, evict_rows) against its definitions in 64 bits. Every place of the pool that no
row fills holds NaN."""

import math

import pytest
import torch

from dual_mod_public_amd import _lib as L
from dual_mod_public_amd import paged
from tests import paged_reference as ref
from tests.hip_helpers import DEV, say

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    L.load()


def make(lengths, counts, h, h_kv, dh, page, dtype, seed=0, spare=2, cols=None):
    """A pool with the sequences' rows in pages of random order, everything else NaN; CPU tensors."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g).tolist()
    table = torch.full((len(lengths), cols or max(max(need), 1)), -1, dtype=torch.int32)
    K, V = (torch.full((total, h_kv, page, dh), math.nan, dtype=dtype) for _ in range(2))
    for b, n in enumerate(lengths):
        for i in range(need[b]):
            table[b, i] = order.pop()
        for r in range(0, n, page):
            m = min(page, n - r)
            for t in (K, V):
                t[table[b, r // page], :, :m] = torch.randn(h_kv, m, dh, generator=g).to(dtype)
    N = sum(counts)
    q = (2 * torch.randn(N, h, dh, generator=g)).to(dtype)
    k, v = (torch.randn(N, h_kv, dh, generator=g).to(dtype) for _ in range(2))
    starts = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32)
    return dict(K=K, V=V, table=table, q=q, k=k, v=v, starts=starts, lengths=torch.tensor(lengths, dtype=torch.int32))


def dev(s):
    return {n: t.to(DEV) for n, t in s.items()}


def near(got, want, bound, what):
    got = got.double().cpu()
    assert not got.isnan().any(), what
    same = got == want
    off = ((got - want).abs() / bound.clamp(min=1e-300)).masked_fill(same, 0.0)
    worst = float(off.max()) if off.numel() else 0.0
    say(f"{what}: worst error / bound {worst:.3f}")
    assert worst <= 1, (what, worst)


def check(s, counts, with_self=False, window=0, scale=None, starts=True, weights=True, q=None):
    d = dev(s)
    pair = dict(k_self=d["k"], v_self=d["v"]) if with_self else {}
    page, cols = s["K"].shape[2], s["table"].shape[1]
    w0 = torch.rand(len(counts), s["K"].shape[1], cols * page, generator=torch.Generator().manual_seed(5)) if weights else None
    w = w0.to(DEV) if weights else None
    r = paged.paged_attention(d["q"] if q is None else q, d["K"], d["V"], d["table"], d["lengths"], d["starts"] if starts else None,
                              window=window, scale=scale, weights=w, **pair)
    torch.cuda.synchronize()
    o, lse, add, bo, bl, bw = ref.attention(s["q"], s["K"], s["V"], s["table"], s["lengths"].tolist(), counts,
                                            s["k"] if with_self else None, s["v"] if with_self else None, window, scale)
    near(r.o, o, bo, "o")
    near(r.lse, lse, bl, "lse")
    if weights:
        near(w, w0.double() + add, bw + 2.0 ** -24 * (w0.double() + add), "weights")
    return r


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("dh,page,h,h_kv", [(64, 16, 4, 4), (128, 64, 4, 1), (64, 32, 6, 2), (128, 16, 3, 3), (64, 1024, 40, 2)])
@pytest.mark.parametrize("with_self", [False, True])
def test_single_tokens(dtype, dh, page, h, h_kv, with_self):
    lengths = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 300, 777]
    s = make(lengths, [1] * len(lengths), h, h_kv, dh, page, DT[dtype], seed=dh + page + h)
    check(s, [1] * len(lengths), with_self, starts=False)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("dh,page,h,h_kv", [(64, 16, 4, 2), (128, 32, 2, 2), (64, 128, 8, 1)])
@pytest.mark.parametrize("with_self,window", [(False, 0), (True, 0), (False, 1), (True, 1), (False, 37), (True, 37), (True, 2)])
def test_chunks(dtype, dh, page, h, h_kv, with_self, window):
    """Chunks of no token, one token, all of the sequence, odd counts across tiles, with windows that end inside them."""
    counts, lengths = [3, 0, 17, 1, 40, 5, 0, 2], [3, 9, 17, 200, 301, 70, 0, 33]
    s = make(lengths, counts, h, h_kv, dh, page, DT[dtype], seed=window + dh)
    check(s, counts, with_self, window)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("new", [60, 64, 200])
def test_long_chunks(dtype, new):
    counts, lengths = [new, 1, new + 3], [new + 190, 77, new + 3]
    s = make(lengths, counts, 4, 2, 64 if new == 60 else 128, 16, DT[dtype], seed=new)
    check(s, counts)
    check(s, counts, True, window=100)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-30, 3.0])
@pytest.mark.parametrize("new", [1, 30, 150])
def test_scales(scale, new):
    counts, lengths = [new, new], [new + 70, new]
    check(make(lengths, counts, 4, 2, 64, 32, torch.bfloat16, seed=new), counts, True, scale=scale)


@pytest.mark.parametrize("with_self", [False, True])
def test_many_sequences(with_self):
    """More sequences than a wave has lanes."""
    lengths = [1 + 7 * b % 143 for b in range(150)]
    s = make(lengths, [1] * 150, 2, 2, 64, 16, torch.bfloat16, seed=3)
    check(s, [1] * 150, with_self)


def test_one_long_sequence():
    """A sequence in many pieces beside short ones."""
    lengths, counts = [20011, 3, 40], [2, 1, 1]
    s = make(lengths, counts, 2, 1, 64, 64, torch.bfloat16, seed=4)
    check(s, counts)


def test_scale_and_strides():
    """q, k and v as slices of one wide projection, K and V pages of one pool, a table wider than the sequences need."""
    counts, lengths = [2, 5], [50, 90]
    s = make(lengths, counts, 4, 2, 64, 32, torch.bfloat16, seed=6, cols=9)
    d = dev(s)
    N = sum(counts)
    wide = torch.full((N, 3 * 8 * 64 + 24), math.nan, device=DEV, dtype=torch.bfloat16)
    q = torch.as_strided(wide, (N, 4, 64), (wide.stride(0), 128, 1), 8)
    q.copy_(d["q"])
    k, v = (torch.as_strided(wide, (N, 2, 64), (wide.stride(0), 256, 1), 8 + 64 + 128 * i) for i in range(2))
    k.copy_(d["k"]), v.copy_(d["v"])
    pool = torch.stack([d["K"], d["V"]], 1)     # [n_pages, 2, h_kv, page, dh]
    K, V = pool[:, 0], pool[:, 1]
    want = check(s, counts, True, scale=0.3)
    r = paged.paged_attention(q, K, V, d["table"], d["lengths"], d["starts"], k_self=k, v_self=v, scale=0.3)
    assert torch.equal(r.o, want.o) and torch.equal(r.lse, want.lse)
    paged.paged_write(k, v, K, V, d["table"], d["lengths"], d["starts"])
    paged.paged_write(d["k"], d["v"], d["K"], d["V"], d["table"], d["lengths"], d["starts"])
    assert torch.equal(K.nan_to_num(7), d["K"].nan_to_num(7)) and torch.equal(V.nan_to_num(7), d["V"].nan_to_num(7))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_write(dtype):
    counts, lengths = [3, 0, 17, 1], [3, 9, 40, 200]
    s = make(lengths, counts, 2, 2, 64, 16, DT[dtype], seed=8)
    d = dev(s)
    paged.paged_write(d["k"], d["v"], d["K"], d["V"], d["table"], d["lengths"], d["starts"])
    t = 0
    for b, (n, m) in enumerate(zip(counts, lengths)):
        for j in range(n):
            r = m - n + j
            for pages, rows in ((s["K"], s["k"]), (s["V"], s["v"])):
                pages[s["table"][b, r // 16], :, r % 16] = rows[t]
            t += 1
    assert torch.equal(d["K"].cpu().nan_to_num(7), s["K"].nan_to_num(7)) and torch.equal(d["V"].cpu().nan_to_num(7), s["V"].nan_to_num(7))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_rows_that_are_not_read_do_not_matter(dtype, dh, value):
    """Rows before the window, after the token and of later tokens hold infinities or NaN; those that the table does not need
    may be anywhere. A long chunk and a short one."""
    counts, lengths = [6, 1, 90], [70, 200, 150]
    window = 20
    s = make(lengths, counts, 2, 1, dh, 16, DT[dtype], seed=9)
    clean = {n: t.clone() for n, t in s.items()}
    for b, (n, m) in enumerate(zip(counts, lengths)):
        for r in list(range(0, m - n - window + 1)) + [m - 1, m - 2][:n - 1]:
            s["K"][s["table"][b, r // 16], :, r % 16] = value
            s["V"][s["table"][b, r // 16], :, r % 16, ::3] = value
    s["table"][1, :(200 - 1 - window) // 16] = -1       # freed
    d, e = dev(s), dev(clean)
    r = paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"], d["starts"], window=window)
    want = paged.paged_attention(e["q"], e["K"], e["V"], e["table"], e["lengths"], e["starts"], window=window)
    bound = ref.attention(clean["q"], clean["K"], clean["V"], clean["table"], lengths, counts, window=window)
    t = 0
    for n, m in zip(counts, lengths):
        fine = max(n - 2, 1) if n > 1 else 1
        near(r.o[t:t + fine], bound[0][t:t + fine], bound[3][t:t + fine], "o")
        assert torch.equal(r.lse[t:t + fine], want.lse[t:t + fine])
        if n > 1:
            assert not torch.isfinite(r.o[t + n - 1].float()).all()     # the last token reads its own row
        t += n


def test_nothing_read():
    """A first token with only its pair, one with a window that leaves nothing, and a token whose scores are all -inf."""
    s = make([1, 5, 40], [1, 1, 1], 2, 2, 64, 16, torch.float32, seed=10)
    d = dev(s)
    r = paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"], k_self=d["k"], v_self=d["v"], window=1)
    assert torch.equal(r.o, d["v"])
    d["K"].fill_(-math.inf)
    r = paged.paged_attention(d["q"].abs(), d["K"], d["V"], d["table"], d["lengths"])
    assert torch.equal(r.o, torch.zeros_like(r.o)) and (r.lse == -math.inf).all()


def test_nonfinite_scores():
    s = make([30, 30, 30], [1, 1, 1], 2, 2, 64, 16, torch.float32, seed=11)
    d = dev(s)
    d["K"][s["table"][0, 0], 0, 3, 0] = math.nan
    d["q"][1, 1] = math.nan
    d["K"][s["table"][2, 1], 1, 2] = math.inf
    q = d["q"].clone()
    q[2] = q[2].abs()
    r = paged.paged_attention(q, d["K"], d["V"], d["table"], d["lengths"])
    nan = r.o.isnan().all(-1).cpu()
    assert nan.tolist() == [[True, False], [False, True], [False, True]]
    assert torch.equal(r.lse.isnan().cpu(), nan)
    assert not r.o[0, 1].isnan().any() and not r.o[2, 0].isnan().any()


def test_bad_sequences_and_pages():
    """Lengths that the table does not hold, lengths below the new tokens, pages outside the pool: NaN there, the others as ever."""
    lengths, counts = [40, 33, 20, 25, 60], [1, 2, 1, 3, 1]
    s = make(lengths, counts, 2, 2, 64, 16, torch.bfloat16, seed=12)
    d = dev(s)
    want = paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"], d["starts"])
    d["lengths"][0] = s["table"].shape[1] * 16 + 1
    d["lengths"][3] = 2
    d["table"][2, 0] = s["K"].shape[0]
    d["table"][4, 3] = -5
    w = torch.zeros(5, 2, s["table"].shape[1] * 16, device=DEV)
    K = d["K"].clone()
    r = paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"], d["starts"], weights=w)
    bad = torch.tensor([1, 0, 0, 1, 1, 1, 1, 1], dtype=torch.bool)
    assert r.o.isnan().flatten(1).all(1).cpu().tolist() == bad.tolist() and r.lse.isnan().all(1).cpu().tolist() == bad.tolist()
    assert torch.equal(r.o[1:3], want.o[1:3])
    assert not w[1].isnan().any() and float(w[1].sum()) == pytest.approx(4, abs=1e-4)
    paged.paged_write(d["k"], d["v"], d["K"], d["V"], d["table"], d["lengths"], d["starts"])
    d["K"][s["table"][1, 1], :, 15], d["K"][s["table"][1, 2], :, 0] = K[s["table"][1, 1], :, 15], K[s["table"][1, 2], :, 0]
    d["K"][s["table"][2, 1], :, 3] = K[s["table"][2, 1], :, 3]
    assert torch.equal(d["K"].nan_to_num(7), K.nan_to_num(7))     # only the rows of whole sequences were written


def test_rows_of_no_sequence_stay():
    s = make([40, 33], [2, 3], 2, 2, 64, 16, torch.bfloat16, seed=13)
    d = dev(s)
    q = torch.cat([d["q"], torch.full((4, 2, 64), math.nan, device=DEV, dtype=torch.bfloat16)])
    out = torch.full_like(q, 5)
    r = paged.paged_attention(q, d["K"], d["V"], d["table"], d["lengths"], d["starts"], out=out)
    want = paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"], d["starts"])
    assert r.o is out and torch.equal(out[:5], want.o) and (out[5:] == 5).all()
    # without starts: an empty place of the batch
    d = dev(make([40, 16], [1, 1], 2, 2, 64, 16, torch.bfloat16, seed=13))
    d["lengths"][1] = 0
    out = torch.full_like(d["q"], 5)
    paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"], out=out)
    assert (out[1] == 5).all() and not (out[0] == 5).all()


def test_attend_one_agrees():
    """The contiguous tape's read of the same rows."""
    from dual_mod_public_amd.attention import DualModAttention
    from dual_mod_public_amd.config import DualModConfig
    cfg = DualModConfig(d_model=256, n_heads=4, ctx_mod="mult_res", max_seq_len=512)
    attn = DualModAttention(cfg).to(DEV)
    P, B = 333, 3
    s = make([P + 1] * B, [1] * B, 4, 4, 64, 64, torch.float32, seed=14)
    d = dev(s)
    rows = [torch.stack([ref.gather(s[n], s["table"], b, P) for b in range(B)]).float().to(DEV) for n in ("K", "V")]
    with torch.no_grad():
        o, _ = attn.attend_one(d["q"][:, :, None], d["k"][:, :, None], d["v"][:, :, None], *rows)
    r = paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"], k_self=d["k"], v_self=d["v"])
    bound = ref.attention(s["q"], s["K"], s["V"], s["table"], [P + 1] * B, [1] * B, s["k"], s["v"])[3]
    assert ((r.o - o[:, :, 0]).abs().cpu() <= 2 * bound).all()


@pytest.mark.parametrize("dtype,dh,page", [("bf16", 64, 16), ("bf16", 128, 64), ("fp32", 64, 32)])
@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (1, 0, 1), (37, 0, 0), (37, 4, 33), (40, 3, 10), (64, 64, 0), (500, 2, 7), (5000, 4, 4)])
def test_evict(dtype, dh, page, keep, sinks, recent):
    lengths = [0, 1, 36, 37, 38, 64, 65, 700, 1500]
    s = make(lengths, [0] * len(lengths), 3, 3, dh, page, DT[dtype], seed=keep, spare=0)
    g = torch.Generator().manual_seed(keep)
    cap = s["table"].shape[1] * page
    w = torch.randn(len(lengths), 3, cap, generator=g).mul(4).exp()
    w[3:6] = (w[3:6] * 2).floor() / 2           # many equal ones
    w[7, 0] = 0.25
    w[7, 1, :400] = 0.0
    w[7, 1, 400:] = -0.0
    w[8, 0, 100:110] = math.nan
    w[8, 0, 200:230] = math.inf
    w[8, 1] -= 3                                # negative ones
    w[8, 2, 5] = -math.inf
    left = [min(n, keep) for n in lengths]
    new_cols = max(1, -(-min(keep, cap) // page)) + 1
    n0, need = s["K"].shape[0], [-(-n // page) for n in left]
    perm = (n0 + torch.randperm(sum(need), generator=g)).tolist()
    new_table = torch.full((len(lengths), new_cols), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        for i in range(n):
            new_table[b, i] = perm.pop()
    pools = [torch.cat([s[n], torch.full((sum(need), *s[n].shape[1:]), 9.0, dtype=s[n].dtype)]).to(DEV) for n in ("K", "V")]
    before = [p.clone() for p in pools]
    r = paged.evict_rows(*pools, w.to(DEV), s["table"].to(DEV), s["lengths"].to(DEV), keep, new_table.to(DEV), sinks=sinks, recent=recent)
    rows = ref.evict(w, lengths, keep, sinks, recent)
    assert r.lengths.tolist() == left
    assert torch.equal(r.rows.cpu(), rows)
    for pool, old in zip(pools, before):
        want = old.cpu()
        for b, n in enumerate(left):
            for c in range(3):
                i = torch.arange(n)
                k = rows[b, c, :n].long()
                want[new_table[b, i // page].long(), c, i % page] = want[s["table"][b, k // page].long(), c, k % page]
        assert torch.equal(pool.cpu().nan_to_num(7), want.nan_to_num(7))
    want = torch.zeros(len(lengths), 3, new_cols * page)
    for b, n in enumerate(left):
        want[b, :, :n] = w[b].gather(1, rows[b, :, :n].long())
    assert torch.equal(r.weights.cpu().nan_to_num(-7), want.nan_to_num(-7))


def test_evict_bad_sequences():
    s = make([40, 60, 50], [0, 0, 0], 2, 2, 64, 16, torch.bfloat16, seed=15, spare=9)
    d = dev(s)
    used = set(s["table"].flatten().tolist())
    free = [p for p in range(s["K"].shape[0]) if p not in used]
    new_table = torch.tensor([free[:2], free[2:4], [free[4], s["K"].shape[0]]], dtype=torch.int32, device=DEV)
    d["lengths"][0] = -3
    d["table"][1, 0] = -1
    w = torch.zeros(3, 2, 64, device=DEV)
    w[1, :, 20] = 1
    K = d["K"].clone()
    r = paged.evict_rows(d["K"], d["V"], w, d["table"], d["lengths"], 32, new_table, recent=20)
    assert r.lengths.tolist() == [0, 32, 32] and (r.rows[0] == -1).all()
    kept = r.rows[1, 0].tolist()
    assert kept == list(range(11)) + [20] + list(range(40, 60))
    got = torch.stack([d["K"][free[2 + i // 16], 0, i % 16] for i in range(32)])
    assert got[:11].isnan().all() and torch.equal(got[12:28], torch.cat([K[s["table"][1, 2], 0, 8:], K[s["table"][1, 3], 0, :8]]))
    for p in free[:2] + sorted(used):
        assert torch.equal(d["K"][p].nan_to_num(7), K[p].nan_to_num(7))


@pytest.mark.parametrize("h,lengths,page", [(8, [13], 16), (8, [125], 128), (16, [77], 128), (4, [200, 45], 16), (8, [1], 16)])
@pytest.mark.parametrize("dh", [64, 128])
def test_sequences_that_end_with_the_pool(h, lengths, page, dh):
    """Prompts whose last page is the pool's last one, not full, so that nothing may be read behind its rows."""
    check(make(lengths, lengths, h, 1, dh, page, torch.bfloat16, seed=h, spare=0), lengths, weights=False)


def test_starts_that_descend():
    """No result is defined, but every place that is read and written lies in the call's tensors, and a right call follows."""
    s = make([64] * 200, [1] * 200, 4, 2, 64, 16, torch.bfloat16, seed=3)
    d = dev(s)
    want = paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"], d["starts"])
    starts = torch.tensor([0, 200] * 100 + [-7], dtype=torch.int32, device=DEV)
    w = torch.zeros(200, 2, s["table"].shape[1] * 16, device=DEV)
    paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"], starts, weights=w)
    got = paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"], d["starts"])
    assert torch.equal(got.o, want.o) and torch.equal(got.lse, want.lse)


def test_many_sequences_and_key_heads():
    """More sequences than lanes with key heads in the thousands: a launch of B h_kv blocks at least."""
    B, h = 130, 1024
    s = make([3] * B, [1] * B, h, h, 64, 16, torch.bfloat16, seed=4, spare=0)
    d = dev(s)
    r = paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"])
    i = torch.tensor([0, 1, 500, h - 1])
    for b in (0, 63, 64, B - 1):
        part = dict(q=s["q"][b:b + 1, i], K=s["K"][:, i], V=s["V"][:, i], table=s["table"][b:b + 1])
        o, lse, _, bo, bl, _ = ref.attention(part["q"], part["K"], part["V"], part["table"], [3], [1])
        near(r.o[b:b + 1, i.to(DEV)], o, bo, "o")
        near(r.lse[b:b + 1, i.to(DEV)], lse, bl, "lse")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("dh,page,h,h_kv", [(64, 64, 2, 2), (128, 16, 4, 1)])
@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [6, 3, 0, 9], [150, 2, 90, 40]])
@pytest.mark.parametrize("with_self,window", [(False, 0), (True, 0), (True, 1301), (False, 700)])
def test_sequences_in_pieces(dtype, dh, page, h, h_kv, counts, with_self, window):
    """Tables of more rows than a tile reads in one piece."""
    s = make([1500, 3, 701, 2303], counts, h, h_kv, dh, page, DT[dtype], seed=sum(counts) + window, cols=-(-4096 // page))
    check(s, counts, with_self, window)

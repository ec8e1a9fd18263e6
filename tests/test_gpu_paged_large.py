"""The paged cache and the drafts' check where offsets pass 31 and 32 bits: pools, weights, kept scores and rows of logits of many
gigabytes, of which a small part is filled and read."""

import math

import pytest
import torch

from dual_mod_public_amd import _lib as L
from dual_mod_public_amd import paged
from dual_mod_public_amd.drafts import verify_drafts
from tests import paged_reference as ref
from tests.hip_helpers import DEV
from tests.test_gpu_drafts import make as make_drafts
from tests.test_gpu_paged import make, near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    L.load()
    yield
    torch.cuda.empty_cache()


def spread(s, n_pages, cols):
    """The sequences of ``make`` in a pool of n_pages pages, the first and the last ones among them, and a table of cols columns."""
    n = s["K"].shape[0]
    at = torch.randperm(n_pages - 2, generator=torch.Generator().manual_seed(n))[:n] + 1
    at[0], at[1] = 0, n_pages - 1
    pools = []
    for name in ("K", "V"):
        t = torch.empty(n_pages, *s[name].shape[1:], device=DEV, dtype=s[name].dtype)
        t[at.to(DEV)] = s[name].to(DEV)
        pools.append(t)
    table = torch.full((s["table"].shape[0], cols), -1, dtype=torch.int32)
    used = s["table"] >= 0
    table[:, :s["table"].shape[1]][used] = at[s["table"][used].long()].int()
    return *pools, table, at


def test_pool_and_scores():
    """Pages of 2 MiB up to the 9th GiB, and more than 2^31 kept scores (16 new tokens of each sequence under a wide table)."""
    n_pages, cols = 4300, 525
    lengths, counts = [20 + 73 * b for b in range(16)], [16] * 16
    s = make(lengths, counts, 16, 8, 128, 1024, torch.bfloat16, seed=21, spare=0)
    K, V, table, at = spread(s, n_pages, cols)
    assert K.numel() > 2 ** 32 and 256 * 16 * cols * 1024 > 2 ** 31
    d = {n: t.to(DEV) for n, t in s.items() if n not in ("K", "V", "table")}
    args = (K, V, table.to(DEV), d["lengths"], d["starts"])
    w = torch.zeros(16, 8, cols * 1024, device=DEV)
    r = paged.paged_attention(d["q"], *args, weights=w)
    o, lse, add, bo, bl, bw = ref.attention(s["q"], s["K"], s["V"], s["table"], lengths, counts)
    near(r.o, o, bo, "o")
    near(r.lse, lse, bl, "lse")
    m = add.shape[2]
    near(w[:, :, :m], add, bw + 2.0 ** -24 * add, "weights")
    assert not w[:, :, m:].any()
    # rows into those pages, then the kept ones to others
    paged.paged_write(d["k"], d["v"], *args)
    for b in (0, 7, 15):
        for j in (0, 15):
            row = lengths[b] - 16 + j
            for pool, t in ((K, s["k"]), (V, s["v"])):
                assert torch.equal(pool[int(table[b, row // 1024]), :, row % 1024].cpu(), t[16 * b + j])
    free = torch.tensor([p for p in range(n_pages - 40, n_pages) if p not in set(at.tolist())][:16], dtype=torch.int32)
    e = paged.evict_rows(K, V, w, *args[2:4], 60, free[:, None].to(DEV), sinks=2, recent=5)
    rows = ref.evict(w[:, :, :m].cpu(), lengths, 60, 2, 5)
    assert torch.equal(e.rows.cpu(), rows)
    for b in (0, 8, 15):
        n = min(60, lengths[b])
        for c in (0, 7):
            i = rows[b, c, :n].long()
            src = table[b, i // 1024].long().to(DEV)
            assert torch.equal(K[int(free[b]), c, :n], K[src, c, (i % 1024).to(DEV)])


@pytest.mark.parametrize("new", [100, 700])
def test_pool_of_a_prompt(new):
    """The same pool read by tiles of many query rows."""
    s = make([1500, 2100], [new, new], 16, 8, 128, 1024, torch.bfloat16, seed=22, spare=0)
    K, V, table, _ = spread(s, 4300, 3)
    d = {n: t.to(DEV) for n, t in s.items()}
    w = [torch.zeros(2, 8, 3 * 1024, device=DEV) for _ in range(2)]
    want = paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"], d["starts"], weights=w[0])
    r = paged.paged_attention(d["q"], K, V, table.to(DEV), d["lengths"], d["starts"], weights=w[1])
    assert torch.equal(r.o, want.o) and torch.equal(r.lse, want.lse) and torch.equal(*w)      # the same plan, the same order


def test_weights_of_wide_tables():
    """Accumulated weights past 2^31 of them."""
    lengths, counts, cols = [5, 7, 2000], [1, 0, 3], 1 << 15
    s = make(lengths, counts, 32, 32, 64, 1024, torch.bfloat16, seed=23, cols=cols)
    d = {n: t.to(DEV) for n, t in s.items()}
    w = torch.zeros(3, 32, cols * 1024, device=DEV)
    assert w[:2].numel() >= 2 ** 31
    r = paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"], d["starts"], weights=w)
    o, lse, add, bo, bl, bw = ref.attention(s["q"], s["K"], s["V"], s["table"][:, :2], lengths, counts)
    near(r.o, o, bo, "o")
    near(w[:, :, :2048], add, bw + 2.0 ** -24 * add, "weights")
    assert not w[:, :, 2048:].any()
    new_table = torch.tensor([[0], [1], [2]], dtype=torch.int32)
    pools = [torch.cat([torch.zeros_like(d[n][:3]), d[n]]) for n in ("K", "V")]
    table = torch.where(d["table"] < 0, d["table"], d["table"] + 3)
    e = paged.evict_rows(*pools, w, table, d["lengths"], 100, new_table.to(DEV), sinks=1, recent=1)
    assert torch.equal(e.rows.cpu(), ref.evict(w[:, :, :2048].cpu(), lengths, 100, 1, 1))
    assert torch.equal(e.weights[2, :, :100].cpu(), w[2, :, :2048].cpu().gather(1, e.rows[2].cpu().long()))


def test_a_sequence_of_millions_of_rows():
    n = (1 << 21) + 12345
    s = make([n, 9], [2, 1], 2, 1, 64, 1024, torch.bfloat16, seed=24)
    d = {m: t.to(DEV) for m, t in s.items()}
    w = torch.zeros(2, 1, s["table"].shape[1] * 1024, device=DEV)
    r = paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"], d["starts"], weights=w)
    o, lse, add, bo, bl, bw = ref.attention(s["q"], s["K"], s["V"], s["table"], [n, 9], [2, 1])
    near(r.o, o, bo, "o")
    near(r.lse, lse, bl, "lse")
    near(w, add, bw + 2.0 ** -24 * add, "weights")


@pytest.mark.parametrize("dh,dtype", [(128, torch.bfloat16), (64, torch.float32), (128, torch.float32)])
def test_more_rows_than_the_last_cache_holds(dh, dtype):
    lengths, counts = [600001, 450000, 77], [1, 2, 3]
    s = make(lengths, counts, 2, 1, dh, 1024, dtype, seed=26)
    assert s["K"].numel() * s["K"].element_size() * 2 > 1 << 28
    d = {m: t.to(DEV) for m, t in s.items()}
    w = torch.zeros(3, 1, s["table"].shape[1] * 1024, device=DEV)
    r = paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"], d["starts"], weights=w)
    o, lse, add, bo, bl, bw = ref.attention(s["q"], s["K"], s["V"], s["table"], lengths, counts)
    near(r.o, o, bo, "o")
    near(r.lse, lse, bl, "lse")
    near(w, add, bw + 2.0 ** -24 * add, "weights")


def test_rows_of_logits_far_apart():
    """A row stride of 2^27 elements: rows past 2^32 elements."""
    counts, V = [20, 3, 17], 5000
    s = make_drafts(counts, V, torch.bfloat16, 25)
    d = {n: t.to(DEV) for n, t in s.items()}
    want = verify_drafts(d["x"], d["ids"], d["u"], d["starts"], draft_logits=d["y"], temperature=d["T"])
    wide = []
    for n in ("x", "y"):
        t = torch.empty(40, 1 << 27, device=DEV, dtype=torch.bfloat16)[:, 7:7 + V]
        t.copy_(d[n])
        wide.append(t)
    r = verify_drafts(wide[0], d["ids"], d["u"], d["starts"], draft_logits=wide[1], temperature=d["T"])
    assert torch.equal(r.tokens, want.tokens) and torch.equal(r.accepted, want.accepted) and torch.equal(r.logp, want.logp)
    assert math.isfinite(float(r.logp.sum()))

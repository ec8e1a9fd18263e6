"""verify_drafts against its definition, row by row in 64 bits."""

import math

import pytest
import torch

from dual_mod_public_amd import _lib as L
from dual_mod_public_amd.drafts import verify_drafts
from tests import paged_reference as ref
from tests.hip_helpers import DEV

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    L.load()


def make(counts, V, dtype, seed, draft=True, sharp=3.0):
    g = torch.Generator().manual_seed(seed)
    N = sum(counts)
    x = sharp * torch.randn(N, V, generator=g)
    y = x + 0.8 * torch.randn(N, V, generator=g)
    x, y = x.to(dtype), y.to(dtype)
    T = 0.5 + torch.rand(len(counts), generator=g)
    ids = torch.randint(0, V, (N,), generator=g)
    for b, t0 in enumerate([sum(counts[:b]) for b in range(len(counts))]):
        for t in range(t0, t0 + counts[b] - 1):
            ids[t + 1] = torch.multinomial(torch.softmax((y if draft else x)[t].double() / T[b], 0), 1, generator=g)
    starts = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32)
    return dict(x=x, y=y if draft else None, ids=ids, u=torch.rand(N, 2, generator=g), T=T, starts=starts)


def check(s, counts, lead=0):
    d = {n: None if t is None else t.to(DEV) for n, t in s.items()}
    r = verify_drafts(d["x"], d["ids"], d["u"], d["starts"], draft_logits=d["y"], temperature=d["T"])
    tokens, accepted, logp = ref.verify(s["x"], s["ids"], s["u"], counts, s["y"], s["T"])
    assert torch.equal(r.accepted.cpu(), accepted)
    assert torch.equal(r.tokens.cpu(), tokens)
    got = r.logp.cpu().double()
    assert torch.equal(got.isnan(), logp.isnan())
    # 64 bits throughout, rounded to fp32 once
    assert ((got - logp).abs() <= 2.0 ** -23 * logp.abs() + 1e-12)[~logp.isnan()].all()
    return r


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [1, 2, 7, 64, 1000, 4095, 4096, 4097, 50257])
@pytest.mark.parametrize("draft", [True, False])
def test_ragged_batches(dtype, V, draft):
    counts = [5, 1, 0, 3, 9, 2, 0, 6]
    for seed in range(2 if V > 5000 else 6):
        s = make(counts, V, dtype, 100 * V + seed, draft, sharp=3.0 if seed % 2 else 0.5)
        s["T"][1 + seed % 4] = 0.0
        r = check(s, counts)
        assert (r.accepted.cpu() <= (torch.tensor(counts) - 1).clamp(min=0)).all()


def test_wide_rows_of_a_buffer():
    """Row strides and odd places of rows in wider buffers."""
    counts = [4, 2]
    s = make(counts, 1001, torch.bfloat16, 5)
    d = {n: t.to(DEV) for n, t in s.items()}
    wide = [torch.full((6, 1040 + i), math.nan, device=DEV, dtype=torch.bfloat16) for i in (1, 2)]
    for t, n in zip(wide, "xy"):
        t[:, 3:1004] = d[n]
    a = verify_drafts(d["x"], d["ids"], d["u"], d["starts"], draft_logits=d["y"], temperature=d["T"])
    b = verify_drafts(wide[0][:, 3:1004], d["ids"], d["u"], d["starts"], draft_logits=wide[1][:, 3:1004], temperature=d["T"])
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("draft", [True, False])
def test_masks_and_rows_without_a_distribution(draft):
    V = 5000
    counts = [4] * 10
    s = make(counts, V, torch.float32, 6, draft)
    x, u = s["x"], s["u"]
    u[:, 0] = 0.0                        # every draft with a probability is accepted
    keep = torch.rand(40, V, generator=torch.Generator().manual_seed(1)) < 0.01
    keep[:, 17] = True
    x.masked_fill_(~keep, -math.inf)
    x[5, 100] = math.nan                 # sequence 1, second row
    x[8] = -math.inf                     # sequence 2, first row
    x[12, 3] = math.inf                  # sequence 3, first row
    s["ids"][17] = V                     # sequence 4: drafts of no token
    s["ids"][21] = -1                    # sequence 5
    x[24] = -math.inf
    x[24, 4444] = 0.0                    # sequence 6: one token is certain
    s["ids"][25] = 4444
    u[28, 1], u[32, 1] = 0.0, 1 - 2.0 ** -24
    s["T"][9] = 0.0
    x[37, 3] = math.inf                  # greedy: it is the largest
    for i in range(40):                  # drafts that the mask leaves
        if 0 <= s["ids"][i] < V and i % 3 and i not in (0,):
            s["ids"][i] = 17
    if draft:
        s["y"][6, 9] = math.nan
        s["y"][33] = -math.inf
    check(s, counts)


def test_equal_distributions_accept_everything_below_one():
    counts = [6] * 8
    s = make(counts, 3000, torch.float32, 7)
    s["y"] = s["x"].clone()
    s["u"][:, 0] = 1 - 2.0 ** -24
    r = check(s, counts)
    assert (r.accepted == 5).all()


def test_places_on_borders():
    """Few equal probabilities: places on and beside the borders between tokens."""
    V, n = 8, 8
    x = torch.zeros(n * 3, V)
    starts = torch.arange(n * 3 + 1, dtype=torch.int32)
    u = torch.zeros(n * 3, 2)
    for i in range(n):
        for k, off in enumerate((0.0, -2.0 ** -20, 2.0 ** -20)):
            u[3 * i + k, 1] = max(0.0, i / n + off)
    s = dict(x=x, y=None, ids=torch.zeros(n * 3, dtype=torch.int64), u=u, T=torch.ones(n * 3), starts=starts)
    r = check(s, [1] * (n * 3))
    assert r.tokens.tolist() == [v for i in range(n) for v in (i, max(i - 1, 0), i)]


def test_frequencies():
    """Tokens of many drawn numbers follow the target, whatever the draft: counts within 5 standard deviations."""
    V, B = 6, 20000
    g = torch.Generator().manual_seed(8)
    x, y = torch.randn(V, generator=g), torch.randn(V, generator=g)
    p = torch.softmax(x.double(), 0)
    ids = torch.zeros(2 * B, dtype=torch.int64)
    ids[1::2] = torch.multinomial(torch.softmax(y.double(), 0), B, replacement=True, generator=g)
    u = torch.rand(2 * B, 2, generator=g)
    count = torch.zeros(V)
    for i in range(0, B, 10000):
        rows = slice(2 * i, 2 * i + 20000)
        r = verify_drafts(x.expand(20000, V).contiguous().to(DEV), ids[rows].to(DEV), u[rows].to(DEV),
                          torch.arange(0, 20001, 2, dtype=torch.int32, device=DEV), draft_logits=y.expand(20000, V).contiguous().to(DEV))
        count += torch.bincount(r.tokens[::2].cpu(), minlength=V)
    sigma = (B * p * (1 - p)).sqrt()
    assert ((count - B * p).abs() <= 5 * sigma).all(), (count, B * p)


def test_rows_of_no_sequence():
    s = make([3, 2], 100, torch.float32, 9)
    d = {n: t.to(DEV) for n, t in s.items()}
    pad = lambda t, n: torch.cat([torch.full((n, *t.shape[1:]), math.nan).to(t) if t.is_floating_point() else t.new_full((n,), 3), t, t])   # noqa: E731
    a = verify_drafts(d["x"], d["ids"], d["u"], d["starts"], draft_logits=d["y"], temperature=d["T"])
    b = verify_drafts(pad(d["x"], 2), pad(d["ids"], 2), pad(d["u"], 2), d["starts"] + 2, draft_logits=pad(d["y"], 2), temperature=d["T"])
    assert torch.equal(b.tokens[2:7], a.tokens) and torch.equal(b.logp[2:7], a.logp) and torch.equal(b.accepted, a.accepted)
    assert (b.tokens[:2] == -1).all() and (b.tokens[7:] == -1).all() and (b.logp[7:] == 0).all()


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_small_and_large_temperatures(draft, dtype):
    """Down to those of which a logit's quotient is far beyond its 64 bits' whole numbers, where only the largest logits have any
    probability, and up to a uniform distribution."""
    counts = [4, 6, 2, 5, 3, 4, 1]
    s = make(counts, 5000, dtype, 77, draft)
    s["T"] = torch.tensor([1e-3, 1e-8, 1e-20, 1e-30, 1e-44, 1e10, 3e38])
    s["x"][5, 10] = s["x"][5, 4200] = s["x"][5].max() + 1      # two largest ones
    s["x"] += 30
    check(s, counts)


@pytest.mark.parametrize("T", [-1.0, -1e-30, math.inf, -math.inf, math.nan])
def test_numbers_that_are_no_temperature(T):
    counts = [4, 3, 5]
    s = make(counts, 700, torch.bfloat16, 78)
    want = check(s, counts)
    d = {n: t.to(DEV) for n, t in s.items()}
    d["T"][1] = T
    r = verify_drafts(d["x"], d["ids"], d["u"], d["starts"], draft_logits=d["y"], temperature=d["T"])
    assert r.accepted[1] == 0 and (r.tokens[4:7] == -1).all() and r.logp[4].isnan() and (r.logp[5:7] == 0).all()
    keep = [0, 1, 2, 3, 7, 8, 9, 10, 11]
    assert torch.equal(r.tokens[keep], want.tokens[keep]) and torch.equal(r.logp[keep], want.logp[keep])

"""dm_logprob_rows / dm_logprob_rows_bwd (logprobs.py) against the definitions in 64 bits on the CPU.

Tolerances count roundings (u = 2^-24) of the fp32 arithmetic: d = x - M (u |d|), e = exp2(d log2 e) (the product and its
constant 1.5 u |d|, the instruction 2 u), sums of n terms in chains of at most n / 64 + 24 additions."""

import math

import pytest
import torch

from dual_mod_public_amd import _lib as L
from dual_mod_public_amd import logprobs as lp
from tests.hip_helpers import DEV, say

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
INF, NAN = float("inf"), float("nan")
DTYPES = [torch.bfloat16, torch.float32]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    L.load()


def oracle(x, t=None, top=0):
    """(logp, entropy, lse, top_logp, top_ids, p, lp) in 64 bits, rows without NaN and +inf."""
    x = x.double().cpu()
    M = x.amax(-1, keepdim=True)
    d = torch.where(x == -INF, -INF, x - M)               # not x - lse: at the type's lowest value log Z is lost in lse
    log_z = d.exp().sum(-1, keepdim=True).log()
    lse = (M + log_z)[..., 0]
    tok = torch.where(x == -INF, -INF, d - log_z)
    p = tok.exp()
    entropy = -(p * torch.where(p == 0, 0.0, tok)).sum(-1)
    logp = None
    if t is not None:
        t = t.cpu()
        logp = tok.gather(-1, t.clamp(0, x.shape[-1] - 1)[..., None])[..., 0]
        logp = torch.where(t < 0, 0.0, torch.where(t >= x.shape[-1], NAN, logp))
    s = x.sort(dim=-1, descending=True, stable=True)
    ids = s.indices[..., :top]
    return logp, entropy, lse, tok.gather(-1, ids), ids, p, tok


def bounds(x):
    """Absolute error bounds per row (shape [...]) of log_z, and of the entropy."""
    x = x.double().cpu()
    M = x.amax(-1, keepdim=True)
    d = torch.where(x == -INF, -1e3, x - torch.where(M == -INF, 0.0, M))
    e = torch.where(x == -INF, 0.0, d.exp())
    Z = e.sum(-1).clamp(min=1e-300)
    chain = x.shape[-1] / 64 + 24
    ad = -torch.where(e == 0, 0.0, d)
    rel = 2.5 * ad + 2                                    # of one e, in u
    log_z = U * ((e * rel).sum(-1) / Z + chain + 2 + 2 * Z.log().abs())
    q = (e * ad).sum(-1) / Z
    ent = log_z + U * ((e * ad * (rel + 2)).sum(-1) / Z + (2 * chain + 4) * q + 2 * Z.log().abs()) + q * log_z
    return log_z, ent


def close(got, want, tol, what):
    got, want = got.double().cpu(), want.double()
    same = torch.isnan(got) == torch.isnan(want)
    inf = torch.isinf(want)
    assert same.all() and (got[inf] == want[inf]).all(), f"{what}: {got.flatten()[:4]} {want.flatten()[:4]}"
    ok = torch.isnan(want) | inf | ((got - want).abs() <= tol)
    bad = (~ok).nonzero()
    assert ok.all(), f"{what}: {len(bad)} off, at {bad[0].tolist()}: {got[tuple(bad[0])]} {want[tuple(bad[0])]}"


def check_values(x, t, top, r, what=""):
    logp, entropy, lse, top_logp, top_ids, _, _ = oracle(x, t, top)
    bz, be = bounds(x)
    if t is not None:
        close(r.logp, logp, bz + 2 * U * (2 * logp.abs().nan_to_num(0, 0, 0) + math.log(x.shape[-1])), what + " logp")
    close(r.lse, lse, bz + U * lse.abs().nan_to_num(0, 0, 0), what + " lse")
    close(r.entropy, entropy, be, what + " entropy")
    if top:
        assert torch.equal(r.top_ids.cpu(), top_ids), what
        close(r.top_logp, top_logp, bz[..., None] + 2 * U * (2 * top_logp.abs().nan_to_num(0, 0, 0) + math.log(x.shape[-1])), what + " top")


def check_grad(x, t, g, gh, dx, what=""):
    """dx of rows without NaN and +inf, targets below the number of columns."""
    _, entropy, lse, _, _, p, tok = oracle(x, t)
    bz, be = bounds(x)
    V = x.shape[-1]
    g = torch.zeros(t.shape, dtype=torch.float64) if g is None else torch.where(t.cpu() < 0, 0.0, g.double().cpu())
    gh = torch.zeros(t.shape, dtype=torch.float64) if gh is None else gh.double().cpu()
    tok = torch.where(p == 0, 0.0, tok)
    inner = g[..., None] + gh[..., None] * (tok + entropy[..., None])
    want = -p * inner
    hot = torch.zeros_like(p).scatter_(-1, t.cpu().clamp(min=0)[..., None], 1.0) * (t.cpu() >= 0)[..., None]
    want = want + hot * g[..., None]
    want[lse == -INF] = 0
    err_lp = bz[..., None] + 2 * U * (2 * tok.abs() + math.log(p.shape[-1]))     # |d| <= |tok| + log Z, log Z <= log V
    size = g.abs()[..., None] + gh.abs()[..., None] * (tok.abs() + entropy[..., None])
    tol = p * (size * (err_lp + U * (2.5 * tok.abs() + 8)) + gh.abs()[..., None] * (err_lp + be[..., None]))
    tol = tol + U * want.abs() + 2 * U * hot * g.abs()[..., None]
    # the stored rounding; exp2 gives 0 below 2^-126, p's error then, and so do stored subnormals
    tol = tol * 1.01 + want.abs() * torch.finfo(dx.dtype).eps / 2 * 1.01 + 2.0 ** -126 * (1 + size)
    close(dx, want, tol, what + " gradient")


def rows_of(M, V, dtype, seed=0, ld=None, scale=3.0, base=0):
    """[M, V] logits with a row stride of ld elements, the first at an offset of base elements; poison around."""
    g = torch.Generator(device=DEV).manual_seed(seed + 7 * V + M)
    ld = ld or V
    buf = torch.full((base + M * ld + 16,), 1e4, device=DEV, dtype=dtype)
    x = buf[base:base + M * ld].view(M, ld)[:, :V]
    x.copy_((scale * torch.randn(M, V, generator=g, device=DEV)).to(dtype))
    t = torch.randint(0, V, (M,), generator=g, device=DEV)
    return x, t, g, buf


SIZES = [(1, 1), (3, 2), (2, 7), (7, 64), (5, 513), (300, 129), (65, 4099), (9, 8192), (4, 32000), (3, 50257), (2, 131073),
         (2, 262147)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,V", SIZES)
def test_values_and_gradient(M, V, dtype):
    say(f"rows {M} x {V} {dtype}")
    for case, (pad, base, top) in enumerate(((0, 0, 0), (3, 1, min(V, 5)), (8, 0, min(V, 32)))):
        x, t, g, buf = rows_of(M, V, dtype, seed=case, ld=V + pad, base=base)
        t[:: 3] = -1
        if case == 2:
            x[:, V // 2:] = x[:, : V - V // 2].clone()       # each value twice or more: the lower id first
        before = buf.clone()
        w, gh = torch.randn(M, generator=g, device=DEV), torch.randn(M, generator=g, device=DEV)
        r = lp.row_logprobs(x, t, top=top)
        check_values(x, t, top, r, f"case {case}")
        r2, dx = lp.row_logprobs_grad(x, t, w, gh, top=top)
        assert all(torch.equal(a, b) for a, b in zip(r, r2) if a is not None)
        check_grad(x, t, w, gh, dx, f"case {case} fused")
        dx2 = lp.row_logprobs_bwd(x, t, r.stats, w, gh)
        check_grad(x, t, w, gh, dx2, f"case {case} backward")
        assert torch.equal(buf, before)
        # one coefficient alone; the gradient in place, its surroundings as they were
        check_grad(x, t, w, None, lp.row_logprobs_bwd(x, t, r.stats, w), f"case {case} logp only")
        check_grad(x, t, None, gh, lp.row_logprobs_grad(x, t, None, gh)[1], f"case {case} entropy only")
        clean = x.clone()
        _, dx3 = lp.row_logprobs_grad(x, t, w, gh, dlogits=x)
        assert dx3.data_ptr() == x.data_ptr() and torch.equal(x, dx)
        x.copy_(clean)
        lp.row_logprobs_bwd(x, t, r.stats, w, gh, dlogits=x)
        assert torch.equal(x, dx2)
        x.copy_(clean)
        assert torch.equal(buf, before)


# the gradient into rows of another stride and alignment than the logits'
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_stride_of_its_own(dtype):
    M, V = 5, 1001
    x, t, g, _ = rows_of(M, V, dtype, ld=1008)
    w = torch.randn(M, generator=g, device=DEV)
    want = lp.row_logprobs_grad(x, t, w)[1]
    for ld, base in ((1001, 1), (1003, 0), (1010, 3)):
        d, _, _, buf = rows_of(M, V, dtype, ld=ld, base=base)
        around = buf.clone()
        around[base:base + M * ld].view(M, ld)[:, :V] = want
        lp.row_logprobs_grad(x, t, w, dlogits=d)
        assert torch.equal(buf, around)
        d.zero_()
        r = lp.row_logprobs(x, t)
        lp.row_logprobs_bwd(x, t, r.stats, w, dlogits=d)
        check_grad(x, t, w, None, d)
        assert torch.equal(buf[:base], around[:base]) and torch.equal(buf[base + M * ld:], around[base + M * ld:])


def special_rows(V, dtype):
    """(name, row, target) of rows at the edges of the definition, without NaN and +inf."""
    g = torch.Generator(device=DEV).manual_seed(V)
    n = torch.randn(V, generator=g, device=DEV)
    low = torch.finfo(dtype).min
    out = [("empty", torch.full((V,), -INF), 0), ("one allowed", torch.full((V,), -INF), V // 2), ("equal", torch.full((V,), 2.5), 1),
           ("zero signs", torch.zeros(V), 1), ("descending", torch.arange(V, 0, -1) / 64.0, 0), ("ascending", torch.arange(V) / 64.0, 0),
           ("lowest", torch.full((V,), low), 2), ("three allowed", torch.full((V,), low), 3), ("masked target", n.clone(), 5),
           ("huge", n * 1e30, 0), ("peaked", n.clone(), 7), ("one lane", n.clone(), 4), ("far", n + 30000.0, 4), ("ignored", n.clone(), -1),
           ("contiguous few", torch.full((V,), -INF), V - 1), ("negative", -5 - n.abs(), 6), ("beside -1e37", n - 3, 2),
           ("all far below", -1e37 * (1 + n.abs()), 2), ("largest number", n.clone(), 3), ("two largest", n.clone(), 3)]
    rows = []
    for name, row, t in out:
        row = row.to(DEV).float()
        if name == "one allowed":
            row[V // 2] = -3.0
        if name == "zero signs":
            row[::3] = -0.0
        if name == "three allowed":
            row[3], row[V // 2], row[V - 1] = 1.0, 2.0, 1.0
        if name == "masked target":
            row[5] = -INF
            row[V // 3:] = -INF
        if name == "peaked":
            row[7] = 200.0
        if name == "one lane":
            row[8 * 64 * 4::8 * 64 * 4] += 50.0       # the largest far apart at one stride
        if name == "beside -1e37":
            row[5::7] = -1e37
            row[torch.arange(V, device=DEV) % 8 != 2] = -1e37
        if name in ("largest number", "two largest"):
            row[3] = 3e38
        if name == "two largest":
            row[V // 2] = 3e38
        if name == "contiguous few":
            row[V - 9:] = n[:9]
        rows.append((name, row.to(dtype), t))
    return rows


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [40, 2048, 32000, 70001])
def test_special_rows(V, dtype):
    rows = special_rows(V, dtype)
    x = torch.stack([r for _, r, _ in rows])
    t = torch.tensor([t for _, _, t in rows], device=DEV)
    w = torch.linspace(-1, 1, len(rows), device=DEV) + 0.01
    gh = torch.linspace(1, 2, len(rows), device=DEV)
    for top in (0, 1, 20, 32):
        r, dx = lp.row_logprobs_grad(x, t, w, gh, top=top)
        for i, (name, _, _) in enumerate(rows):
            s = slice(i, i + 1)
            check_values(x[s], t[s], top, lp.RowLogprobs(*[None if v is None else v[s] for v in r]), f"{name} top={top}")
            check_grad(x[s], t[s], w[s], gh[s], dx[s], f"{name} top={top}")
    dx = lp.row_logprobs_bwd(x, t, r.stats, w, gh)
    for i, (name, _, _) in enumerate(rows):
        check_grad(x[i:i + 1], t[i:i + 1], w[i:i + 1], gh[i:i + 1], dx[i:i + 1], name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [33, 5000, 70001])
def test_nan_and_infinity(V, dtype):
    """NaN rows, +inf rows, targets past the columns: as documented, and the rows between them untouched by it."""
    x, t, g, _ = rows_of(8, V, dtype)
    clean, ones = x.clone(), torch.ones(8, device=DEV)
    x[1, V // 2] = NAN
    x[3, 4], x[3, 20] = INF, INF
    x[4, 4], x[4, 9] = INF, NAN
    t[3], t[4], t[5], t[6] = 4, 0, V, -1
    x[6, 0] = NAN
    r, dx = lp.row_logprobs_grad(x, t, ones, 0.5 * ones, top=4)
    for i in (0, 2, 7):
        s = slice(i, i + 1)
        check_values(clean[s], t[s], 4, lp.RowLogprobs(*[v[s] for v in r]))
        check_grad(clean[s], t[s], ones[s], 0.5 * ones[s], dx[s])
    assert torch.isnan(r.logp[[1, 3, 4, 5]]).all() and r.logp[6] == 0
    assert torch.isnan(r.lse[[1, 4, 6]]).all() and r.lse[3] == INF
    assert torch.isnan(r.entropy[[1, 3, 4, 6]]).all() and torch.isfinite(r.entropy[5])
    assert torch.isnan(dx[[1, 3, 4, 5, 6]]).all()
    assert torch.isnan(lp.row_logprobs_bwd(x, t, r.stats, ones, 0.5 * ones)[[1, 3, 4, 5, 6]]).all()
    # NaN before every number, then infinities, the lower id first; finite tokens beside an infinite one
    assert r.top_ids[1, 0] == V // 2 and r.top_ids[3, :2].tolist() == [4, 20] and r.top_ids[4, :2].tolist() == [9, 4]
    assert torch.isnan(r.top_logp[1]).all() and torch.isnan(r.top_logp[3, :2]).all() and (r.top_logp[3, 2:] == -INF).all()
    t[3] = 5
    assert lp.row_logprobs(x, t).logp[3] == -INF
    # rows whose coefficients are 0 are zeros, whatever they hold
    zero = lp.row_logprobs_grad(x, t, 0 * ones)[1]
    assert (zero == 0).all()
    assert (lp.row_logprobs_bwd(x, t, r.stats, 0 * ones, 0 * ones) == 0).all()
    assert (lp.row_logprobs_grad(x, t, ones)[1][6] == 0).all()          # ignored


@pytest.mark.parametrize("dtype", DTYPES)
def test_autograd(dtype):
    """token_logprobs: leading dimensions, strided and broadcast logits, either output alone, and the gradient against
    differences of the 64-bit definition."""
    g = torch.Generator(device=DEV).manual_seed(3)
    wide = torch.randn(2, 5, 120, generator=g, device=DEV).to(dtype).requires_grad_()
    t = torch.randint(0, 100, (2, 5), generator=g, device=DEV)
    t[0, 1] = -1
    w, gh = torch.randn(2, 5, generator=g, device=DEV), torch.randn(2, 5, generator=g, device=DEV)
    logp, ent = lp.token_logprobs(wide[..., :100], t)
    d, = torch.autograd.grad((logp, ent), wide, (w, gh))
    assert (d[..., 100:] == 0).all()
    check_grad(wide.detach()[..., :100], t, w, gh, d[..., :100])
    # differences: f = sum(w logp + gh ent), d/dh f(x + h v); the third derivative's term h^2 / 6 sup|f'''| |v|^3 and
    # the cancellation 2^-52 |f| / h are far below the gradient's own bf16 / fp32 rounding of sum |d v|
    x64 = wide.detach()[..., :100].double().cpu()
    v = torch.randn(x64.shape, generator=torch.Generator().manual_seed(1), dtype=torch.float64)

    def f(x):
        o = oracle(x, t)
        return (w.double().cpu() * o[0] + gh.double().cpu() * o[1]).sum()

    h = 1e-4
    want = (f(x64 + h * v) - f(x64 - h * v)) / (2 * h)
    got = (d[..., :100].double().cpu() * v).sum()
    assert abs(got - want) <= (torch.finfo(dtype).eps + 1e-6) * (d[..., :100].double().cpu() * v).abs().sum()
    # one output alone
    logp, ent = lp.token_logprobs(wide[..., :100], t)
    check_grad(wide.detach()[..., :100], t, torch.ones_like(w), None, torch.autograd.grad(logp.sum(), wide)[0][..., :100])
    logp, ent = lp.token_logprobs(wide[..., :100], t)
    check_grad(wide.detach()[..., :100], t, None, torch.ones_like(w), torch.autograd.grad(ent.sum(), wide)[0][..., :100])
    # one row for all positions: its gradient is the sum over them
    row = torch.randn(1, 64, generator=g, device=DEV).to(dtype).requires_grad_()
    t4 = torch.tensor([0, 5, 5, 63], device=DEV)
    logp, _ = lp.token_logprobs(row.expand(4, 64), t4)
    d, = torch.autograd.grad(logp, row, torch.ones(4, device=DEV))
    p = row.detach().double().softmax(-1).cpu()
    want = torch.zeros(1, 64, dtype=torch.float64).index_add_(1, t4.cpu(), torch.ones(1, 4, dtype=torch.float64)) - 4 * p
    # four stored gradients, each rounded once, and their sum's roundings
    tol = (4 * torch.finfo(dtype).eps) * (p * 4 + (want + 4 * p)) + 1e-6
    assert ((d.double().cpu() - want).abs() <= tol).all()
    # differentiable once; nothing written into what autograd keeps
    logp, _ = lp.token_logprobs(wide[..., :100], t)
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(logp.sum(), wide, create_graph=True)
    logp, _ = lp.token_logprobs(wide[..., :100].contiguous(), t)
    assert logp.grad_fn is not None and not lp.row_logprobs(wide.detach()[..., :100], t).logp.requires_grad


def test_rows_past_32_bits():
    """A buffer of more than 2^32 bytes and 2^31 elements: the last rows are read and written in their place."""
    M, V = 33000, 65601
    x = torch.zeros(M, V, device=DEV, dtype=torch.bfloat16)
    t = torch.full((M,), 7, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(0)
    x[-1] = torch.randn(V, generator=g, device=DEV).to(x.dtype)
    r, dx = lp.row_logprobs_grad(x, t, torch.ones(M, device=DEV), top=1)
    check_values(x[-1:], t[-1:], 1, lp.RowLogprobs(*[v[-1:] for v in r]))
    check_grad(x[-1:], t[-1:], torch.ones(1, device=DEV), None, dx[-1:])
    check_values(x[-2:-1], t[-2:-1], 1, lp.RowLogprobs(*[v[-2:-1] for v in r]))
    want = lp.row_logprobs_bwd(x, t, r.stats, torch.ones(M, device=DEV), dlogits=x)
    check_grad(torch.zeros(1, V), t[:1], torch.ones(1, device=DEV), None, want[:1])
    assert torch.equal(want[-1], dx[-1]) or (want[-1].float() - dx[-1].float()).abs().max() <= 2.0 ** -8 * dx[-1].float().abs().max()


def test_many_short_rows():
    """More rows than a launch has blocks."""
    M, V = (1 << 20) + 70000, 9
    x, t, g, _ = rows_of(M, V, torch.float32)
    w = torch.randn(M, generator=g, device=DEV)
    r, dx = lp.row_logprobs_grad(x, t, w, top=2)
    check_values(x, t, 2, r)
    check_grad(x, t, w, None, dx)
    check_grad(x, t, w, None, lp.row_logprobs_bwd(x, t, r.stats, w))


def test_rows_do_not_depend_on_the_batch():
    """A row alone gives the values it has among others, whatever form its number of rows takes; a call repeated gives
    its bits again."""
    for V, dtype in ((32000, torch.bfloat16), (50257, torch.float32), (700, torch.bfloat16)):
        x, t, g, _ = rows_of(600, V, dtype)
        w = torch.randn(600, generator=g, device=DEV)
        r, dx = lp.row_logprobs_grad(x, t, w, top=8)
        again, dx2 = lp.row_logprobs_grad(x, t, w, top=8)
        assert torch.equal(dx, dx2) and all(torch.equal(a, b) for a, b in zip(r, again))
        one = lp.row_logprobs(x[5:6], t[5:6], top=8)
        check_values(x[5:6], t[5:6], 8, one)
        assert torch.equal(one.top_ids[0], r.top_ids[5])


@pytest.mark.parametrize("M,V", [(3, 50257), (300, 2000)])
def test_streams_and_graph(M, V):
    """On another stream, and captured: every replay, with new inputs and eager work between, equals the eager call."""
    x, t, g, _ = rows_of(M, V, torch.bfloat16)
    w, gh = torch.randn(M, generator=g, device=DEV), torch.randn(M, generator=g, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    want = lp.row_logprobs_grad(x, t, w, gh, top=6)
    with torch.cuda.stream(s):
        got = lp.row_logprobs_grad(x, t, w, gh, top=6)
    s.synchronize()
    assert torch.equal(got[1], want[1]) and all(torch.equal(a, b) for a, b in zip(got[0], want[0]))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        r, dx = lp.row_logprobs_grad(x, t, w, gh, top=6)
        dx2 = lp.row_logprobs_bwd(x, t, r.stats, w, gh)
    for k in range(4):
        x.copy_(torch.randn(M, V, generator=g, device=DEV).to(x.dtype))
        graph.replay()
        want = lp.row_logprobs_grad(x, t, w, gh, top=6)
        want2 = lp.row_logprobs_bwd(x, t, want[0].stats, w, gh)
        torch.cuda.synchronize()
        assert torch.equal(dx, want[1]) and torch.equal(dx2, want2)
        assert all(torch.equal(a, b) for a, b in zip(r, want[0]))


def test_given_outputs():
    """out=: the given tensors hold what new ones would, the fields left out nothing; wrong ones are refused."""
    x, t, g, _ = rows_of(6, 333, torch.bfloat16)
    w = torch.randn(6, generator=g, device=DEV)
    want = lp.row_logprobs(x, t, top=4)
    out = lp.RowLogprobs(*[torch.zeros_like(v) for v in want])
    assert lp.row_logprobs(x, t, top=4, out=out) is out and all(torch.equal(a, b) for a, b in zip(out, want))
    few = lp.RowLogprobs(None, torch.zeros(6, device=DEV), None, None, None, None)
    _, dx = lp.row_logprobs_grad(x, t, w, out=few)
    assert torch.equal(few.entropy, want.entropy) and torch.equal(dx, lp.row_logprobs_grad(x, t, w)[1])
    none = few._replace(entropy=None)
    assert torch.equal(lp.row_logprobs_grad(x, t, w, out=none)[1], dx)
    for bad, top in ((out, 0), (out, 3), (few, 2), (few._replace(top_ids=out.top_ids), 4), (few._replace(lse=w[:5]), 0),
                     (few._replace(lse=w.double()), 0), (few._replace(lse=w.cpu()), 0), (few._replace(stats=out.stats[:, :2]), 0)):
        with pytest.raises(ValueError, match="out"):
            lp.row_logprobs(x, t, top=top, out=bad)
    with pytest.raises(ValueError, match="out.logp"):
        lp.row_logprobs(x, None, out=few._replace(logp=w))


def test_written_tensors_are_known_to_autograd():
    """A graph that saved the logits refuses to use them after a gradient in their place."""
    x, t, g, _ = rows_of(4, 50, torch.float32)
    w = torch.randn(4, generator=g, device=DEV)
    leaf = x.clone().requires_grad_()
    z = leaf * 1.0
    loss, kept = z.square().sum(), z.detach()
    out = lp.RowLogprobs(None, w.clone(), None, None, None, None)
    versions = z._version, out.entropy._version
    lp.row_logprobs_grad(kept, t, w, dlogits=kept, out=out)
    assert z._version > versions[0] and out.entropy._version > versions[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_no_rows():
    x = torch.zeros(0, 10, device=DEV)
    t = torch.zeros(0, dtype=torch.int64, device=DEV)
    r, dx = lp.row_logprobs_grad(x, t, torch.zeros(0, device=DEV), top=3)
    assert r.logp.shape == (0,) and r.top_ids.shape == (0, 3) and dx.shape == (0, 10)
    logp, ent = lp.token_logprobs(torch.zeros(2, 0, 10, device=DEV, requires_grad=True), torch.zeros(2, 0, dtype=torch.int64, device=DEV))
    assert logp.shape == (2, 0)
    r = lp.row_logprobs(torch.zeros(10, device=DEV), torch.tensor(3, device=DEV), top=2)      # one row, no leading dims
    assert r.logp.shape == () and r.top_ids.tolist() == [0, 1]


def test_refusals():
    x, t, g, _ = rows_of(4, 100, torch.float32)
    w = torch.ones(4, device=DEV)
    bad = [lambda: lp.row_logprobs(x, t, top=33), lambda: lp.row_logprobs(x, t, top=-1), lambda: lp.row_logprobs(x[:, :5], t, top=6),
           lambda: lp.row_logprobs(x, t.int()), lambda: lp.row_logprobs(x, t[:3]), lambda: lp.row_logprobs(x, t.cpu()),
           lambda: lp.row_logprobs(x.cpu(), t.cpu()), lambda: lp.row_logprobs(x.t(), torch.zeros(100, dtype=torch.int64, device=DEV)),
           lambda: lp.row_logprobs(x[:1].expand(4, 100), t), lambda: lp.row_logprobs(x[:, :0], t),
           lambda: lp.row_logprobs(x.half(), t), lambda: lp.row_logprobs_grad(x, t, None), lambda: lp.row_logprobs_grad(x, None, w),
           lambda: lp.row_logprobs_grad(x, t, w.double()), lambda: lp.row_logprobs_grad(x, t, w, dlogits=x.bfloat16()),
           lambda: lp.row_logprobs_grad(x, t, w, dlogits=torch.empty(4, 101, device=DEV)),
           lambda: lp.row_logprobs_bwd(x, t, lp.row_logprobs(x[:3], t[:3]).stats, w), lambda: lp.row_logprobs_bwd(x, t, w, w),
           lambda: lp.row_logprobs(torch.zeros(2, 3, 8, device=DEV).transpose(0, 1), torch.zeros(3, 2, dtype=torch.int64, device=DEV))]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, NotImplementedError)):
            f()
            pytest.fail(f"call {i} was not refused")
    leaf = x.clone().requires_grad_()
    for f in (lambda: lp.row_logprobs(leaf, t), lambda: lp.row_logprobs_grad(leaf, t, w, dlogits=leaf)):
        with pytest.raises(NotImplementedError, match="token_logprobs"):
            f()
    with torch.no_grad():
        assert not lp.row_logprobs(leaf, t).logp.requires_grad
    wide = torch.zeros(4, 200, device=DEV)
    with pytest.raises(L.DMError, match="overlaps"):
        lp.row_logprobs_grad(wide[:, :100], t, w, dlogits=wide[:, 50:150])

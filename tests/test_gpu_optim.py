"""optim.AdamW (dm_adamw_step, dm_grad_norm, dm_adamw_values) against the definitions in 64 bits, and its 8-bit codes
against the same arithmetic in numpy, bit for bit.

Tolerances count roundings (u = 2^-24): m = b1 m + c1 (c g): a rounded constant and a product per term, one more each
for c and c g, and the sum: u (3 |b1 m| + 5 |c1 c g|); v: u (3 b2 v + 8 c2 (c g)^2); p: see ``p_bound``."""

import math

import numpy as np
import pytest
import torch

from dual_mod_public_amd import _lib as L
from dual_mod_public_amd.optim import AdamW
from tests.hip_helpers import DEV, say

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
B1, B2, EPS, LR = 0.9, 0.999, 1e-8, 3e-3


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    L.load()


def make(sizes, g_dtype=torch.float32, seed=0, shift=0, scale=1e-2):
    """Parameters and gradients of these sizes as views at odd places (shift elements from an aligned one) of buffers with
    poison between; two groups."""
    g = torch.Generator(device=DEV).manual_seed(seed + sum(sizes))
    n = sum(sizes) + (len(sizes) + 1) * (shift + 4)
    P, G = torch.full((n,), 1e3, device=DEV), torch.full((n,), 1e3, device=DEV, dtype=g_dtype)
    ps, gs, at = [], [], 0
    for k in sizes:
        at += -at % 4 + shift
        ps.append(P[at:at + k])
        gs.append(G[at:at + k])
        ps[-1].copy_(torch.randn(k, generator=g, device=DEV))
        gs[-1].copy_((scale * torch.randn(k, generator=g, device=DEV)).to(g_dtype))
        at += k
    half = len(ps) // 2
    groups = [dict(params=ps[:half], weight_decay=0.1), dict(params=ps[half:], weight_decay=0.0, lr_scale=0.5)]
    return ps, gs, groups, P, G


def hyper(i, n):
    """(weight decay, lr_scale) of tensor i of n."""
    return (0.1, 1.0) if i < n // 2 else (0.0, 0.5)


def coef_of(gs, max_norm):
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
    return (min(1.0, max_norm / (norm + 1e-6)) if max_norm else 1.0), norm


def p_bound(p, wd, ls, m, v, dm, dv, t):
    """The bound of p's error, and p itself, from m and v (64 bits) with errors dm, dv."""
    rate, s2 = LR * ls / (1 - B1 ** t), 1 / math.sqrt(1 - B2 ** t)
    denom = v.sqrt() * s2 + EPS
    dden = s2 * (((v + dv).sqrt() - v.sqrt()) + 4 * U * v.sqrt()) + 2 * U * denom
    upd = rate * m / denom
    want = p * (1 - LR * ls * wd) - upd
    # rate is three roundings (lr, the quotient, lr_scale), the division and the product five more
    return want, U * (3 * p.abs() + want.abs()) + rate * dm / denom + upd.abs() * (dden / denom + 10 * U)


# lengths around a wave's block, a launched block, and odd ones; empty tensors between
SIZES = [[1], [3, 0, 255, 256, 257, 1000], [4095, 4096, 4097, 1, 12289], [70001, 5, 512]]


@pytest.mark.parametrize("g_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("max_norm", [None, 0.05, 1e6])
@pytest.mark.parametrize("sizes", SIZES)
def test_step32(sizes, max_norm, g_dtype):
    for shift in (0, 1, 3):
        ps, gs, groups, P, G = make(sizes, g_dtype, shift=shift)
        before = P.clone()
        inside = torch.zeros_like(P, dtype=torch.bool)
        for p in ps:
            inside[p.storage_offset():p.storage_offset() + p.numel()] = True
        opt = AdamW(groups, grads=gs, lr=LR, betas=(B1, B2), eps=EPS, max_norm=max_norm)
        ref = [[p.double().cpu(), torch.zeros(p.numel(), dtype=torch.float64), torch.zeros(p.numel(), dtype=torch.float64)] for p in ps]
        for t in (1, 2, 3):
            c, norm = coef_of(gs, max_norm)
            got = opt.step()
            assert (got is None) == (max_norm is None)
            if got is not None:
                assert abs(float(got) - norm) <= U * norm * 1.001
            for i, (p, g, r) in enumerate(zip(ps, gs, ref)):
                gc = c * g.double().cpu()
                dm = U * (3 * (B1 * r[1]).abs() + 5 * ((1 - B1) * gc).abs())
                dv = U * (3 * B2 * r[2] + 8 * (1 - B2) * gc * gc)
                r[1], r[2] = B1 * r[1] + (1 - B1) * gc, B2 * r[2] + (1 - B2) * gc * gc
                m, v = (opt.views(s)[i].double().cpu() for s in (opt.exp_avg, opt.exp_avg_sq))
                assert ((m - r[1]).abs() <= dm).all() and ((v - r[2]).abs() <= dv + 1e-44).all(), (t, i)
                want, tol = p_bound(r[0], *hyper(i, len(ps)), r[1], r[2], dm, dv, t)
                assert ((p.double().cpu() - want).abs() <= tol).all(), (t, i)
                r[0], r[1], r[2] = p.double().cpu(), m, v       # the next step from what is there
            for g in gs:
                g.copy_((g.float() * 0.7 - 1e-3).to(g.dtype))
        assert int(opt.steps) == 3 and torch.equal(P[~inside], before[~inside])


# ---- 8-bit states ---------------------------------------------------------------------------------------------------

def mix(x):
    x = x.astype(np.uint32).copy()
    x ^= x >> np.uint32(16)
    x *= np.uint32(0x9E3779B1)
    x ^= x >> np.uint32(13)
    x *= np.uint32(0xBB67AE85)
    return x ^ (x >> np.uint32(16))


G32 = np.uint32(0x9E3779B1)


def hashes(seed, t, block0, blocks):
    with np.errstate(over="ignore"):
        key = mix(np.array([seed], np.uint32) + np.array([t], np.uint32) * G32)
        key = mix(key + (block0 + np.arange(blocks, dtype=np.uint32)) * G32)
        return mix(key[:, None] + np.arange(256, dtype=np.uint32)[None] * G32)


def value(code, e, second):
    """The numbers of codes [blocks, 256] with block exponents e [blocks], in 64 bits."""
    code = code.astype(np.int64)
    neg, c = (code * 0, code) if second else (code >> 7, code & 127)
    E, M, low = c >> 3, c & 7, -31 if second else -15
    a = np.where(E > 0, np.ldexp(1 + M / 8, E + low - 1), np.ldexp(M / 8, low))
    return np.where(e[:, None] == 255, np.nan, np.ldexp(a, e[:, None].astype(np.int64) - 125) * np.where(neg, -1, 1))


def code_of(x, r, second):
    """Codes and block exponents of x [blocks, 256] (fp32), rounded by the hashes r, in exact arithmetic."""
    mag = np.abs(x)
    e = np.maximum(mag.max(1).view(np.uint32) >> 23, 1).astype(np.int64)
    low, r16 = (-31, r >> 16) if second else (-15, r & 0xffff)
    frac = (r16.astype(np.float64) * 16 + 8) / 2 ** 20
    a = np.ldexp(mag.astype(np.float64), (125 - e)[:, None])
    E = np.where(a == 0, low, np.maximum(np.frexp(a)[1] - 1, low))           # the binade, the lowest one at least
    code = np.floor(np.ldexp(a, 3 - E) + frac).astype(np.int64) + 8 * (E - low)   # 0..16 steps of it, 8 per one below
    if second:
        code = np.where((mag > 0) & (code == 0), 1, code)
    else:
        code = np.where((x < 0) & (code > 0), code + 128, code)
    return code.astype(np.uint8), e.astype(np.uint8)


def blocks_of(x, n):
    out = np.zeros(-(-n // 256) * 256, np.float32)
    out[:n] = x
    return out.reshape(-1, 256)


@pytest.mark.parametrize("g_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("max_norm", [None, 0.05])
@pytest.mark.parametrize("sizes", SIZES)
def test_step8(sizes, max_norm, g_dtype):
    """Three steps: the codes equal numpy's in every bit, the parameters 64-bit ones."""
    ps, gs, groups, P, _ = make(sizes, g_dtype, shift=1)
    gs[0][:: 2] = 0
    gs[-1] *= torch.logspace(-6, 3, gs[-1].numel(), device=DEV).to(g_dtype)     # every code, and blocks of one value
    opt = AdamW(groups, grads=gs, lr=LR, betas=(B1, B2), eps=EPS, max_norm=max_norm, state_bits=8, seed=77)
    nb = opt.n_blocks
    codes = [(np.zeros((nb, 256), np.uint8), np.ones(nb, np.uint8)) for _ in range(2)]
    f32 = np.float32
    for t in (1, 2, 3):
        c, _ = coef_of(gs, max_norm)
        p0 = [p.double().cpu() for p in ps]
        opt.step()
        m_all, v_all = (value(*codes[k], k == 1).astype(f32) for k in (0, 1))
        for i, (p, g) in enumerate(zip(ps, gs)):
            n, b = p.numel(), opt._block0[i]
            if n == 0:
                continue
            rows = slice(b, b - (-n // 256))
            gc = blocks_of(g.float().cpu().numpy(), n) * f32(c)
            m = m_all[rows] * f32(B1) + gc * f32(1 - B1)
            v = v_all[rows] * f32(B2) + (gc * gc) * f32(1 - B2)
            r = hashes(77, t, b, m.shape[0])
            for k, x in ((0, m), (1, v)):
                codes[k][0][rows], codes[k][1][rows] = code_of(x, r, k == 1)
            wd, ls = hyper(i, len(ps))
            m64, v64 = (torch.from_numpy(x.reshape(-1)[:n].astype(np.float64)) for x in (m, v))
            want, tol = p_bound(p0[i], wd, ls, m64, v64, 0 * m64, 0 * v64, t)
            assert ((p.double().cpu() - want).abs() <= tol).all(), (t, i)
        for k, (have, exps) in enumerate(((opt.exp_avg, opt.exp_avg_exponent), (opt.exp_avg_sq, opt.exp_avg_sq_exponent))):
            assert np.array_equal(exps.cpu().numpy(), codes[k][1]), (t, k)
            assert np.array_equal(have.view(nb, 256).cpu().numpy(), codes[k][0]), (t, k)
        for k, x in enumerate(opt.state_values()):
            assert np.array_equal(x.float().cpu().numpy().reshape(nb, 256), value(*codes[k], k == 1).astype(f32))


def test_every_code_has_its_value():
    codes = torch.arange(256, device=DEV, dtype=torch.uint8).repeat(254)
    e = torch.cat([torch.arange(1, 254), torch.tensor([255])]).to(DEV, torch.uint8)
    for second in (0, 1):
        out = torch.empty(codes.numel(), device=DEV, dtype=torch.bfloat16)
        L.check(L.lib().dm_adamw_values(codes.data_ptr(), e.data_ptr(), 254, second, out.data_ptr(), L.stream_ptr()))
        want = torch.from_numpy(value(codes.view(254, 256).cpu().numpy(), e.cpu().numpy(), second == 1).reshape(-1))
        got = out.double().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        fine = ~torch.isnan(want)
        # exact down to bf16's smallest number, half of it off below
        assert ((got - want).abs()[fine] <= torch.where(want.abs() >= 2.0 ** -126, 0.0, 2.0 ** -134 * 1.01)[fine]).all()


def test_second_moment_follows_its_average():
    """Stochastic rounding keeps the mean: 300 steps of decay to nothing (each 0.1%, a code an eighth) leave b2^300 of v on
    average. An element's relative step has variance at most (change) (code) = 0.001 * 0.125; over 300 steps, with
    N independent elements, six sigma of the mean are 6 sqrt(300 * 0.001 * 0.125 / N) of v."""
    N = 1 << 16
    p, g = torch.zeros(N, device=DEV), torch.zeros(N, device=DEV)
    opt = AdamW([p], grads=[g], lr=0.0, betas=(B1, B2), weight_decay=0.0, state_bits=8, seed=5)
    g.copy_(1.0 + torch.rand(N, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV))
    opt.step()
    v0 = opt.state_values()[1].double().mean()
    g.zero_()
    for _ in range(300):
        opt.step()
    v = opt.state_values()[1].double().mean()
    want = v0 * B2 ** 300
    say(f"mean second moment after 300 steps of decay: {float(v / want):.5f} of the exact one")
    assert abs(v / want - 1) <= 6 * math.sqrt(300 * 0.001 * 0.125 / N) * 1.4      # 1.4: v's spread over its elements, at most
    assert (opt.state_values()[1] > 0).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_not_finite(bits):
    """A NaN gradient reaches its own element (8 bits: its block's states), through the norm everything; skip_nonfinite
    leaves the whole step out."""
    for bad in (float("nan"), float("inf")):
        ps, gs, groups, P, _ = make([1000, 300])
        opt = AdamW(groups, grads=gs, lr=LR, state_bits=bits)
        opt.step()
        keep = gs[0][300].clone()
        gs[0][300] = bad
        opt.step()
        nan = torch.isnan(ps[0])
        assert nan.nonzero().flatten().tolist() == [300] and not torch.isnan(ps[1]).any()
        m, v = (opt.views(s)[0].float() for s in opt.state_values())
        hit = torch.zeros(1000, dtype=torch.bool, device=DEV)
        hit[300 if bits == 32 else slice(256, 512)] = True
        if bits == 32:
            assert not torch.isfinite(m[300]) and torch.isfinite(m[~hit]).all() and torch.isfinite(v[~hit]).all()
        else:
            assert torch.equal(torch.isnan(m), hit) and torch.equal(torch.isnan(v), hit)
        opt = AdamW(groups, grads=gs, lr=LR, max_norm=1.0, state_bits=bits)
        ps[0][300] = 0
        opt.step()
        assert torch.isnan(ps[0]).any() if math.isinf(bad) else torch.isnan(P[:1000]).any()

        ps, gs, groups, P, _ = make([1000, 300])
        opt = AdamW(groups, grads=gs, lr=LR, max_norm=1.0, skip_nonfinite=True, state_bits=bits)
        opt.step()
        state = [P.clone()] + [t.clone() for t in (opt.exp_avg, opt.exp_avg_sq, opt.steps)]
        gs[0][300] = bad
        norm = opt.step()
        assert not math.isfinite(float(norm)) and int(opt.skipped) == 1
        assert all(torch.equal(a, b) for a, b in zip(state, (P, opt.exp_avg, opt.exp_avg_sq, opt.steps)))
        gs[0][300] = keep
        opt.step()
        assert int(opt.steps) == 2 and int(opt.skipped) == 1 and torch.isfinite(ps[0]).all()


def test_norm_alone():
    for sizes, g_dtype in (([1], torch.float32), ([5000, 0, 77, 4096 * 1500 + 3], torch.bfloat16), ([3, 9, 1 << 20], torch.float32)):
        ps, gs, groups, P, _ = make(sizes, g_dtype, shift=1)
        before = P.clone()
        opt = AdamW(groups, grads=gs)
        norm = coef_of(gs, None)[1]
        assert abs(float(opt.grad_norm()) - norm) <= U * norm * 1.001
        assert torch.equal(P, before) and int(opt.steps) == 0
        for g in gs:
            g.zero_()
        assert float(opt.grad_norm()) == 0
        gs[-1].fill_(1e30)                            # squares past fp32's range
        norm = coef_of(gs, None)[1]
        assert abs(float(opt.grad_norm()) - norm) <= U * norm * 1.001


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_own_gradients(bits):
    """Without ``grads``: .grad at each step, wherever it lies then; a parameter without one stays as it is."""
    a, b, c = (torch.nn.Parameter(torch.randn(n, device=DEV)) for n in (300, 70, 5))
    copy = [p.detach().clone().requires_grad_() for p in (a, b, c)]
    opt = AdamW([a, b, c], lr=LR, state_bits=bits, seed=3)
    fixed = [torch.zeros_like(p) for p in copy]
    opt2 = AdamW(copy, grads=fixed, lr=LR, state_bits=bits, seed=3, weight_decay=0.01)
    with pytest.raises(ValueError, match="no parameter has a gradient"):
        opt.step()
    keep = []
    for k in range(3):
        for p, f in zip((a, b, c), fixed):
            f.normal_(generator=torch.Generator(device=DEV).manual_seed(10 * k + p.numel()))
            p.grad = f.clone()
            keep.append(p.grad)                      # each step's gradients elsewhere
        version = a._version
        opt.step()
        opt2.step()
        assert a._version > version
        assert all(torch.equal(p, q) for p, q in zip((a, b, c), copy))
    b.grad = None
    before = b.detach().clone()
    states = [s.clone() for s in opt.state_values()]
    opt.step()
    assert torch.equal(b, before) and not torch.equal(a, copy[0])
    for s, t in zip(states, opt.state_values()):
        assert torch.equal(opt.views(s)[1], opt.views(t)[1])
    a.grad = torch.zeros(600, device=DEV)[::2]
    with pytest.raises(ValueError, match="gradient 0"):
        opt.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step(bits):
    """Replays with new gradients, another learning rate and eager steps between equal an eager optimizer's steps."""
    runs = []
    for captured in (False, True):
        ps, gs, groups, P, _ = make([3000, 17, 260])
        opt = AdamW(groups, grads=gs, lr=LR, max_norm=0.1, state_bits=bits, seed=9)
        opt.step()
        if captured:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
                norm = opt.step()
        seen = []
        for k in range(6):
            for g in gs:
                g.mul_(0.9).add_(1e-3)
            if k == 3:
                opt.set_lr(LR / 3)
            if captured and k != 4:
                version = ps[0]._version
                graph.replay()
                opt.mark_updated()
                assert ps[0]._version > version
            else:
                norm = opt.step()
            torch.cuda.synchronize()
            seen.append((P.clone(), norm.clone(), opt.exp_avg.clone(), opt.exp_avg_sq.clone(), opt.steps.clone()))
        runs.append(seen)
    for a, b in zip(*runs):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_grad_of_another_order_at_an_old_address():
    """A .grad that is new in the place of an old one is looked at again: strides that are not rows are refused."""
    p = torch.nn.Parameter(torch.ones(8, 8, device=DEV))
    p.grad = torch.arange(64.0, device=DEV).view(8, 8)
    opt = AdamW([p], lr=0.5, weight_decay=0.0)
    opt.step()
    before = p.detach().clone()
    p.grad = p.grad.t()
    with pytest.raises(ValueError, match="gradient 0"):
        opt.step()
    assert torch.equal(p.detach(), before)
    p.grad = p.grad.t()
    opt.step()
    assert not torch.equal(p.detach(), before) and int(opt.steps) == 2


def test_old_graph_after_parameters_moved():
    """A captured step keeps writing the storage that it was captured with, which stays allocated."""
    p = torch.nn.Parameter(torch.ones(1000, device=DEV))
    opt = AdamW([p], grads=[torch.ones(1000, device=DEV)], lr=0.5, weight_decay=0.0)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    old = p.data_ptr()
    p.data = p.data.clone()
    opt.step()
    others = [torch.zeros(1000, device=DEV) for _ in range(64)]
    assert old not in [t.data_ptr() for t in others]
    kept = p.detach().clone()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(p.detach(), kept) and not any(bool(t.any()) for t in others)


def test_capture_needs_a_plan():
    p = torch.nn.Parameter(torch.ones(10, device=DEV))
    opt = AdamW([p])
    p.grad = torch.ones(10, device=DEV)
    opt.step()
    first = opt._plan
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        opt.step()
    kept = p.grad
    p.grad = torch.full((10,), 2.0, device=DEV)       # the eager step's plan is another; the graph keeps its own
    opt.step()
    assert opt._plan is not first and any(t is first for t in opt._in_graphs)
    before = p.detach().clone()
    graph.replay()
    torch.cuda.synchronize()
    assert kept.sum() == 10 and not torch.equal(p, before) and int(opt.steps) == 3
    p.grad = torch.full((10,), 3.0, device=DEV)
    with pytest.raises(RuntimeError, match="moved"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=torch.cuda.Stream()):
            opt.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_continues(bits):
    ps, gs, groups, P, _ = make([3000, 17])
    opt = AdamW(groups, grads=gs, lr=LR, state_bits=bits, seed=4)
    opt.step()
    opt.step()
    saved = {k: v.clone() if torch.is_tensor(v) else v for k, v in opt.state_dict().items()}
    p0 = P.clone()
    opt.step()
    want = P.clone()
    P.copy_(p0)
    opt2 = AdamW(groups, grads=gs, lr=1.0, state_bits=bits, seed=4)
    opt2.load_state_dict(saved)
    opt2.step()
    assert torch.equal(P, want) and int(opt2.steps) == 3
    with pytest.raises(ValueError):
        AdamW(groups, grads=gs, state_bits=40 - bits).load_state_dict(saved)
    with pytest.raises(ValueError):
        AdamW(ps[:1], grads=gs[:1], state_bits=bits).load_state_dict(saved)


@pytest.mark.parametrize("bits", [32, 8])
def test_elements_past_32_bits(bits):
    """A tensor of more than 2^31 elements: its first and last ones are updated as a short tensor's."""
    n = (1 << 31) + 777
    p, g = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV, dtype=torch.bfloat16)
    ends = [slice(0, 300), slice(n - 300, n)]
    for s in ends:
        p[s] = torch.linspace(-1, 1, 300, device=DEV)
        g[s] = torch.linspace(-2, 1, 300, device=DEV).bfloat16()
    small = p[ends[1]].clone()
    opt = AdamW([p], grads=[g], lr=LR, max_norm=1.0, state_bits=bits)
    other = AdamW([small], grads=[g[ends[1]].clone()], lr=LR)
    norm = math.sqrt(sum(float(g[s].double().square().sum()) for s in ends))
    got = opt.step()
    assert abs(float(got) - norm) <= U * norm * 1.001
    other.step()
    # the first step moves by lr g / (|g| + eps / c): the clipping cancels but for eps, below 1e-6 of it
    for s in ends:
        assert ((p[s] - small).abs() <= LR * 1e-4 + 4 * U).all()
    m, v = opt.state_values()
    assert (m[n - 100:n] != 0).all() and (v[n - 100:n] != 0).any() and float(p[300:n - 300].abs().max()) == 0


def test_other_stream():
    ps, gs, groups, P, _ = make([5000, 3])
    ps2, gs2, groups2, P2, _ = make([5000, 3])
    a = AdamW(groups, grads=gs, lr=LR, max_norm=0.1)
    b = AdamW(groups2, grads=gs2, lr=LR, max_norm=0.1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    a.step()
    with torch.cuda.stream(s):
        b.step()
    s.synchronize()
    assert torch.equal(P, P2)


def test_refusals():
    p = torch.zeros(10, device=DEV)
    bad = [lambda: AdamW([p.bfloat16()]), lambda: AdamW([torch.zeros(4, 4, device=DEV).t()]), lambda: AdamW([p, p]),
           lambda: AdamW([p[:6], p[5:]]), lambda: AdamW([p], grads=[p[:9]]), lambda: AdamW([p], grads=[p.cpu()]),
           lambda: AdamW([p], grads=[torch.zeros(20, device=DEV)[::2]]), lambda: AdamW([p], grads=[p, p]),
           lambda: AdamW([p, torch.zeros(3)]), lambda: AdamW([p], grads=[p.half()])]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, NotImplementedError)):
            f()
            pytest.fail(f"call {i} was not refused")
    # a group's parameters may be an iterator or one tensor
    opt = AdamW([dict(params=(t for t in (p[:3], p[3:])), weight_decay=0.5), dict(params=torch.zeros(4, device=DEV))])
    assert len(opt.params) == 3 and opt._decay == [0.5, 0.5, 0.01] and opt._scale == [1.0] * 3
    q = torch.zeros(10, device=DEV)
    AdamW([p[:5], p[5:]], grads=[q[:5], q[:5]])       # neighbours are not overlaps, and gradients may be shared
    both = torch.zeros(20, device=DEV)
    AdamW([both[:10]], grads=[both[10:]])
    for g in (both[:10], both[9:19]):
        with pytest.raises(ValueError, match="shares memory"):
            AdamW([both[:10]], grads=[g])

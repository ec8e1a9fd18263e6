"""The optimizer where a program changes beneath it: parameters that grow, gradients that come late or go while a captured
step lives, very small moments, states of another model. Bounds as in test_gpu_optim.py."""

import math

import pytest
import torch

from dual_mod_public_amd import _lib as L
from dual_mod_public_amd.optim import AdamW
from tests.hip_helpers import DEV
from tests.test_gpu_optim import B1, B2, EPS, LR, U, p_bound

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    L.load()


def noise(n, seed):
    return torch.randn(n, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


@pytest.mark.parametrize("bits", [32, 8])
def test_parameter_of_another_size(bits):
    """The states are laid out once: a parameter that holds another number of elements later is refused, and nothing
    is written."""
    a, b = (torch.nn.Parameter(noise(n, n)) for n in (300, 700))
    opt = AdamW([a, b], lr=LR, state_bits=bits)
    a.grad, b.grad = torch.ones(300, device=DEV), torch.ones(700, device=DEV)
    opt.step()
    kept = b.detach().clone()
    for n in (5000, 100):
        a.grad = None
        a.data = noise(n, 1)
        a.grad = torch.ones(n, device=DEV)
        with pytest.raises(ValueError, match="parameter 0"):
            opt.step()
        with pytest.raises(ValueError, match="parameter 0"):
            opt.grad_norm()
    assert torch.equal(b.detach(), kept) and int(opt.steps) == 1
    a.grad = None
    a.data = noise(300, 2)
    both = torch.ones(300, device=DEV)
    a.grad = both
    opt.step()
    a.grad = None
    a.data = a.data[:100]                            # fewer elements at the old address, and their gradient too
    a.grad = both[:100]
    with pytest.raises(ValueError, match="parameter 0"):
        opt.step()
    assert int(opt.steps) == 2
    a.grad = None
    a.data = noise(300, 2).view(20, 15)              # another shape of as many elements is laid out the same
    a.grad = torch.ones(20, 15, device=DEV)
    opt.step()
    assert int(opt.steps) == 3


def test_captured_gradients_stay():
    """A captured step reads the gradients that it was captured with; they stay allocated when the parameters let go of
    them."""
    p, q = (torch.nn.Parameter(torch.zeros(n, device=DEV)) for n in (1000, 50))
    opt = AdamW([p, q], lr=0.5, weight_decay=0.0, betas=(0.0, B2), max_norm=1e6)
    p.grad, q.grad = torch.ones(1000, device=DEV), torch.ones(50, device=DEV)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        norm = opt.step()
    held = {p.grad.data_ptr(), q.grad.data_ptr()}
    p.grad = None
    q.grad = None
    others = [torch.full((n,), -7.0, device=DEV) for n in (1000, 50) for _ in range(64)]
    assert not held & {t.data_ptr() for t in others}
    graph.replay()
    torch.cuda.synchronize()
    assert abs(float(norm) - math.sqrt(1050)) <= 1e-5 * math.sqrt(1050)
    # three steps against gradients of 1, the second captured but not run: two of them in all
    assert (p + 1.0).abs().max() <= 1e-5 and (q + 1.0).abs().max() <= 1e-5
    # a later plan's gradients are not kept by the graph's
    p.grad, q.grad = torch.ones(1000, device=DEV), torch.ones(50, device=DEV)
    opt.step()
    assert int(opt.steps) == 3


def _follow(opt, params, counts, decay):
    """One step, every parameter against 64-bit AdamW with its own step count (counts, advanced here)."""
    before = [p.detach().double().cpu() for p in params]
    m0, v0 = ([t.double().cpu().flatten() for t in opt.views(s)] for s in opt.state_values())
    opt.step()
    m1, v1 = ([t.double().cpu().flatten() for t in opt.views(s)] for s in opt.state_values())
    for i, p in enumerate(params):
        if p.grad is None:
            assert torch.equal(p.detach().double().cpu(), before[i]) and torch.equal(m1[i], m0[i]) and torch.equal(v1[i], v0[i])
            continue
        counts[i] += 1
        g = p.grad.double().cpu()
        m, v = B1 * m0[i] + (1 - B1) * g, B2 * v0[i] + (1 - B2) * g * g
        dm = U * (3 * (B1 * m0[i]).abs() + 5 * ((1 - B1) * g).abs())
        dv = U * (3 * B2 * v0[i] + 8 * (1 - B2) * g * g)
        want, tol = p_bound(before[i], decay, 1.0, m, v, dm, dv, counts[i])
        assert ((p.detach().double().cpu() - want).abs() <= tol).all(), (i, counts)
        if opt.state_bits == 32:
            assert ((m1[i] - m).abs() <= dm).all() and ((v1[i] - v).abs() <= dv + 1e-44).all()
    assert opt.tensor_steps.tolist() == counts


@pytest.mark.parametrize("bits", [32, 8])
def test_gradient_first_appears_later(bits):
    """A parameter's bias corrections count the steps that it took part in: one whose first gradient comes late moves by
    the learning rate as any other does, not by 0.1 / sqrt(0.001) of it; one that pauses goes on where it was."""
    params = [torch.nn.Parameter(noise(n, n)) for n in (300, 70, 5000, 1)]
    opt = AdamW(params, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=0.1, state_bits=bits, seed=3)
    counts = [0] * 4
    taking_part = ((0, 2), (0, 2), (0, 2, 3), (0, 1, 2), (1, 3), (0, 1, 2, 3), (1,), (0, 1, 2, 3))
    for k, who in enumerate(taking_part):
        for i, p in enumerate(params):
            p.grad = noise(p.numel(), 100 * k + i) if i in who else None
        _follow(opt, params, counts, 0.1)
    assert int(opt.steps) == len(taking_part) and counts == [6, 5, 6, 4]


def test_late_gradient_with_skipped_and_captured_steps():
    """Steps left out count for no parameter, replayed ones for those that the captured plan holds."""
    a, b = (torch.nn.Parameter(noise(n, n)) for n in (4100, 9))
    opt = AdamW([a, b], lr=LR, betas=(B1, B2), eps=EPS, weight_decay=0.0, skip_nonfinite=True)
    a.grad = torch.full((4100,), float("inf"), device=DEV)
    opt.step()
    assert opt.tensor_steps.tolist() == [0, 0] and int(opt.skipped) == 1
    counts = [0, 0]
    a.grad.fill_(0.5)
    _follow(opt, [a, b], counts, 0.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        opt.step()
    only_a = a.grad
    for k in range(3):
        graph.replay()
        counts[0] += 1
        a.grad, b.grad = noise(4100, k), noise(9, 10 + k)
        _follow(opt, [a, b], counts, 0.0)
        a.grad, b.grad = only_a, None
    assert counts == [7, 3] and int(opt.steps) == 7


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_keeps_the_counts(bits):
    def make():
        params = [torch.nn.Parameter(noise(n, n)) for n in (300, 70)]
        return params, AdamW(params, lr=LR, state_bits=bits, seed=3)

    (p, opt), (q, other) = make(), make()
    for k in range(3):
        p[0].grad, p[1].grad = noise(300, k), noise(70, k) if k == 2 else None
        opt.step()
    other.load_state_dict(opt.state_dict())
    assert other.tensor_steps.tolist() == [3, 1] and other.tensor_steps.data_ptr() != opt.tensor_steps.data_ptr()
    for a, b in zip(p, q):
        b.data.copy_(a.data)
        a.grad = noise(a.numel(), 7)
        b.grad = a.grad.clone()
    opt.step()
    other.step()
    assert all(torch.equal(a, b) for a, b in zip(p, q)) and other.tensor_steps.tolist() == [4, 2]
    # without the counts: every parameter took part in every step
    d = opt.state_dict()
    del d["tensor_steps"]
    other.load_state_dict(d)
    assert other.tensor_steps.tolist() == [4, 4] and int(other.steps) == 4
    with pytest.raises(ValueError, match="tensor_steps"):
        other.load_state_dict(dict(opt.state_dict(), tensor_steps=torch.zeros(3, dtype=torch.int64)))


def test_counts_of_many_tensors():
    """More tensors than the counting block has threads, every third of them from the second step on."""
    params = [torch.nn.Parameter(noise(1 + k % 3, k)) for k in range(700)]
    opt = AdamW(params, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=0.1)
    counts = [0] * 700
    for t in (1, 2):
        for k, p in enumerate(params):
            p.grad = noise(p.numel(), 1000 * t + k) if t == 2 or k % 3 else None
        _follow(opt, params, counts, 0.1)


@pytest.mark.parametrize("bits", [32, 8])
def test_without_counts_every_tensor_is_as_old(bits):
    """dm_adamw_step, which takes no counts: the step count is every tensor's."""
    runs = []
    for counts in (True, False):
        ps, gs = [noise(n, n) for n in (300, 5000)], [noise(n, n + 1) for n in (300, 5000)]
        opt = AdamW(ps, grads=gs, lr=LR, max_norm=0.5, state_bits=bits, seed=2)
        a = opt._args()
        if not counts:
            a.workspace_bytes = L.DM_ADAMW_WORKSPACE
        for _ in range(3):
            opt.step() if counts else L.check(L.lib().dm_adamw_step(L.byref(a), L.stream_ptr()))
        torch.cuda.synchronize()
        assert opt.tensor_steps.tolist() == ([3, 3] if counts else [0, 0]) and int(opt.steps) == 3
        runs.append(ps + [opt.exp_avg, opt.exp_avg_sq])
    assert all(torch.equal(x, y) for x, y in zip(*runs))


@pytest.mark.parametrize("eps", [1e-8, 1e-15, 1e-30, 2.0 ** -126])
def test_very_small_gradients(eps):
    """Second moments below fp32's normal numbers: their square root is as exact as any other's."""
    g = torch.logspace(-22, -15, 3000, device=DEV) * torch.where(noise(3000, 1) < 0, -1.0, 1.0)
    g[::5] = 0
    p = torch.zeros(3000, device=DEV)
    opt = AdamW([p], grads=[g], lr=LR, betas=(B1, B2), eps=eps, weight_decay=0.0)
    m, v = (torch.zeros(3000, dtype=torch.float64) for _ in range(2))
    for t in (1, 2):
        before = p.double().cpu()
        opt.step()
        g64 = g.double().cpu()
        # the square, its product with 1 - b2 and the product with b2 each round to a multiple of 2^-149 at best
        sub = 2.0 ** -150 * 3
        dm = U * (3 * (B1 * m).abs() + 5 * ((1 - B1) * g64).abs())
        dv = U * (3 * B2 * v + 8 * (1 - B2) * g64 * g64) + sub
        m, v = B1 * m + (1 - B1) * g64, B2 * v + (1 - B2) * g64 * g64
        have_m, have_v = opt.exp_avg.double().cpu()[:3000], opt.exp_avg_sq.double().cpu()[:3000]
        assert ((have_m - m).abs() <= dm).all() and ((have_v - v).abs() <= dv).all()
        # the update of the moments that are there: a square root, a quotient and a few products
        rate, s2 = LR / (1 - B1 ** t), 1 / math.sqrt(1 - B2 ** t)
        denom = have_v.sqrt() * s2 + eps
        upd = rate * have_m / denom
        assert ((p.double().cpu() - (before - upd)).abs() <= U * (16 * upd.abs() + 4 * before.abs()) + 2.0 ** -149).all(), t
        m, v = have_m, have_v


@pytest.mark.parametrize("bits", [32, 8])
def test_state_of_other_parameters(bits):
    """States of parameters of other sizes or another order are refused, also where they fill as many blocks."""
    def make(*sizes, seed=0):
        params = [torch.zeros(n, device=DEV) for n in sizes]
        return params, AdamW(params, grads=[noise(n, n) for n in sizes], lr=LR, state_bits=bits, seed=seed)

    _, opt = make(100, 300)
    opt.step()
    saved = opt.state_dict()
    for sizes in ((300, 100), (101, 300), (100, 300, 0)):
        other = make(*sizes)[1]
        assert other.exp_avg.shape == opt.exp_avg.shape
        with pytest.raises(ValueError, match="sizes"):
            other.load_state_dict(saved)
        assert int(other.steps) == 0 and not other.exp_avg.any()
    _, other = make(100, 300)
    other.load_state_dict({k: v for k, v in saved.items() if k not in ("sizes", "seed")})    # states without them
    assert torch.equal(other.exp_avg, opt.exp_avg) and other.seed == 0


def test_state_keeps_the_seed():
    """The rounding's seed belongs to the states: a run that is taken up again repeats bit for bit."""
    def make(seed):
        p = torch.zeros(1000, device=DEV)
        return p, AdamW([p], grads=[noise(1000, 5)], lr=LR, state_bits=8, seed=seed)

    (p, opt), (q, other) = make(11), make(0)
    opt.step()
    other.step()                                      # its plan is there already
    other.load_state_dict(opt.state_dict())
    q.copy_(p)
    for _ in range(2):
        opt.step()
        other.step()
    assert torch.equal(p, q) and torch.equal(opt.exp_avg, other.exp_avg) and torch.equal(opt.exp_avg_sq, other.exp_avg_sq)

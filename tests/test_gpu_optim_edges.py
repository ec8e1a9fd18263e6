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

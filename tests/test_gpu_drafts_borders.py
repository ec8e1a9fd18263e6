"""verify_drafts where a random number lies within 10^-12 of the border that it is compared with."""

import numpy as np
import pytest
import torch

from dual_mod_public_amd import _lib as L
from dual_mod_public_amd.drafts import verify_drafts
from tests.hip_helpers import DEV, say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    L.load()


def cases(T, seed, n=4_000_000):
    """(x, u, u < p) with p = 1 / (1 + e^(x / T)) and u, both fp32, relatively 2 10^-14 to 10^-12 apart: by 64 significant bits. (A
    difference of a few units of 2^-53 times 1 + |x / T| may be any correct computation's in 64 bits: 2 10^-15 here.)"""
    rng = np.random.default_rng(seed)
    x = (rng.uniform(-6, 3, n) * T).astype(np.float32)
    t = np.float64(np.float32(T))
    p = 1 / (1 + np.exp(x.astype(np.float64) / t))
    near = p.astype(np.float32)
    close = np.abs(near - p) < 4e-12 * p
    x, near = x[close], near[close]
    exact = 1 / (1 + np.exp(x.astype(np.longdouble) / np.longdouble(t)))
    off = (near.astype(np.longdouble) - exact) / exact
    use = (np.abs(off) > 2e-14) & (np.abs(off) < 1e-12) & (near < 1)
    return x[use], near[use], off[use] < 0


@pytest.mark.parametrize("T", [1.0, 0.7, 3.0])
def test_acceptance(T):
    """A draft looked up in a vocabulary of two tokens is accepted where u < p."""
    x, u, want = cases(T, seed=1)
    B = min(len(x), 30000)
    assert B > 100
    logits = torch.zeros(2 * B, 2)
    logits[0::2, 1] = torch.from_numpy(x[:B])
    uniforms = torch.zeros(2 * B, 2)
    uniforms[0::2, 0] = torch.from_numpy(u[:B])
    r = verify_drafts(logits.to(DEV), torch.zeros(2 * B, dtype=torch.int64, device=DEV), uniforms.to(DEV),
                      torch.arange(0, 2 * B + 1, 2, dtype=torch.int32, device=DEV), temperature=T)
    wrong = int((r.accepted.cpu().bool() != torch.from_numpy(want[:B])).sum())
    say(f"T={T}: {wrong} of {B} on the other side")
    assert wrong == 0


@pytest.mark.parametrize("T", [1.0, 0.7, 3.0])
def test_places(T):
    """The token of two drawn by u: the first one where u < p."""
    x, u, want = cases(T, seed=2)
    B = min(len(x), 30000)
    logits = torch.zeros(B, 2)
    logits[:, 1] = torch.from_numpy(x[:B])
    uniforms = torch.zeros(B, 2)
    uniforms[:, 1] = torch.from_numpy(u[:B])
    r = verify_drafts(logits.to(DEV), torch.zeros(B, dtype=torch.int64, device=DEV), uniforms.to(DEV),
                      torch.arange(B + 1, dtype=torch.int32, device=DEV), temperature=T)
    wrong = int((r.tokens.cpu() != torch.from_numpy(~want[:B]).long()).sum())
    say(f"T={T}: {wrong} of {B} on the other side")
    assert wrong == 0

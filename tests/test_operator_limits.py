"""CPU checks of the limits of the logit-row and optimizer calls: sizes that no 32-bit count holds, settings at the ends of
fp32's range."""

import pytest
import torch

from dual_mod_public_amd import _lib as L
from dual_mod_public_amd import logprobs as lp
from tests.test_operator_refusals import plan, step_args, tensor


def test_step_counts_need_their_place():
    """The tensors' own step counts: aligned, and with room for their rates behind the workspace."""
    lib = L.load()
    assert lib.dm_adamw_step_counted(L.byref(step_args(workspace_bytes=1 << 20)), 0x80004, None) == -1
    for n in (1, 5):
        for have in (L.DM_ADAMW_WORKSPACE, L.DM_ADAMW_WORKSPACE + 8 * n - 1):
            a = step_args(n_tensors=n, workspace_bytes=have)
            assert lib.dm_adamw_step_counted(L.byref(a), 0x80000, None) == -3


@pytest.mark.parametrize("eps", [1e-39, 1e-45, 2.0 ** -127, 1e39])
def test_eps_out_of_range_is_refused(eps):
    """eps is the least denominator of an update, in fp32: one that is no normal number there is refused."""
    from dual_mod_public_amd.optim import AdamW
    assert L.load().dm_adamw_step(L.byref(step_args(eps=eps)), None) == -1
    with pytest.raises(ValueError, match="eps"):
        AdamW([torch.zeros(3)], eps=eps)


def test_plan_of_lengths_past_64_bits():
    """Lengths whose sum of launched blocks would pass 64 bits are refused one by one."""
    big = (1 << 63) - 1
    for ts in ([tensor(big)], [tensor(big), tensor((1 << 63) - 4096), tensor(5 * 4096)], [tensor(big, block0=1), tensor(4)],
               [tensor(4, block0=big)]):
        assert plan(*ts) is None


@pytest.mark.parametrize("shape", [((1 << 31), 1), ((1 << 32) + 4, 3), (2, 1 << 30, 2), (4, (1 << 27) + 1), (1, (1 << 32) + 5), (0, 1 << 32)])
def test_rows_and_columns_past_their_limits(shape):
    """More rows than a 32-bit count holds, or more columns than a row may have, are refused by size, not cut off."""
    with pytest.raises(ValueError, match="at most"):
        lp._rows(torch.empty(shape, device="meta", dtype=torch.bfloat16), "logits")


def test_rows_at_their_limits():
    assert lp._rows(torch.empty((1 << 31) - 1, 5, device="meta", dtype=torch.bfloat16), "logits") == ((1 << 31) - 1, 5)
    assert lp._rows(torch.empty(2, 1 << 27, device="meta"), "logits") == (2, 1 << 27)

"""CPU checks of the limits of the logit-row and optimizer calls: sizes that no 32-bit count holds, settings at the ends of
fp32's range."""

import pytest

from dual_mod_public_amd import _lib as L
from tests.test_operator_refusals import step_args


def test_step_counts_need_their_place():
    """The tensors' own step counts: aligned, and with room for their rates behind the workspace."""
    lib = L.load()
    assert lib.dm_adamw_step_counted(L.byref(step_args(workspace_bytes=1 << 20)), 0x80004, None) == -1
    for n in (1, 5):
        for have in (L.DM_ADAMW_WORKSPACE, L.DM_ADAMW_WORKSPACE + 8 * n - 1):
            a = step_args(n_tensors=n, workspace_bytes=have)
            assert lib.dm_adamw_step_counted(L.byref(a), 0x80000, None) == -3

"""The learning paths of the trunk at the ends of what they take."""

import pytest
import torch

from dual_mod_public_amd import _lib as L
from dual_mod_public_amd.trunk import HipTrunk
from tests.hip_helpers import DEV
from tests.test_gpu_learning import B, SCHED, T
from tests.test_gpu_trunk import _batch, _cfg, _model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    L.load()


def test_score_refuses_targets_of_another_shape():
    """Targets of more or fewer tokens than the batch would be taken row by row for others' places."""
    cfg = _cfg()
    m, _ = _model(cfg, torch.float32)
    tr = HipTrunk(m, B, T, schedule=SCHED, loss_chunk=48)
    idx, tg = _batch(cfg, B, T)
    idx = idx.to(DEV)
    want = tr.score(idx, tg).logp
    for bad in (torch.cat([tg, tg[:, :1]], 1), torch.cat([tg, tg]), tg[:, 1:], tg.reshape(-1), tg.t()):
        with pytest.raises(ValueError, match="targets"):
            tr.score(idx, bad)
    assert torch.equal(tr.score(idx, tg).logp, want)

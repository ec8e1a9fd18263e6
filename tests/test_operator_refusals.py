"""CPU checks of what the logit-row and optimizer entry points refuse before they touch a device, and of the optimizer's
launch plan."""

import ctypes

import pytest
import torch

from dual_mod_public_amd import _lib as L
from dual_mod_public_amd import logprobs as lp
from dual_mod_public_amd.optim import AdamW


def rows_args(**kw):
    a = L.dm_logprob_args()
    for k, v in dict(dict(dtype=L.DM_F32, rows=4, cols=10, ld=10, logits=0x10000, target=0x20000, lse=0x30000, entropy=0x30100, stats=0x30300,
                          logp=0x30200), **kw).items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [dict(dtype=2), dict(rows=-1), dict(cols=0), dict(cols=(1 << 27) + 1, ld=1 << 40), dict(ld=9), dict(logits=None), dict(logits=0x10002),
                                dict(target=None), dict(top=33), dict(top=-1), dict(top=3), dict(cols=2, top=3, top_logp=1, top_ids=1),
                                dict(dlogits=0x40000, ld_d=10), dict(dlogits=0x40000, ld_d=9, g_logp=0x50000),
                                dict(dlogits=0x40001, ld_d=10, g_logp=0x50000),
                                dict(dlogits=0x10004, ld_d=10, g_logp=0x50000), dict(dlogits=0x10000, ld_d=11, g_logp=0x50000),
                                dict(dlogits=0x10000 - 40, ld_d=10, g_logp=0x50000),
                                dict(target=None, logp=None, dlogits=0x40000, ld_d=10, g_logp=0x50000),
                                # outputs over inputs and over each other (rows take 160 bytes, targets 32, values 16, stats 48)
                                dict(lse=0x10000 + 156), dict(logp=0x20000 - 12), dict(stats=0x20000 + 28), dict(entropy=0x30000 + 12),
                                dict(stats=0x30100 - 44), dict(top=2, top_logp=0x60000, top_ids=0x60000 + 28),
                                dict(top=2, top_ids=0x60000, top_logp=0x10000 - 28),
                                dict(dlogits=0x10000, ld_d=10, g_logp=0x10000 + 80), dict(dlogits=0x40000, ld_d=10, g_logp=0x40000 + 156),
                                dict(dlogits=0x20000 + 28, ld_d=10, g_entropy=0x50000),
                                dict(dlogits=0x40000, ld_d=10, g_logp=0x30000)])
def test_logprob_rows_refuses(kw):
    lib = L.load()
    assert lib.dm_logprob_rows(L.byref(rows_args(**kw)), None) == -1 and lib.dm_last_error()


@pytest.mark.parametrize("kw", [dict(dlogits=None), dict(stats=None), dict(g_logp=None), dict(stats=0x40000 + 156),
                                dict(dlogits=0x10000, stats=0x10000 - 44)])
def test_logprob_bwd_refuses(kw):
    a = rows_args(**dict(dict(dlogits=0x40000, ld_d=10, g_logp=0x50000), **kw))
    assert L.load().dm_logprob_rows_bwd(L.byref(a), None) == -1


def test_no_rows_is_no_launch():
    lib = L.load()
    assert lib.dm_logprob_rows(L.byref(rows_args(rows=0, logits=None)), None) == 0
    assert lib.dm_logprob_rows_bwd(L.byref(rows_args(rows=0)), None) == 0
    assert lib.dm_logprob_rows(None, None) == -1 and lib.dm_logprob_rows_bwd(None, None) == -1


def tensor(n, p=0x10000, g=0x20000, dtype=L.DM_F32, block0=0):
    return L.dm_adamw_tensor(p, g, n, block0, 0.1, 1.0, dtype, 0)


def plan(*ts):
    arr = (L.dm_adamw_tensor * len(ts))(*ts)
    lib = L.load()
    nb, n = lib.dm_adamw_plan_bytes(arr, len(ts)), ctypes.c_int64()
    if nb == 0:
        return None
    buf = ctypes.create_string_buffer(nb)
    assert lib.dm_adamw_plan(arr, len(ts), buf, nb - 1, ctypes.byref(n)) == -3
    assert lib.dm_adamw_plan(arr, len(ts), buf, nb, ctypes.byref(n)) == 0
    return n.value


def test_plan_covers_every_element():
    one = plan(tensor(1))
    assert one == 1
    size = next(n for n in range(256, 1 << 20, 256) if plan(tensor(n + 1)) == 2)     # elements per launched block
    assert size % L.DM_ADAMW_BLOCK == 0
    assert plan(tensor(size)) == 1 and plan(tensor(3 * size + 1)) == 4
    assert plan(tensor(5), tensor(0, p=None, g=None), tensor(2 * size), tensor(size + 1)) == 1 + 2 + 2


@pytest.mark.parametrize("ts", [[tensor(0)], [tensor(-1)], [tensor(4, p=None)], [tensor(4, g=None)], [tensor(4, p=0x10002)],
                                [tensor(4, g=0x20002)], [tensor(4, g=0x20001, dtype=L.DM_BF16)], [tensor(4, dtype=2)],
                                [tensor(4, block0=-1)], [tensor(1 << 50)]])
def test_plan_refuses(ts):
    assert plan(*ts) is None


def step_args(**kw):
    a = L.dm_adamw_args()
    for k, v in dict(dict(plan=0x10000, n_chunks=1, n_tensors=1, state_bits=8, exp_avg=0x20000, exp_avg_sq=0x30000,
                          exp_avg_exponent=0x40000, exp_avg_sq_exponent=0x50000, beta1=0.9, beta2=0.999, eps=1e-8, max_norm=1.0,
                          lr=0x60000, steps=0x60010, norm=0x60020, skipped=0x60030, workspace=0x70000,
                          workspace_bytes=L.DM_ADAMW_WORKSPACE), **kw).items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,rc", [(dict(plan=None), -1), (dict(n_chunks=0), -1), (dict(n_tensors=0), -1), (dict(state_bits=16), -1),
                                   (dict(exp_avg=0x20004), -1), (dict(exp_avg_sq=None), -1), (dict(exp_avg_exponent=None), -1),
                                   (dict(beta1=1.0), -1), (dict(beta2=-0.1), -1), (dict(eps=0.0), -1), (dict(eps=1e-60), -1),
                                   (dict(eps=float("nan")), -1), (dict(max_norm=float("inf")), -1), (dict(max_norm=float("nan")), -1),
                                   (dict(lr=None), -1), (dict(steps=None), -1), (dict(norm=None), -1),
                                   (dict(skipped=None, skip_nonfinite=1), -1), (dict(workspace=None), -3),
                                   (dict(workspace=0x70008), -3), (dict(workspace_bytes=L.DM_ADAMW_WORKSPACE - 1), -3)])
def test_step_refuses(kw, rc):
    assert L.load().dm_adamw_step(L.byref(step_args(**kw)), None) == rc
    assert L.load().dm_adamw_step(None, None) == -1


def test_norm_and_values_refuse():
    lib = L.load()
    assert lib.dm_grad_norm(L.byref(step_args(norm=None)), None) == -1
    assert lib.dm_grad_norm(L.byref(step_args(workspace=None)), None) == -3
    assert lib.dm_adamw_values(None, None, 1, 0, None, None) == -1
    assert lib.dm_adamw_values(0x1000, 0x2000, 1, 0, 0x3004, None) == -1
    assert lib.dm_adamw_values(None, None, -1, 0, None, None) == -1
    assert lib.dm_adamw_values(None, None, 0, 0, None, None) == 0


def test_python_refuses_cpu_tensors_and_bad_settings():
    x = torch.zeros(2, 5)
    t = torch.zeros(2, dtype=torch.int64)
    for f in (lambda: lp.row_logprobs(x, t), lambda: lp.token_logprobs(x, t), lambda: lp.row_logprobs_grad(x, t, torch.ones(2)),
              lambda: AdamW([x]), lambda: AdamW([]), lambda: AdamW([x], state_bits=16), lambda: AdamW([x], betas=(1.0, 0.9)),
              lambda: AdamW([x], eps=0.0), lambda: AdamW([x], max_norm=0.0), lambda: AdamW([x], max_norm=float("nan")),
              lambda: AdamW([dict(params=[x], lr=1.0)]), lambda: AdamW([dict(weight_decay=0.1)]), lambda: AdamW([x], grads=[])):
        with pytest.raises(ValueError):
            f()

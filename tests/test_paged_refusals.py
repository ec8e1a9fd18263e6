"""CPU checks of what the paged cache's and the drafts' entry points refuse before they touch a device."""

import pytest
import torch

from dual_mod_public_amd import _lib as L
from dual_mod_public_amd import drafts, paged


def paged_args(**kw):
    a = L.dm_paged_args()
    base = dict(dtype=L.DM_BF16, B=2, h=4, h_kv=2, dh=64, page=16, n_pages=5, table_cols=3, n_tokens=2, window=0, scale=0.125, q=0x10000,
                q_token=256, q_head=64, K=0x20000, V=0x30000, k_page=2048, v_page=2048, table=0x40000, lengths=0x50000, o=0x60000,
                lse=0x70000, workspace=0x100000, workspace_bytes=1 << 40)
    for k, v in dict(base, **kw).items():
        setattr(a, k, v)
    return a


PAGES = [(dict(dtype=2), -1), (dict(dh=96), -2), (dict(page=8), -2), (dict(page=48), -2), (dict(page=2048), -2), (dict(n_pages=0), -1),
         (dict(table_cols=0), -1), (dict(B=0), -1), (dict(B=65536, n_tokens=65536), -1), (dict(h_kv=0), -1), (dict(K=None), -1),
         (dict(V=0x30008), -1), (dict(k_page=2040), -1), (dict(v_page=2052), -1), (dict(table_cols=1 << 23), -1), (dict(table=None), -1),
         (dict(lengths=None), -1)]


@pytest.mark.parametrize("kw,rc", PAGES + [
    (dict(n_tokens=3), -1), (dict(n_tokens=-1), -1), (dict(h=3), -1), (dict(h=0), -1), (dict(q=None), -1), (dict(q=0x10008), -1),
    (dict(q_token=252), -1), (dict(q_head=-64), -1), (dict(window=-1), -1), (dict(scale=float("inf")), -1), (dict(scale=float("nan")), -1),
    (dict(o=None), -1), (dict(o=0x60004), -1), (dict(lse=None), -1), (dict(k_rows=0x80000), -1), (dict(v_rows=0x80000), -1),
    (dict(k_rows=0x80000, v_rows=0x90008, k_token=128, k_head=64, v_token=128, v_head=64), -1),
    (dict(workspace=None, table_cols=200), -3), (dict(workspace=0x100008, table_cols=200), -3), (dict(workspace_bytes=16, table_cols=200), -3),
    (dict(starts=0x51000, n_tokens=1 << 26), -1)])
def test_attention_refuses(kw, rc):
    lib = L.load()
    assert lib.dm_paged_attention(L.byref(paged_args(**kw)), None) == rc and lib.dm_last_error()


@pytest.mark.parametrize("kw,rc", PAGES + [(dict(k_rows=None), -1), (dict(v_rows=0x90004), -1), (dict(k_token=4), -1)])
def test_write_refuses(kw, rc):
    base = dict(k_rows=0x80000, v_rows=0x90000, k_token=128, k_head=64, v_token=128, v_head=64)
    assert L.load().dm_paged_write(L.byref(paged_args(**dict(base, **kw))), None) == rc


def test_no_tokens_is_no_launch():
    lib = L.load()
    a = paged_args(n_tokens=0, starts=0x51000, q=None, o=None)
    assert lib.dm_paged_attention(L.byref(a), None) == 0 and lib.dm_paged_write(L.byref(a), None) == 0
    assert lib.dm_paged_attention(None, None) == -1 and lib.dm_paged_write(None, None) == -1 and lib.dm_paged_evict(None, None) == -1
    assert lib.dm_paged_workspace_bytes(None) == 0 and lib.dm_verify_workspace_bytes(None) == 0


@pytest.mark.parametrize("kw,rc", [p for p in PAGES if "n_tokens" not in p[0]] + [
    (dict(B=65536), -1), (dict(keep=0), -1), (dict(sinks=-1), -1), (dict(recent=-1), -1), (dict(sinks=20, recent=13), -1),
    (dict(new_cols=1), -1), (dict(new_cols=0), -1), (dict(new_cols=1 << 23), -1), (dict(weights=None), -1), (dict(weights_out=None), -1),
    (dict(weights_out=0x60000), -1), (dict(lengths_out=0x50000), -1), (dict(rows=None), -1), (dict(new_table=None), -1)])
def test_evict_refuses(kw, rc):
    a = L.dm_evict_args()
    base = dict(dtype=L.DM_BF16, B=2, h_kv=2, dh=64, page=16, n_pages=5, table_cols=3, new_cols=2, keep=32, sinks=2, recent=4, K=0x20000,
                V=0x30000, k_page=2048, v_page=2048, table=0x40000, lengths=0x50000, new_table=0x41000, weights=0x60000,
                weights_out=0x61000, rows=0x62000, lengths_out=0x63000)
    for k, v in dict(base, **kw).items():
        setattr(a, k, v)
    assert L.load().dm_paged_evict(L.byref(a), None) == rc


@pytest.mark.parametrize("kw,rc", [(dict(dtype=2), -1), (dict(rows=-1), -1), (dict(rows=65536), -1), (dict(B=65536), -1), (dict(B=-1), -1),
                                   (dict(rows=0), -1), (dict(B=0), -1), (dict(cols=0), -1), (dict(cols=(1 << 27) + 1), -1), (dict(ld=99), -1),
                                   (dict(draft_logits=0x20000, ld_draft=99), -1), (dict(logits=None), -1), (dict(logits=0x10001), -1),
                                   (dict(draft_logits=0x20001, ld_draft=100), -1), (dict(ids=None), -1), (dict(uniforms=None), -1),
                                   (dict(temperature=None), -1), (dict(starts=None), -1), (dict(tokens=None), -1), (dict(accepted=None), -1),
                                   (dict(logp=None), -1), (dict(workspace=None), -3), (dict(workspace=0x80008), -3),
                                   (dict(workspace_bytes=100), -3)])
def test_verify_refuses(kw, rc):
    a = L.dm_verify_args()
    base = dict(dtype=L.DM_BF16, rows=6, cols=100, B=2, logits=0x10000, ld=100, ids=0x30000, uniforms=0x40000, temperature=0x50000,
                starts=0x51000, tokens=0x60000, accepted=0x61000, logp=0x62000, workspace=0x80000, workspace_bytes=1 << 30)
    for k, v in dict(base, **kw).items():
        setattr(a, k, v)
    assert L.load().dm_verify_drafts(L.byref(a), None) == rc


def test_python_refuses_tensors_of_the_cpu():
    K, V = paged.new_pages(4, 2, 16, 64, device="cpu")
    table, lengths = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    for f in (lambda: paged.paged_attention(q, K, V, table, lengths), lambda: paged.paged_write(q, q, K, V, table, lengths),
              lambda: paged.evict_rows(K, V, torch.zeros(1, 2, 32), table, lengths, 8, table),
              lambda: drafts.verify_drafts(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64), torch.zeros(2, 2),
                                           torch.tensor([0, 2], dtype=torch.int32))):
        with pytest.raises(ValueError):
            f()
    with pytest.raises(NotImplementedError, match="no autograd"):
        paged.paged_attention(q.requires_grad_(), K, V, table, lengths)


def test_more_blocks_than_a_launch_has():
    """B h_kv blocks are the least of a launch; of 2^22 and more of them a launch's threads would pass 32 bits."""
    lib = L.load()
    big = dict(B=4097, h_kv=1024, h=1024, n_tokens=4097, k_page=1024 * 16 * 64, v_page=1024 * 16 * 64)
    rows = dict(k_rows=0x80000, v_rows=0x90000, k_token=1024 * 64, k_head=64, v_token=1024 * 64, v_head=64)
    assert lib.dm_paged_attention(L.byref(paged_args(**big)), None) == -1 and b"in all" in lib.dm_last_error()
    assert lib.dm_paged_write(L.byref(paged_args(**big, **rows)), None) == -1


def test_workspaces():
    """None where every tile's rows lie in one piece and no scores are kept; else enough for twice the pieces wanted."""
    size = L.load().dm_paged_workspace_bytes
    assert size(L.byref(paged_args())) == 0 and size(L.byref(paged_args(table_cols=64))) == 0
    assert size(L.byref(paged_args(table_cols=200))) > 0 and size(L.byref(paged_args(weights=0x90000, n_pages=4096))) > 0
    assert size(L.byref(paged_args(table_cols=200, window=64))) == 0

"""CPU checks of the paged calls' limits: numbers at the ends of their ranges, workspaces."""

import pytest

from dual_mod_public_amd import _lib as L


def evict_args(**kw):
    a = L.dm_evict_args()
    base = dict(dtype=L.DM_BF16, B=2, h_kv=2, dh=64, page=16, n_pages=5, table_cols=3, new_cols=3, keep=32, sinks=2, recent=4, K=0x20000,
                V=0x30000, k_page=2048, v_page=2048, table=0x40000, lengths=0x50000, new_table=0x41000, weights=0x60000,
                weights_out=0x61000, rows=0x62000, lengths_out=0x63000)
    for k, v in dict(base, **kw).items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("keep", [L.DM_PAGED_ROWS + 1, 2 ** 31 - 1024, 2 ** 31 - 1])
def test_more_kept_rows_than_a_table_has(keep):
    """A block's threads step through the keep places of a sequence by 1024: past 2^31 - 1024 their count would leave 32 bits, and the
    places behind the kept rows be written before the buffer."""
    lib = L.load()
    assert lib.dm_paged_evict(L.byref(evict_args(keep=keep)), None) == -1 and b"keep" in lib.dm_last_error()


def attention_args(**kw):
    a = L.dm_paged_args()
    base = dict(dtype=L.DM_BF16, B=64, h=32, h_kv=8, dh=128, page=64, n_pages=1 << 20, table_cols=1 << 11, n_tokens=64, scale=0.125,
                q=0x10000, q_token=4096, q_head=128, K=0x20000, V=0x30000, k_page=65536, v_page=65536, table=0x40000, lengths=0x50000,
                o=0x60000, lse=0x70000, weights=0x80000)
    for k, v in dict(base, **kw).items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [{}, dict(n_tokens=512, starts=0x51000), dict(dtype=L.DM_F32, n_tokens=4096, starts=0x51000),
                                dict(window=256), dict(table_cols=1 << 20)])
def test_kept_scores_have_a_bound_of_their_own(kw):
    """Not the table's width times the tokens (here 1 GiB to 0.5 TiB) up to the size of the pool's keys (128 GiB)."""
    size = L.load().dm_paged_workspace_bytes
    assert size(L.byref(attention_args(**kw))) <= (1 << 30) + size(L.byref(attention_args(**kw, weights=None)))


def test_scores_are_kept_within_the_bound():
    size = L.load().dm_paged_workspace_bytes
    kept = size(L.byref(attention_args())) - size(L.byref(attention_args(weights=None)))
    assert kept == 64 * 32 * (1 << 17) * 4 == 1 << 30


@pytest.mark.parametrize("scale", [2.4e38, -3.4e38])
def test_scales_whose_product_with_log2_e_is_infinite(scale):
    """Scores are held in units of ln 2: the scale times log2 e has to be a number, or scores of 0 become NaN."""
    lib = L.load()
    a = attention_args(weights=None, scale=scale, workspace=0x100000, workspace_bytes=1 << 40)
    assert lib.dm_paged_attention(L.byref(a), None) == -1 and b"scale" in lib.dm_last_error()

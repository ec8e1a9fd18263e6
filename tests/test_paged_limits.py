"""CPU checks of the paged calls' limits: numbers at the ends of their ranges, workspaces."""

import math
import random

import pytest

from dual_mod_public_amd import _lib as L


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


def plan(lengths, starts, N, g, rows, cap, want, least, with_self=False, window=0):
    """The kernels' plan on the host: (sequence, tile, piece, pieces, slot) of each item, in order. It counts tiles of 64 cached
    rows per query tile of ``rows`` query rows, and cuts a sequence into pieces of ``each`` of them."""
    seqs = []
    for b, length in enumerate(lengths):
        first = min(max(starts[b], 0), N)
        n = min(max(starts[b + 1], first), N) - first
        bad = length < n or length > cap
        length = n if bad else length
        tiles_k = 0
        if n and not bad:
            low = max(0, length - n - window + 1) if window else 0
            high = length - 1 + (0 if with_self else 1)
            tiles_k = (max(0, high - low // 64 * 64) + 63) // 64
        seqs.append((-(-n * g // rows), tiles_k))
    cost = sum(tq * tk for tq, tk in seqs) * (1 + 1e-4)
    each = max(least, math.ceil(cost / want))
    items, slots = [], 0
    for b, (tq, tk) in enumerate(seqs):
        pieces = max(1, -(-tk // each))
        for tile in range(tq - 1, -1, -1):
            for piece in range(pieces):
                items.append((b, tile, piece, pieces, slots + tile * pieces if pieces > 1 else 0))
        slots += tq * pieces if pieces > 1 else 0
    return items


@pytest.mark.parametrize("seed", range(20))
def test_pieces_have_their_places_whatever_the_starts(seed):
    """Every piece of a query tile has a place of its own in the workspace, also where starts descend and sequences share tokens."""
    rng = random.Random(seed)
    B, h_kv, g, dh, page = rng.choice([1, 7, 200]), 2, rng.choice([1, 2]), 64, 16
    cols = rng.choice([200, 500])
    N = rng.randint(1, 16 * B // g)
    a = attention_args(B=B, h=h_kv * g, h_kv=h_kv, dh=dh, page=page, table_cols=cols, n_tokens=N, starts=0x51000, weights=None,
                       k_page=h_kv * page * dh, v_page=h_kv * page * dh)
    want = L.load().dm_paged_workspace_bytes(L.byref(a)) // (2 * h_kv * 16 * (dh + 2) * 4)      # tiles of 16 query rows
    assert want > 0
    for _ in range(5):
        starts = [rng.randint(-3, N + 3) for _ in range(B + 1)] if rng.random() < 0.5 else [0, N] * (B // 2 + 1)
        lengths = [rng.choice([0, rng.randint(0, cols * page), cols * page, cols * page + 1]) for _ in range(B)]
        places = set()
        for b, tile, piece, pieces, slot in plan(lengths, starts, N, g, 16, cols * page, want, 2):
            if pieces > 1:
                assert 0 <= slot + piece < 2 * want and (slot + piece) not in places
                places.add(slot + piece)

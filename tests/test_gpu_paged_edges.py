"""The paged operators' results in bits and at odd values, against their definitions in 64 bits."""

import math

import pytest
import torch
from torch.autograd import forward_ad

from dual_mod_public_amd import _lib as L
from dual_mod_public_amd import paged
from dual_mod_public_amd.drafts import verify_drafts
from tests import paged_reference as ref
from tests.hip_helpers import DEV
from tests.test_gpu_paged import dev, make, near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    L.load()


def bounds_without_rounded_probabilities(s, lengths, counts, pair):
    """(o, its bound) where probabilities keep 16 bits. One of two bf16 parts: the first is p cut to 8 bits, what is left is below
    2^-7 p and rounded by at most 2^-8 of that, or 2^-24 p where it is less. (ref.attention counts 2^-8 for a probability; the share
    that it multiplies is what the magnitudes of the values give.)"""
    k, v = (s["k"], s["v"]) if pair else (None, None)
    o, _, _, bo, _, _ = ref.attention(s["q"], s["K"], s["V"], s["table"], lengths, counts, k, v)
    share = ref.attention(s["q"], s["K"], s["V"].abs(), s["table"], lengths, counts, k, None if v is None else v.abs())[0]
    return o, bo + share * (2.0 ** -15 + 2.0 ** -24 - 2.0 ** -8)


@pytest.mark.parametrize("dh,page,h,h_kv", [(64, 64, 4, 4), (128, 16, 4, 1), (64, 16, 8, 2)])
@pytest.mark.parametrize("new", [1, 5])
@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("cols", [None, 1024])
def test_probabilities_of_few_query_rows_keep_16_bits(dh, page, h, h_kv, new, pair, cols):
    """Outputs whose terms cancel show a probability's rounding: it is relative to the terms. In one piece and in several."""
    lengths = [5, 17, 40, 64, 100, 300, 1100]
    counts = [new] * len(lengths)
    s = make(lengths, counts, h, h_kv, dh, page, torch.bfloat16, seed=dh + h, cols=cols)
    s["q"] *= 0.25
    o, bound = bounds_without_rounded_probabilities(s, lengths, counts, pair)
    d = dev(s)
    kw = dict(k_self=d["k"], v_self=d["v"]) if pair else {}
    near(paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"], d["starts"], **kw).o, o, bound, "o")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("new", [1, 3, 90, 600])
def test_infinite_values_that_are_read(dtype, dh, new):
    """An infinite value of a row that all tokens read makes its column infinite, in steps without a mask too, and no other one."""
    lengths, counts = [700 + new], [new]
    s = make(lengths, counts, 2, 1, dh, 16, dtype, seed=new)
    s["q"] *= 0.25
    o, _, _, bo, _, _ = ref.attention(s["q"], s["K"], s["V"], s["table"], lengths, counts)
    for r, c, x in ((3, 1, math.inf), (70, 9, -math.inf), (400, 33, math.inf), (401, 33, math.inf), (699, 40, -math.inf),
                    (130, 50, math.nan), (200, 60, math.inf), (201, 60, -math.inf)):
        s["V"][s["table"][0, r // 16], :, r % 16, c] = x
    d = dev(s)
    got = paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"], d["starts"]).o.cpu()
    assert (got[..., [1, 33]] == math.inf).all() and (got[..., [9, 40]] == -math.inf).all() and got[..., [50, 60]].isnan().all()
    rest = [c for c in range(dh) if c not in (1, 9, 33, 40, 50, 60)]
    near(got[..., rest], o[..., rest], bo[..., rest], "o")


@pytest.mark.parametrize("keep", [2 ** 32 + 5, 2 ** 31])
def test_keep_past_32_bits(keep):
    """Refused before the rows are allocated: the call would take the lower bits."""
    K, V = paged.new_pages(4, 2, 16, 64)
    table, w = torch.zeros(1, 2, dtype=torch.int32, device=DEV), torch.zeros(1, 2, 32, device=DEV)
    with pytest.raises(ValueError, match="keep="):
        paged.evict_rows(K, V, w, table, torch.ones(1, dtype=torch.int32, device=DEV), keep, table + 2)


@pytest.mark.parametrize("keep", [2 ** 26 + 1, 2 ** 31 - 1])
def test_keep_of_more_than_there_is(keep):
    """All rows stay, and all places behind them hold -1. A block's threads step through the places by 1024: within 1024 of 2^31 a
    count of 32 bits would wrap, and go on before the buffer."""
    K, V = paged.new_pages(4, 1, 16, 64)
    K[1] = torch.randn(1, 16, 64)
    table, w = torch.tensor([[1]], dtype=torch.int32, device=DEV), torch.rand(1, 1, 16, device=DEV)
    r = paged.evict_rows(K, V, w, table, torch.tensor([13], dtype=torch.int32, device=DEV), keep, table + 2)
    assert r.rows.shape == (1, 1, keep) and r.rows[0, 0, :13].tolist() == list(range(13)) and r.lengths.tolist() == [13]
    assert all((part == -1).all() for part in r.rows[0, 0, 13:].split(1 << 28))
    assert torch.equal(K[3, 0, :13], K[1, 0, :13]) and torch.equal(r.weights[0, 0, :13], w[0, 0, :13])


def test_more_tokens_than_32_bits_count():
    """Refused, where the library would see the lower 32 bits of their number (here 2 tokens)."""
    K, V = paged.new_pages(4, 2, 16, 64)
    table, lengths = torch.zeros(1, 2, dtype=torch.int32, device=DEV), torch.full((1,), 2, dtype=torch.int32, device=DEV)
    k = torch.ones(1, 2, 64, device=DEV, dtype=torch.bfloat16).expand(2 ** 32 + 2, 2, 64)
    with pytest.raises(ValueError, match="too many"):
        paged.paged_write(k, k, K, V, table, lengths, torch.tensor([0, 2], dtype=torch.int32, device=DEV))
    assert not K.any()


def test_tangents_and_graphs_are_refused():
    """Tensors with a forward-mode tangent have no requires_grad; the calls would drop the tangent. Weights and temperatures with
    a graph."""
    K, V = paged.new_pages(4, 2, 16, 64, dtype=torch.float32)
    table, lengths = torch.zeros(1, 2, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    q, pair, w = torch.zeros(1, 4, 64, device=DEV), torch.zeros(1, 2, 64, device=DEV), torch.zeros(1, 2, 32, device=DEV)
    x, ids, u = torch.zeros(2, 9, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV), torch.zeros(2, 2, device=DEV)
    starts, T = torch.tensor([0, 2], dtype=torch.int32, device=DEV), torch.ones(1, device=DEV)
    calls = {
        "attend": (lambda **kw: paged.paged_attention(**dict(dict(q=q, K=K, V=V, table=table, lengths=lengths, k_self=pair, v_self=pair,
                                                                  weights=w), **kw)), dict(q=q, K=K, V=V, k_self=pair, v_self=pair, weights=w)),
        "write": (lambda **kw: paged.paged_write(**dict(dict(k=pair, v=pair, K=K, V=V, table=table, lengths=lengths), **kw)),
                  dict(k=pair, v=pair, K=K, V=V)),
        "evict": (lambda **kw: paged.evict_rows(**dict(dict(K=K, V=V, weights=w, table=table, lengths=lengths, keep=8, new_table=table + 2),
                                                       **kw)), dict(K=K, V=V, weights=w)),
        "verify": (lambda **kw: verify_drafts(**dict(dict(logits=x, ids=ids, uniforms=u, starts=starts, draft_logits=x, temperature=T), **kw)),
                   dict(logits=x, draft_logits=x, temperature=T)),
    }
    for name, (call, tensors) in calls.items():
        call()
        for n, t in tensors.items():
            with forward_ad.dual_level():
                call()
                with pytest.raises(NotImplementedError, match="tangent"):
                    call(**{n: forward_ad.make_dual(t.clone(), torch.ones_like(t))})
                with torch.no_grad(), pytest.raises(NotImplementedError, match="tangent"):
                    call(**{n: forward_ad.make_dual(t.clone(), torch.ones_like(t))})
            with pytest.raises(NotImplementedError, match="graph"):
                call(**{n: t.clone().requires_grad_()})
            with torch.no_grad():
                call(**{n: t.clone().requires_grad_()})


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 90, 600])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_scale_of_zero_times_queries_that_are_not_finite(dtype, new, value):
    """0 times NaN or infinity is NaN, whichever read a call takes; the other query rows are means of the rows read."""
    lengths, counts = [40 + new], [new]
    s = make(lengths, counts, 2, 1, 64, 16, dtype, seed=new)
    o, _, _, bo, _, _ = ref.attention(s["q"], s["K"], s["V"], s["table"], lengths, counts, scale=0.0)
    s["q"][new // 2, 1, 7] = value
    d = dev(s)
    r = paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"], d["starts"], scale=0.0)
    nan = torch.zeros(new, 2, dtype=torch.bool)
    nan[new // 2, 1] = True
    assert torch.equal(r.lse.isnan().cpu(), nan) and torch.equal(r.o.isnan().all(-1).cpu(), nan)
    near(r.o.cpu()[~nan], o[~nan], bo[~nan], "o")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new,g", [(3, 1), (60, 2), (300, 4)])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("bad", [0, 7, -1])
def test_chunks_with_a_page_outside_the_pool(dtype, new, g, window, bad):
    """The tokens that read a row of it get NaN, the others NaN or what they get without it; and so do the weights of the rows
    that those read. The other sequence is as ever."""
    lengths, counts, page = [200 + new, 90], [new, 2], 16
    s = make(lengths, counts, g, 1, 64, page, dtype, seed=new)
    d = dev(s)
    cap = s["table"].shape[1] * page
    w, v = torch.zeros(2, 1, cap, device=DEV), torch.zeros(2, 1, cap, device=DEV)
    want = paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"], d["starts"], window=window, weights=w)
    at = bad if bad >= 0 else (lengths[0] - 1) // page
    d["table"][0, at] = s["K"].shape[0]
    r = paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"], d["starts"], window=window, weights=v)
    reads_it = torch.zeros(new + 2, dtype=torch.bool)
    read_by_it = torch.zeros(cap, dtype=torch.bool)
    for j in range(new):
        p = 200 + j
        low = max(0, p - window + 1) if window else 0
        reads_it[j] = p >= page * at and low < page * (at + 1)
        if reads_it[j]:
            read_by_it[low:p + 1] = True
    nan = r.o.isnan().flatten(1).all(1).cpu()
    assert nan[reads_it].all() and not nan[new:].any() and torch.equal(r.lse.isnan().all(1).cpu(), nan)
    assert torch.equal(r.o[~nan], want.o[~nan]) and torch.equal(r.lse[~nan], want.lse[~nan])
    v, w = v.cpu(), w.cpu()
    assert v[0, 0, read_by_it].isnan().all() and torch.equal(v[1], w[1]) and not v[0, 0, lengths[0]:].any()


def guarded(n_bytes, fill=0xa5):
    """n_bytes in the middle of a buffer of a pattern: (the buffer, their address)."""
    t = torch.full((n_bytes + 2 * GUARD,), fill, dtype=torch.uint8, device=DEV)
    return t, t.data_ptr() + GUARD


GUARD = 1 << 16


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,N,g", [(200, 200, 2), (5, 150, 4), (3, 400, 4)])
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("starts", ["ascending", "turning", "negative"])
def test_nothing_around_the_outputs_is_written(dtype, B, N, g, weights, starts):
    """Outputs, weights and workspace inside buffers of a pattern, which stays, also where starts descend: sequences then share
    tokens, and no result is defined."""
    h_kv, dh, page, cols = 2, 64, 16, 200
    lengths = [(37 * b) % 3000 + N for b in range(B)]
    rng = torch.Generator().manual_seed(B)
    table = torch.randint(0, 64, (B, cols), generator=rng, dtype=torch.int32).to(DEV)
    K, V = (torch.randn(64, h_kv, page, dh, generator=rng).to(dtype).to(DEV) for _ in range(2))
    q = torch.randn(N, h_kv * g, dh, generator=rng).to(dtype).to(DEV)
    cut = {"ascending": [N * b // B for b in range(B + 1)], "turning": ([0, N] * B)[:B + 1],
           "negative": [N - 2 * b for b in range(B)] + [-7]}[starts]
    cut = torch.tensor(cut, dtype=torch.int32, device=DEV)
    length = torch.tensor([min(n, cols * page) for n in lengths], dtype=torch.int32, device=DEV)
    sizes = dict(o=N * h_kv * g * dh * q.element_size(), lse=N * h_kv * g * 4)
    if weights:
        sizes["weights"] = B * h_kv * cols * page * 4
    a = L.dm_paged_args(L.dtype_code(dtype), B, h_kv * g, h_kv, dh, page, 64, cols, N, 0, 0.125, 0, q.data_ptr(), q.stride(0), q.stride(1),
                        K.data_ptr(), V.data_ptr(), K.stride(0), V.stride(0), table.data_ptr(), length.data_ptr(), cut.data_ptr())
    if weights:
        a.weights = 1
    sizes["workspace"] = L.lib().dm_paged_workspace_bytes(L.byref(a))
    buffers = {}
    for n, size in sizes.items():
        buffers[n], at = guarded(size)
        setattr(a, n, at)
    a.workspace_bytes = sizes["workspace"]
    if weights:
        buffers["weights"][GUARD:-GUARD] = 0
    L.call_on(K.device, L.lib().dm_paged_attention, L.byref(a))
    torch.cuda.synchronize()
    for n, t in buffers.items():
        assert (t[:GUARD] == 0xa5).all() and (t[-GUARD:] == 0xa5).all(), n
    if starts == "ascending":
        w = torch.zeros(B, h_kv, cols * page, device=DEV) if weights else None
        want = paged.paged_attention(q, K, V, table, length, cut, scale=0.125, weights=w)
        assert torch.equal(buffers["o"][GUARD:-GUARD].view(dtype).view_as(want.o), want.o)
        assert torch.equal(buffers["lse"][GUARD:-GUARD].view(torch.float32).view_as(want.lse), want.lse)
        assert not weights or torch.equal(buffers["weights"][GUARD:-GUARD].view(torch.float32).view_as(w), w)


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("new", [1, 3])
def test_sums_of_fp32_scores_are_short_chains(dh, new):
    """The 2-norm of fp32 outputs' errors over 4096 rows, of queries of standard deviation 2 and keys of 1, in u = 2^-24. A sum's
    rounding is u / sqrt(3) of the partial sum, which after i products is 2 sqrt(i): two chains of 16 products take turns, each gives a
    variance of 4 / 3 (1 + .. + 16) = 181, and adding them (at 32, and at 64, 96, 128 in all) 4 / 3 (4 * 32 + 288) more: for 128
    products 2000 in all, 45 u, times the scale 4.0 u; for 64 3.9 u. An exponential's argument (of about 2 and up to 8 below the
    maximum) and the exponential itself give 2 u, sums over 64 steps of 16 rows in each of four waves 3 u. Together 5.4 u = 3.2e-7;
    twice that is the bound. One chain of all products gives 9.4 u (128) for the first alone."""
    lengths, counts = [4096] * 6, [new] * 6
    s = make(lengths, counts, 8, 2, dh, 64, torch.float32, seed=dh + new)
    d = dev(s)
    o, lse, _, _, _, _ = ref.attention(s["q"], s["K"], s["V"], s["table"], lengths, counts)
    r = paged.paged_attention(d["q"], d["K"], d["V"], d["table"], d["lengths"], d["starts"])
    err = float((r.o.double().cpu() - o).norm() / o.norm())
    assert err < 6.4e-7, err
    # lse: rounded once, beside a sum's and a maximum's few units
    assert float((r.lse.double().cpu() - lse).abs().max()) < 12 * 2.0 ** -24 * float(lse.abs().max())

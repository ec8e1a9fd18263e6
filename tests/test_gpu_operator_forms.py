"""Every kernel form that the number and length of rows (logits) or the number of elements (optimizer) chooses, against the
definitions in 64 bits, with the bounds of test_gpu_logprobs.py and test_gpu_optim.py."""

import math

import numpy as np
import pytest
import torch

from dual_mod_public_amd import _lib as L
from dual_mod_public_amd import logprobs as lp
from dual_mod_public_amd.optim import AdamW
from tests.hip_helpers import DEV, say
from tests.test_gpu_logprobs import check_grad, check_values, rows_of
from tests.test_gpu_optim import B1, B2, EPS, LR, U, coef_of, code_of, hashes, make, value

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    L.load()


# Around 256 rows; row lengths of each tile, in 16-byte vectors (8 bf16, 4 fp32): up to 256, 512, 1024, 4096, 8192, 16384, more
ROWS = [(M, V, BF16) for M in (255, 256) for V in (2048, 3001, 8000, 32000, 50257, 70001)] + \
       [(M, V, FP32) for M in (255, 256) for V in (1023, 2047, 3001, 16000, 32000, 50257)] + \
       [(300, 140001, BF16), (300, 70001, FP32), (1000, 50257, BF16)]


@pytest.mark.parametrize("M,V,dtype", ROWS)
def test_many_rows(M, V, dtype):
    say(f"rows {M} x {V} {dtype}")
    for seed, (pad, base, top) in enumerate(((0, 0, 0), (5, 1, 8))):
        x, t, g, buf = rows_of(M, V, dtype, seed=seed, ld=V + pad, base=base)
        t[::7] = -1
        before = buf.clone()
        w, gh = torch.randn(M, generator=g, device=DEV), torch.randn(M, generator=g, device=DEV)
        r = lp.row_logprobs(x, t, top=top)
        r2, dx = lp.row_logprobs_grad(x, t, w, gh, top=top)
        dx2 = lp.row_logprobs_bwd(x, t, r.stats, w, gh)
        assert torch.equal(buf, before)
        pick = torch.unique(torch.cat([torch.arange(0, M, 17), torch.tensor([1, 127, 128, M - 2, M - 1])])).to(DEV)
        xs, ts, ws, ghs = x[pick], t[pick], w[pick], gh[pick]
        for what, q in (("values", r), ("fused", r2)):
            check_values(xs, ts, top, lp.RowLogprobs(*[None if v is None else v[pick] for v in q]), f"{what} top={top}")
        check_grad(xs, ts, ws, ghs, dx[pick], "fused")
        check_grad(xs, ts, ws, ghs, dx2[pick], "after the values")
        # the rows between them: the same numbers from the other form
        scale = dx2.float().abs().amax(1, keepdim=True)
        assert ((dx.float() - dx2.float()).abs() <= 2 * torch.finfo(dtype).eps * dx2.float().abs() + 1e-4 * scale).all()
        lp.row_logprobs_grad(x, t, w, gh, dlogits=x)
        assert torch.equal(x, dx)


# Elements up to about 5M (8-bit states: 8M) stay in the caches, above 67M nothing does
@pytest.mark.parametrize("n", [6_000_001, 20_000_003, 70_000_001])
@pytest.mark.parametrize("g_dtype", [FP32, BF16])
@pytest.mark.parametrize("max_norm", [None, 0.05])
def test_large_steps32(n, g_dtype, max_norm):
    sizes = [5, 4097, n, 300]
    ps, gs, groups, P, _ = make(sizes, g_dtype, shift=1)
    inside = torch.zeros_like(P, dtype=torch.bool)
    for p in ps:
        inside[p.storage_offset():p.storage_offset() + p.numel()] = True
    around = P[~inside].clone()
    opt = AdamW(groups, grads=gs, lr=LR, betas=(B1, B2), eps=EPS, max_norm=max_norm)
    for t in (1, 2):
        c, norm = coef_of(gs, max_norm)
        before = [p.clone() for p in ps]
        m0, v0 = ([s.clone() for s in opt.views(f)] for f in (opt.exp_avg, opt.exp_avg_sq))
        got = opt.step()
        assert max_norm is None or abs(float(got) - norm) <= U * norm * 1.001
        for i, (p, g) in enumerate(zip(ps, gs)):
            wd, ls = (0.1, 1.0) if i < 2 else (0.0, 0.5)
            gc, m, v = c * g.double(), m0[i].double(), v0[i].double()
            dm = U * (3 * (B1 * m).abs() + 5 * ((1 - B1) * gc).abs())
            dv = U * (3 * B2 * v + 8 * (1 - B2) * gc * gc)
            m, v = B1 * m + (1 - B1) * gc, B2 * v + (1 - B2) * gc * gc
            have_m, have_v = (opt.views(f)[i].double() for f in (opt.exp_avg, opt.exp_avg_sq))
            assert ((have_m - m).abs() <= dm).all() and ((have_v - v).abs() <= dv + 1e-44).all(), (t, i)
            rate, s2 = LR * ls / (1 - B1 ** t), 1 / math.sqrt(1 - B2 ** t)
            denom = have_v.sqrt() * s2 + EPS
            upd = rate * have_m / denom
            want = before[i].double() * (1 - LR * ls * wd) - upd
            tol = U * (3 * before[i].double().abs() + want.abs() + 16 * upd.abs())
            assert ((p.double() - want).abs() <= tol).all(), (t, i)
        for g in gs:
            g.copy_((g.float() * 0.7 - 1e-3).to(g.dtype))
    assert torch.equal(P[~inside], around)


@pytest.mark.parametrize("n", [6_000_001, 20_000_003, 70_000_001])
@pytest.mark.parametrize("g_dtype", [FP32, BF16])
def test_large_steps8(n, g_dtype):
    """The codes of some thousand blocks at the ends and inside, bit for bit, and their elements' parameters."""
    ps, gs, groups, P, _ = make([300, n], g_dtype, shift=1)
    opt = AdamW(groups, grads=gs, lr=LR, betas=(B1, B2), eps=EPS, state_bits=8, seed=77)
    nb, f32 = -(-n // 256), np.float32
    b0 = opt._block0[1]
    runs = [slice(k, min(k + 500, nb)) for k in (0, 7777, nb // 2 + 3, nb - 500)]
    codes = {(r.start, k): (np.zeros((r.stop - r.start, 256), np.uint8), np.ones(r.stop - r.start, np.uint8)) for r in runs for k in (0, 1)}
    for t in (1, 2):
        before = ps[1].clone()
        opt.step()
        for r in runs:
            at = slice(256 * r.start, min(256 * r.stop, n))
            k, full = at.stop - at.start, 256 * (r.stop - r.start)
            g, p0, p1 = (np.pad(x[at].float().cpu().numpy(), (0, full - k)).reshape(-1, 256) for x in (gs[1], before, ps[1]))
            m = value(*codes[r.start, 0], False).astype(f32) * f32(B1) + g * f32(1 - B1)
            v = value(*codes[r.start, 1], True).astype(f32) * f32(B2) + (g * g) * f32(1 - B2)
            h = hashes(77, t, np.uint32(b0 + r.start), r.stop - r.start)
            for j, x, have, exps in ((0, m, opt.exp_avg, opt.exp_avg_exponent), (1, v, opt.exp_avg_sq, opt.exp_avg_sq_exponent)):
                codes[r.start, j] = code_of(x, h, j == 1)
                rows = slice(b0 + r.start, b0 + r.stop)
                assert np.array_equal(exps[rows].cpu().numpy(), codes[r.start, j][1]), (t, r, j)
                assert np.array_equal(have.view(-1, 256)[rows].cpu().numpy(), codes[r.start, j][0]), (t, r, j)
            rate, s2 = LR * 0.5 / (1 - B1 ** t), 1 / math.sqrt(1 - B2 ** t)
            upd = rate * m.astype(np.float64) / (np.sqrt(v.astype(np.float64)) * s2 + EPS)
            want = p0.astype(np.float64) - upd
            assert (np.abs(p1 - want) <= U * (3 * np.abs(p0) + np.abs(want) + 16 * np.abs(upd))).all(), (t, r)
        for g in gs:
            g.copy_((g.float() * 0.7 - 1e-3).to(g.dtype))


@pytest.mark.parametrize("bits", [32, 8])
def test_clipped_step_spreads_nan(bits):
    """A NaN gradient makes the norm, and through it every element, NaN; an infinite one leaves the others where their own
    moments take them (the clipped gradients are zeros)."""
    for bad in (float("nan"), float("inf")):
        ps, gs, groups, P, _ = make([1000, 300])
        opt = AdamW(groups, grads=gs, lr=LR, max_norm=1.0, state_bits=bits)
        gs[0][300] = bad
        norm = opt.step()
        assert not math.isfinite(float(norm))
        if math.isnan(bad):
            assert torch.isnan(ps[0]).all() and torch.isnan(ps[1]).all()
        else:
            assert torch.isnan(ps[0]).nonzero().flatten().tolist() == [300] and not torch.isnan(ps[1]).any()

"""The logit-row operators and the optimizer on the framework's own paths: HipTrunk's weighted objective, score() and
optimizer(), GraphDecoder's log probabilities, DualModLM.token_logprobs, and a run of them together. fp32 against the
oracle's 64-bit model within 1e-5, bf16 within 2e-2 (the bars of the trunk's other tests)."""

import math

import pytest
import torch

import oracle as O
from dual_mod_public_amd import _lib as L
from dual_mod_public_amd.engine import uniform_chunks
from dual_mod_public_amd.graph_decode import GraphDecoder
from dual_mod_public_amd.logprobs import row_logprobs
from dual_mod_public_amd.trunk import HipTrunk
from tests.hip_helpers import DEV, record, relerr, say
from tests.test_gpu_trunk import _batch, _cfg, _memsets, _model

pytestmark = pytest.mark.gpu

B, T = 2, 64
SCHED = uniform_chunks(T, 16, 4)


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    L.load()
    torch.backends.cuda.matmul.allow_tf32 = False


def _weights(seed=4):
    return torch.randn(B, T, generator=torch.Generator().manual_seed(seed))


def _lm(cfg, sd, idx):
    """(leaves, log probabilities of every token [B, T, V]) of the oracle's 64-bit model."""
    leaves = {k: v.double().cpu().clone().requires_grad_(True) for k, v in sd.items() if k != "lm_head.weight"}
    c64, s64 = O.build_rope_cache(T, cfg.head_dim, cfg.rope_theta, dtype=torch.float64)
    logits = O.lm_forward(cfg, dict(leaves, **{"lm_head.weight": leaves["tok_emb.weight"]}), idx.cpu(), c64, s64, schedule=SCHED)
    return leaves, torch.log_softmax(logits, -1)


def _weighted(cfg, sd, idx, tg, w, coef):
    """Loss, gradients, token log probabilities and entropies of the weighted objective."""
    leaves, lp = _lm(cfg, sd, idx)
    valid = tg >= 0
    logp = torch.where(valid, lp.gather(-1, tg.clamp(min=0)[..., None])[..., 0], 0.0)
    ent = -(lp.exp() * lp).sum(-1)
    loss = (-(w.double() * logp) - coef * ent * valid)[valid].sum() / valid.sum()
    loss.backward()
    return loss.detach(), {k: v.grad for k, v in leaves.items()}, logp.detach(), ent.detach()


@pytest.mark.parametrize("dtype,tol,coef,wavefront", [(torch.float32, 1e-5, 0.0, False), (torch.float32, 1e-5, 0.1, False),
                                                      (torch.float32, 1e-5, 0.1, True), (torch.bfloat16, 2e-2, 0.1, False)])
def test_weighted_step_matches_oracle(dtype, tol, coef, wavefront):
    cfg = _cfg()
    m, sd = _model(cfg, dtype)
    tr = HipTrunk(m, B, T, schedule=SCHED, loss_chunk=48, objective="weighted", entropy_coef=coef, wavefront=wavefront)
    idx, tg = _batch(cfg, B, T)
    w = _weights() if dtype == torch.float32 else 0.5 + _weights().abs()   # bf16: no cancellation between tokens
    tr.train_step(idx.to(DEV), tg.to(DEV), w.to(DEV))
    torch.cuda.synchronize()
    loss, grads, logp, ent = _weighted(cfg, sd, idx, tg, w, coef)
    errs = dict({k: relerr(tr.grad[k], v) for k, v in grads.items()}, loss=relerr(tr.loss, loss), logp=relerr(tr.logp, logp),
                entropy=relerr(tr.entropy, ent))
    worst = max(errs, key=errs.get)
    say(f"weighted step {dtype} entropy_coef={coef}: worst {worst} {errs[worst]:.2e}")
    record(f"weighted step {dtype}", errs, tol)
    assert errs[worst] < tol, (worst, errs[worst])


def test_weight_one_is_cross_entropy():
    cfg = _cfg()
    m, _ = _model(cfg, torch.float32)
    idx, tg = (t.to(DEV) for t in _batch(cfg, B, T))
    a = HipTrunk(m, B, T, schedule=SCHED)
    b = HipTrunk(m, B, T, schedule=SCHED, objective="weighted")
    a.train_step(idx, tg)
    b.train_step(idx, tg, _weights().to(DEV))
    assert relerr(a.flat, b.flat) > 0.1
    b.train_step(idx, tg)
    assert relerr(b.loss, a.loss) < 1e-6 and relerr(b.flat, a.flat) < 1e-5


def test_weighted_step_captured():
    """Replays with other batches and weights, eager steps between, equal eager steps bit for bit; no memset recorded."""
    cfg = _cfg()
    m, _ = _model(cfg, torch.bfloat16)
    tr = HipTrunk(m, B, T, schedule=SCHED, loss_chunk=48, objective="weighted", entropy_coef=0.01)
    data = [tuple(t.to(DEV) for t in (*_batch(cfg, B, T, seed=s), _weights(s))) for s in (1, 2, 3)]
    ref = []
    for d in data:
        tr.train_step(*d)
        torch.cuda.synchronize()
        ref.append([t.clone() for t in (tr.loss, tr.flat, tr.logp, tr.entropy)])
    assert _memsets(tr._run) == 0
    tr.capture()
    graph = tr.graph
    for rep in range(2):
        for i in range(3):
            for tr.graph, k in ((graph, i), (None, (i + 1) % 3)):
                tr.train_step(*data[k])
                torch.cuda.synchronize()
                assert all(torch.equal(x, y) for x, y in zip((tr.loss, tr.flat, tr.logp, tr.entropy), ref[k])), (rep, i, k)


def test_objective_refusals():
    cfg = _cfg()
    m, _ = _model(cfg, torch.float32)
    for kw in (dict(objective="other"), dict(entropy_coef=0.1)):
        with pytest.raises(ValueError):
            HipTrunk(m, B, T, schedule=SCHED, **kw)
    idx, tg = (t.to(DEV) for t in _batch(cfg, B, T))
    with pytest.raises(ValueError, match="weights"):
        HipTrunk(m, B, T, schedule=SCHED).train_step(idx, tg, torch.ones(B, T, device=DEV))
    with pytest.raises(ValueError, match="top"):
        GraphDecoder(m, 1, 8, top=33)


@pytest.mark.parametrize("dtype,tol,wavefront", [(torch.float32, 1e-5, False), (torch.bfloat16, 2e-2, True)])
def test_score_matches_oracle(dtype, tol, wavefront):
    cfg = _cfg()
    m, sd = _model(cfg, dtype)
    tr = HipTrunk(m, B, T, schedule=SCHED, loss_chunk=48, wavefront=wavefront)
    idx, tg = _batch(cfg, B, T)
    tr.train_step(idx.to(DEV), tg.to(DEV))
    flat = tr.flat.clone()
    r = tr.score(idx.to(DEV), tg, top=3)
    _, lp = _lm(cfg, sd, idx)
    lp = lp.detach()
    logp = torch.where(tg >= 0, lp.gather(-1, tg.clamp(min=0)[..., None])[..., 0], 0.0)
    errs = dict(logp=relerr(r.logp, logp), entropy=relerr(r.entropy, -(lp.exp() * lp).sum(-1)),
                top=relerr(r.top_logp, lp.topk(3, -1).values))
    record(f"score {dtype}", errs, tol)
    assert max(errs.values()) < tol, errs
    # the tokens themselves where the next one is further off than twice the largest error
    top = lp.topk(4, -1)
    clear = (top.values[..., :3] - top.values[..., 1:]).amin(-1) > 2 * (r.top_logp.double().cpu() - top.values[..., :3]).abs().max()
    assert clear.any() and torch.equal(r.top_ids.cpu()[clear], top.indices[..., :3][clear])
    assert torch.equal(tr.flat, flat) and tr.score(idx.to(DEV), tg).top_ids is None
    tr.train_step(idx.to(DEV), tg.to(DEV))
    assert torch.equal(tr.flat, flat)


@pytest.mark.parametrize("bits", [32, 8])
def test_training_run(bits):
    """Three captured steps of the weighted objective with the optimizer: the parameters against AdamW in 64 bits on the
    trunk's own gradients, the loss after each update against the oracle on the updated parameters; then decoding with
    log probabilities from the trained weights. Twice, with the same bits."""
    cfg = _cfg()
    runs = []
    for repeat in range(2):
        m, _ = _model(cfg, torch.float32)
        tr = HipTrunk(m, B, T, schedule=SCHED, objective="weighted", entropy_coef=0.01)
        opt = tr.optimizer(lr=1e-2, weight_decay=0.1, max_norm=0.5, state_bits=bits, seed=6)
        dec = GraphDecoder(m, B, 16, top=4).capture()
        idx, tg = _batch(cfg, B, T)
        w = _weights()
        tr.capture()
        params = dict(m.named_parameters())
        ref = {n: [p.detach().double().cpu(), 0.0, 0.0] for n, p in params.items()}
        losses = []
        for t in (1, 2, 3):
            losses.append(float(tr.train_step(idx.to(DEV), tg.to(DEV), w.to(DEV))))
            if repeat == 0:
                loss, *_ = _weighted(cfg, {n: p.detach() for n, p in params.items()}, idx, tg, w, 0.01)
                assert relerr(tr.loss, loss) < 1e-5, t
            grads = {n: tr.grad[n].double().cpu() for n in params}
            norm = math.sqrt(sum(float(g.square().sum()) for g in grads.values()))
            got = opt.step()
            assert abs(float(got) - norm) <= 2.0 ** -23 * norm
            tr.refresh()
            if bits == 32:
                for n, (p, mm, v) in ref.items():
                    g = grads[n] * min(1.0, 0.5 / (norm + 1e-6))
                    mm, v = 0.9 * mm + 0.1 * g, 0.999 * v + 0.001 * g * g
                    p = p * (1 - 1e-2 * (0.1 if p.dim() >= 2 else 0.0))
                    p = p - 1e-2 * (mm / (1 - 0.9 ** t)) / ((v / (1 - 0.999 ** t)).sqrt() + 1e-8)
                    ref[n] = [p, mm, v]
                    # an update is at most a few lr; its relative error and that of p are a few 2^-24 a step
                    assert (params[n].double().cpu() - p).abs().max() <= t * 2.0 ** -20 * (p.abs().max() + 1e-2), (t, n)
        assert int(opt.steps) == 3
        # the decoder saw the parameters change
        gen, k = dec.generate(idx[:, :4].to(DEV), 6)
        assert dec.gen_logp.shape == (B, 6) and torch.equal(dec.top_ids[..., 0], dec.next)
        full = torch.cat([idx[:, :4], gen], 1)
        pad = torch.cat([full, torch.zeros(B, T - 10, dtype=torch.long)], 1)
        tg2 = torch.full((B, T), -1)
        tg2[:, 3:9] = full[:, 4:]
        runs.append((losses, [p.detach().clone() for p in params.values()], gen, dec.gen_logp))
        if repeat == 0:
            lp = torch.log_softmax(m(pad.to(DEV))[0].double(), -1).cpu()        # exact scan, as the decoder's
            assert relerr(dec.gen_logp, lp.gather(-1, tg2.clamp(min=0)[..., None])[:, 3:9, 0]) < 1e-5
    assert runs[0][0] == runs[1][0] and torch.equal(runs[0][2], runs[1][2]) and torch.equal(runs[0][3], runs[1][3])
    assert all(torch.equal(a, b) for a, b in zip(runs[0][1], runs[1][1]))


@pytest.mark.parametrize("dtype,top", [(torch.bfloat16, 5), (torch.float32, 0)])
def test_decoder_logprobs(dtype, top):
    """Each replayed step's log probability, entropy and alternatives are its logits'; the tokens are those of a decoder
    without them."""
    cfg = _cfg(vocab_size=521)        # odd: rows without alignment
    m, _ = _model(cfg, dtype)
    plain, dec = GraphDecoder(m, 3, 16).capture(), GraphDecoder(m, 3, 16, top=top).capture()
    prompt = torch.randint(0, 521, (3, 4), generator=torch.Generator().manual_seed(0)).to(DEV)
    for p in range(10):
        for d in (plain, dec):
            d.tok.copy_(prompt[:, p:p + 1] if p < 4 else d.next)
            d.step()
        assert torch.equal(plain.logits, dec.logits) and torch.equal(plain.next, dec.next)
        r = row_logprobs(dec.logits.to(dtype), dec.next, top=top)
        assert torch.equal(dec.logp, r.logp) and torch.equal(dec.entropy, r.entropy)
        if top:
            assert torch.equal(dec.top_ids, r.top_ids) and torch.equal(dec.top_logp, r.top_logp)
            assert torch.equal(dec.top_ids[..., 0], dec.next) and torch.equal(dec.top_logp[..., 0], dec.logp)
    gen, k = dec.generate(prompt, 5)
    gen2, _ = plain.generate(prompt, 5)
    assert torch.equal(gen, gen2) and dec.gen_logp.shape == (3, 5) and plain.gen_logp is None


def test_module_token_logprobs():
    """DualModLM.token_logprobs under autograd: minus its mean over the targets has the loss's value and gradients."""
    cfg = _cfg(n_layers=1)
    m, _ = _model(cfg, torch.float32)
    idx, tg = (t.to(DEV) for t in _batch(cfg, B, T))
    _, loss = m(idx, tg)
    want = torch.autograd.grad(loss, list(m.parameters()))
    logp, ent = m.token_logprobs(idx, tg)
    mine = -logp.sum() / (tg >= 0).sum()
    got = torch.autograd.grad(mine, list(m.parameters()))
    assert relerr(mine, loss) < 1e-6 and ent.shape == (B, T)
    assert all(relerr(a, b) < 1e-5 for a, b in zip(got, want))

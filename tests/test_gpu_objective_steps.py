"""Training steps of the GPT on a policy loss and on a preference loss, against differentiation through the oracle's forward pass in 64 bits."""
import ctypes as C
import math

import pytest
import torch

import femtochat_b200 as fb
from femtochat_b200 import _lib
from oracle import femto_oracle as fo
from test_gpu_step import MID, TC, cosine, inputs

pytestmark = pytest.mark.gpu


def setup(kw, B, dtype, seed=0, **options):
    cfg, ocfg = fb.GPTConfig(**kw), fo.GPTConfig(**kw)
    lay, olay = fb.parameter_layout(cfg), fo.parameter_layout(ocfg)
    th = torch.zeros(lay.nparams)
    fo.initialize(th, ocfg, olay, 5, all_nonzero=True)
    # logits of a model that has seen some text: the initial ones are nearly all zero
    g = torch.Generator().manual_seed(seed)
    head = lay.lm_head
    th[head.offset:head.offset + head.size] = 0.6 * kw["n_embed"] ** -0.5 * torch.randn(head.size, generator=g)
    tok, tgt, pos = inputs(kw, B, seed)
    params = fb.Params(th.cuda())
    st = fb.gradient_state(params, cfg, lay, tok, tgt, pos, compute_type=dtype, **options)
    M = fo.Model(ocfg, fo.StepOptions(eps=fo.EPS_BF16 if dtype == "bfloat16" else fo.EPS_F32, **options))
    return cfg, lay, th, (tok, tgt, pos), params, st, M


def oracle(M, th, batch, objective, temperature=1.0):
    """(loss, gradient, log-probabilities) of objective(logp, valid) by differentiation in 64 bits."""
    tok, tgt, pos = batch
    theta, c = th.double().requires_grad_(), {}
    M.forward(theta, tok, tgt, pos, attention="naive", cache=c)
    ls = torch.log_softmax(c["z"] / temperature, -1)
    lp = torch.where(c["valid"], ls.gather(-1, c["tgt"][..., None])[..., 0], 0.0)
    loss = objective(lp, c["valid"])
    loss.backward()
    return float(loss.detach()), theta.grad, lp.detach()


def numbers(lp, seed, edges=(0.8, 1.28), noise=0.2):
    g = torch.Generator().manual_seed(seed)
    old = lp.double() - noise * torch.randn(lp.shape, generator=g, dtype=torch.float64)
    for e in edges:      # away from where the clipping begins: there two right answers differ
        old = torch.where(((lp - old).exp() / e - 1).abs() < 5e-3, old + 0.02, old)
    A = torch.randn(lp.shape[0], 1, generator=g).expand(lp.shape).contiguous()
    w = torch.rand(lp.shape, generator=g)
    return old.float(), A, (lp + 0.3 * torch.randn(lp.shape, generator=g)).float(), w


def policy(old, A, ref, w, lo, hi, kl, mean):
    def f(lp, valid):
        r = (lp - old.double()).exp()
        loss = -torch.minimum(r * A, r.clamp(1 - lo, 1 + hi) * A)
        if kl:
            gap = ref.double() - lp
            loss = loss + kl * (torch.expm1(gap) - gap)
        if w is not None:
            loss = loss * w
        return torch.where(valid, loss, 0.0).sum() / (valid.sum() if mean else 1)
    return f


def preference(ref, offsets, beta, margin, smoothing, normalised):
    def f(lp, valid):
        gap, v = (lp - ref.double()).flatten(), valid.flatten().double()
        rho = torch.stack([(gap * v)[a:b].sum() / (v[a:b].sum().clamp(min=1) if normalised else 1) for a, b in zip(offsets[:-1], offsets[1:])])
        h = beta * (rho[0::2] - rho[1::2]) - margin
        return (-(1 - smoothing) * torch.nn.functional.logsigmoid(h) - smoothing * torch.nn.functional.logsigmoid(-h)).mean()
    return f


@pytest.mark.parametrize("chunk", ["", "256"])      # one chunk of the lm_head tail, or two
@pytest.mark.parametrize("temperature,kl,reduction", [(1.0, 0.0, "sum"), (0.875, 0.125, "mean")])
def test_policy_step_fp32(chunk, temperature, kl, reduction, monkeypatch):
    if chunk:
        monkeypatch.setenv("FEMTO_XENT_CHUNK", chunk)
    cfg, lay, th, batch, params, st, M = setup(MID, 3, "float32", short_window=32)
    logp = fb.forward_token_logprobs(params, st, lay, *batch, temperature=temperature)
    old, A, ref, w = numbers(logp.cpu(), 1)
    loss, grad, lp = oracle(M, th, batch, policy(old, A, ref, w, 0.2, 0.28, kl, reduction == "mean"), temperature)
    assert float((logp.cpu() - lp).abs().max()) < 1e-5 * (1 + float(lp.abs().max()))
    r = fb.policy_loss_and_gradient_(params, st, lay, batch[0], batch[1], old.cuda(), A.cuda(), positions=batch[2], ref_logp=ref.cuda(), weights=w.cuda(),
                                     clip_low=0.2, clip_high=0.28, kl_coef=kl, temperature=temperature, reduction=reduction)
    g1 = params.delta.cpu()
    assert torch.equal(r.logp, logp) and int(r.n_valid) == int((batch[1] != -1).sum())
    assert 0 < int(r.n_clipped) < int(r.n_valid)
    assert float(r.loss) == pytest.approx(loss, rel=2e-5, abs=2e-5 * float((A.abs() * w).sum() if reduction == "sum" else 1.0))
    assert cosine(grad, g1) >= 0.999999 and float((grad - g1).abs().max()) <= 5e-5 * float(grad.abs().max())
    # a second step adds
    fb.policy_loss_and_gradient_(params, st, lay, batch[0], batch[1], old.cuda(), A.cuda(), positions=batch[2], ref_logp=ref.cuda(), weights=w.cuda(),
                                 clip_low=0.2, clip_high=0.28, kl_coef=kl, temperature=temperature, reduction=reduction, accumulate=True)
    assert float((params.delta.cpu() - 2 * g1).abs().max()) <= 1e-5 * float(g1.abs().max())
    assert st.status_word() == 0


@pytest.mark.parametrize("chunk", ["", "256"])
@pytest.mark.parametrize("normalised", [False, True])
def test_preference_step_fp32(chunk, normalised, monkeypatch):
    if chunk:
        monkeypatch.setenv("FEMTO_XENT_CHUNK", chunk)
    cfg, lay, th, batch, params, st, M = setup(MID, 4, "float32", seed=2, short_window=32)
    T = MID["sequence_len"]
    offsets = [0, 40, 90, 200, 200, 250, 330] if not normalised else [0, T, 2 * T, 3 * T, 4 * T]      # any runs of rows; or a column each
    logp = fb.forward_token_logprobs(params, st, lay, *batch)
    g = torch.Generator().manual_seed(3)
    ref = (logp.cpu() + 0.2 * torch.randn(logp.shape, generator=g)).float()
    beta = 2.0 if normalised else 0.25
    loss, grad, lp = oracle(M, th, batch, preference(ref, offsets, beta, 0.25, 0.125, normalised))
    r = fb.preference_loss_and_gradient_(params, st, lay, batch[0], batch[1], torch.tensor(offsets, dtype=torch.int32, device="cuda"), positions=batch[2],
                                         ref_logp=ref.cuda(), beta=beta, margin=0.25, label_smoothing=0.125, length_normalised=normalised)
    assert torch.equal(r.logp, logp)
    assert float(r.loss) == pytest.approx(loss, rel=1e-4)
    g1 = params.delta.cpu()
    assert cosine(grad, g1) >= 0.99999 and float((grad - g1).abs().max()) <= 5e-4 * float(grad.abs().max())
    # the same numbers from the stand-alone call
    q = fb.preference_loss(logp, torch.tensor(offsets, dtype=torch.int32, device="cuda"), targets0=batch[1].cuda(), ref_logp=ref.cuda(), beta=beta, margin=0.25,
                           label_smoothing=0.125, length_normalised=normalised)
    assert torch.equal(q.loss, r.loss) and torch.equal(q.ratios, r.ratios) and torch.equal(q.pair_losses, r.pair_losses)


@pytest.mark.parametrize("chunk", ["", "256"])
def test_steps_in_bf16_on_the_tensor_cores(chunk, monkeypatch):
    if chunk:
        monkeypatch.setenv("FEMTO_XENT_CHUNK", chunk)
    cfg, lay, th, batch, params, st, M = setup(TC, 4, "bfloat16", seed=4, short_window=128)
    T = TC["sequence_len"]
    logp = fb.forward_token_logprobs(params, st, lay, *batch, temperature=0.75)
    old, A, ref, w = numbers(logp.cpu(), 5, edges=(), noise=0.1)
    # no clipping: in bf16 the oracle's ratios are a few hundredths off
    loss, grad, lp = oracle(M, th, batch, policy(old, A, ref, None, 1.0, 1e9, 0.125, True), 0.75)
    args = dict(positions=batch[2], ref_logp=ref.cuda(), clip_low=1.0, clip_high=None, kl_coef=0.125, temperature=0.75, reduction="mean")
    r = fb.policy_loss_and_gradient_(params, st, lay, batch[0], batch[1], old.cuda(), A.cuda(), **args)
    g1 = params.delta.cpu().clone()
    assert torch.equal(r.logp, logp)      # the very log-probabilities that the call without a gradient gives
    assert float((logp.cpu() - lp).abs().max()) < 0.1 and abs(float(r.loss) - loss) <= 2e-2 * (1 + abs(loss))
    assert cosine(grad, g1) >= 0.995 and abs(float(g1.norm() / grad.norm()) - 1) < 0.03
    fb.policy_loss_and_gradient_(params, st, lay, batch[0], batch[1], old.cuda(), A.cuda(), **args)
    assert torch.equal(g1, params.delta.cpu())
    offsets = [b * T for b in range(5)]
    one = fb.forward_token_logprobs(params, st, lay, *batch)
    ref = one.cpu()
    loss, grad, _ = oracle(M, th, batch, preference(ref, offsets, 0.125, 0.0, 0.0, False))
    q = fb.preference_loss_and_gradient_(params, st, lay, batch[0], batch[1], torch.tensor(offsets, dtype=torch.int32, device="cuda"), positions=batch[2],
                                         ref_logp=ref.cuda(), beta=0.125)
    # the reference is this model: every ratio is exactly 1
    assert torch.equal(q.logp, one) and bool((q.ratios == 0).all()) and float(q.loss) == pytest.approx(math.log(2), rel=1e-6)
    assert cosine(grad, params.delta.cpu()) >= 0.99
    assert st.status_word() == 0


@pytest.mark.parametrize("kw,dtype", [(MID, "float32"), (TC, "bfloat16"), (dict(TC, sequence_len=200), "bfloat16"), (dict(TC, sequence_len=2048), "bfloat16")])
def test_first_update_is_the_plain_policy_gradient(kw, dtype):
    """On the answers' own log-probabilities every ratio is 1, nothing is clipped, and with unit advantages the step is the cross-entropy's."""
    cfg, lay, th, batch, params, st, M = setup(kw, 2, dtype, seed=6)
    loss = fb.loss_and_gradient_(params, st, lay, *batch)
    want = params.delta.clone()
    logp = fb.forward_token_logprobs(params, st, lay, *batch)
    r = fb.policy_loss_and_gradient_(params, st, lay, batch[0], batch[1], logp, torch.ones_like(logp), positions=batch[2])
    n = int((batch[1] != -1).sum())
    assert float(r.loss) == -n and int(r.n_clipped) == 0
    assert -float(logp.double().sum()) == pytest.approx(loss, rel=1e-5 if dtype == "float32" else 2e-3)
    if dtype == "float32":
        assert float((params.delta - want).abs().max()) <= 1e-5 * float(want.abs().max())
    else:      # the cross-entropy takes its statistics from the stored logits, bf16 2^-8 off each
        assert cosine(want, params.delta) >= 0.9999


def test_confident_tokens_in_bf16():
    """Of tokens that the model is all but sure of, softmax - 1 is smaller than the rounding of a stored logit.  With unit advantages and the answers' own
    log-probabilities the step is the cross-entropy's, whose softmax is that of the stored logits.  These are off by half a bf16 step, 2^-9 of x, which
    softcap15 scales by 1 - tanh^2(x / 15): at most 6.8 2^-9 = 0.014, and tanh.approx by 15 2^-11 = 0.008.  A factor e^(z - lse) takes the error of
    two logits, so an element of the two gradients differs by at most 0.044 of itself in either, 0.09 together; its parts of one sign add up in dx, and the
    cosine is 1 - 0.09^2 / 2 at the least where they do not cancel."""
    cfg, lay, th, batch, params, st, M = setup(TC, 8, "bfloat16", seed=10)
    tok, tgt, pos = batch
    g = torch.Generator().manual_seed(11)
    head = slice(lay.lm_head.offset, lay.lm_head.offset + lay.lm_head.size)
    D, V = TC["n_embed"], lay.lm_head.size // TC["n_embed"]
    # the rows that enter the lm_head, read through a head that is the identity; the head that is used gives 64 of them a token each
    th[head] = torch.eye(D, V).flatten()
    x = 15 * torch.atanh(fb.GPT(fb.Params(th.cuda()), cfg, lay, compute_type="bfloat16").logits(tok, pos)[..., :D].cpu().flatten(0, 1) / 15)
    W = D ** -0.5 * torch.randn(D, V, generator=g)
    rows = torch.randperm(x.shape[0], generator=g)[:64]
    W[:, :64] = ((16 + 10 * torch.rand(64, 1, generator=g)) * torch.nn.functional.normalize(x[rows], dim=1)).T * D ** -0.5
    th[head] = W.flatten()
    best = torch.full((x.shape[0],), -1, dtype=torch.int32)
    best[rows] = torch.arange(1, 65, dtype=torch.int32)
    best = best.view(tok.shape)
    params = fb.Params(th.cuda())
    st = fb.gradient_state(params, cfg, lay, tok, tgt, pos, compute_type="bfloat16")
    logp = fb.forward_token_logprobs(params, st, lay, tok, best, pos)
    left = -torch.expm1(logp.double()).cpu()
    chosen = torch.where((left > 2e-4) & (left < 8e-3), best, -1).int()
    assert int((chosen > 0).sum()) >= 8
    fb.loss_and_gradient_(params, st, lay, tok, chosen, pos)
    want = params.delta.clone()
    r = fb.policy_loss_and_gradient_(params, st, lay, tok, chosen, logp, torch.ones_like(logp), positions=pos)
    got = params.delta
    assert int(r.n_valid) == int((chosen > 0).sum()) and int(r.n_clipped) == 0
    assert cosine(want[head], got[head]) >= 0.99 and abs(float(got[head].norm() / want[head].norm()) - 1) < 0.09
    assert cosine(want, got) >= 0.98


def test_a_policy_step_trains_a_model():
    """Log-probabilities, steps and updates in turn, as a training loop calls them, on another stream than the default."""
    cfg, lay, th, batch, params, st, M = setup(TC, 4, "bfloat16", seed=7)
    opt = fb.MuonAdamW(params, lay, st, compute_type="bfloat16")
    A = torch.tensor([1.0, -1.0, 0.5, -0.5], device="cuda")[:, None].expand(4, TC["sequence_len"])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        old = fb.forward_token_logprobs(params, st, lay, *batch)
        for _ in range(3):
            r = fb.policy_loss_and_gradient_(params, st, lay, batch[0], batch[1], old, A, positions=batch[2], kl_coef=0.01, ref_logp=old, reduction="mean")
            assert math.isfinite(float(r.loss)) and bool(params.delta.isfinite().all())
            opt.step(eta=0.1, Nt=float(r.n_valid))
        new = fb.forward_token_logprobs(params, st, lay, *batch)
    side.synchronize()
    assert not torch.equal(old, new) and bool(new.isfinite().all())
    assert st.status_word() == 0


def test_the_step_and_the_call_on_the_model_s_logits_agree():
    """The model's logits through `policy_loss` and `preference_loss`, against the steps that never hold them all."""
    cfg, lay, th, batch, params, st, M = setup(MID, 2, "float32", seed=8, short_window=32)
    tok, tgt, pos = batch
    z = fb.GPT(params, cfg, lay, short_window=32).logits(tok, pos)
    t0 = (torch.where(tgt > 0, tgt - 1, tgt)).int().cuda()
    old, A, ref, w = (x.cuda() for x in numbers(fb.token_logprobs(z, t0).logp.cpu(), 9))
    args = dict(ref_logp=ref, weights=w, clip_low=0.2, clip_high=0.28, kl_coef=0.125, reduction="mean")
    reference = fb.GPT(fb.Params(params.theta.clone()), cfg, lay, short_window=32)      # a model of its own, whose weights it casts itself
    assert torch.equal(reference.token_logprobs(tok, tgt, pos, temperature=0.75), fb.forward_token_logprobs(params, st, lay, tok, tgt, pos, temperature=0.75))
    a = fb.policy_loss(z, t0, old, A, **args)
    b = fb.policy_loss_and_gradient_(params, st, lay, tok, tgt, old, A, positions=pos, **args)
    assert torch.equal(a.n_valid, b.n_valid) and torch.equal(a.n_clipped, b.n_clipped)
    assert float((a.logp - b.logp).abs().max()) < 2e-5 and float(a.loss) == pytest.approx(float(b.loss), rel=1e-4, abs=1e-6)
    offsets = torch.tensor([0, 60, 150], dtype=torch.int32, device="cuda")
    p = fb.preference_loss(a.logp, offsets, targets0=t0, ref_logp=ref, beta=0.5)
    q = fb.preference_loss_and_gradient_(params, st, lay, tok, tgt, offsets, positions=pos, ref_logp=ref, beta=0.5)
    assert float(p.loss) == pytest.approx(float(q.loss), rel=1e-3)
    # one token of a request: its logits from the cache, its log-probability as the whole text has it
    cache = fb.KVCache(st, 2, MID["sequence_len"])
    one = fb.prefill(fb.GPT(params, cfg, lay, short_window=32), cache, tok[:, :10], pos[:, :10])
    assert float((fb.token_logprobs(one, t0[:, 9].contiguous()).logp - b.logp[:, 9]).abs().max()) < 1e-3


def test_steps_refuse_a_decoder():
    layers = [fb.LayerConfig(mixer="lightning", heads=2, dim=16, vdim=16, decay=(0.9, 0.8), ff=64)]
    cfg = fb.DecoderConfig(vocab_size=50, width=32, norm_eps=1e-5, layers=layers)
    st = fb.DecoderState(cfg, max_batch=1, max_rows=8)
    x = torch.zeros(1024, device="cuda")
    i = torch.zeros(8, dtype=torch.int32, device="cuda")
    L, p = _lib.lib(), _lib.ptr
    c, q = C.byref(_lib.PolicyConfigC(1.0, 0.2, 0.2, 0.0, 0)), C.byref(_lib.PreferenceConfigC(0, 0.1, 0.0, 0.0, 0, 1))
    assert L.femto_policy_loss_and_gradient(st.h, p(x), p(x), p(i), p(i), None, 1, p(x), p(x), None, None, c, 0, p(x), p(i), None, None, None) == -5
    assert L.femto_preference_loss_and_gradient(st.h, p(x), p(x), p(i), p(i), None, 1, None, p(i), 1, q, 0, p(x), p(x), p(x), None, None) == -5
    assert L.femto_forward_token_logprobs(st.h, p(x), p(i), p(i), None, 1, 1.0, p(x), None) == -5


def test_steps_refuse():
    cfg, lay, th, batch, params, st, M = setup(MID, 2, "float32")
    z = torch.zeros(2, MID["sequence_len"], device="cuda")
    with pytest.raises(_lib.FemtoError, match="kl_coef needs ref_logp"):
        fb.policy_loss_and_gradient_(params, st, lay, batch[0], batch[1], z, z, kl_coef=0.1)
    with pytest.raises(_lib.FemtoError, match="temperature"):
        fb.policy_loss_and_gradient_(params, st, lay, batch[0], batch[1], z, z, temperature=0.0)
    with pytest.raises(_lib.FemtoError, match="temperature"):
        fb.forward_token_logprobs(params, st, lay, *batch, temperature=-1.0)
    with pytest.raises(ValueError, match="advantages has shape"):
        fb.policy_loss_and_gradient_(params, st, lay, batch[0], batch[1], z, z[:1])
    with pytest.raises(ValueError, match="offsets"):
        fb.preference_loss_and_gradient_(params, st, lay, batch[0], batch[1], torch.zeros(4, dtype=torch.int32, device="cuda"))
    big = torch.cat([batch[0]] * 3)
    with pytest.raises(_lib.FemtoError, match="max_batch"):
        fb.policy_loss_and_gradient_(params, st, lay, big, big, torch.zeros(big.shape, device="cuda"), torch.zeros(big.shape, device="cuda"))
    assert torch.equal(fb.forward_token_logprobs(params, st, lay, *batch), fb.forward_token_logprobs(params, st, lay, *batch))

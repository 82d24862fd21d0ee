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


def rows_of_the_head(params, st, lay, cfg, batch, targets, rows):
    """The bf16 rows that enter the lm_head of a step, as it has them (another pass, as the model call's, may take other kernels and differ by roundings).
    With one target in the batch, in row r, the head's gradient is x_r d, each product of two bf16 numbers exact in fp32: of the numbers that d may be
    at the target, by the row's norm, which is 1 per element within some percent, one makes every x_r a bf16 number."""
    D, Vp = cfg.n_embed, lay.lm_head.size // cfg.n_embed
    out = []
    for r in rows:
        only = torch.full_like(targets, -1).flatten()
        only[r] = targets.flatten()[r]
        only = only.view(targets.shape)
        old = fb.forward_token_logprobs(params, st, lay, batch[0], only, batch[2])
        fb.policy_loss_and_gradient_(params, st, lay, batch[0], only, old, torch.ones_like(old), positions=batch[2])
        column = params.delta[lay.lm_head.offset:lay.lm_head.offset + lay.lm_head.size].view(D, Vp)[:, int(only.flatten()[r]) - 1].cpu().double()
        guess = -float(column.norm()) / D ** 0.5      # the gradient at the target is negative
        first = torch.tensor(1.03 * guess).bfloat16()
        found, d = [], first
        while abs(float(d)) > 0.97 * abs(guess):
            x = column / float(d)      # correctly rounded on the host
            if torch.equal(x, x.bfloat16().double()):
                found.append(x)
            d = torch.nextafter(d, torch.zeros_like(d))
        assert len(found) == 1, (r, len(found))
        out.append(found[0])
    return torch.stack(out).cuda()


@pytest.mark.parametrize("chunk", ["", "256"])
@pytest.mark.parametrize("temperature", [1.0, 0.125, 0.03125])
def test_log_probabilities_and_gradient_at_low_temperatures_in_bf16(chunk, temperature, monkeypatch):
    """The lm_head's product of bf16 numbers, softcapped and divided by the temperature, against 64 bits.  Tolerances: a product's sum of D exact terms has
    at most D / 8 roundings of 2^-23 of sum |x w| in the tensor cores; tanh_fp32 is 5e-7 off, 8e-6 of a logit: `dz` together, divided by the temperature
    in a log-probability, of the target and of the others.  An element of the gradient is made from a logit stored in fp16: half a step, 2^-11 of x,
    or x (1 - tanh^2) 2^-11 behind the softcap; and twice that relative to x in 1 - tanh^2.  It is rounded to bf16, 2^-8."""
    if chunk:
        monkeypatch.setenv("FEMTO_XENT_CHUNK", chunk)
    cfg, lay, th, batch, params, st, M = setup(TC, 2, "bfloat16", seed=12)
    tok, tgt, pos = batch
    D, Vp, V = TC["n_embed"], lay.lm_head.size // TC["n_embed"], TC["vocab_size"]
    head = slice(lay.lm_head.offset, lay.lm_head.offset + lay.lm_head.size)
    rows = [0, 1, 130, 255, 256, 300, 301, 511]
    targets = torch.randint(1, V + 1, tok.shape, generator=torch.Generator().manual_seed(3), dtype=torch.int32).cuda()
    x = rows_of_the_head(params, st, lay, cfg, batch, targets, rows)
    W = th[head].view(D, Vp)[:, :V].cuda().bfloat16().double()
    y = x @ W
    th15 = torch.tanh(y / 15)
    ls = torch.log_softmax(15 * th15 / temperature, 1)
    # half of the tokens are the likeliest, the others what was drawn
    t0 = targets.flatten()[rows].long() - 1
    t0[::2] = torch.argmax(y, 1)[::2]
    targets.view(-1)[rows] = t0.int() + 1
    lp = ls.gather(1, t0[:, None])[:, 0]
    dz = float((x.abs() @ W.abs()).max()) * D / 8 * 2.0 ** -23 + 8e-6
    got = fb.forward_token_logprobs(params, st, lay, tok, targets, pos, temperature=temperature)
    error = (got.double().flatten()[rows] - lp).abs()
    tol = 2 * dz / temperature + 2.0 ** -23 * (lp.abs() + 16) + 1e-6
    assert not bool((error > tol).any()), (float(error.max()), float(tol.min()))
    # one row at a time has a target: with ratios of 1 and an advantage of 1 its column of the head's gradient is x (p - 1[target]) (1 - tanh^2) / temperature
    for k, r in enumerate(rows):
        only = torch.full_like(targets, -1).flatten()
        only[r] = targets.flatten()[r]
        only = only.view(tok.shape)
        q = fb.policy_loss_and_gradient_(params, st, lay, tok, only, got, torch.ones_like(got), positions=pos, temperature=temperature)
        assert float(q.loss) == -1 and int(q.n_valid) == 1 and float(q.logp.flatten()[r]) == float(got.flatten()[r])
        i, t = int(torch.argmax(x[k].abs())), int(t0[k])
        d = params.delta[head].view(D, Vp)[i, :V].double() / x[k, i]
        slope = 1 - th15[k] ** 2
        want = ls[k].exp() * slope / temperature
        want[t] = torch.expm1(lp[k]) * slope[t] / temperature
        off = (y[k].abs() * slope * 2.0 ** -11 + 2 * dz) / temperature      # of the exponent
        rel = torch.expm1(off) + 2 * 2.0 ** -11 * y[k].abs() / 15 + 2.0 ** -8 * 1.01 + 1e-5
        rel[t] = 2 * 2.0 ** -11 * y[k, t].abs() / 15 + 2.0 ** -8 * 1.01 + 1e-5
        tol = rel * want.abs() + 1e-30
        tol[t] += tolerance_of_p(lp[k], 2 * dz / temperature) * slope[t] / temperature
        bad = (d - want).abs() > tol
        assert not bad.any(), (r, int(bad.sum()), float(((d - want).abs() / (want.abs() + 1e-30))[bad].max()))
    assert st.status_word() == 0


def tolerance_of_p(lp, off):
    """How far p is off where log p + log(1 / (1 - p)), the target's logit relative to the others', is `off`: p (1 - p) off, and the second order."""
    p = torch.exp(lp)
    return p * (1 - p) * torch.expm1(torch.tensor(off))


@pytest.mark.parametrize("kw,dtype", [(MID, "float32"), (TC, "bfloat16")])
def test_steps_on_confident_tokens(kw, dtype):
    """Tokens of 1 - p from 1e-8 to 1e-2: the step's -log p has its own precision, where a difference of logsumexp and logit in fp32 would leave 1e-6.  The
    head gives chosen rows a token each; what the model then gives them is compared with 64 bits for the rows that enter the head in bf16, or in fp32 for the
    logits of the model call: another pass in fp32, whose logits, 15 at most, are within 2^-17 of themselves (1e-4) of the step's."""
    cfg, lay, th, batch, params, st, M = setup(kw, 2, dtype, seed=13)
    tok, tgt, pos = batch
    D, Vp, V = kw["n_embed"], lay.lm_head.size // kw["n_embed"], kw["vocab_size"]
    head = slice(lay.lm_head.offset, lay.lm_head.offset + lay.lm_head.size)
    t = th.clone()
    t[head] = torch.eye(D, Vp).flatten()
    x = 15 * torch.atanh(fb.GPT(fb.Params(t.cuda()), cfg, lay, compute_type=dtype).logits(tok, pos)[..., :D].double().flatten(0, 1) / 15)
    n = 32
    W = D ** -0.5 * torch.randn(D, V, generator=torch.Generator().manual_seed(1)) * 0.5
    rows = torch.randperm(x.shape[0], generator=torch.Generator().manual_seed(2))[:n].tolist()
    W[:, :n] = (torch.linspace(10, 40, n)[:, None] * torch.nn.functional.normalize(x[rows].float().cpu(), dim=1)).T * D ** -0.5
    full = torch.zeros(D, Vp)
    full[:, :V] = W
    th[head] = full.flatten()
    params = fb.Params(th.cuda())
    st = fb.gradient_state(params, cfg, lay, tok, tgt, pos, compute_type=dtype)
    targets = torch.full((tok.numel(),), -1, dtype=torch.int32)
    targets[rows] = torch.arange(1, n + 1, dtype=torch.int32)
    targets = targets.view(tok.shape).cuda()
    if dtype == "bfloat16":
        x = rows_of_the_head(params, st, lay, cfg, batch, targets, rows)
        W = W.cuda().bfloat16().double()
        z = 15 * torch.tanh(x @ W / 15)
        dz = float((x.abs() @ W.abs()).max()) * D / 8 * 2.0 ** -23 + 8e-6
    else:
        z, dz = fb.GPT(params, cfg, lay).logits(tok, pos).double().flatten(0, 1)[rows], 1e-4
    ls = torch.log_softmax(z, 1)
    own = torch.arange(n, device="cuda")
    want = ls[own, own]
    ls[own, own] = -math.inf
    left = ls.exp().sum(1)
    got = fb.forward_token_logprobs(params, st, lay, tok, targets, pos)
    lp = got.flatten()[rows].double()
    sure = (left > 1e-8) & (left < 1e-2)
    assert int(sure.sum()) >= 5
    # every logit dz off: 1 - p by 2 dz of itself; and the roundings of a sum of V exponentials
    rel = 2 * dz * 1.01 + 2.0 ** -20 + V * 2.0 ** -24
    assert not bool(((lp - want).abs() > rel * want.abs())[sure].any()), float(((lp - want) / want)[sure].abs().max())
    step = fb.policy_loss_and_gradient_(params, st, lay, tok, targets, got, torch.ones_like(got), positions=pos)
    assert torch.equal(step.logp, got)


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


@pytest.mark.parametrize("kw,dtype", [(MID, "float32"), (TC, "bfloat16")])
def test_captured_steps(kw, dtype):
    """A step in a graph, replayed on other tokens while eager steps run in between, gives what the eager step gives."""
    cfg, lay, th, batch, params, st, M = setup(kw, 2, dtype, seed=14)
    tok, tgt, pos = (x.cuda() for x in batch)
    other, theirs, _ = (x.cuda() for x in inputs(kw, 2, 15))
    T = kw["sequence_len"]
    old = fb.forward_token_logprobs(params, st, lay, tok, tgt, pos) + 0.1
    A, offsets = torch.randn(old.shape, device="cuda"), torch.tensor([0, T, 2 * T], dtype=torch.int32, device="cuda")
    calls = [lambda: fb.policy_loss_and_gradient_(params, st, lay, tok, tgt, old, A, positions=pos, reduction="mean"),
             lambda: fb.preference_loss_and_gradient_(params, st, lay, tok, tgt, offsets, positions=pos, ref_logp=old),
             lambda: (fb.forward_token_logprobs(params, st, lay, tok, tgt, pos),)]
    graphs = []
    for call in calls:
        call()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    tok.copy_(other), tgt.copy_(theirs)
    for _ in range(2):
        for call, (g, out) in zip(calls, graphs):
            params.delta.zero_()
            g.replay()
            got, delta = [x.clone() for x in out], params.delta.clone()
            params.delta.zero_()
            assert all(torch.equal(a, b) for a, b in zip(got, call())) and torch.equal(delta, params.delta)
    assert st.status_word() == 0


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

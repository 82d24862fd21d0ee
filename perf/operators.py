"""The operators that train a model on its own answers, as cases that can be timed and checked: log-probabilities of chosen tokens with
their entropy and the gradient of both, the clipped policy loss with a KL term on logits, and the paired preference loss.

`listed()` names cases over the range of sizes, `draw(rng)` gives others of the same ranges.  `prepare` builds what a program holds
before the call, `run` makes one pass through one operator: with `own` through the framework's entry points, else in elementary torch
operations in 32 bits.  `exact` gives the results in 64 bits, written from the definitions."""
import math

import torch

own = False

LN2 = math.log(2.0)
CLIP = (0.2, 0.28)      # how far the ratio may fall and rise


def case_logprobs(name, dtype, N, V, pitch=0, temperature=1.0, entropy=False, masked=0.0):
    return dict(name=name, op="logprobs", dtype=dtype, N=N, V=V, pitch=pitch, temperature=temperature, entropy=entropy, masked=masked)


def case_gradient(name, dtype, N, V, pitch=0, temperature=1.0, entropy=False, masked=0.0):
    return dict(name=name, op="gradient", dtype=dtype, N=N, V=V, pitch=pitch, temperature=temperature, entropy=entropy, masked=masked)


def case_policy(name, dtype, B, T, V, pitch=0, temperature=1.0, kl=0.0, prompt=0.25, reduction="sum", gradient=True):
    return dict(name=name, op="policy", dtype=dtype, B=B, T=T, V=V, pitch=pitch, temperature=temperature, kl=kl, prompt=prompt,
                reduction=reduction, gradient=gradient)


def case_preference(name, pairs, length, kind="sigmoid", reference=True, normalised=False, masked=0.0):
    return dict(name=name, op="preference", pairs=pairs, length=length, kind=kind, reference=reference, normalised=normalised, masked=masked)


def listed():
    return [
        # one sampled token of one request: the logits of a decode step, whose latency counts
        case_logprobs("logprobs f32 1x65536", "float32", 1, 65536),
        # sixteen requests in step, sampled at a temperature, with the entropy that is watched
        case_logprobs("logprobs f32 16x65536 entropy", "float32", 16, 65536, temperature=0.8, entropy=True),
        # scoring finished answers under a reference model: many tokens, half of them prompt
        case_logprobs("logprobs bf16 4096x65536", "bfloat16", 4096, 65536, masked=0.5),
        # an objective written by the user on log-probabilities and entropies: its way back to logits whose rows start anywhere
        case_gradient("gradient f32 999x50021 entropy", "float32", 999, 50021, temperature=0.8, entropy=True, masked=0.3),
        # the same of a batch
        case_gradient("gradient bf16 4096x65536", "bfloat16", 4096, 65536, masked=0.25),
        # a small model in the default type
        case_policy("policy f32 2x100x4096", "float32", 2, 100, 4096, kl=0.05),
        # evaluation of the objective only, token mean
        case_policy("policy f32 4x256x32768 loss only", "float32", 4, 256, 32768, kl=0.05, reduction="mean", gradient=False),
        # answers of a batch, logits cut from a padded vocabulary whose size is odd
        case_policy("policy f32 3x333x50021", "float32", 3, 333, 50021, pitch=43, temperature=0.8, reduction="mean"),
        # the benchmark's vocabulary, a full batch of answers in bf16
        case_policy("policy bf16 8x512x65536", "bfloat16", 8, 512, 65536, kl=0.02),
        # one pair of short answers
        case_preference("preference 1x24", 1, 24),
        # a batch of pairs of ragged answers, prompts masked
        case_preference("preference 16x1000 normalised", 16, 1000, reference=False, normalised=True, masked=0.5),
        # many pairs of long answers at once, as log-probabilities kept of a whole epoch
        case_preference("preference 1024x2048", 1024, 2048, masked=0.25),
    ]


def log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    case = draw_any(rng)
    del case["name"]
    return case


def draw_any(rng):
    op = rng.choice(("logprobs", "gradient", "policy", "policy", "preference"))
    if op == "preference":
        pairs, length = log_int(rng, 1, 1024), log_int(rng, 2, 2048)
        return case_preference(None, pairs, length, kind=rng.choice(("sigmoid", "sigmoid", "squared")), reference=rng.random() < 0.7,
                               normalised=rng.random() < 0.3, masked=rng.choice((0.0, 0.3, 0.6))) | dict(shape_seed=rng.randrange(1 << 30))
    dtype = rng.choice(("float32", "bfloat16"))
    V = rng.choice((4096, 32768, 65536)) if rng.random() < 0.3 else log_int(rng, 200, 130000)
    most = max(2, min(8192, (120_000_000 if dtype == "float32" else 240_000_000) // V))
    pitch = 0 if rng.random() < 0.5 else rng.randrange(1, 64)
    temperature = rng.choice((1.0, 1.0, 0.7, 1.3))
    if op == "policy":
        B = log_int(rng, 1, min(16, most))
        return case_policy(None, dtype, B, log_int(rng, 1, most // B), V, pitch=pitch, temperature=temperature, kl=rng.choice((0.0, 0.05)),
                           prompt=rng.choice((0.0, 0.25, 0.6)), reduction=rng.choice(("sum", "mean")), gradient=rng.random() < 0.8)
    make = case_logprobs if op == "logprobs" else case_gradient
    return make(None, dtype, log_int(rng, 1, most), V, pitch=pitch, temperature=temperature, entropy=rng.random() < 0.4, masked=rng.choice((0.0, 0.3, 0.6)))


# ---- what a program holds before the call ---------------------------------------------------------------------------------------------
def generator(seed, salt=0):
    return torch.Generator(device="cuda").manual_seed(1000 * seed + salt)


def rows_of(case):
    return case["B"] * case["T"] if case["op"] == "policy" else case["N"]


def masked_of(case):
    """Rows without a target: the prompt of every answer, or the first rows."""
    if case["op"] == "policy":
        return case["B"] * int(case["prompt"] * case["T"])
    return int(case["masked"] * case["N"])


def make_logits(case, seed):
    """Soft-capped logits as the model gives them, a token drawn from each row's softmax, and that token's log-probability in 64 bits.
    The rows are the first V columns of a wider buffer where the case has a pitch."""
    N, V = rows_of(case), case["V"]
    g = generator(seed)
    logits = torch.empty(N, V + case["pitch"], device="cuda", dtype=getattr(torch, case["dtype"]))[:, :V]
    targets = torch.empty(N, device="cuda", dtype=torch.int32)
    logp = torch.empty(N, device="cuda", dtype=torch.float64)
    common = 2.0 * torch.randn(V, device="cuda", generator=g)         # some tokens are frequent everywhere
    step = max(1, (1 << 26) // V)
    for i in range(0, N, step):
        n = min(step, N - i)
        x = 2.5 * torch.randn(n, V, device="cuda", generator=g) + common
        logits[i:i + n] = (15.0 * torch.tanh(x / 15.0)).to(logits.dtype)
        s = logits[i:i + n].double() / case["temperature"]
        u = torch.rand(n, V, device="cuda", generator=g).clamp_(1e-20, 1.0)
        t = torch.argmax(s.float() - torch.log(-torch.log(u)), dim=1)
        targets[i:i + n] = t.int()
        logp[i:i + n] = s.gather(1, t[:, None])[:, 0] - torch.logsumexp(s, dim=1)
    return logits, targets, logp


def prepare(case, seed):
    if case["op"] == "preference":
        return prepare_preference(case, seed)
    logits, targets, logp = make_logits(case, seed)
    N = rows_of(case)
    st = dict(case=case, logits=logits)
    g = generator(seed, 1)
    if case["op"] != "policy":
        targets[:masked_of(case)] = -1
        st["targets"] = targets
        if case["op"] == "gradient":
            # the gradient of the user's objective
            st["dlogp"] = torch.randn(N, device="cuda", generator=g) / N
            st["dentropy"] = 0.1 * torch.randn(N, device="cuda", generator=g) / N if case["entropy"] else None
        return st
    B, T = case["B"], case["T"]
    targets.view(B, T)[:, :int(case["prompt"] * T)] = -1
    # log-probabilities from some updates ago, and of the reference.  The objective has a kink where the ratio leaves its range, and there
    # two right answers differ: tokens within 0.2 percent of it are moved off.
    old = logp - 0.15 * torch.randn(N, device="cuda", generator=g, dtype=torch.float64)
    for edge in (1.0 - CLIP[0], 1.0 + CLIP[1]):
        old = torch.where((torch.exp(logp - old) / edge - 1.0).abs() < 2e-3, old + 0.01, old)
    rewards = torch.randn(B, 1, device="cuda", generator=g)
    st.update(targets=targets.view(B, T), logits=logits.unflatten(0, (B, T)), old=old.float().view(B, T),
              advantages=rewards.expand(B, T).contiguous(),
              ref=(logp + 0.3 * torch.randn(N, device="cuda", generator=g, dtype=torch.float64)).float().view(B, T) if case["kl"] else None,
              # a sum over tokens is one over answers, each divided by its length
              weights=torch.full((B, T), 1.0 / (B * (T - int(case["prompt"] * T))), device="cuda") if case["reduction"] == "sum" else None)
    return st


def lengths_of(case):
    """Lengths of the chosen and the rejected answers in turn: ragged, up to the case's, one in fifty empty where there are many."""
    g = torch.Generator().manual_seed(case["pairs"] * 65537 + case["length"] + case.get("shape_seed", 0))
    n = torch.randint(max(1, case["length"] // 2), case["length"] + 1, (2 * case["pairs"],), generator=g)
    if case["pairs"] > 8:
        n[torch.rand(2 * case["pairs"], generator=g) < 0.02] = 0
    return n


def prepare_preference(case, seed):
    g = generator(seed, 2)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(lengths_of(case), 0)]).int().cuda()
    N = int(lengths_of(case).sum())
    logp = -torch.empty(N, device="cuda").exponential_(0.7, generator=g)
    ref = logp + 0.1 * torch.randn(N, device="cuda", generator=g) if case["reference"] else None
    targets = torch.randint(0, 65536, (N,), device="cuda", dtype=torch.int32, generator=g)
    if case["masked"]:
        targets[torch.rand(N, device="cuda", generator=g) < case["masked"]] = -1
        logp[targets < 0] = 0.0
    return dict(case=case, logp=logp, ref=ref, targets=targets if case["masked"] else None, offsets=offsets)


# ---- one pass -------------------------------------------------------------------------------------------------------------------------
def run(state):
    return (run_own if own else run_plain)(state)


def beta_of(case):
    return 2.0 if case["normalised"] else 0.1


def run_own(state):
    import femtochat_b200 as fb
    case = state["case"]
    op = case["op"]
    if op == "logprobs":
        r = fb.token_logprobs(state["logits"], state["targets"], temperature=case["temperature"], entropy=case["entropy"])
        return (r.logp, r.entropy) if case["entropy"] else r.logp
    if op == "gradient":
        return fb.token_logprobs_gradient(state["logits"], state["targets"], state["dlogp"], dentropy=state["dentropy"], temperature=case["temperature"])
    if op == "policy":
        r = fb.policy_loss(state["logits"], state["targets"], state["old"], state["advantages"], ref_logp=state["ref"], weights=state["weights"],
                           clip_low=CLIP[0], clip_high=CLIP[1], kl_coef=case["kl"], temperature=case["temperature"], reduction=case["reduction"],
                           gradient=case["gradient"])
        out = (r.loss, r.n_valid, r.n_clipped, r.token_losses, r.logp)
        return out + (r.dlogits,) if case["gradient"] else out
    r = fb.preference_loss(state["logp"], state["offsets"], targets0=state["targets"], ref_logp=state["ref"], kind=case["kind"], beta=beta_of(case),
                           margin=0.5 if case["normalised"] and case["kind"] == "sigmoid" else 0.0,
                           label_smoothing=0.1 if case["kind"] == "sigmoid" else 0.0, length_normalised=case["normalised"], reduction="mean")
    return r.loss, r.pair_losses, r.ratios, r.dlogp


def softmax_parts(logits, targets, temperature):
    """Scaled logits, their log-sum-exp, the target's log-probability (0 without a target), in 32 bits."""
    s = logits.float() * (1.0 / temperature)
    m = s.max(dim=-1).values
    lse = m + torch.log(torch.exp(s - m[..., None]).sum(-1))
    has = targets >= 0
    st = s.gather(-1, targets.clamp(min=0).long()[..., None])[..., 0]
    return s, lse, torch.where(has, st - lse, 0.0), has


def run_plain(state):
    case = state["case"]
    op = case["op"]
    if op == "preference":
        return plain_preference(state)
    if op == "logprobs":
        s, lse, logp, has = softmax_parts(state["logits"], state["targets"], case["temperature"])
        if not case["entropy"]:
            return logp
        ls = s - lse[:, None]
        return logp, torch.where(has, -(torch.exp(ls) * ls).sum(1), 0.0)
    targets = state["targets"]
    if op == "gradient":
        s, lse, _, _ = softmax_parts(state["logits"], targets, case["temperature"])
        ls = s - lse[:, None]
        p = torch.exp(ls)
        d = -p * state["dlogp"][:, None]
        d.scatter_add_(1, targets.clamp(min=0).long()[:, None], state["dlogp"][:, None])
        if case["entropy"]:
            d -= state["dentropy"][:, None] * p * (ls - (p * ls).sum(1)[:, None])
        return torch.where((targets >= 0)[:, None], d * (1.0 / case["temperature"]), 0.0).to(state["logits"].dtype)
    s, lse, logp, has = softmax_parts(state["logits"], targets, case["temperature"])
    A = state["advantages"]
    n_valid = has.sum()
    ratio = torch.exp(logp - state["old"])
    clipped = torch.where(A > 0, ratio > 1.0 + CLIP[1], (A < 0) & (ratio < 1.0 - CLIP[0])) & has
    token = -torch.minimum(ratio * A, ratio.clamp(1.0 - CLIP[0], 1.0 + CLIP[1]) * A)
    slope = torch.where(clipped, 0.0, -ratio * A)
    if case["kl"]:
        gap = state["ref"] - logp
        token = token + case["kl"] * (torch.exp(gap) - gap - 1.0)
        slope = slope + case["kl"] * (1.0 - torch.exp(gap))
    scale = state["weights"] if case["reduction"] == "sum" else 1.0 / n_valid.float()
    raw = torch.where(has, token * (state["weights"] if state["weights"] is not None else 1.0), 0.0)
    loss = raw.sum() * (1.0 if case["reduction"] == "sum" else scale)
    out = (loss.reshape(1), n_valid.int().reshape(1), clipped.sum().int().reshape(1), raw, logp)
    if not case["gradient"]:
        return out
    coef = torch.where(has, slope * scale, 0.0) * (1.0 / case["temperature"])
    d = -coef[..., None] * torch.exp(s - lse[..., None])
    d.scatter_add_(-1, targets.clamp(min=0).long()[..., None], coef[..., None])
    return out + (d.to(state["logits"].dtype),)


def plain_preference(state):
    case = state["case"]
    offsets = state["offsets"].long()
    N, S = state["logp"].shape[0], 2 * case["pairs"]
    counted = (state["targets"] >= 0) if state["targets"] is not None else torch.ones(N, device="cuda", dtype=torch.bool)
    owner = torch.repeat_interleave(torch.arange(S, device="cuda"), offsets[1:] - offsets[:-1], output_size=N)
    gap = state["logp"] - state["ref"] if state["ref"] is not None else state["logp"]
    # long sums that nearly cancel: in 64 bits
    rho = torch.zeros(S, device="cuda", dtype=torch.float64).scatter_add_(0, owner, torch.where(counted, gap, 0.0).double())
    count = torch.zeros(S, device="cuda", dtype=torch.float64).scatter_add_(0, owner, counted.double())
    per = 1.0 / count.clamp(min=1.0) if case["normalised"] else torch.ones_like(count)
    rho = rho * per
    delta = rho[0::2] - rho[1::2]
    beta = beta_of(case)
    if case["kind"] == "sigmoid":
        h = beta * delta - (0.5 if case["normalised"] else 0.0)
        e = 0.1
        softplus = torch.log1p(torch.exp(-h.abs()))
        losses = (1 - e) * (softplus + (-h).clamp(min=0)) + e * (softplus + h.clamp(min=0))
        slope = beta * (1.0 / (1.0 + torch.exp(-h)) - (1 - e))
    else:
        losses = (delta - 0.5 / beta) ** 2
        slope = 2.0 * (delta - 0.5 / beta)
    per_sequence = torch.stack([slope, -slope], 1).flatten() * per / case["pairs"]
    dlogp = torch.where(counted, per_sequence[owner], 0.0)
    return losses.mean().float().reshape(1), losses.float(), rho.float(), dlogp.float()


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "preference":
        return exact_preference(state)
    V = case["V"]
    logits, targets = state["logits"].flatten(0, -2), state["targets"].flatten()
    N = targets.shape[0]
    has = targets >= 0
    index = targets.clamp(min=0).long()
    logp = torch.zeros(N, device="cuda", dtype=torch.float64)
    entropy = torch.zeros_like(logp)
    step = max(1, (1 << 26) // V)
    for i in range(0, N, step):
        rows = slice(i, min(N, i + step))
        ls = torch.log_softmax(logits[rows].double() / case["temperature"], dim=1)
        logp[rows] = ls[torch.arange(ls.shape[0], device="cuda"), index[rows]]
        entropy[rows] = -(ls.exp() * ls).sum(1)
    zero = torch.zeros_like(logp)
    if op == "logprobs":
        return (torch.where(has, logp, zero), torch.where(has, entropy, zero)) if case["entropy"] else torch.where(has, logp, zero)

    def gradient(dlogp, dentropy=None):
        """Through log p(target) and the entropy to the logits."""
        d = torch.empty(N, V, device="cuda", dtype=torch.float64)
        for i in range(0, N, step):
            rows = slice(i, min(N, i + step))
            ls = torch.log_softmax(logits[rows].double() / case["temperature"], dim=1)
            p = ls.exp()
            onehot = torch.nn.functional.one_hot(index[rows], V)
            d[rows] = dlogp[rows, None] * (onehot - p)
            if dentropy is not None:
                d[rows] -= dentropy[rows, None] * p * (ls + entropy[rows, None])
        return d.mul_(1.0 / case["temperature"])

    if op == "gradient":
        return gradient(torch.where(has, state["dlogp"].double(), zero), torch.where(has, state["dentropy"].double(), zero) if case["entropy"] else None)
    old, A = state["old"].flatten().double(), state["advantages"].flatten().double()
    w = state["weights"].flatten().double() if state["weights"] is not None else torch.ones_like(logp)
    ratio = (logp - old).exp()
    lo, hi = 1.0 - CLIP[0], 1.0 + CLIP[1]
    unclipped, bounded = ratio * A, ratio.clamp(lo, hi) * A
    clipped = has & (bounded < unclipped)
    token, slope = -torch.minimum(unclipped, bounded), torch.where(clipped, zero, -unclipped)
    if case["kl"]:
        ref = state["ref"].flatten().double()
        token = token + case["kl"] * (torch.expm1(ref - logp) - (ref - logp))
        slope = slope - case["kl"] * torch.expm1(ref - logp)
    n = int(has.sum())
    mean = 1.0 / n if case["reduction"] == "mean" else 1.0
    raw = torch.where(has, w * token, zero)
    shape = state["targets"].shape
    out = ((raw.sum() * mean).reshape(1), torch.tensor([n], device="cuda", dtype=torch.int32), clipped.sum().int().reshape(1), raw.view(shape),
           torch.where(has, logp, zero).view(shape))
    if not case["gradient"]:
        return out
    return out + (gradient(torch.where(has, w * mean * slope, zero)).view(shape + (V,)),)


def exact_preference(state):
    case = state["case"]
    lp = state["logp"].double()
    if state["ref"] is not None:
        lp = lp - state["ref"].double()
    counted = (state["targets"] >= 0).double() if state["targets"] is not None else torch.ones_like(lp)
    starts = state["offsets"].long()
    lengths = starts[1:] - starts[:-1]

    def per_answer(x):
        total = torch.cat([torch.zeros(1, device="cuda", dtype=torch.float64), torch.cumsum(x, 0)])
        return total[starts[1:]] - total[starts[:-1]]

    rho, count = per_answer(lp * counted), per_answer(counted)
    scale = torch.ones_like(count)
    if case["normalised"]:
        scale = torch.where(count > 0, 1.0 / count.clamp(min=1), 0.0)
    rho = rho * scale
    delta = (rho[0::2] - rho[1::2]).requires_grad_()
    beta = beta_of(case)
    if case["kind"] == "sigmoid":
        h = beta * delta - (0.5 if case["normalised"] else 0.0)
        losses = -0.9 * torch.nn.functional.logsigmoid(h) - 0.1 * torch.nn.functional.logsigmoid(-h)
    else:
        losses = (delta - 0.5 / beta).square()
    slope, = torch.autograd.grad(losses.mean(), delta)
    d = torch.stack([slope, -slope], 1).flatten() * scale
    return losses.mean().detach().reshape(1), losses.detach(), rho, torch.repeat_interleave(d, lengths, output_size=lp.shape[0]) * counted


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "preference":
        N, P = int(lengths_of(case).sum()), case["pairs"]
        arrays = 2 + (1 if case["reference"] else 0) + (1 if case["masked"] else 0)      # log-probabilities in, gradient out, ...
        return {"bytes": 4 * N * arrays + 4 * (2 * P + 1) + 12 * P, "flops": 4 * N}
    N, V, size = rows_of(case), case["V"], 4 if case["dtype"] == "float32" else 2
    live = N - masked_of(case)
    if case["op"] == "logprobs":      # a scale, an exponential, a sum
        return {"bytes": live * V * size + 4 * N * (3 if case["entropy"] else 2), "flops": (5 if case["entropy"] else 3) * live * V}
    if case["op"] == "gradient":
        return {"bytes": (live + N) * V * size + 4 * N * (3 if case["entropy"] else 2), "flops": (9 if case["entropy"] else 6) * live * V}
    rows = 4 * N * (5 + (1 if case["kl"] else 0) + (1 if case["reduction"] == "sum" else 0))
    return {"bytes": (live + (N if case["gradient"] else 0)) * V * size + rows, "flops": (7 if case["gradient"] else 3) * live * V}

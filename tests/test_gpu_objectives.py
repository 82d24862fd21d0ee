"""Objectives on a model's own answers against their definitions in 64 bits.

Tolerances.  A log-probability is ln2 u - log l with l a sum of V exponentials.  Relative errors of l: 2^-22 of an exponential, 2^-24 ln2 |u|
of its argument (|u| < 64 wherever 2^u counts), and at most one rounding per addition; a chain of additions is no longer than V / 256 + 48 in any
form of the kernels.  The scale log2(e) / temperature is rounded once, which moves a log-probability by at most 2^-24 of its distance from the
row's mean of log p, |lp| + H; the result is rounded to fp32.  So an error of `slack(V)` + 2^-23 (|lp| + H + 1), slack(V) = 2^-22 + 2^-24 (V / 256 + 96).
A probability has the relative error of l, twice (its own exponential, and 1 / l)."""
import ctypes as C
import math

import pytest
import torch

import femtochat_b200 as fb
from femtochat_b200 import _lib

pytestmark = pytest.mark.gpu
LO, HI = 0.2, 0.28


def slack(V):
    return 2.0 ** -22 + 2.0 ** -24 * (V / 256 + 96)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def status():
    out = C.c_int32(0)
    _lib.check(_lib.lib().femto_status_word(None, C.byref(out)))
    return out.value


def make(N, V, dtype, pitch=0, offset=0, seed=0, spread=3.0, masked=0.0, temperature=1.0):
    """Logits in a buffer of their own pitch that starts `offset` elements in, targets drawn from the softmax, some rows without."""
    g = torch.Generator(device="cuda").manual_seed(1009 * seed + 31 * N + V)
    buf = torch.full((offset + N * (V + pitch) + 64,), 7.0, device="cuda", dtype=dtype)
    z = buf[offset:offset + N * (V + pitch)].view(N, V + pitch)[:, :V]
    z.copy_(spread * torch.randn(N, V, device="cuda", generator=g))
    t = torch.multinomial(torch.softmax(z.float() / temperature, 1), 1, generator=g)[:, 0].int() if V <= 1 << 20 else torch.zeros(N, device="cuda", dtype=torch.int32)
    if masked:
        t[torch.rand(N, device="cuda", generator=g) < masked] = -1
    return z, t


def reference(z, t, temperature=1.0):
    """(logp, entropy, log p of every token) in 64 bits; 0 in rows without a target."""
    s = z.double() / temperature
    lse = torch.logsumexp(s, 1)
    ls = torch.where(lse[:, None] == -math.inf, -math.inf, s - lse[:, None])
    h = -torch.where(ls == -math.inf, 0.0, ls.exp() * ls).sum(1)
    has = t >= 0
    lp = ls.gather(1, t.clamp(min=0).long()[:, None])[:, 0]
    return torch.where(has, lp, 0.0), torch.where(has, h, 0.0), ls


def near(got, want, tol, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~same & ~((got - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, largest {float((got - want).abs().nan_to_num(1e300).max()):.3e}"


# a row that fits a thread, a warp, a block; odd; past every size that one block, or eight together, hold of it; many wide rows, which
# come through a ring that holds them (20011, 40000) or not
SHAPES = [(200, 9001), (300, 1), (400, 5), (700, 20011), (310, 40000), (320, 150001), (1, 1), (3, 2), (5, 7), (2, 33), (7, 255), (4, 1000), (9, 4099), (150, 4096), (600, 300), (3, 50021), (2, 65536), (1, 131073), (2, 300007)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V", SHAPES)
@pytest.mark.parametrize("pitch,offset,temperature", [(0, 0, 1.0), (3, 1, 0.75)])
def test_token_logprobs(dtype, N, V, pitch, offset, temperature):
    z, t = make(N, V, dtype, pitch, offset, masked=0.3 if N > 3 else 0.0)
    lp, h, _ = reference(z, t, temperature)
    for entropy in (False, True):
        r = fb.token_logprobs(z, t, temperature=temperature, entropy=entropy)
        near(r.logp, lp, slack(V) + 2.0 ** -23 * (lp.abs() + h + 1), "logp")
        if entropy:     # the mean of -log p: as far off as a log-probability, and p as above
            near(r.entropy, h, 3 * slack(V) * (h + 1), "entropy")
    again = fb.token_logprobs(z, t, temperature=temperature, entropy=True)
    assert torch.equal(r.logp, again.logp) and torch.equal(r.entropy, again.entropy)
    assert status() == 0


def check_gradient(d, z, coef, t, ls, V, dtype, inv_t, extra=0.0, what="dlogits"):
    """d = inv_t coef (onehot - p), within the roundings of p, of the coefficient and of the result."""
    p = ls.exp()
    onehot = torch.nn.functional.one_hot(t.clamp(min=0).long(), V).double() * (t >= 0)[:, None]
    want = inv_t * coef[:, None] * (onehot - p)
    tol = half_step(dtype) * 1.01 * want.abs() + inv_t * coef.abs()[:, None] * (p + onehot) * (2 * slack(V) + 2.0 ** -21) + extra + 1e-38
    near(d, want, tol, what)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V", SHAPES)
@pytest.mark.parametrize("pitch,offset,temperature", [(0, 0, 1.0), (5, 3, 1.25)])
def test_token_logprobs_gradient(dtype, N, V, pitch, offset, temperature):
    z, t = make(N, V, dtype, pitch, offset, seed=1, masked=0.3 if N > 3 else 0.0)
    g = torch.Generator(device="cuda").manual_seed(N + V)
    dlogp, dent = torch.randn(2, N, device="cuda", generator=g)
    _, h, ls = reference(z, t, temperature)
    has, inv = (t >= 0), 1.0 / temperature
    d = fb.token_logprobs_gradient(z, t, dlogp, temperature=temperature)
    check_gradient(d, z, torch.where(has, dlogp.double(), 0.0), t, ls, V, dtype, inv)
    # with the entropy: - dH p (log p + H)
    d2 = fb.token_logprobs_gradient(z, t, dlogp, dentropy=dent, temperature=temperature)
    p = ls.exp()
    onehot = torch.nn.functional.one_hot(t.clamp(min=0).long(), V).double()
    k = dlogp.double()[:, None] + dent.double()[:, None] * (ls + h[:, None])
    want = torch.where(has[:, None], inv * (dlogp.double()[:, None] * onehot - k * p), 0.0)
    size = dlogp.double().abs()[:, None] * (onehot + p) + dent.double().abs()[:, None] * p * (ls.abs() + h[:, None] + 2)
    near(d2, want, half_step(dtype) * 1.01 * want.abs() + inv * size * (4 * slack(V) + 2.0 ** -20) + 1e-38, "with the entropy")
    assert status() == 0


def tokens_of(N, lp, seed, ref=True):
    """Old log-probabilities away from where the clipping begins, advantages of both signs and 0, a reference, weights (one of them 0)."""
    g = torch.Generator(device="cuda").manual_seed(7 * seed + N)
    old = lp - 0.25 * torch.randn(N, device="cuda", generator=g, dtype=torch.float64)
    for edge in (1 - LO, 1 + HI):
        old = torch.where(((lp - old).exp() / edge - 1).abs() < 1e-3, old + 0.01, old)
    A = torch.randn(N, device="cuda", generator=g)
    w = torch.rand(N, device="cuda", generator=g)
    if N > 2:
        A[1], w[2] = 0.0, 0.0
    return old.float(), A, (lp + 0.4 * torch.randn(N, device="cuda", generator=g, dtype=torch.float64)).float(), w


def policy_reference(lp, has, old, A, ref, w, kl):
    """Token losses and their slopes by lp, where the minimum is the bounded product; and how far an error of lp moves them."""
    r = (lp - old.double()).exp()
    A, w = A.double(), (w.double() if w is not None else torch.ones_like(lp))
    bounded = r.clamp(1 - LO, 1 + HI) * A
    clipped = has & (bounded < r * A)
    loss, slope = -torch.minimum(r * A, bounded), torch.where(clipped, 0.0, -r * A)
    size = r * A.abs() + A.abs()
    if kl:
        gap = ref.double() - lp
        loss = loss + kl * (torch.expm1(gap) - gap)
        slope = slope - kl * torch.expm1(gap)
        size = size + kl * (gap.exp() + gap.abs() + 1)
    zero = torch.zeros_like(lp)
    return torch.where(has, w * loss, zero), torch.where(has, w * slope, zero), clipped, torch.where(has, w * size, zero)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V", SHAPES)
@pytest.mark.parametrize("pitch,offset,temperature,kl,reduction", [(0, 0, 1.0, 0.0, "sum"), (8, 0, 0.8125, 0.125, "mean"), (1, 5, 1.0, 0.0625, "sum")])
def test_policy_loss(dtype, N, V, pitch, offset, temperature, kl, reduction):
    z, t = make(N, V, dtype, pitch, offset, seed=2, masked=0.4 if N > 3 else 0.0, temperature=temperature)
    lp, h, ls = reference(z, t, temperature)
    old, A, ref, w = tokens_of(N, lp, V)
    w = w if offset else None
    has = t >= 0
    loss, slope, clipped, size = policy_reference(lp, has, old, A, ref, w, kl)
    n = int(has.sum())
    scale = 1.0 / max(n, 1) if reduction == "mean" else 1.0
    dlp = slack(V) + 2.0 ** -23 * (lp.abs() + h + 1)
    term = size * (2 * dlp + 2.0 ** -21)      # ratio and e^gap: the error of lp, of exp and of the products
    kwargs = dict(ref_logp=ref if kl else None, weights=w, clip_low=LO, clip_high=HI, kl_coef=kl, temperature=temperature, reduction=reduction)
    r = fb.policy_loss(z, t, old, A, **kwargs)
    near(r.logp, lp, dlp, "logp")
    near(r.token_losses, loss, term, "token losses")
    near(r.loss, (scale * loss.sum()).reshape(1), scale * (term.sum() + loss.abs().sum() * 2.0 ** -24 * (N / 1024 + 16)), "loss")
    assert int(r.n_valid) == n and int(r.n_clipped) == int(clipped.sum())
    p = ls.exp()
    onehot = torch.nn.functional.one_hot(t.clamp(min=0).long(), V).double()
    check_gradient(r.dlogits, z, scale * slope, t, ls, V, dtype, 1 / temperature, scale / temperature * term[:, None] * (p + onehot))
    # the loss alone is the same, and so is the gradient in the logits' place
    only = fb.policy_loss(z, t, old, A, gradient=False, **kwargs)
    near(only.loss, r.loss, scale * (2 * term.sum() + loss.abs().sum() * 2.0 ** -23 * (N / 1024 + 16)), "loss alone")
    assert only.dlogits is None and torch.equal(only.n_clipped, r.n_clipped)
    keep = z.clone()
    inplace = fb.policy_loss(z, t, old, A, out=z, **kwargs)
    assert inplace.dlogits is z and torch.equal(z, r.dlogits) and torch.equal(inplace.loss, r.loss)
    z.copy_(keep)
    assert status() == 0


# every number of warps a row and of rows a block that narrow rows have, each group with several rows in turn
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,words", [(7200, 40), (7000, 255), (6500, 301), (5500, 341), (5000, 401), (4700, 450), (3700, 513), (2900, 641), (2500, 801), (1900, 902), (1900, 1050),
                                     (1900, 1151), (1300, 1281), (1300, 1399), (1300, 1401), (1100, 1699), (1100, 1701)])
def test_narrow_rows(dtype, N, words):
    V = words * 16 // torch.finfo(dtype).bits * 8 + 1
    N = N if V < 2000 else N // 2
    test_token_logprobs(dtype, N, V, 3, 1, 0.75)
    test_token_logprobs_gradient(dtype, N, V, 0, 0, 1.25)
    test_policy_loss(dtype, N, V, 5, 3, 1.0, 0.125, "mean")


@pytest.mark.parametrize("V", [37, 5000, 70001])
def test_rows_around_the_gradient_stay(V):
    """What lies between and behind the rows of a padded gradient is not written; rows start anywhere."""
    N, pad = 5, 11
    for dtype in (torch.float32, torch.bfloat16):
        for offset in (0, 1, 4):
            z, t = make(N, V, dtype)
            buf = torch.full((offset + N * (V + pad) + 40,), 5.0, device="cuda", dtype=dtype)
            out = buf[offset:offset + N * (V + pad)].view(N, V + pad)[:, :V]
            old = torch.zeros(N, device="cuda")
            r = fb.policy_loss(z, t, old, torch.ones_like(old), clip_high=None, out=out)
            d = fb.policy_loss(z, t, old, torch.ones_like(old), clip_high=None).dlogits
            assert torch.equal(out, d)
            out.fill_(5.0)
            assert bool((buf == 5.0).all())
            fb.token_logprobs_gradient(z, t, old + 1, out=out)
            assert torch.equal(out, fb.token_logprobs_gradient(z, t, old + 1))
            out.fill_(5.0)
            assert bool((buf == 5.0).all())
            assert r.dlogits is out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [9, 3001, 12001, 66000, 140001])
@pytest.mark.parametrize("copies", [1, 51])      # few rows and many take different kernels
def test_masked_rows_and_masked_tokens(dtype, V, copies):
    """Rows without a target may hold anything; logits of -inf are tokens that cannot be chosen; a row of them has no distribution."""
    N = 6
    z, t = make(N, V, dtype, seed=3)
    g = torch.Generator(device="cuda").manual_seed(V)
    hidden = torch.rand(N, V, device="cuda", generator=g) < 0.6
    hidden.scatter_(1, t.long()[:, None], False)
    z.masked_fill_(hidden, -math.inf)
    t[0], z[0] = -1, math.nan
    z[1] = -math.inf
    z[2] = torch.finfo(dtype).min        # the lowest value, everywhere: a uniform distribution
    z[3, :] = -math.inf
    z[3, int(t[3])] = 1.0                # one token left: it is certain
    t[4] = -5
    numbers = torch.tensor([math.nan, 0.5, -0.5, 1.0, math.inf, 0.25], device="cuda")
    lp, h, ls = reference(z, t)
    lp[2], h[2] = -math.log(V), math.log(V)
    many_z, many_t, many_numbers = z.repeat(copies, 1), t.repeat(copies), numbers.repeat(copies)

    def every(x):      # [copies][row]...
        return x.unflatten(0, (copies, N))

    r = fb.token_logprobs(many_z, many_t, entropy=True)
    near(r.logp, lp.repeat(copies), slack(V) + 2.0 ** -23 * (lp.abs() + h + 1).repeat(copies), "logp")
    near(r.entropy, h.repeat(copies), 3 * slack(V) * (h + 1).repeat(copies), "entropy")
    assert bool((every(r.logp)[:, 1] == -math.inf).all() and (every(r.logp)[:, 3] == 0.0).all() and (every(r.entropy)[:, 3] == 0.0).all())
    d = fb.token_logprobs_gradient(many_z, many_t, many_numbers, dentropy=many_numbers)
    assert not d.isnan().any()
    assert bool((every(d)[:, [0, 1, 4]] == 0).all())
    impossible = hidden & (t >= 0)[:, None] & (torch.arange(N, device="cuda") != 2)[:, None]
    assert bool((every(d)[:, impossible] == 0).all())
    finite = torch.tensor([math.nan, 0.0, 0.0, 0.0, math.nan, -2.0], device="cuda")
    q = fb.policy_loss(many_z, many_t, finite.repeat(copies), many_numbers, ref_logp=torch.where(many_t < 0, math.nan, -3.0),
                       weights=torch.where(many_t < 0, math.nan, 1.0))
    assert bool((every(q.dlogits)[:, [0, 1, 4]] == 0).all() and (every(q.token_losses)[:, [0, 1, 4]] == 0).all())
    assert not q.dlogits.isnan().any() and math.isfinite(float(q.loss)) and int(q.n_valid) == 4 * copies
    assert status() == 0


def test_not_a_number_stays_in_its_row():
    for N, V in ((4, 50), (4, 40000), (300, 50), (300, 9000), (300, 40000), (300, 140000)):
        z, t = make(N, V, torch.float32, seed=4)
        z[1, 3], z[2, 4] = math.nan, math.inf
        rest = torch.arange(N, device="cuda") % N
        rest = rest[(rest != 1) & (rest != 2)]
        r = fb.token_logprobs(z, t, entropy=True)
        assert r.logp[1:3].isnan().all() and r.entropy[1:3].isnan().all() and not r.logp[rest].isnan().any()
        q = fb.policy_loss(z, t, torch.zeros(N, device="cuda"), torch.ones(N, device="cuda"), clip_high=None)
        assert q.dlogits[1:3].isnan().all() and not q.dlogits[rest].isnan().any()


@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 60007), (torch.bfloat16, 214001), (torch.float32, 33001), (torch.float32, 110003)])
@pytest.mark.parametrize("pitch,offset", [(0, 0), (7, 5)])
def test_wide_rows_in_place(dtype, V, pitch, offset):
    """A row that two blocks share, written over its logits: the target in either half and where they meet; rows that their ring holds, and wider."""
    N = 260
    z, t = make(N, V, dtype, pitch, offset, seed=6, masked=0.3)
    half = V // 2
    t[:12] = torch.tensor([0, V - 1, half, half - 1, half + 1, half - 9, half + 9, half - 17, half + 17, -1, 1, V - 2], device="cuda", dtype=t.dtype)
    g = torch.Generator(device="cuda").manual_seed(V)
    lp = reference(z, t, 1.0)[0]
    old, A, _, w = tokens_of(N, lp, 6)
    apart = fb.policy_loss(z, t, old, A, weights=w, out=torch.full_like(z, 3.0))
    dlogp, dent = torch.randn(2, N, device="cuda", generator=g)
    want = fb.token_logprobs_gradient(z, t, dlogp, dentropy=dent)
    over = z.as_strided(z.shape, z.stride(), z.storage_offset())
    keep = z.clone()
    r = fb.policy_loss(over, t, old, A, weights=w, out=over)
    assert torch.equal(r.logp, apart.logp) and torch.equal(r.loss, apart.loss)
    near(over, apart.dlogits.double(), 0, "the same pass")
    z.copy_(keep)
    d = fb.token_logprobs_gradient(over, t, dlogp, dentropy=dent, out=over)
    near(d, want.double(), 0, "the same pass, with the entropy")
    near(r.logp, torch.where(t >= 0, lp, 0.0), slack(V) + 2.0 ** -23 * (lp.abs() + 13), "logp")
    assert status() == 0


def test_no_rows_and_rows_without_targets():
    empty = torch.empty(0, 5, device="cuda")
    i32, f32 = torch.empty(0, device="cuda", dtype=torch.int32), torch.empty(0, device="cuda")
    assert fb.token_logprobs(empty, i32, entropy=True).logp.shape == (0,)
    assert fb.token_logprobs_gradient(empty, i32, f32).shape == (0, 5)
    for reduction in ("sum", "mean"):
        r = fb.policy_loss(empty, i32, f32, f32, reduction=reduction)
        assert float(r.loss) == 0 and int(r.n_valid) == 0 and int(r.n_clipped) == 0
        for N, V in ((3, 4000), (300, 1000), (700, 9001), (333, 70003)):
            z = torch.randn(N, V, device="cuda")
            out = torch.full_like(z, 3.0)
            r = fb.policy_loss(z, torch.full((N,), -1, device="cuda", dtype=torch.int32), torch.zeros(N, device="cuda"), torch.ones(N, device="cuda"),
                               reduction=reduction, out=out)
            assert float(r.loss) == 0 and int(r.n_valid) == 0 and bool((out == 0).all()) and bool((r.logp == 0).all())


def test_target_outside_the_vocabulary():
    z, t = make(4, 1000, torch.bfloat16)
    want = fb.token_logprobs(z, t).logp
    bad = t.clone()
    bad[2] = 1000
    r = fb.token_logprobs(z, bad)
    assert status() == 1 and status() == 0
    assert float(r.logp[2]) == 0 and torch.equal(r.logp[[0, 1, 3]], want[[0, 1, 3]])
    q = fb.policy_loss(z, bad, torch.zeros(4, device="cuda"), torch.ones(4, device="cuda"), reduction="mean")
    assert status() == 1 and int(q.n_valid) == 3 and bool((q.dlogits[2] == 0).all())
    fb.token_logprobs_gradient(z, bad, torch.ones(4, device="cuda"))
    assert status() == 1


def test_rows_past_32_bits():
    """Row offsets beyond 2^32 bytes and 2^31 elements."""
    pitch, V = (1 << 30) + 16, 5000
    buf = torch.empty(2 * pitch + V, device="cuda", dtype=torch.bfloat16)
    z = torch.as_strided(buf, (3, V), (pitch, 1))
    small, t = make(3, V, torch.bfloat16, seed=5)
    z.copy_(small)
    assert torch.equal(fb.token_logprobs(z, t).logp, fb.token_logprobs(small, t).logp)
    old, A = torch.full((3,), -5.0, device="cuda"), torch.ones(3, device="cuda")
    want = fb.policy_loss(small, t, old, A).dlogits
    assert torch.equal(fb.policy_loss(z, t, old, A, out=z).dlogits, want)


@pytest.mark.parametrize("N,V", [(64, 9000), (320, 2000), (320, 9000), (320, 70000)])
def test_streams_and_graphs(N, V):
    """Two calls at once on two streams, and a captured call replayed on other inputs while another graph of the same call lives."""
    z, t = make(N, V, torch.bfloat16, seed=6, masked=0.2)
    y, u = make(N, V, torch.bfloat16, seed=7, masked=0.2)
    old, A = torch.full((N,), -4.0, device="cuda"), torch.linspace(-1, 1, N, device="cuda")
    want, other = (fb.policy_loss(a, b, old, A, reduction="mean") for a, b in ((z, t), (y, u)))
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s1):
            a = fb.policy_loss(z, t, old, A, reduction="mean")
        with torch.cuda.stream(s2):
            b = fb.policy_loss(y, u, old, A, reduction="mean")
        torch.cuda.synchronize()
        for got, ref in ((a, want), (b, other)):
            assert all(torch.equal(x, y) for x, y in zip(got, ref))
    x, v, runs = z.clone(), t.clone(), torch.arange(0, N + 1, N // 4, device="cuda", dtype=torch.int32)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            p = fb.policy_loss(x, v, old, A, reduction="mean")
            lp = fb.token_logprobs(x, v, entropy=True)
            d = fb.token_logprobs_gradient(x, v, old, dentropy=A)
            q = fb.preference_loss(lp.logp, runs, targets0=v, beta=0.375)
        graphs.append((g, p, lp, d, q))
    x.copy_(y), v.copy_(u)
    for g, p, lp, d, q in graphs:
        g.replay()
    torch.cuda.synchronize()
    fresh = fb.token_logprobs(y, u, entropy=True)
    for g, p, lp, d, q in graphs:
        assert all(torch.equal(a, b) for a, b in zip(p, other))
        assert torch.equal(lp.entropy, fresh.entropy)
        assert all(torch.equal(a, b) for a, b in zip(q, fb.preference_loss(fresh.logp, runs, targets0=u, beta=0.375)))
        assert torch.equal(d, fb.token_logprobs_gradient(y, u, old, dentropy=A))


def test_first_call_of_a_process_inside_a_capture():
    """Nothing is allocated or looked up on a call's way that a capture would refuse, not even the first time."""
    import subprocess
    import sys
    code = """
import torch, femtochat_b200 as fb
z = torch.randn(300, 70000, device="cuda"); t = torch.zeros(300, device="cuda", dtype=torch.int32); f = torch.randn(300, device="cuda")
o = torch.tensor([0, 100, 300], device="cuda", dtype=torch.int32)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    p = fb.policy_loss(z, t, f, f, reduction="mean")
    a = fb.token_logprobs(z[:, :3000], t, entropy=True)
    d = fb.token_logprobs_gradient(z[:9], t[:9], f[:9])
    q = fb.preference_loss(a.logp, o)
g.replay(); torch.cuda.synchronize()
r = fb.policy_loss(z, t, f, f, reduction="mean")
assert all(torch.equal(x, y) for x, y in zip(p, r)) and torch.equal(q.loss, fb.preference_loss(a.logp, o).loss)
assert torch.equal(d, fb.token_logprobs_gradient(z[:9], t[:9], f[:9]))
"""
    subprocess.run([sys.executable, "-c", code], check=True, cwd=__file__.rsplit("/tests/", 1)[0], timeout=300)


def test_temperatures_at_the_ends_of_their_range():
    z, t = make(5, 700, torch.float32, seed=11)
    for temperature in (1e-6, 1e6):
        r = fb.token_logprobs(z, t, temperature=temperature, entropy=True)
        T = float(torch.tensor(temperature, dtype=torch.float32))
        lp, h, _ = reference(z, t, T)
        near(r.logp, lp, slack(700) + 2.0 ** -22 * (lp.abs() + h + 1), "logp")
        assert bool(fb.token_logprobs_gradient(z, t, torch.ones(5, device="cuda"), temperature=temperature).isfinite().all())
    low = torch.full((1, 700), torch.finfo(torch.float32).min, device="cuda")
    near(fb.token_logprobs(low, t[:1], temperature=1e-6).logp, torch.tensor([-math.log(700)], device="cuda", dtype=torch.float64), slack(700) + 1e-6, "lowest")
    high = torch.full((1, 700), 1e30, device="cuda")
    near(fb.token_logprobs(high, t[:1], temperature=1e-6).logp, torch.tensor([-math.log(700)], device="cuda", dtype=torch.float64), slack(700) + 1e-6, "highest")


def test_gradient_against_differences():
    """The gradient of the reduced loss against central differences of the definition in 64 bits."""
    N, V, kl = 4, 11, 0.125
    z, t = make(N, V, torch.float32, seed=8)
    lp, _, _ = reference(z, t, 0.875)
    old, A, ref, w = tokens_of(N, lp, 3)
    r = fb.policy_loss(z, t, old, A, ref_logp=ref, weights=w, clip_low=LO, clip_high=HI, kl_coef=kl, temperature=0.875)

    def f(x):
        return policy_reference(reference(x, t, 0.875)[0], t >= 0, old, A, ref, w, kl)[0].sum()

    step = 1e-5
    for i in range(N):
        for j in range(V):
            e = torch.zeros(N, V, device="cuda", dtype=torch.float64)
            e[i, j] = step
            slope = float((f(z.double() + e) - f(z.double() - e)) / (2 * step))
            # differences: step^2 times a third derivative of a few, and roundings 2^-52 / step
            assert abs(float(r.dlogits[i, j]) - slope) < 1e-5 * (1 + abs(slope))


# ---- pairs ----------------------------------------------------------------------------------------------------------------------------------
def pairs(P, longest, seed, ref=True, masked=0.0, before=0, behind=0):
    g = torch.Generator().manual_seed(1000 * seed + 17 * P + longest)
    n = torch.randint(0, longest + 1, (2 * P,), generator=g)
    offsets = (before + torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(n, 0)])).int()
    N = int(offsets[-1]) + behind
    logp = -torch.empty(N).exponential_(0.7, generator=g)
    t = torch.randint(0, 9, (N,), generator=g, dtype=torch.int32)
    if masked:
        t[torch.rand(N, generator=g) < masked] = -1
    return logp.cuda(), (logp + 0.2 * torch.randn(N, generator=g)).cuda() if ref else None, t.cuda(), offsets.cuda()


def preference_reference(logp, ref, t, offsets, kind, beta, margin, smoothing, normalised, reduction):
    gap = logp.double() - (ref.double() if ref is not None else 0.0)
    P = offsets.shape[0] // 2
    o = offsets.tolist()
    rho, size, per, d = [], [], [], torch.zeros_like(gap)
    for k in range(2 * P):
        rows = slice(o[k], o[k + 1])
        m = (t[rows] >= 0).double() if t is not None else torch.ones_like(gap[rows])
        c = max(float(m.sum()), 1.0) if normalised else 1.0
        x = torch.where(m > 0, gap[rows], 0.0)
        rho.append(x.sum() / c), size.append(x.abs().sum() / c), per.append(m / c)
    rho = torch.stack(rho) if rho else torch.zeros(0, device="cuda", dtype=torch.float64)
    D = (rho[0::2] - rho[1::2]).requires_grad_()
    if kind == "sigmoid":
        h = beta * D - margin
        losses = -(1 - smoothing) * torch.nn.functional.logsigmoid(h) - smoothing * torch.nn.functional.logsigmoid(-h)
    else:
        losses = (D - 0.5 / beta) ** 2
    loss = losses.sum() / (P if reduction == "mean" and P else 1)
    slope = torch.autograd.grad(loss, D)[0] if P else D
    for k in range(2 * P):
        d[o[k]:o[k + 1]] = per[k] * slope[k // 2] * (1 if k % 2 == 0 else -1)
    return loss.detach().reshape(1), losses.detach(), rho, d, (torch.stack(size) if P else rho)


@pytest.mark.parametrize("P,longest", [(0, 4), (1, 1), (1, 24), (3, 200), (2, 5000), (1, 70000), (300, 40), (1500, 3)])
@pytest.mark.parametrize("kind,ref,masked,normalised,reduction", [("sigmoid", True, 0.0, False, "mean"), ("sigmoid", False, 0.4, True, "sum"),
                                                                  ("squared", True, 0.3, False, "mean")])
def test_preference_loss(P, longest, kind, ref, masked, normalised, reduction):
    logp, ref_logp, t, offsets = pairs(P, longest, 1, ref, masked, before=3, behind=9001)
    beta = 1.5 if normalised else 0.125
    margin, smoothing = (0.25, 0.125) if kind == "sigmoid" else (0.0, 0.0)
    targets = t if masked else None
    loss, losses, rho, d, size = preference_reference(logp, ref_logp, targets, offsets, kind, beta, margin, smoothing, normalised, reduction)
    r = fb.preference_loss(logp, offsets, targets0=targets, ref_logp=ref_logp, kind=kind, beta=beta, margin=margin, label_smoothing=smoothing,
                           length_normalised=normalised, reduction=reduction)
    # each difference is rounded to fp32, everything else is in 64 bits until it is stored
    drho = 2.0 ** -24 * size * 1.01
    near(r.ratios, rho, drho + 2.0 ** -24 * rho.abs(), "ratios")
    dD = drho[0::2] + drho[1::2]
    slope = beta if kind == "sigmoid" else 2 * (rho[0::2] - rho[1::2]).abs() + 1 / beta
    dl = slope * dD + dD ** 2 + 2.0 ** -23 * (losses.abs() + beta + abs(margin))
    near(r.pair_losses, losses, dl, "pair losses")
    near(r.loss, loss, (dl.sum() + 2.0 ** -24 * losses.sum()) / (P if reduction == "mean" and P else 1) + 1e-30, "loss")
    curve = beta * beta / 4 if kind == "sigmoid" else 2.0
    worst = float((curve * dD).max()) if P else 0.0
    near(r.dlogp, d, 2.0 ** -22 * d.abs() + (worst + 2.0 ** -24 * beta) * (1.0 / P if reduction == "mean" and P else 1.0), "dlogp")
    assert bool((r.dlogp[:3] == 0).all()) and bool((r.dlogp[logp.shape[0] - 9001:] == 0).all())
    only = fb.preference_loss(logp, offsets, targets0=targets, ref_logp=ref_logp, kind=kind, beta=beta, margin=margin, label_smoothing=smoothing,
                              length_normalised=normalised, reduction=reduction, gradient=False)
    assert only.dlogp is None and torch.equal(only.loss, r.loss) and torch.equal(only.ratios, r.ratios)
    assert status() == 0


def test_preference_extremes():
    """Answers that are far apart: the loss is linear there, not infinite; masked tokens may hold anything."""
    logp = torch.tensor([-1e4, -1.0, math.nan, -2.0], device="cuda")
    t = torch.tensor([3, 3, -1, 3], device="cuda", dtype=torch.int32)
    offsets = torch.tensor([0, 1, 4], device="cuda", dtype=torch.int32)
    r = fb.preference_loss(logp, offsets, targets0=t, beta=1.0)
    assert float(r.loss) == pytest.approx(9997.0, rel=1e-6) and r.dlogp.tolist() == [-1.0, 1.0, 0.0, 1.0]
    r = fb.preference_loss(logp, torch.tensor([1, 4, 4], device="cuda", dtype=torch.int32), targets0=t, beta=500.0)
    assert float(r.loss) == pytest.approx(1500.0) and r.ratios.tolist() == [-3.0, 0.0]
    r = fb.preference_loss(logp[1:2], torch.tensor([0, 0, 0], device="cuda", dtype=torch.int32), reduction="sum")
    assert float(r.loss) == pytest.approx(math.log(2)) and r.dlogp.tolist() == [0.0]


def test_bad_offsets_are_flagged():
    logp = -torch.ones(10, device="cuda")
    for bad in ([0, 4, 11], [0, 6, 5], [-1, 4, 6]):
        r = fb.preference_loss(logp, torch.tensor(bad, device="cuda", dtype=torch.int32))
        assert status() == 8 and math.isfinite(float(r.loss))
    assert status() == 0


@pytest.mark.parametrize("N,offsets", [(10, [0, 4, 11]), (10, [0, 6, 5]), (10, [-1, 4, 6]), (12, [0, -5, 8, 10, 12]), (12, [3, 2147483647, 5, 6, 7]), (12, [-2147483648, 2147483647, -1]),
                                       (60000, [100, 70000, 50000]), (60000, [0, 20000, 70000])])
def test_every_row_gets_a_gradient_behind_bad_offsets(N, offsets):
    """The output's memory held something else before: a row that no good answer holds gets 0, one that a good answer holds a finite number."""
    logp = -torch.rand(N, device="cuda")
    o = torch.tensor(offsets, device="cuda", dtype=torch.int32)
    P = len(offsets) // 2
    dlogp, losses, ratios, loss = torch.full((N,), math.nan, device="cuda"), torch.empty(P, device="cuda"), torch.empty(2 * P, device="cuda"), torch.empty(1, device="cuda")
    cfg = _lib.PreferenceConfigC(0, 0.1, 0.0, 0.0, 0, 0)
    _lib.check(_lib.lib().femto_preference_loss(logp.data_ptr(), None, None, N, o.data_ptr(), P, C.byref(cfg), loss.data_ptr(), losses.data_ptr(), ratios.data_ptr(),
                                                dlogp.data_ptr(), _lib.stream_ptr()))
    held = torch.zeros(N, dtype=torch.bool, device="cuda")
    for k, (a, b) in enumerate(zip(offsets, offsets[1:])):
        if 0 <= a <= b <= N:
            held[a:b] = True
        else:
            assert float(ratios[k]) == 0
    assert status() == 8
    assert bool(dlogp.isfinite().all()) and bool((dlogp[~held] == 0).all())


def test_the_count_of_clipped_tokens_is_that_of_the_gradient():
    """Ratios within a rounding of the bound: a token counts as clipped where, and only where, it has no gradient."""
    N, V = 4000, 50
    z, t = make(N, V, torch.float32, seed=12)
    lp = fb.token_logprobs(z, t).logp
    old = lp - math.log(1.25)
    turn = torch.arange(N, device="cuda") % 3
    for way in (1, 2):
        old = torch.where(turn == way, torch.nextafter(old, torch.full_like(old, 90.0 if way == 1 else -90.0)), old)
    r = fb.policy_loss(z, t, old, torch.ones(N, device="cuda"), clip_high=0.25)
    none = (r.dlogits == 0).all(1)
    assert 0 < int(none.sum()) < N and int(r.n_clipped) == int(none.sum())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_preference_from_logits_to_logits(dtype):
    """The three calls in a row, as a step makes them, against the gradient of the whole by differentiation in 64 bits."""
    B, T, V = 6, 40, 3000
    z, t = make(B * T, V, dtype, pitch=8, seed=9, masked=0.3)
    offsets = (torch.arange(B + 1) * T).int().cuda()
    ref = fb.token_logprobs(z + 0.1 * torch.randn_like(z), t).logp
    s = fb.token_logprobs(z, t, temperature=0.875)
    r = fb.preference_loss(s.logp, offsets, targets0=t, ref_logp=ref, beta=0.375)
    d = fb.token_logprobs_gradient(z, t, r.dlogp, temperature=0.875)
    x = z.double().requires_grad_()
    ls = torch.log_softmax(x / 0.875, 1).gather(1, t.clamp(min=0).long()[:, None])[:, 0]
    gap = torch.where(t >= 0, ls - ref.double(), 0.0).view(B, T).sum(1)
    loss = -torch.nn.functional.logsigmoid(0.375 * (gap[0::2] - gap[1::2])).mean()
    want, = torch.autograd.grad(loss, x)
    loss = loss.detach()
    p, onehot = torch.softmax(x.detach() / 0.875, 1), torch.nn.functional.one_hot(t.clamp(min=0).long(), V)
    size = 0.125 / 0.875 * (p + onehot)      # |d loss / d lp| <= beta / pairs
    dlp = T * 2 * (slack(V) + 2.0 ** -23 * 30)
    assert abs(float(r.loss) - float(loss)) <= 0.375 * 2 * dlp + 1e-6
    near(d, want, half_step(dtype) * 1.01 * want.abs() + size * (dlp + 4 * slack(V) + 2.0 ** -20), "dlogits")


def test_tensors_as_the_model_gives_them():
    """[B][T][V] logits of the model call, slices of a padded vocabulary, and arrays that are not contiguous."""
    z, t = make(6, 500, torch.float32, pitch=12, seed=10)
    z3, t3 = z.unflatten(0, (2, 3)), t.view(2, 3)
    A = torch.tensor([1.0, -1.0], device="cuda")[:, None].expand(2, 3)
    old = torch.full((3, 2), -6.0, device="cuda").t()
    r = fb.policy_loss(z3, t3, old, A)
    want = fb.policy_loss(z.contiguous(), t, old.flatten(), A.flatten())
    assert r.dlogits.shape == z3.shape and torch.equal(r.dlogits.flatten(0, 1), want.dlogits) and torch.equal(r.loss, want.loss)
    one = fb.token_logprobs(z[0], t[0])
    assert one.logp.shape == () and torch.equal(one.logp, fb.token_logprobs(z, t).logp[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V", [(7, 300), (9, 9001), (5, 66001), (300, 37), (300, 701), (400, 4003), (300, 9001), (310, 20011), (300, 60007), (300, 140001)])
@pytest.mark.parametrize("offset,temperature", [(0, 1.0), (3, 0.75)])
def test_confident_tokens(dtype, N, V, offset, temperature):
    """Of a token that the model is all but sure of, 1 - p and -log p are small numbers, right to some roundings of their own.  With q the sum of the
    others' exponentials over the token's: q has the relative error of l above, and that of the scale's rounding, 2^-24 of the exponent (|u| < 64, so
    2^-24 48); with_token() takes one more exponential, log1p, the quotient and the products some roundings: `rel` for each number that is made of q."""
    z, t = make(N, V, dtype, 5, offset, seed=21)
    g = torch.Generator(device="cuda").manual_seed(V + N)
    t = torch.randint(0, V, (N,), device="cuda", generator=g).int()
    t[:4] = torch.tensor([0, V - 1, 1, V // 2], device="cuda", dtype=torch.int32)
    rows = torch.arange(N, device="cuda")
    s = z.double() / temperature
    s[rows, t.long()] = -math.inf
    left = torch.logspace(-7, -3, N, device="cuda", dtype=torch.float64)[torch.randperm(N, device="cuda", generator=g)]      # 1 - p
    z[rows, t.long()] = (temperature * (torch.logsumexp(s, 1) + torch.log1p(-left) - left.log())).to(dtype)
    lp, h, ls = reference(z, t, temperature)
    q = torch.where(torch.nn.functional.one_hot(t.long(), V) > 0, 0.0, ls.exp()).sum(1)      # 1 - p
    assert float(q.max()) < 0.01
    rel = slack(V) + 2.0 ** -24 * 48 + 2.0 ** -20
    r = fb.token_logprobs(z, t, temperature=temperature, entropy=True)
    near(r.logp, lp, rel * lp.abs(), "logp")
    near(r.entropy, h, 3 * rel * h, "entropy")
    near(fb.token_logprobs(z, t, temperature=temperature).logp, r.logp, 0, "logp without the entropy")
    dlogp, dent = torch.randn(2, N, device="cuda", generator=g)
    inv, at = 1 / temperature, (rows, t.long())
    d = fb.token_logprobs_gradient(z, t, dlogp, temperature=temperature)[at]
    want = inv * dlogp.double() * q
    near(d, want, (half_step(dtype) * 1.01 + rel) * want.abs(), "at the target")
    d = fb.token_logprobs_gradient(z, t, dlogp, dentropy=dent, temperature=temperature)[at]
    second = inv * dent.double() * lp.exp() * (lp + h)
    near(d, want - second, half_step(dtype) * 1.01 * (want - second).abs() + 3 * rel * (want.abs() + inv * dent.double().abs() * h), "with the entropy")
    # ratios of 1: the slope by log p is -A, right to the error of log p and of the exponential
    A = torch.randn(N, device="cuda", generator=g)
    keep = z.clone()
    for out in (None, z):
        got = fb.policy_loss(z, t, r.logp, A, temperature=temperature, out=out).dlogits[at]
        want = -inv * A.double() * q
        near(got, want, (half_step(dtype) * 1.01 + 2 * rel) * want.abs(), "policy")
    z.copy_(keep)
    assert status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V", [(6, 50), (6, 9001), (6, 66001), (330, 50), (330, 4003), (330, 20011), (330, 70001), (330, 300001)])
@pytest.mark.parametrize("reduction", ["sum", "mean"])
def test_a_weight_of_0_counts_nothing(dtype, N, V, reduction):
    """Rows that a user drops by their weight, an overflow in their logits or in another of their numbers: no loss, no gradient."""
    z, t = make(N, V, dtype, 3, 1, seed=22)
    lp, _, _ = reference(z, t)
    old, A, ref, w = tokens_of(N, lp, V)
    w = torch.where(torch.arange(N, device="cuda") % 3 == 0, w + 0.25, 0.0)
    args = dict(clip_low=LO, clip_high=HI, kl_coef=0.125, reduction=reduction)
    clean = fb.policy_loss(z, t, old, A, ref_logp=ref, weights=w, **args)
    dropped = w == 0
    g = torch.Generator(device="cuda").manual_seed(V)
    kind = torch.randint(0, 5, (N,), device="cuda", generator=g)
    spot = torch.randint(0, V, (N,), device="cuda", generator=g)
    rows = torch.arange(N, device="cuda")
    z[rows[dropped & (kind == 0)], spot[dropped & (kind == 0)]] = math.nan
    z[rows[dropped & (kind == 1)], t.long()[dropped & (kind == 1)]] = math.inf
    z[rows[dropped & (kind == 2)]] = math.nan
    old, A, ref = (torch.where(dropped & (kind >= 3 - i), bad, x) for i, (x, bad) in enumerate(((old, math.nan), (A, math.inf), (ref, -math.inf))))
    for out in (None, z):
        r = fb.policy_loss(z, t, old, A, ref_logp=ref, weights=w, out=out, **args)
        assert torch.equal(r.loss, clean.loss) and torch.equal(r.token_losses, clean.token_losses) and torch.equal(r.n_valid, clean.n_valid)
        assert bool((r.dlogits[dropped] == 0).all()) and torch.equal(r.dlogits[~dropped], clean.dlogits[~dropped])
    assert status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [9, 3001, 12001, 66000, 140001])
@pytest.mark.parametrize("copies", [1, 51])      # few rows and many take different kernels
@pytest.mark.parametrize("offset", [0, 1])       # of the gradient: rows that lie as the logits do, or not
def test_kl_term_of_tokens_that_the_model_rules_out(dtype, V, copies, offset):
    """A chosen token of probability 0 has g = ref - log p = +inf: its KL term and the loss are +inf by the definition, e^g - g - 1, and no NaN.  Its row's
    gradient is -inf at the token, +inf at tokens of p > 0, and 0 where p = 0; a row without a distribution has none."""
    N, kl = 6, 0.125
    z, t = make(N, V, dtype, seed=23)
    g = torch.Generator(device="cuda").manual_seed(V)
    hidden = torch.rand(N, V, device="cuda", generator=g) < 0.5
    hidden[:, V - 1] = False
    t[:] = torch.tensor([V // 2, -1, 0, 3, V // 3, 5], device="cuda", dtype=torch.int32)
    hidden.scatter_(1, t.clamp(min=0).long()[:, None], False)
    hidden[0, V // 2] = hidden[4, V // 3] = True      # ruled out
    z.masked_fill_(hidden, -math.inf)
    z[3], z[1] = -math.inf, math.nan                  # a row without a distribution; one without a target
    lp, _, ls = reference(z, t)
    ref = torch.tensor([-3.0, math.nan, -2.0, -4.0, -0.5, -1.0], device="cuda")
    old = torch.tensor([-3.0, math.nan, -2.5, -4.0, -0.5, -1.5], device="cuda")
    A = torch.tensor([1.0, math.nan, 0.5, -1.0, -2.0, 1.5], device="cuda")
    many = lambda x: x.repeat(copies, *[1] * (x.dim() - 1))
    buf = torch.full((offset + N * copies * V,), 5.0, device="cuda", dtype=dtype)
    r = fb.policy_loss(many(z), many(t), many(old), many(A), ref_logp=many(ref), clip_low=LO, clip_high=HI, kl_coef=kl, out=buf[offset:].view(-1, V))
    losses, d, logp = r.token_losses.view(copies, N), r.dlogits.view(copies, N, V), r.logp.view(copies, N)
    assert float(r.loss) == math.inf and not losses.isnan().any() and not d.isnan().any()
    assert bool((losses[:, [0, 3, 4]] == math.inf).all()) and bool((logp[:, [0, 3, 4]] == -math.inf).all()) and bool((losses[:, 1] == 0).all())
    assert bool((d[:, [1, 3]] == 0).all())
    for i in (0, 4):
        at = int(t[i])
        assert bool((d[:, i, at] == -math.inf).all())
        rest = torch.arange(V, device="cuda") != at
        assert bool((d[:, i, rest & hidden[i]] == 0).all()) and bool((d[:, i, rest & ~hidden[i]] == math.inf).all())
    # the other rows are what they are without these
    keep = torch.tensor([2, 5], device="cuda")
    alone = fb.policy_loss(z[keep], t[keep], old[keep], A[keep], ref_logp=ref[keep], clip_low=LO, clip_high=HI, kl_coef=kl)
    h = -torch.where(ls[keep] == -math.inf, 0.0, ls[keep].exp() * ls[keep]).sum(1)
    term = policy_reference(lp[keep], t[keep] >= 0, old[keep], A[keep], ref[keep], None, kl)[3] * (2 * (slack(V) + 2.0 ** -23 * (lp[keep].abs() + h + 1)) + 2.0 ** -21)
    near(losses[:, keep], alone.token_losses.expand(copies, 2).double(), 2 * term, "other rows")
    assert bool(alone.dlogits.isfinite().all()) and bool(d[:, keep].isfinite().all())
    assert status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V", [(5, 300), (300, 300), (300, 9001), (320, 40001), (300, 150001)])
@pytest.mark.parametrize("logits_first", [True, False])
def test_gradient_beside_the_logits_in_one_buffer(dtype, N, V, logits_first):
    """Rows of both in turn, nothing shared, a gap of one element before the next pair."""
    small, t = make(N, V, dtype, seed=24, masked=0.3)
    buf = torch.full((N, 2 * V + 1), 7.0, device="cuda", dtype=dtype)
    z, d = (buf[:, :V], buf[:, V:2 * V]) if logits_first else (buf[:, V:2 * V], buf[:, :V])
    z.copy_(small)
    old, A = torch.full((N,), -4.0, device="cuda"), torch.linspace(-1, 1, N, device="cuda")
    r, want = fb.policy_loss(z, t, old, A, reduction="mean", out=d), fb.policy_loss(small, t, old, A, reduction="mean")
    near(d, want.dlogits.double(), 2 * slack(V) * want.dlogits.double().abs() + 2 * half_step(dtype) * want.dlogits.double().abs(), "policy")
    assert torch.equal(r.n_valid, want.n_valid) and torch.equal(z, small) and bool((buf[:, 2 * V] == 7.0).all())
    fb.token_logprobs_gradient(z, t, A, dentropy=old, out=d)
    g = fb.token_logprobs_gradient(small, t, A, dentropy=old)
    _, h, ls = reference(small, t)
    size = A.double().abs()[:, None] * (torch.nn.functional.one_hot(t.clamp(min=0).long(), V) + ls.exp()) + 4 * ls.exp() * (ls.abs() + h[:, None] + 2)
    near(d, g.double(), 2 * half_step(dtype) * 1.01 * g.double().abs() + 2 * size * (4 * slack(V) + 2.0 ** -20) + 1e-38, "gradient")
    assert torch.equal(z, small) and bool((buf[:, 2 * V] == 7.0).all()) and status() == 0


def test_python_reads_what_the_device_found():
    z, t = make(4, 100, torch.float32)
    logp = fb.token_logprobs(z, t).logp
    assert fb.status_word() == 0
    t[1] = 100
    fb.token_logprobs(z, t)
    assert fb.status_word(z.device) == 1 and fb.status_word() == 0
    fb.preference_loss(logp, torch.tensor([0, 3, 2], device="cuda", dtype=torch.int32))
    fb.token_logprobs(z, t)
    assert fb.status_word() == 9 and fb.status_word() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V", [(400, 37), (400, 701), (1500, 4003), (400, 20011), (500, 60007), (300, 150001)])      # every kernel that waits, rows that its ring holds or not
@pytest.mark.parametrize("polls", [0, 1, 50])
def test_waits_that_run_out(dtype, N, V, polls):
    """Waits that give up, at once or early, while copies are on their way: the kernels raise bit 2, wait for these and return.  Nothing but the rows of the
    gradient is written, and the calls that follow are right."""
    z, t = make(N, V, dtype, 3, 1, seed=25, masked=0.2)
    dlogp = torch.randn(N, device="cuda", generator=torch.Generator(device="cuda").manual_seed(V))
    code = _lib.F32 if dtype is torch.float32 else _lib.BF16
    pitch = z.stride(0)
    buf = torch.full((N * pitch + 64,), 5.0, device="cuda", dtype=dtype)
    d = buf[1:1 + N * pitch].view(N, pitch)[:, :V]
    logp = torch.full((N + 2,), 5.0, device="cuda")
    word = C.c_int32(-1)

    def run(limit, gradient):
        _lib.check(_lib.lib().femto_selftest_rows_wait(code, d.data_ptr() if gradient else None, z.data_ptr(), pitch, t.data_ptr(), N, V, dlogp.data_ptr(),
                                                       logp[1:].data_ptr(), limit, C.byref(word), _lib.stream_ptr()))
        return word.value

    for gradient in (True, False):
        for _ in range(3):
            found = run(polls, gradient)
            assert found == 2 or (polls > 0 and found == 0)
        assert status() == 0
        # with the ordinary limit the same entry gives what the calls give
        assert run(1 << 22, gradient) == 0
    assert torch.equal(d, fb.token_logprobs_gradient(z, t, dlogp)) and torch.equal(logp[1:-1], fb.token_logprobs(z, t).logp)
    d.fill_(5.0)
    assert bool((buf == 5.0).all()) and float(logp[0]) == float(logp[-1]) == 5.0
    lp, h, _ = reference(z, t)
    near(logp[1:-1], lp, slack(V) + 2.0 ** -23 * (lp.abs() + h + 1), "logp")
    assert status() == 0


@pytest.mark.parametrize("smoothing", [0.0, 0.25, 1.0])
def test_pairs_with_an_answer_that_the_model_rules_out(smoothing):
    """log p = -inf in the rejected answer: D = h = +inf and -(1 - e) log sigma(h) = 0; in the chosen one h = -inf and the loss is +inf; with e the other way
    round.  A factor of 0 counts nothing.  The slopes by D are the limits, beta (sigma(h) - (1 - e))."""
    logp = torch.tensor([-1.0, -2.0, -1.5, -math.inf, -0.5, -math.inf, -1.0, -1.0], device="cuda")
    offsets = torch.tensor([0, 2, 4, 6, 8], device="cuda", dtype=torch.int32)
    r = fb.preference_loss(logp, offsets, beta=0.5, label_smoothing=smoothing, reduction="sum")
    inf = math.inf
    assert r.ratios.tolist() == [-3.0, -inf, -inf, -2.0]
    assert r.pair_losses.tolist() == [0.0 if smoothing == 0 else inf, 0.0 if smoothing == 1 else inf] and float(r.loss) == inf
    a, b = 0.5 * smoothing, 0.5 * (smoothing - 1)
    assert r.dlogp.tolist() == [a, a, -a, -a, b, b, -b, -b]
    assert status() == 0


@pytest.mark.parametrize("N,V", [(3, 50), (5, 66001), (330, 50), (330, 9001), (330, 70001)])
def test_rows_of_weight_0_alone_end_behind_the_count(N, V):
    """A mean whose rows all have weight 0 asks for no count of the targets; the call still ends behind the kernel that counts them, so that what follows in
    the stream may write over the targets."""
    z, t = make(N, V, torch.float32, seed=26, masked=0.3)
    old, zero = torch.full((N,), -4.0, device="cuda"), torch.zeros(N, device="cuda")
    n = int((t >= 0).sum())
    for _ in range(20):
        u = t.clone()
        r = fb.policy_loss(z, u, old, zero + 1, weights=zero, reduction="mean")
        u.fill_(-1)
        assert int(r.n_valid) == n and float(r.loss) == 0 and bool((r.dlogits == 0).all())
    assert status() == 0

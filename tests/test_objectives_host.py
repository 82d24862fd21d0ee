"""What the objectives refuse, checked without a GPU: no call below reaches a launch."""
import ctypes as C
import math

import pytest
import torch

import femtochat_b200 as fb
from femtochat_b200 import _lib

BASE = 1 << 20      # stands for device memory that nobody reads


def at(i):
    return C.c_void_p(BASE * (i + 1))


def rows(**change):
    a = dict(dtype=1, logits=at(0), ldl=100, targets0=at(1), N=4, V=100)
    a.update(change)
    return a


def logprobs(temperature=1.0, logp=at(2), **change):
    a = rows(**change)
    return _lib.lib().femto_token_logprobs(a["dtype"], a["logits"], a["ldl"], a["targets0"], a["N"], a["V"], temperature, logp, None, None)


def gradient(dlogits=at(3), ldd=100, dlogp=at(4), dentropy=None, temperature=1.0, **change):
    a = rows(**change)
    return _lib.lib().femto_token_logprobs_gradient(a["dtype"], dlogits, ldd, a["logits"], a["ldl"], a["targets0"], a["N"], a["V"], temperature, dlogp, dentropy,
                                                    None)


def policy(old=at(2), adv=at(3), ref=None, token_losses=at(4), logp=at(5), loss=at(6), n_valid=at(7), dlogits=at(8), ldd=100, cfg=(1.0, 0.2, 0.2, 0.0, 0), **change):
    a = rows(**change)
    c = None if cfg is None else C.byref(_lib.PolicyConfigC(*cfg))
    return _lib.lib().femto_policy_loss(a["dtype"], a["logits"], a["ldl"], a["targets0"], a["N"], a["V"], old, adv, ref, None, c, dlogits, ldd, token_losses, logp,
                                        loss, n_valid, None, None)


def preference(logp=at(0), N=10, offsets=at(1), P=2, cfg=(0, 0.1, 0.0, 0.0, 0, 1), loss=at(2), pair_losses=at(3), ratios=at(4)):
    c = None if cfg is None else C.byref(_lib.PreferenceConfigC(*cfg))
    return _lib.lib().femto_preference_loss(logp, None, None, N, offsets, P, c, loss, pair_losses, ratios, None, None)


ARG, SHAPE, ALIGN = -1, -2, -3


@pytest.mark.parametrize("call", [logprobs, gradient, policy])
@pytest.mark.parametrize("change,code", [(dict(dtype=2), ARG), (dict(dtype=-1), ARG), (dict(logits=None), ARG), (dict(targets0=None), ARG), (dict(N=-1), SHAPE),
                                         (dict(V=0), SHAPE), (dict(ldl=99), SHAPE), (dict(logits=C.c_void_p(BASE + 1)), ALIGN)])
def test_rows_that_are_refused(call, change, code):
    assert call(**change) == code
    assert _lib.lib().femto_last_error(None)


def test_log_probabilities_refuse():
    for t in (0.0, -1.0, 1e-7, 1e7, math.inf, math.nan):
        assert logprobs(temperature=t) == ARG and gradient(temperature=t) == ARG
    assert logprobs(logp=None) == ARG
    assert gradient(dlogits=None) == ARG and gradient(dlogp=None) == ARG
    assert gradient(ldd=99) == SHAPE
    assert gradient(dlogits=C.c_void_p(3 * BASE + 1)) == ALIGN


def test_a_gradient_in_place_has_the_same_rows():
    for call in (gradient, policy):
        assert call(dlogits=at(0), ldd=101) == ARG                          # the logits' place with another pitch
        assert call(dlogits=C.c_void_p(BASE + 2)) == ARG                    # one element on
        assert call(dlogits=C.c_void_p(BASE - 2 * 399)) == ARG              # its last element is the first logit


def test_rows_of_the_gradient_and_the_logits_in_turn_do_not_overlap():
    """In one buffer with one pitch, 250 elements of 2 bytes: a row of 100 logits, and one of the gradient in what is left."""
    for call in (gradient, policy):
        for d in (0, 2, 198, 302, 498):           # bytes behind the logits' first row: 0 and 498 within a pitch of the row's own place
            for turns in (0, 1, 2):               # the gradient's first row may be that many pitches on
                if d or turns:
                    assert call(ldl=250, ldd=250, dlogits=C.c_void_p(BASE + d + 500 * turns)) == ARG, (d, turns)
        assert call(ldl=250, ldd=251, dlogits=C.c_void_p(BASE + 200)) == ARG      # of two pitches some rows meet, or may
        assert call(ldl=199, ldd=199, dlogits=C.c_void_p(BASE + 200)) == ARG      # one element short


def test_policy_refuses():
    for name in ("old", "adv", "token_losses", "logp", "loss", "n_valid", "cfg"):
        assert policy(**{name: None}) == ARG, name
    for cfg in ((0.0, 0.2, 0.2, 0.0, 0), (1.0, -0.1, 0.2, 0.0, 0), (1.0, 1.1, 0.2, 0.0, 0), (1.0, 0.2, -0.2, 0.0, 0), (1.0, math.nan, 0.2, 0.0, 0),
                (1.0, 0.2, math.nan, 0.0, 0), (1.0, 0.2, 0.2, -1.0, 0), (1.0, 0.2, 0.2, math.inf, 0), (1.0, 0.2, 0.2, 0.1, 0), (1.0, 0.2, 0.2, 0.0, 2)):
        assert policy(cfg=cfg) == ARG, cfg


def test_preference_refuses():
    for name in ("logp", "offsets", "loss", "pair_losses", "ratios", "cfg"):
        assert preference(**{name: None}) == ARG, name
    assert preference(N=-1) == SHAPE and preference(P=-1) == SHAPE and preference(P=1 << 30) == SHAPE
    for cfg in ((2, 0.1, 0, 0, 0, 1), (0, 0.0, 0, 0, 0, 1), (0, math.nan, 0, 0, 0, 1), (0, 0.1, math.inf, 0, 0, 1), (0, 0.1, 0, 1.5, 0, 1), (0, 0.1, 0, -0.1, 0, 1),
                (1, 0.1, 0.5, 0, 0, 1), (1, 0.1, 0, 0.1, 0, 1), (0, 0.1, 0, 0, 0, 2)):
        assert preference(cfg=cfg) == ARG, cfg


def test_python_refuses_what_is_not_on_the_device():
    z, t = torch.zeros(2, 5), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        fb.token_logprobs(z, t)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        fb.token_logprobs(z.double(), t)
    with pytest.raises(ValueError, match="CUDA"):
        fb.preference_loss(torch.zeros(3), torch.tensor([0, 1, 3], dtype=torch.int32))


def test_policy_loss_refuses_a_place_for_a_gradient_that_it_does_not_compute():
    z, t, f = torch.zeros(2, 5), torch.zeros(2, dtype=torch.int32), torch.zeros(2)
    with pytest.raises(ValueError, match="gradient=False"):
        fb.policy_loss(z, t, f, f, gradient=False, out=z)


def test_python_refuses_options():
    from femtochat_b200 import objectives
    with pytest.raises(ValueError, match="reduction"):
        objectives._policy_config(0.2, 0.2, 0.0, 1.0, "none")
    with pytest.raises(ValueError, match="kind"):
        objectives._preference_config("hinge", 0.1, 0.0, 0.0, False, "mean")
    assert objectives._policy_config(0.2, None, 0.0, 1.0, "sum").clip_high == math.inf


def test_steps_refuse_without_a_handle():
    L, c, q = _lib.lib(), C.byref(_lib.PolicyConfigC(1.0, 0.2, 0.2, 0.0, 0)), C.byref(_lib.PreferenceConfigC(0, 0.1, 0.0, 0.0, 0, 1))
    assert L.femto_forward_token_logprobs(None, at(0), at(1), at(2), None, 1, 1.0, at(3), None) == ARG
    assert L.femto_policy_loss_and_gradient(None, at(0), at(1), at(2), at(3), None, 1, at(4), at(5), None, None, c, 0, at(6), at(7), None, None, None) == ARG
    assert L.femto_preference_loss_and_gradient(None, at(0), at(1), at(2), at(3), None, 1, None, at(4), 1, q, 0, at(5), at(6), at(7), None, None) == ARG


T = 8


def steps_of(tokens, targets, positions=None):
    """The three steps on a batch; the model is one without a handle, so that a call that is not refused cannot launch anything."""
    from types import SimpleNamespace
    params = SimpleNamespace(theta=torch.zeros(16), delta=torch.zeros(16))
    state = SimpleNamespace(h=None, config=SimpleNamespace(sequence_len=T))
    rows, offsets = torch.zeros(tokens.shape), torch.tensor([0, 1, 2], dtype=torch.int32)
    return (lambda: fb.forward_token_logprobs(params, state, None, tokens, targets, positions),
            lambda: fb.policy_loss_and_gradient_(params, state, None, tokens, targets, rows, rows, positions=positions),
            lambda: fb.preference_loss_and_gradient_(params, state, None, tokens, targets, offsets, positions=positions))


def ids(*shape):
    return torch.ones(shape, dtype=torch.int32)


@pytest.mark.parametrize("tokens,targets,positions,match", [
    (ids(2, T - 1), ids(2, T - 1), None, "tokens must be"), (ids(2, T + 1), ids(2, T + 1), None, "tokens must be"), (ids(2 * T), ids(2 * T), None, "tokens must be"),
    (ids(1, 2, T), ids(1, 2, T), None, "tokens must be"), (ids(2, T), ids(2, T - 1), None, "targets has shape"), (ids(2, T), ids(1, T), None, "targets has shape"),
    (ids(2, T), ids(2 * T), None, "targets has shape"), (ids(2, T), ids(2, T), ids(2, T - 1), "positions has shape"), (ids(2, T), ids(2, T), ids(T), "positions has shape")])
def test_steps_refuse_a_batch_of_another_shape(tokens, targets, positions, match):
    """The library reads and writes B x sequence_len entries of every array."""
    for step in steps_of(tokens, targets, positions):
        with pytest.raises(ValueError, match=match):
            step()


@pytest.mark.parametrize("tokens,targets,positions,match", [
    (ids(2, T - 1), ids(2, T - 1), None, "tokens must be"), (ids(2, T + 1), ids(2, T + 1), None, "tokens must be"), (ids(2, T), ids(2, T - 1), None, "targets has shape"),
    (ids(2, T), ids(2, T), ids(2, T - 1), "positions has shape")])
def test_model_calls_refuse_a_batch_of_another_shape(tokens, targets, positions, match):
    """As above: the losses of all tokens and the logits have B x sequence_len entries too."""
    from types import SimpleNamespace
    params = SimpleNamespace(theta=torch.zeros(16), delta=torch.zeros(16))
    config = SimpleNamespace(sequence_len=T, vocab_size=9)
    state = SimpleNamespace(h=None, config=config)
    model = fb.GPT(params, config, None)
    model.state = lambda B: pytest.fail("the batch was not refused")
    calls = [lambda: fb.loss_and_gradient_(params, state, None, tokens, targets, positions), lambda: model(tokens, targets, positions),
             lambda: model(tokens, targets, positions, reduction="none"), lambda: model.token_logprobs(tokens, targets, positions),
             lambda: fb.loss_and_gradient_host_(params, state, tokens, targets, positions)]
    if "targets" not in match:
        calls.append(lambda: model.logits(tokens, positions))
    for call in calls:
        with pytest.raises(ValueError, match=match):
            call()


def test_steps_refuse_no_targets():
    for step in steps_of(ids(2, T), None):
        with pytest.raises(ValueError, match="targets is None"):
            step()


def test_self_test_of_the_waits_refuses():
    word = C.c_int32(0)

    def call(dtype=0, d=at(0), z=at(1), ldl=9, t=at(2), N=3, V=9, dlogp=at(3), logp=at(4), polls=0, out=C.byref(word)):
        return _lib.lib().femto_selftest_rows_wait(dtype, d, z, ldl, t, N, V, dlogp, logp, polls, out, None)

    for change in (dict(dtype=2), dict(z=None), dict(t=None), dict(dlogp=None), dict(d=None, logp=None), dict(out=None)):
        assert call(**change) == ARG, change
    for change in (dict(N=0), dict(V=0), dict(ldl=8), dict(polls=-1)):
        assert call(**change) == SHAPE, change


def test_steps_refuse_a_decoder_by_name():
    """A decoder that lists its layers has no sequence_len, so that there is no shape to hold its batch to."""
    from types import SimpleNamespace
    params, state = SimpleNamespace(theta=torch.zeros(16), delta=None), SimpleNamespace(h=None, config=SimpleNamespace(sequence_len=None))
    with pytest.raises(ValueError, match="decoder"):
        fb.forward_token_logprobs(params, state, None, ids(2, T), ids(2, T))

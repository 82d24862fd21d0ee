"""Objectives on a model's own answers (femto_token_logprobs*, femto_policy_loss, femto_preference_loss): what a host calls after
pretraining, when answers have rewards or come in pairs.  No counterpart in the reference.  Every call is asynchronous on the current
stream and returns device tensors; nothing is read back, so a call may be captured into a graph.  What only the device can see, targets
outside the vocabulary or offsets that descend, is taken as nothing and reported by `status_word()`.

Logits are [..., V] with unit stride along V and one pitch between rows, as `GPT.logits` and `decode_step` give them, or cut from a wider
buffer; float32 or bfloat16.  Targets are 0-based here (`targets0`; the model's own ids may start at 1), negative where a row counts for
nothing.  Arrays of one number per token have the logits' leading shape and are float32."""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional

from . import _lib
from .gpt import _batch

PREFERENCES = {"sigmoid": 0, "squared": 1}


class TokenLogprobs(NamedTuple):
    logp: object
    entropy: Optional[object]


class PolicyLoss(NamedTuple):
    loss: object            # [1]
    n_valid: object         # [1] int32, tokens with a target
    n_clipped: object       # [1] int32, those that the clipping held
    token_losses: object
    logp: object
    dlogits: Optional[object]


class PreferenceLoss(NamedTuple):
    loss: object            # [1]
    pair_losses: object     # [P]
    ratios: object          # [2 P]: rho of the chosen and the rejected answer in turn
    dlogp: Optional[object]


def _on_device(name, t, dtype, shape, device):
    """A contiguous array of `shape` on `device`, or an error that names it."""
    if t is None:
        return None
    if t.dtype is dtype and t.shape == shape and t.device == device:
        return t if t.is_contiguous() else t.contiguous()
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    raise ValueError(f"{name} has shape {tuple(t.shape)}, not {tuple(shape)}")


def _address(t):
    return None if t is None else t.data_ptr()


def _rows(name, t):
    """(rows, V, pitch, type) of [..., V] logits whose rows lie one pitch apart."""
    import torch
    code = _lib.F32 if t.dtype is torch.float32 else _lib.BF16 if t.dtype is torch.bfloat16 else None
    if code is None:
        raise ValueError(f"{name} must be float32 or bfloat16, not {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device")
    shape = t.shape
    if not shape or shape[-1] == 0:
        raise ValueError(f"{name} must be [..., V]")
    V, n = shape[-1], t.numel() // shape[-1]
    if n >= 1 << 31 or V >= 1 << 31:
        raise ValueError(f"{name}: {n} rows of {V}")
    if n == 0 or t.is_contiguous():
        return n, V, V, code
    strides = t.stride()
    if V > 1 and strides[-1] != 1:
        raise ValueError(f"{name} must have unit stride along the vocabulary")
    pitch, reach = None, 1
    for size, stride in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if size == 1:
            continue
        if pitch is None:
            pitch = stride
        elif stride != pitch * reach:
            raise ValueError(f"the rows of {name} must lie one pitch apart")
        reach *= size
    if pitch is None:
        pitch = V
    if pitch < V:
        raise ValueError(f"the rows of {name} overlap")
    return n, V, pitch, code


def _gradient_of(logits, n, V, pitch, out):
    """The tensor that takes the gradient, and its pitch: the logits' own where that wastes little, so that rows of both start alike."""
    import torch
    if out is None:
        if pitch == V:
            return torch.empty_like(logits, memory_format=torch.contiguous_format), V
        if pitch - V > V // 8 + 64:
            return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device), V
        return torch.empty((n, pitch), dtype=logits.dtype, device=logits.device)[:, :V].view(logits.shape), pitch
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        raise ValueError("out must have the logits' shape, type and device")
    return out, _rows("out", out)[2]


class PolicyStep(NamedTuple):
    loss: object            # [1]
    n_valid: object         # [1] int32
    n_clipped: object       # [1] int32
    logp: object            # [B][T]


class PreferenceStep(NamedTuple):
    loss: object            # [1]
    pair_losses: object     # [P]
    ratios: object          # [2 P]
    logp: object            # [B][T]


def _call(device, name, *args):
    """The library's call on the current stream of the tensors' device."""
    import torch
    if device.index == torch.cuda.current_device():
        _lib.check(getattr(_lib.lib(), name)(*args, _lib.stream_ptr()))
    else:
        with torch.cuda.device(device):
            _lib.check(getattr(_lib.lib(), name)(*args, _lib.stream_ptr()))


def token_logprobs(logits, targets0, temperature: float = 1.0, entropy: bool = False) -> TokenLogprobs:
    """Log-probabilities of the targets under softmax(logits / temperature), and the entropy where asked for."""
    import torch
    n, V, pitch, code = _rows("logits", logits)
    shape, device = logits.shape[:-1], logits.device
    targets0 = _on_device("targets0", targets0, torch.int32, shape, device)
    if targets0 is None:
        raise ValueError("targets0 is None")
    logp = torch.empty_like(targets0, dtype=torch.float32)
    ent = torch.empty_like(logp) if entropy else None
    _call(device, "femto_token_logprobs", code, logits.data_ptr(), pitch, _address(targets0), n, V, temperature, logp.data_ptr(), _address(ent))
    return TokenLogprobs(logp, ent)


def token_logprobs_gradient(logits, targets0, dlogp, dentropy=None, temperature: float = 1.0, out=None):
    """d objective / d logits from d objective / d logp (and / d entropy).  `out` may be the logits themselves."""
    import torch
    n, V, pitch, code = _rows("logits", logits)
    shape, f32, device = logits.shape[:-1], torch.float32, logits.device
    targets0 = _on_device("targets0", targets0, torch.int32, shape, device)
    dlogp, dentropy = _on_device("dlogp", dlogp, f32, shape, device), _on_device("dentropy", dentropy, f32, shape, device)
    out, out_pitch = _gradient_of(logits, n, V, pitch, out)
    _call(device, "femto_token_logprobs_gradient", code, out.data_ptr(), out_pitch, logits.data_ptr(), pitch, _address(targets0), n, V, temperature,
          _address(dlogp), _address(dentropy))
    return out


def _policy_config(clip_low, clip_high, kl_coef, temperature, reduction):
    if reduction not in _lib.REDUCTION:
        raise ValueError(f"reduction must be 'sum' or 'mean', not {reduction!r}")
    return _lib.PolicyConfigC(temperature, clip_low, math.inf if clip_high is None else clip_high, kl_coef, _lib.REDUCTION[reduction])


def policy_loss(logits, targets0, old_logp, advantages, ref_logp=None, weights=None, clip_low: float = 0.2, clip_high: Optional[float] = 0.2,
                kl_coef: float = 0.0, temperature: float = 1.0, reduction: str = "sum", gradient: bool = True, out=None) -> PolicyLoss:
    """Clipped policy loss with a KL term, and its gradient by the logits in the same pass:
    weight (-min(r A, clamp(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (e^g - g - 1)) per token, r = exp(logp - old_logp) and
    g = ref_logp - logp.  clip_high=None bounds the ratio below only.  `out` may be the logits themselves."""
    import torch
    if out is not None and not gradient:
        raise ValueError("out takes the gradient, which gradient=False leaves out")
    n, V, pitch, code = _rows("logits", logits)
    shape, f32, device = logits.shape[:-1], torch.float32, logits.device
    targets0 = _on_device("targets0", targets0, torch.int32, shape, device)
    old_logp, advantages = _on_device("old_logp", old_logp, f32, shape, device), _on_device("advantages", advantages, f32, shape, device)
    ref_logp, weights = _on_device("ref_logp", ref_logp, f32, shape, device), _on_device("weights", weights, f32, shape, device)
    cfg = _policy_config(clip_low, clip_high, kl_coef, temperature, reduction)
    d, d_pitch = _gradient_of(logits, n, V, pitch, out) if gradient else (None, V)
    if targets0 is None or old_logp is None or advantages is None:
        raise ValueError("targets0, old_logp or advantages is None")
    token_losses, logp = torch.empty_like(old_logp), torch.empty_like(old_logp)
    loss, n_valid, n_clipped = old_logp.new_empty(1), targets0.new_empty(1), targets0.new_empty(1)
    _call(device, "femto_policy_loss", code, logits.data_ptr(), pitch, _address(targets0), n, V, _address(old_logp), _address(advantages),
          _address(ref_logp), _address(weights), C.byref(cfg), _address(d), d_pitch, token_losses.data_ptr(), logp.data_ptr(), loss.data_ptr(),
          n_valid.data_ptr(), n_clipped.data_ptr())
    return PolicyLoss(loss, n_valid, n_clipped, token_losses, logp, d)


def _preference_config(kind, beta, margin, label_smoothing, length_normalised, reduction):
    if kind not in PREFERENCES:
        raise ValueError(f"kind must be 'sigmoid' or 'squared', not {kind!r}")
    if reduction not in _lib.REDUCTION:
        raise ValueError(f"reduction must be 'sum' or 'mean', not {reduction!r}")
    return _lib.PreferenceConfigC(PREFERENCES[kind], beta, margin, label_smoothing, 1 if length_normalised else 0, _lib.REDUCTION[reduction])


def _offsets(offsets, device):
    import torch
    if offsets.dim() != 1 or offsets.shape[0] % 2 != 1:
        raise ValueError(f"offsets must be [2 P + 1], not {tuple(offsets.shape)}")
    return _on_device("offsets", offsets, torch.int32, offsets.shape, device), offsets.shape[0] // 2


def preference_loss(logp, offsets, targets0=None, ref_logp=None, kind: str = "sigmoid", beta: float = 0.1, margin: float = 0.0,
                    label_smoothing: float = 0.0, length_normalised: bool = False, reduction: str = "mean", gradient: bool = True) -> PreferenceLoss:
    """Preference loss of pairs of answers from their tokens' log-probabilities (any shape, taken in order): answer k is the rows
    offsets[k] .. offsets[k + 1] - 1 (int32 [2 P + 1], ascending), chosen and rejected in turn; tokens with a negative target do not count.
    `dlogp` is what `token_logprobs_gradient` takes."""
    import torch
    if not logp.is_cuda:
        raise ValueError("logp must be on a CUDA device")
    f32, device, shape = torch.float32, logp.device, logp.shape
    logp, ref_logp = _on_device("logp", logp, f32, shape, device), _on_device("ref_logp", ref_logp, f32, shape, device)
    targets0 = _on_device("targets0", targets0, torch.int32, shape, device)
    offsets, P = _offsets(offsets, device)
    n = logp.numel()
    if n >= 1 << 31:
        raise ValueError(f"{n} tokens")
    cfg = _preference_config(kind, beta, margin, label_smoothing, length_normalised, reduction)
    loss, pair_losses, ratios = logp.new_empty(1), logp.new_empty(P), logp.new_empty(2 * P)
    dlogp = torch.empty_like(logp) if gradient else None
    _call(device, "femto_preference_loss", logp.data_ptr(), _address(ref_logp), _address(targets0), n, offsets.data_ptr(), P, C.byref(cfg),
          loss.data_ptr(), pair_losses.data_ptr(), ratios.data_ptr(), _address(dlogp))
    return PreferenceLoss(loss, pair_losses, ratios, dlogp)


# ---- the GPT's steps ----------------------------------------------------------------------------------------------------------------------
def forward_token_logprobs(params, state, layout, tokens, targets, positions=None, temperature: float = 1.0):
    """Log-probabilities [B][T] that the model gives the targets (0 where ignored), at a temperature: those of answers before an update, or
    under a reference model.  Tokens, targets and positions as for `loss_and_gradient_`: [B][sequence_len]; shorter answers are padded, their targets
    ignored there."""
    import torch
    tok, tgt, pos = _batch(state.config, params.theta.device, tokens, targets, positions)
    logp = torch.empty(tok.shape, dtype=torch.float32, device=tok.device)
    _call(tok.device, "femto_forward_token_logprobs", state.h, _lib.ptr(params.theta), _lib.ptr(tok), _lib.ptr(tgt), _lib.ptr(pos), tok.shape[0],
          temperature, _lib.ptr(logp))
    return logp


def policy_loss_and_gradient_(params, state, layout, tokens, targets, old_logp, advantages, positions=None, ref_logp=None, weights=None,
                              clip_low: float = 0.2, clip_high: Optional[float] = 0.2, kl_coef: float = 0.0, temperature: float = 1.0,
                              reduction: str = "sum", accumulate: bool = False) -> PolicyStep:
    """A training step on `policy_loss`: fills params.delta (or adds to it), as `loss_and_gradient_` does for the cross-entropy.  old_logp,
    advantages, ref_logp and weights are [B][T]."""
    import torch
    tok, tgt, pos = _batch(state.config, params.theta.device, tokens, targets, positions)
    f32, device = torch.float32, tok.device
    old_logp, advantages, ref_logp, weights = (_on_device(name, t, f32, tok.shape, device) for name, t in
                                               (("old_logp", old_logp), ("advantages", advantages), ("ref_logp", ref_logp), ("weights", weights)))
    cfg = _policy_config(clip_low, clip_high, kl_coef, temperature, reduction)
    loss, logp = torch.empty(1, dtype=f32, device=device), torch.empty(tok.shape, dtype=f32, device=device)
    n_valid, n_clipped = torch.empty(1, dtype=torch.int32, device=device), torch.empty(1, dtype=torch.int32, device=device)
    _call(device, "femto_policy_loss_and_gradient", state.h, _lib.ptr(params.theta), _lib.ptr(params.delta), _lib.ptr(tok), _lib.ptr(tgt), _lib.ptr(pos),
          tok.shape[0], _lib.ptr(old_logp), _lib.ptr(advantages), _lib.ptr(ref_logp), _lib.ptr(weights), C.byref(cfg), 1 if accumulate else 0,
          _lib.ptr(loss), _lib.ptr(n_valid), _lib.ptr(n_clipped), _lib.ptr(logp))
    return PolicyStep(loss, n_valid, n_clipped, logp)


def preference_loss_and_gradient_(params, state, layout, tokens, targets, offsets, positions=None, ref_logp=None, kind: str = "sigmoid",
                                  beta: float = 0.1, margin: float = 0.0, label_smoothing: float = 0.0, length_normalised: bool = False,
                                  reduction: str = "mean", accumulate: bool = False) -> PreferenceStep:
    """A training step on `preference_loss`: fills params.delta (or adds to it).  offsets [2 P + 1] (int32) count rows of the flattened [B][T]
    arrays; with one answer a column, chosen and rejected in turn, they are the multiples of T."""
    import torch
    tok, tgt, pos = _batch(state.config, params.theta.device, tokens, targets, positions)
    f32, device = torch.float32, tok.device
    ref_logp = _on_device("ref_logp", ref_logp, f32, tok.shape, device)
    offsets, P = _offsets(offsets, device)
    cfg = _preference_config(kind, beta, margin, label_smoothing, length_normalised, reduction)
    loss, logp = torch.empty(1, dtype=f32, device=device), torch.empty(tok.shape, dtype=f32, device=device)
    pair_losses, ratios = torch.empty(P, dtype=f32, device=device), torch.empty(2 * P, dtype=f32, device=device)
    _call(device, "femto_preference_loss_and_gradient", state.h, _lib.ptr(params.theta), _lib.ptr(params.delta), _lib.ptr(tok), _lib.ptr(tgt), _lib.ptr(pos),
          tok.shape[0], _lib.ptr(ref_logp), _lib.ptr(offsets), P, C.byref(cfg), 1 if accumulate else 0, _lib.ptr(loss), _lib.ptr(pair_losses),
          _lib.ptr(ratios), _lib.ptr(logp))
    return PreferenceStep(loss, pair_losses, ratios, logp)

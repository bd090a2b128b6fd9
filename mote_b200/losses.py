"""Losses on logits for post-training, with their gradients: what the reference's preference and policy loops
(mote/train/dpo.py, kto.py, rlvr.py) compute between the model and the clip + AdamW step (dpo.py:217, kto.py:151,
rlvr.py:308) that `fused_step` replaces.

    r = policy_loss(logits, targets, advantages, old_logprobs, ref_logprobs, kl_coef=0.04)
    logits.backward(r.grad)
    fused_step(opt, max_norm=1.0, grad_divisor=r.count)      # the losses are sums: divided here, over any micro-batches

The calls read logits and write their gradient in the logits' type; nothing is recorded for autograd, so the gradient is
handed on with `logits.backward(grad)` (a step that is captured into a CUDA graph captures that too).

Logits are [S, T, V] (S sequences of T positions) or [N, V] (packed positions), fp32 or bf16, on the GPU. The last axis has
to be contiguous; the others may be strided (`logits[:, :-1]` needs no copy). A position whose target is negative does not
count: it is not read, its log-probability and its gradient are 0, whatever its logits hold. A target of V or more makes its
position NaN. `targets` is int64, one shape with the logits' leading axes; the label of a position stands at that position
(shift the targets, or the logits, by one for next-token prediction).

Two calls on the same inputs give the same bits. Scratch memory is allocated per call on the current stream.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib as L
from .functional import _device_divisor

Divisor = Union[None, float, torch.Tensor]


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor   # fp32, the targets' shape
    lse: torch.Tensor        # fp32, the targets' shape


class PolicyLoss(NamedTuple):
    loss: torch.Tensor       # fp32 0-dim
    count: torch.Tensor      # fp32 0-dim: the counted positions' weights, summed
    kl: torch.Tensor         # fp32 0-dim: the KL terms, weighted and divided as the loss is, without their coefficient
    clipped: torch.Tensor    # fp32 0-dim: the weights of the positions whose ratio is clipped, summed
    logprobs: torch.Tensor   # fp32, the targets' shape
    grad: Optional[torch.Tensor]


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor       # fp32 0-dim
    rewards: torch.Tensor    # fp32 [S]: beta * (logprobs - ref_logprobs)
    logprobs: torch.Tensor   # fp32 [S]: the sequences' summed (or mean) log-probabilities
    grad: Optional[torch.Tensor]


_DTYPES = {torch.bfloat16: L.DTYPE_BF16, torch.float32: L.DTYPE_F32}
_NONE = L.Positions(None, 0, 0)
_raw_stream = torch._C._cuda_getCurrentRawStream   # torch.cuda.current_stream(i).cuda_stream without the Stream object


def _logits(logits: torch.Tensor, targets: torch.Tensor) -> Tuple[L.Logits, L.Positions]:
    code = _DTYPES.get(logits.dtype)
    if code is None:
        raise TypeError(f"logits must be fp32 or bf16, got {logits.dtype}")
    if not logits.is_cuda:
        raise ValueError("logits must be a CUDA tensor (the losses run only on the GPU)")
    if targets.dtype != torch.int64:
        raise TypeError(f"targets must be int64, got {targets.dtype}")
    shape, st, ty = logits.shape, logits.stride(), targets.stride()
    n = len(shape)
    if n not in (2, 3):
        raise ValueError(f"logits must be [S, T, V] or [N, V], got {tuple(shape)}")
    if targets.shape != shape[:-1]:
        raise ValueError(f"targets {tuple(targets.shape)} do not match logits {tuple(shape)}")
    if targets.get_device() != logits.get_device():
        raise ValueError("targets must be on the logits' device")
    if shape[-1] == 0:
        raise ValueError("logits have no vocabulary")
    if st[-1] != 1 and shape[-1] > 1:
        raise ValueError("the logits' last axis must be contiguous")
    if n == 3:
        return (L.Logits(logits.data_ptr(), code, shape[0], shape[1], shape[2], st[0], st[1]),
                L.Positions(targets.data_ptr(), ty[0], ty[1]))
    return (L.Logits(logits.data_ptr(), code, 1, shape[0], shape[1], 0, st[0]),
            L.Positions(targets.data_ptr(), 0, ty[0]))


def _positions(t: Optional[torch.Tensor], targets: torch.Tensor, what: str, per_sequence: bool = False) -> L.Positions:
    """fp32 values of the targets' shape, or [S] for [S, T] targets where `per_sequence`; none for None."""
    if t is None:
        return _NONE
    if t.dtype != torch.float32:
        raise TypeError(f"{what} must be fp32, got {t.dtype}")
    if t.get_device() != targets.get_device():
        raise ValueError(f"{what} must be on the logits' device")
    st = t.stride()
    if t.shape == targets.shape:
        return L.Positions(t.data_ptr(), st[0], st[1]) if len(st) == 2 else L.Positions(t.data_ptr(), 0, st[0])
    if per_sequence and targets.ndim == 2 and t.shape == targets.shape[:1]:
        return L.Positions(t.data_ptr(), st[0], 0)
    raise ValueError(f"{what} {tuple(t.shape)} does not match targets {tuple(targets.shape)}")


def _divisor(divisor: Divisor, dev: torch.device) -> Tuple[float, Optional[torch.Tensor]]:
    if divisor is None:
        return 1.0, None
    if isinstance(divisor, torch.Tensor):
        return 0.0, _device_divisor(divisor, dev)
    return float(divisor), None


def _call(fn, what: str, index: int, *args) -> None:
    """One library call on the current stream of device `index`, with that device current."""
    if torch.cuda.current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc != 0:
        L.check(rc, what)


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, *, temperature: float = 1.0) -> TokenLogprobs:
    """log_softmax(logits / temperature) at the targets, and the log of the sum of exponentials, in one read of the
    logits: the old and reference log-probabilities of policy_loss, the reference sums of preference_loss
    (`r.logprobs.sum(-1)`), or a loss of the caller's own with token_logprobs_backward."""
    z, y = _logits(logits, targets)
    logp = torch.empty(targets.shape, dtype=torch.float32, device=logits.device)
    lse = torch.empty_like(logp)
    _call(L.lib.moteopt_token_logprobs, "moteopt_token_logprobs", logits.get_device(), z, y, temperature, logp.data_ptr(),
          lse.data_ptr())
    return TokenLogprobs(logp, lse)


def token_logprobs_backward(logits: torch.Tensor, targets: torch.Tensor, logprobs: torch.Tensor, lse: torch.Tensor,
                            grad_logprobs: torch.Tensor, *, temperature: float = 1.0) -> torch.Tensor:
    """The gradient in the logits of sum(grad_logprobs * logprobs), from what token_logprobs gave for the same logits,
    targets and temperature: grad ([j == y] - softmax_j) / temperature. Positions whose grad_logprobs is 0 are not read
    and get 0. `grad_logprobs` is the targets' shape, or [S] for [S, T] targets."""
    z, y = _logits(logits, targets)
    lp, ls = _positions(logprobs, targets, "logprobs"), _positions(lse, targets, "lse")
    g = _positions(grad_logprobs, targets, "grad_logprobs", True)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    _call(L.lib.moteopt_token_logprobs_backward, "moteopt_token_logprobs_backward", logits.get_device(), z, y, temperature,
          lp, ls, g, grad.data_ptr())
    return grad


def policy_loss(logits: torch.Tensor, targets: torch.Tensor, advantages: torch.Tensor, old_logprobs: torch.Tensor,
                ref_logprobs: Optional[torch.Tensor] = None, *, weights: Optional[torch.Tensor] = None,
                clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0, temperature: float = 1.0,
                divisor: Divisor = None, grad: bool = True) -> PolicyLoss:
    """The clipped policy loss with a KL term, and its gradient in the logits (rlvr.py's loop). Per counted position:

        r = exp(logp - old),  d = ref - logp
        loss += w (-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(d) - d - 1)) / divisor

    `advantages` and `weights` are the targets' shape, or [S] (one per sequence) for [S, T] targets; a position of weight 0
    does not count. The loss is a sum: divide by a number, by a one-element tensor (read on the device), or later by
    `fused_step(grad_divisor=count)`; weights of 1 / length with divisor S give the mean over sequences of their means.
    Without `ref_logprobs` there is no KL term (kl_coef must be 0); with it and kl_coef 0 the KL is only measured.
    `grad=False` leaves the gradient out."""
    z, y = _logits(logits, targets)
    dev, index = logits.device, logits.get_device()
    if kl_coef != 0.0 and ref_logprobs is None:
        raise ValueError("policy_loss: kl_coef needs ref_logprobs")
    div, div_t = _divisor(divisor, dev)
    p = L.Policy(_positions(advantages, targets, "advantages", True), _positions(old_logprobs, targets, "old_logprobs"),
                 _positions(ref_logprobs, targets, "ref_logprobs"), _positions(weights, targets, "weights", True),
                 clip_low, clip_high, kl_coef, div, None if div_t is None else div_t.data_ptr())
    nbytes = L.lib.moteopt_policy_loss_workspace_size(z)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    sums = torch.empty(4, dtype=torch.float32, device=dev)
    logp = torch.empty(targets.shape, dtype=torch.float32, device=dev)
    g = torch.empty(logits.shape, dtype=logits.dtype, device=dev) if grad else None
    _call(L.lib.moteopt_policy_loss, "moteopt_policy_loss", index, z, y, p, temperature, sums.data_ptr(), logp.data_ptr(),
          g.data_ptr() if grad else None, ws.data_ptr(), nbytes)
    loss, count, kl, clipped = sums.unbind(0)
    return PolicyLoss(loss, count, kl, clipped, logp, g)


def preference_loss(logits: torch.Tensor, targets: torch.Tensor, ref_logprobs: Optional[torch.Tensor] = None, *,
                    cu_seqlens: Optional[torch.Tensor] = None, beta: float = 0.1, label_smoothing: float = 0.0,
                    average: bool = False, temperature: float = 1.0, divisor: Divisor = None,
                    grad: bool = True) -> PreferenceLoss:
    """The paired preference loss, and its gradient in the logits (dpo.py's loop). The sequences are the chosen ones, then
    the rejected ones in the same order: [S, T, V] logits with S even, or [N, V] with `cu_seqlens` (int32, S + 1 ascending
    row offsets on the device; rows outside them do not count). With s a sequence's summed log-probability (its mean with
    `average`; 0 where no position counts) and ref_logprobs [S] the reference model's (none: 0):

        u = beta ((s_i - ref_i) - (s_j - ref_j)),  j = i + S / 2
        loss = sum_i (-(1 - label_smoothing) log sigmoid(u) - label_smoothing log sigmoid(-u)) / divisor

    The loss is a sum over pairs (divisor=S / 2 for the mean; a one-element tensor is read on the device). `grad=False`
    leaves the gradient out."""
    z, y = _logits(logits, targets)
    dev, index = logits.device, logits.get_device()
    if cu_seqlens is not None:
        if logits.ndim != 2:
            raise ValueError("preference_loss: cu_seqlens goes with [N, V] logits")
        if cu_seqlens.dtype != torch.int32 or cu_seqlens.ndim != 1 or not cu_seqlens.is_contiguous():
            raise TypeError("cu_seqlens must be a contiguous int32 vector")
        if cu_seqlens.get_device() != index:
            raise ValueError("cu_seqlens must be on the logits' device")
        seqs = cu_seqlens.numel() - 1
    else:
        if logits.ndim != 3:
            raise ValueError("preference_loss: [N, V] logits need cu_seqlens")
        seqs = logits.shape[0]
    if seqs < 0 or seqs % 2:
        raise ValueError(f"preference_loss: chosen and rejected sequences come in pairs, got {seqs}")
    if ref_logprobs is not None:
        if ref_logprobs.dtype != torch.float32:
            raise TypeError(f"ref_logprobs must be fp32, got {ref_logprobs.dtype}")
        if ref_logprobs.shape != (seqs,) or ref_logprobs.get_device() != index or not ref_logprobs.is_contiguous():
            raise ValueError(f"ref_logprobs must be a contiguous vector of {seqs} on the logits' device")
    div, div_t = _divisor(divisor, dev)
    p = L.Preference(seqs, None if cu_seqlens is None else cu_seqlens.data_ptr(),
                     None if ref_logprobs is None else ref_logprobs.data_ptr(), beta, label_smoothing, bool(average), div,
                     None if div_t is None else div_t.data_ptr())
    nbytes = L.lib.moteopt_preference_loss_workspace_size(z, seqs)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    rewards = torch.empty(seqs, dtype=torch.float32, device=dev)
    logp = torch.empty_like(rewards)
    g = torch.empty(logits.shape, dtype=logits.dtype, device=dev) if grad else None
    _call(L.lib.moteopt_preference_loss, "moteopt_preference_loss", index, z, y, p, temperature, loss.data_ptr(),
          rewards.data_ptr(), logp.data_ptr(), g.data_ptr() if grad else None, ws.data_ptr(), nbytes)
    return PreferenceLoss(loss, rewards, logp, g)

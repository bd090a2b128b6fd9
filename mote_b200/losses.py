"""Losses on logits for post-training, with their gradients: what stands between a model and the clip + AdamW step that
`fused_step` replaces in loops like the reference's (mote/train/dpo.py:217, kto.py:151, rlvr.py:308).

    r = policy_loss(logits, targets, advantages, old_logprobs, ref_logprobs, kl_coef=0.04)
    logits.backward(r.grad)
    fused_step(opt, max_norm=1.0, grad_divisor=r.count)      # the losses are sums: divided here, over any micro-batches

The calls read logits and write their gradient in the logits' type; nothing is recorded for autograd, so the gradient is
handed on with `logits.backward(grad)` (a step that is captured into a CUDA graph captures that too). Tensors with a
forward-mode tangent are refused.

Logits are [S, T, V] (S sequences of T positions) or [N, V] (packed positions), fp32 or bf16, on the GPU. The last axis has
to be contiguous; the others may be strided (`logits[:, :-1]` needs no copy). A position whose target is negative does not
count: it is not read, its log-probability and its gradient are 0, whatever its logits hold. A target of V or more makes its
position NaN. `targets` is int64, one shape with the logits' leading axes; the label of a position stands at that position
(shift the targets, or the logits, by one for next-token prediction).

`temperature` divides the logits as torch divides fp32 by a number: a product with its fp32 reciprocal.

Two calls on the same inputs give the same bits. Scratch memory is allocated per call on the current stream. The argument
checks and allocations are in C++ (csrc/torch_losses.cpp, mote_b200/_torch_losses.so).
"""

from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib as L
from . import build
from .functional import _device_divisor

Divisor = Union[None, float, torch.Tensor]


def _load():
    import importlib.util
    if not build.BINDING.exists():
        raise ImportError(f"{build.BINDING.name} not found at {build.BINDING}: build it with `python -m mote_b200.build`")
    if not build.binding_fits():
        raise ImportError(f"{build.BINDING} was not built for {build.built_for()}: build it again with `python -m mote_b200.build`")
    spec = importlib.util.spec_from_file_location("mote_b200._torch_losses", build.BINDING)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    names = ("moteopt_last_error", "moteopt_token_logprobs_workspace_size", "moteopt_token_logprobs", "moteopt_token_logprobs_backward",
             "moteopt_policy_loss_workspace_size", "moteopt_policy_loss", "moteopt_preference_loss_workspace_size",
             "moteopt_preference_loss")
    mod.init(*[C.cast(getattr(L.lib, n), C.c_void_p).value for n in names], L.MoteoptError, torch.OutOfMemoryError)
    return mod


_torch = _load()


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


def _divisor(divisor: Divisor, logits: torch.Tensor) -> Tuple[float, Optional[torch.Tensor]]:
    if divisor is None:
        return 1.0, None
    if isinstance(divisor, torch.Tensor):
        return 0.0, _device_divisor(divisor, logits.device)
    return divisor, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, *, temperature: float = 1.0) -> TokenLogprobs:
    """log_softmax(logits / temperature) at the targets, and the log of the sum of exponentials, in one read of the
    logits: the old and reference log-probabilities of policy_loss, the reference sums of preference_loss
    (`r.logprobs.sum(-1)`), or a loss of the caller's own with token_logprobs_backward."""
    return TokenLogprobs(*_torch.token_logprobs(logits, targets, temperature))


def token_logprobs_backward(logits: torch.Tensor, targets: torch.Tensor, logprobs: torch.Tensor, lse: torch.Tensor,
                            grad_logprobs: torch.Tensor, *, temperature: float = 1.0) -> torch.Tensor:
    """The gradient in the logits of sum(grad_logprobs * logprobs), from what token_logprobs gave for the same logits,
    targets and temperature: grad ([j == y] - exp(x_j - lse)) / temperature. Positions whose grad_logprobs is 0 get 0, whatever
    their logits hold. lse is fp32: where it is of size L, the probabilities are off by 6e-8 L. `grad_logprobs` is the targets' shape, or [S] for [S, T] targets."""
    return _torch.token_logprobs_backward(logits, targets, logprobs, lse, grad_logprobs, temperature)


def policy_loss(logits: torch.Tensor, targets: torch.Tensor, advantages: torch.Tensor, old_logprobs: torch.Tensor,
                ref_logprobs: Optional[torch.Tensor] = None, *, weights: Optional[torch.Tensor] = None,
                clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0, temperature: float = 1.0,
                divisor: Divisor = None, grad: bool = True) -> PolicyLoss:
    """The clipped policy loss with a KL term, and its gradient in the logits (for a loop like rlvr.py). Per counted position:

        r = exp(logp - old),  d = ref - logp
        loss += w (-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(d) - d - 1)) / divisor

    `advantages` and `weights` are the targets' shape, or [S] (one per sequence) for [S, T] targets; a position of weight 0
    does not count. The loss is a sum: divide by a number, by a one-element tensor (read on the device), or later by
    `fused_step(grad_divisor=count)`; weights of 1 / length with divisor S give the mean over sequences of their means.
    Without `ref_logprobs` there is no KL term (kl_coef must be 0); with it and kl_coef 0 the KL is only measured.
    `grad=False` leaves the gradient out."""
    div, div_t = _divisor(divisor, logits)
    return PolicyLoss(*_torch.policy_loss(logits, targets, advantages, old_logprobs, ref_logprobs, weights, clip_low,
                                          clip_high, kl_coef, temperature, div, div_t, grad))


def preference_loss(logits: torch.Tensor, targets: torch.Tensor, ref_logprobs: Optional[torch.Tensor] = None, *,
                    cu_seqlens: Optional[torch.Tensor] = None, beta: float = 0.1, label_smoothing: float = 0.0,
                    average: bool = False, temperature: float = 1.0, divisor: Divisor = None,
                    grad: bool = True) -> PreferenceLoss:
    """The paired preference loss, and its gradient in the logits (for a loop like dpo.py). The sequences are the chosen ones,
    then the rejected ones in the same order: [S, T, V] logits with S even, or [N, V] with `cu_seqlens` (int32, S + 1 ascending
    row offsets on the device, held to [0, N]; rows outside them do not count; where offsets descend, a row of several
    sequences has the coefficient of one of them). With s a sequence's summed log-probability (its mean with `average`; 0 where
    no position counts) and ref_logprobs [S] the reference model's (none: 0):

        u = beta ((s_i - ref_i) - (s_j - ref_j)),  j = i + S / 2
        loss = sum_i (-(1 - label_smoothing) log sigmoid(u) - label_smoothing log sigmoid(-u)) / divisor

    The loss is a sum over pairs (divisor=S / 2 for the mean; a one-element tensor is read on the device). `grad=False`
    leaves the gradient out."""
    div, div_t = _divisor(divisor, logits)
    return PreferenceLoss(*_torch.preference_loss(logits, targets, ref_logprobs, cu_seqlens, beta, label_smoothing, average,
                                                  temperature, div, div_t, grad))

"""The training step that makes the weights an update carries, in hand-written HIP kernels (csrc/step.hip):

    logp = token_logprobs(logits, tokens, mask)              # also under the old and the reference policy
    out = policy_loss(logits, tokens, old_logp, advantages, mask, ref_logp, kl_coef=0.04)
    out.loss.backward()
    norm = grad_norm(grads)
    adamw_step(weights, masters, exp_avg, exp_avg_sq, grads, step=1, lr=1e-6, grad_norm=norm, max_norm=1.0)
    update = encode_update(previous, weights)

The reference leaves this step to its caller (its training loop, bench/grpo.py:57-100, is plain torch).

- All tensors lie on one HIP device.  Work is enqueued on the current stream; nothing waits for the device
  or reads from it, so the calls can be captured into a HIP graph.  Tracers (torch.jit.trace, make_fx) do not see
  kernels: under one the calls raise RuntimeError; torch.compile runs them between its graphs.
- Wrong arguments raise ValueError before anything is enqueued, and so do dual tensors (there are no
  forward-mode derivatives).  What depends on values on the device cannot: a token id outside
  the vocabulary makes its position's results and gradient NaN (and with them the loss).
- A position whose mask is 0 takes no part: its logits and token id are not read (they may hold anything),
  its results are 0 and its gradient is 0.
- Logits that are -inf, or the type's lowest value beside larger ones, have probability 0.  A row without a
  finite logit, with a NaN or with +inf gives NaN, as the formula does.
"""

from __future__ import annotations

import os
import threading
from collections.abc import Mapping
from dataclasses import dataclass

import torch

from . import _native

_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "crx_step.so")
_ENTRIES = ("crx_rows_scratch", "crx_token_logprobs", "crx_token_logprobs_grad", "crx_policy_loss", "crx_policy_loss_grad",
            "crx_norm_scratch", "crx_grad_norm", "crx_clip_grads", "crx_adamw_step")
_ANY_DEVICE = False  # the CPU model of the library takes tensors in host memory
_front = None
_lock = threading.Lock()


def _load():
    """The C++ front (csrc/step_front.cpp), with the entry points of the loaded library."""
    global _front
    with _lock:
        if _front is None:
            if not os.path.exists(_PATH):
                raise _native.NativeLibraryMissing(
                    f"{_PATH} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'`")
            import ctypes
            import importlib.util
            L = _native.lib()
            spec = importlib.util.spec_from_file_location("crx_step", _PATH)
            mod = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(mod)
            raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
            mod.init({name: ctypes.cast(getattr(L, name), ctypes.c_void_p).value for name in _ENTRIES},
                     raw or (lambda index: torch.cuda.current_stream(index).cuda_stream), _ANY_DEVICE)
            _front = mod
    return _front


def _tensor(name: str, t) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name}: expected a torch tensor, got {type(t).__name__}")


def _are_tensors(named) -> None:
    for name, t in named:
        if t is not None:
            _tensor(name, t)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, mask: torch.Tensor | None = None, *,
                   temperature: float = 1.0, entropy: bool = False):
    """log softmax(logits / temperature) at every position's token, in float32; with `entropy`, a pair with the
    entropy of the whole distribution (nats).  Differentiable by the logits.

    logits: [tokens, vocabulary] or [sequences, tokens, vocabulary], bf16, fp16 or fp32, the vocabulary
    contiguous and the other dimensions at any stride (logits[:, :-1] is taken as it is).  tokens: int64 or
    int32 of the leading shape.  mask: bool or uint8 of that shape; positions with 0 score 0."""
    front = _front or _load()
    try:
        return front.token_logprobs(logits, tokens, mask, temperature, entropy)
    except TypeError:
        _tensor("logits", logits), _tensor("tokens", tokens), _are_tensors([("mask", mask)])
        raise


@dataclass
class PolicyLoss:
    """loss: a 0-d float32 tensor; logprobs: of the sampled tokens under the trained policy; kl: the weighted
    mean (by the loss's reduction; "sum": the sum) of exp(ref - logprob) - 1 - (ref - logprob); clipped: that of
    the positions whose ratio is outside the clip range on the side that the advantage pushes to."""
    loss: torch.Tensor
    logprobs: torch.Tensor
    kl: torch.Tensor
    clipped: torch.Tensor


def _policy(logits, tokens, old, advantages, mask, ref, clip, kl_coef, temperature, reduction, scale, direct):
    front = _front or _load()
    try:
        return front.policy_loss(logits, tokens, old, advantages, mask, ref, clip, kl_coef, temperature, reduction, scale, direct)
    except TypeError:
        for name, t in (("logits", logits), ("tokens", tokens), ("old_logprobs", old), ("advantages", advantages)):
            _tensor(name, t)
        _are_tensors([("mask", mask), ("ref_logprobs", ref)])
        raise


def policy_loss(logits: torch.Tensor, tokens: torch.Tensor, old_logprobs: torch.Tensor, advantages: torch.Tensor,
                mask: torch.Tensor | None = None, ref_logprobs: torch.Tensor | None = None, *, clip=(0.2, 0.2),
                kl_coef: float = 0.0, temperature: float = 1.0, reduction: str = "token",
                scale: float = 1.0) -> PolicyLoss:
    """The clipped policy loss of sampled tokens, with a KL penalty against a reference policy.  With r =
    exp(logprob - old) and d = ref - logprob, a position's loss is

        -min(r * A, clamp(r, 1 - clip[0], 1 + clip[1]) * A) + kl_coef * (exp(d) - 1 - d)

    and the loss is `scale` times their mean over the unmasked positions ("token"), the mean over the sequences
    that have an unmasked position of the sequence's mean ("sequence"), or their sum ("sum"; 2-d logits are one
    sequence).  Without any unmasked position it is 0.  Differentiable by the logits only; at a clip limit itself
    a position counts as not clipped.  logits, tokens and mask as in token_logprobs; old_logprobs, advantages and
    ref_logprobs float32, with as many dimensions as tokens, each of its size or of size 1 (advantages of
    [sequences, 1]: one for all tokens of a sequence)."""
    return PolicyLoss(*_policy(logits, tokens, old_logprobs, advantages, mask, ref_logprobs, clip, kl_coef, temperature,
                               reduction, scale, False))


def policy_loss_grad(logits: torch.Tensor, tokens: torch.Tensor, old_logprobs: torch.Tensor, advantages: torch.Tensor,
                     mask: torch.Tensor | None = None, ref_logprobs: torch.Tensor | None = None, *, clip=(0.2, 0.2),
                     kl_coef: float = 0.0, temperature: float = 1.0, reduction: str = "token",
                     scale: float = 1.0) -> tuple[PolicyLoss, torch.Tensor]:
    """policy_loss and its gradient with respect to the logits (of their shape and type) in one call, without
    autograd: for a head that is run a chunk of positions at a time ("sum" with `scale` = 1 / all positions)."""
    r = _policy(logits, tokens, old_logprobs, advantages, mask, ref_logprobs, clip, kl_coef, temperature, reduction, scale,
                True)
    return PolicyLoss(*r[:4]), r[4]


def _items(tensors):
    """A mapping as a dict, a sequence as a list."""
    if isinstance(tensors, (dict, list)):
        return tensors
    return dict(tensors) if isinstance(tensors, Mapping) else list(tensors)


def grad_norm(grads) -> torch.Tensor:
    """The 2-norm of all elements of all gradients together, a 0-d float32 tensor on their device.  grads: a mapping
    or a sequence of contiguous bf16, fp16 or fp32 tensors.  Squares are summed in 64 bits.  The norm itself carries no
    gradient, also where the tensors require one."""
    return (_front or _load()).grad_norm(_items(grads), torch.cuda.current_device)


def clip_grad_norm(grads, max_norm: float) -> torch.Tensor:
    """Scales every gradient, in place, by min(1, max_norm / (norm + 1e-6)), and returns the norm that they had
    (grad_norm).  An infinite norm scales by 0, a NaN makes every gradient NaN.  No two tensors may overlap: a tensor
    listed twice counts twice in the norm and may be scaled twice."""
    return (_front or _load()).clip_grad_norm(_items(grads), max_norm, torch.cuda.current_device)


def adamw_step(weights: Mapping[str, torch.Tensor], masters: Mapping[str, torch.Tensor], exp_avg: Mapping[str, torch.Tensor],
               exp_avg_sq: Mapping[str, torch.Tensor], grads: Mapping[str, torch.Tensor], *, step: int, lr: float,
               betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01, grad_norm: torch.Tensor | None = None,
               max_norm: float | None = None) -> None:
    """One AdamW step, in place, of all tensors together:

        g = c * grad;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
        w = w (1 - lr * weight_decay) - lr / (1 - b1^step) * m / (sqrt(v / (1 - b2^step)) + eps)

    w, m and v are the float32 masters, exp_avg and exp_avg_sq; the weights (bf16, which encode_update
    takes, fp16 or fp32) become the new masters, rounded to nearest even.  With grad_norm (a 0-d float32 tensor
    from grad_norm(), or one reduced over ranks) and max_norm the gradients are clipped on the way, without being
    written: c = min(1, max_norm / (grad_norm + 1e-6)).  `step` counts from 1.  All mappings hold the same names
    and shapes; no two tensors may overlap."""
    if (grad_norm is None) != (max_norm is None):
        raise ValueError("grad_norm and max_norm go together")
    dicts = [d if type(d) is dict else dict(d) for d in (weights, masters, exp_avg, exp_avg_sq, grads)]
    (_front or _load()).adamw_step(dicts, step, lr, betas[0], betas[1], eps, weight_decay, grad_norm,
                                   0.0 if max_norm is None else max_norm)

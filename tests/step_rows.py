"""Gradients of the training step's rows, held element by element to what each may be away from its definition in 64 bits.

In units of u = 2^-24, with s the relative error of a softmax's sum (step_reference.softmax_error):
- a probability p_j = 2^((x_j - m) c) / sum is off by s and by its own exponent's rounding, 3u * |x_j - m| log2(e) / T, of
  itself; below 2^-126 it is 0;
- a log probability by e = s + 4u (its magnitude + ln V), so a ratio by e + 8u of itself, and e^d - 1 by e e^d + 8u |e^d - 1|;
- so the slope a of a row by E = |w scale / T| ((e + 8u) |r A| + kl (e e^d + 8u |e^d - 1|)) + 8u |a|, whatever cancels in it;
- an element a (1[j = y] - p_j) by E |1[j = y] - p_j| + |a| p_j (error of p_j), by 4u |a| more at the token itself (where 1 and p
  cancel), and by the rounding to its own type;
- the entropy's part h p_j (ln p_j + H) by |h| p_j ((error of p_j) |ln p_j + H| + (error of p_j) + 2 (s + 4u) (ln V + 8)).
Nothing is measured against another row or another element."""

from __future__ import annotations

import math

import torch

import step_reference as ref
from step_reference import U


def _softmax(x, tokens, temperature):
    """p, its relative error, ln p (0 where p is 0) and 1[j = y]."""
    z = x.double() / temperature
    z = z - z.amax(-1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    p = e / total
    off = ref.softmax_error(x.shape[-1]) + 3 * U * 1.4427 * torch.where(p > 0, -z, 0.0)
    hit = torch.zeros_like(p).scatter_(-1, tokens.long()[..., None], 1.0)
    return p, off, torch.where(p > 0, z - total.log(), 0.0), hit


def _slope_error(x, tokens, old, adv, mask, rf, kl_coef, temperature, scale, want):
    lp = want["logprobs"]
    e = ref.softmax_error(x.shape[-1]) + 4 * U * (lp.abs() + math.log(x.shape[-1] + 1))
    at = lambda t: t.expand(lp.shape).double()  # noqa: E731
    r = torch.exp(lp - at(old))
    parts = (e + 8 * U) * (r * at(adv)).abs()
    if rf is not None:
        d = at(rf) - lp
        parts = parts + kl_coef * (e * d.exp() + 8 * U * torch.special.expm1(d).abs())
    return parts * want["weight"] * abs(scale) / temperature + 8 * U * want["slope"].abs()


def _weights(on, reduction):
    if reduction == "token":
        return on.double() / max(1, int(on.sum()))
    if reduction == "sequence":
        per = on if on.dim() == 2 else on[None]
        n = per.sum(1, keepdim=True)
        return (per.double() / n.clamp(min=1) / max(1, int((n > 0).sum()))).view(on.shape)
    return on.double()


def check_policy_gradient(grad, x, tokens, old, adv, mask=None, rf=None, *, clip=(0.2, 0.2), kl_coef=0.0, temperature=1.0,
                          reduction="token", scale=1.0):
    """grad against the gradient of the policy loss; clipped rows and masked ones are exactly 0."""
    want = ref.policy(x, tokens, old, adv, mask, rf, clip, kl_coef, temperature, reduction, scale)
    a, on = want["slope"], want["on"]
    want["weight"] = _weights(on, reduction)
    p, off, _, hit = _softmax(x, tokens, temperature)
    wrong = _slope_error(x, tokens, old, adv, mask, rf, kl_coef, temperature, scale, want)
    rel, tiny = ref.round_error(grad.dtype)
    a, wrong = a.abs()[..., None], wrong[..., None]
    tol = rel * want["grad"].abs() + tiny + wrong * (hit - p).abs() + a * (p * off + 2.0 ** -126 + hit * 4 * U)
    live = on & (want["slope"] != 0)
    ref.same(grad[live], want["grad"][live], tol[live], "grad")
    assert not grad[~live].any()


def check_score_gradient(grad, x, tokens, up, up_entropy, mask=None, temperature=1.0):
    p, off, lnp, hit = _softmax(x, tokens, temperature)
    on = torch.ones(p.shape[:-1], dtype=torch.bool, device=p.device) if mask is None else mask.bool()
    want = ref.scores_grad(x, tokens, up, up_entropy, mask, temperature)
    rel, tiny = ref.round_error(grad.dtype)
    tol = rel * want.abs() + tiny
    if up is not None:
        a = up.double().abs()[..., None] / temperature
        tol = tol + a * (4 * U * (hit - p).abs() + p * off + 2.0 ** -126 + hit * 4 * U)
    if up_entropy is not None:
        h = up_entropy.double().abs()[..., None] / temperature
        H = -(p * lnp).sum(-1, keepdim=True)
        more = 2 * (ref.softmax_error(x.shape[-1]) + 4 * U) * (math.log(x.shape[-1] + 1) + 8)
        tol = tol + h * (p * (off * (lnp + H).abs() + off + more) + 2.0 ** -120)
    ref.same(grad[on], want[on], tol[on], "grad")
    assert not grad[~on].any()

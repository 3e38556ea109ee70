"""The element-by-element check of tests/step_rows.py sees what a lost vector, a lost tail or a row of a wrong weight leaves:
on gradients made in 64 bits, with mistakes planted in them.  No device."""

from __future__ import annotations

import pytest
import torch

import step_cases as cases
import step_reference as ref
import step_rows as rows

OPTS = {"clip": (0.2, 0.28), "kl_coef": 0.05, "reduction": "sequence"}


def _lost_tail(g, y):
    g[..., -8:] = 0


def _lost_vector(g, y):
    at = g.shape[-1] // 16 * 8
    g[1, 2, at:at + 16 // g.element_size()] = 0


def _lost_element(g, y):
    g[2, 3, (int(y[2, 3]) + 1) % g.shape[-1]] = 0


def _row_of_another_weight(g, y):
    g[0, 1] *= 1.01


def _token_missed(g, y):
    g[2, 1, y[2, 1]] -= g[2, 1, y[2, 1]].sign() * 0.05 * g[2, 1, y[2, 1]].abs()


def _neighbours_exchanged(g, y):
    at = (int(y[0, 2]) + 1) % (g.shape[-1] - 1)
    g[0, 2, [at, at + 1]] = g[0, 2, [at + 1, at]]


MISTAKES = [_lost_tail, _lost_vector, _lost_element, _row_of_another_weight, _token_missed, _neighbours_exchanged]


def _case(dtype, vocab):
    x, y = cases.logits((3, 4, vocab), dtype, vocab, "cpu")
    y[2, 3] %= vocab - 16
    old, rf, adv = cases.policies(x, y, vocab)
    mask = torch.ones((3, 4), dtype=torch.bool)
    mask[0, 0] = False
    return x, y, old, rf, adv, mask, 1024.0 if dtype == "fp16" else 1.0  # a loss scale, without which fp16 holds little


@pytest.mark.parametrize("dtype", sorted(cases.TYPES))
@pytest.mark.parametrize("vocab", [515, 20011, 65537, 151936])
def test_mistakes_in_policy_gradients_are_seen(dtype, vocab):
    x, y, old, rf, adv, mask, scale = _case(dtype, vocab)
    adv = torch.full_like(adv, 0.3)  # no row is clipped away that a mistake is planted in
    lp = ref.scores(x, y)[0]
    old = (lp - 0.1).float()
    opts = {**OPTS, "scale": scale}
    right = ref.policy(x, y, old, adv, mask, rf, **opts)["grad"].to(cases.TYPES[dtype])
    rows.check_policy_gradient(right, x, y, old, adv, mask, rf, **opts)
    for plant in MISTAKES:
        wrong = right.clone()
        plant(wrong, y)
        assert not torch.equal(wrong, right)
        with pytest.raises(AssertionError, match="off by"):
            rows.check_policy_gradient(wrong, x, y, old, adv, mask, rf, **opts)


@pytest.mark.parametrize("dtype", sorted(cases.TYPES))
@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("vocab", [515, 20011, 151936])
def test_mistakes_in_score_gradients_are_seen(dtype, vocab, entropy):
    x, y, _, _, _, mask, scale = _case(dtype, vocab)
    g = torch.Generator().manual_seed(1)
    up = torch.randn((3, 4), generator=g).abs() * scale + scale
    uh = torch.randn((3, 4), generator=g) * scale if entropy else None
    right = ref.scores_grad(x, y, up, uh, mask, 0.8).to(cases.TYPES[dtype])
    rows.check_score_gradient(right, x, y, up, uh, mask, 0.8)
    for plant in MISTAKES:
        wrong = right.clone()
        plant(wrong, y)
        with pytest.raises(AssertionError, match="off by"):
            rows.check_score_gradient(wrong, x, y, up, uh, mask, 0.8)

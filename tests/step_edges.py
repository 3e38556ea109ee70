"""Checks of the training step's operators that run on any device: on the GPU in tests/test_step_edges.py, and on the CPU
model of the library in tests/model/run_step_edges.py.  Each takes the device's name."""

from __future__ import annotations

import pytest
import torch

import crukx_sync
import step_cases as cases
import step_reference as ref
import step_rows as rows

EDGES = {}


def edge(check):
    EDGES[check.__name__] = check
    return check


def _generator(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ AdamW

@edge
def small_decays_shrink_the_masters(dev):
    """lr * weight_decay far below the spacing of 32-bit numbers at 1, as at lr = 1e-6: a single master hardly shows it,
    the projection of all changes on the masters does.

    Every master is rounded once, by at most u |w|, in directions that do not depend on one another (the updates are random
    and many times a last place); so the projection sum(w dw) / sum(w^2) is off by more than 8 u sqrt(sum w^4) / sum(w^2)
    with a probability below 1e-13.  The decay itself is held to 1e-6 of itself beside that."""
    n = 120_000 if dev == "cpu" else 4_000_000
    g = _generator(1)
    w0 = torch.randn(n, generator=g) * 0.02
    m0, g0 = torch.randn(n, generator=g) * 1e-3, torch.randn(n, generator=g) * 1e-2
    v0 = torch.rand(n, generator=g) * 1e-5
    for wd in (0.01, 0.1, 0.0):
        s = [{"p": t.clone().to(dev)} for t in (w0.bfloat16(), w0, m0, v0, g0)]
        crukx_sync.adamw_step(*s, step=7, lr=1e-6, weight_decay=wd)
        want = ref.adamw(w0, m0, v0, g0, 7, 1e-6, (0.9, 0.999), 1e-8, wd)[0]
        got, w = s[1]["p"].cpu().double(), w0.double()
        off = float(((got - want) * w).sum() / (w * w).sum())
        allowed = 8 * ref.U * float((w ** 4).sum().sqrt() / (w * w).sum()) + 1e-6 * 1e-6 * wd
        assert abs(off) <= allowed, f"decay {wd}: {off / (1e-6 * wd or 1):+.3f} of it too little (allowed {allowed / (1e-6 * wd or 1):.3f})"


@edge
def infinite_masters_stay_infinite(dev):
    """As in the formula, with and without a decay; the neighbours are stepped as ever."""
    w0 = torch.tensor([1.0, float("inf"), -2.0, float("-inf"), 0.0, 3e38])
    for wd in (0.0, 0.1):
        s = [{"p": t.clone().to(dev)} for t in (w0.bfloat16(), w0, torch.ones(6), torch.ones(6), torch.ones(6))]
        crukx_sync.adamw_step(*s, step=3, lr=1e-3, weight_decay=wd)
        one = torch.ones(6)
        want = ref.adamw(w0, one, one, one, 3, 1e-3, (0.9, 0.999), 1e-8, wd)[0]
        ref.same(s[1]["p"], want, 4 * ref.U * torch.where(w0.isfinite(), w0.abs() + 1e-2, 0.0))


# ------------------------------------------------------------------ tensors that are more than their data

def _positions(dev, shape=(3,), vocab=9, seed=2):
    g = _generator(seed)
    x = torch.randn((*shape, vocab), generator=g).to(dev)
    y = torch.randint(0, vocab, shape, generator=g).to(dev)
    f = torch.zeros(shape, device=dev)
    return x, y, f


def _calls(x, y, f):
    """Every entry point by what it takes of a tensor: name -> (call of a tensor put in that place, the place's tensor)."""
    state = [t.clone() for t in (f, f, f, f, f)]

    def adamw(k, t):
        crukx_sync.adamw_step(*({"p": t if i == k else s} for i, s in enumerate(state)), step=1, lr=1e-3)

    return {
        "scores": (lambda t: crukx_sync.token_logprobs(t, y), x),
        "entropies": (lambda t: crukx_sync.token_logprobs(t, y, entropy=True), x),
        "loss": (lambda t: crukx_sync.policy_loss(t, y, f, f), x),
        "loss and gradient": (lambda t: crukx_sync.policy_loss_grad(t, y, f, f), x),
        "old": (lambda t: crukx_sync.policy_loss(x, y, t, f), f),
        "advantages": (lambda t: crukx_sync.policy_loss(x, y, f, t), f),
        "ref": (lambda t: crukx_sync.policy_loss_grad(x, y, f, f, None, t), f),
        "norm": (lambda t: crukx_sync.grad_norm([f, t]), f),
        "norm of a mapping": (lambda t: crukx_sync.grad_norm({"a": t}), f),
        "clip": (lambda t: crukx_sync.clip_grad_norm([t, f], 1.0), f),
        "adamw weights": (lambda t: adamw(0, t), f), "adamw masters": (lambda t: adamw(1, t), f),
        "adamw exp_avg": (lambda t: adamw(2, t), f), "adamw exp_avg_sq": (lambda t: adamw(3, t), f),
        "adamw grads": (lambda t: adamw(4, t), f),
    }


@edge
def forward_mode_derivatives_are_refused(dev):
    """No operator has a forward-mode derivative: a dual tensor in any place raises, with and without requires_grad, and
    does not come back as a result without a tangent."""
    import torch.autograd.forward_ad as fwd
    x, y, f = _positions(dev)
    for name, (call, at) in _calls(x, y, f).items():
        call(at.clone())
        with fwd.dual_level():
            for leaf in (False, True):
                dual = fwd.make_dual(at.clone().requires_grad_(leaf and not name.startswith(("clip", "adamw"))), torch.ones_like(at))
                with pytest.raises((ValueError, RuntimeError), match="forward-mode|jvp"):
                    call(dual)
            call(at.clone())  # a level by itself changes nothing
    leaf = x.clone().requires_grad_()
    with fwd.dual_level():
        up = fwd.make_dual(f + 1, torch.ones_like(f))
        for r, u in ((crukx_sync.token_logprobs(leaf, y), up), (crukx_sync.policy_loss(leaf, y, f, f).loss, up[0])):
            with pytest.raises((ValueError, RuntimeError), match="forward-mode"):
                torch.autograd.grad(r, leaf, u)


@edge
def traced_calls_are_refused(dev):
    """A trace would hold the allocation of the results and not the kernels that write them."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    x, y, f = _positions(dev)
    for call, at in _calls(x, y, f).values():
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(call, (at.clone(),), check_trace=False)
        for mode in ("real", "fake"):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                make_fx(call, tracing_mode=mode)(at.clone())
        with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(RuntimeError, match="cannot be traced"):
            call(at.clone())
        call(at.clone())
    leaf = x.clone().requires_grad_()
    for r in (crukx_sync.token_logprobs(leaf, y).sum(), crukx_sync.policy_loss(leaf, y, f, f).loss):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(lambda u: torch.autograd.grad(r, leaf, u, retain_graph=True)[0])(torch.ones_like(r))
        assert torch.autograd.grad(r, leaf)[0].isfinite().all()
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(lambda t: t + crukx_sync.grad_norm([]))(f)


@edge
def observed_calls_answer(dev):
    """A dispatch mode that only looks on (a profiler's) changes nothing, and a compiled function calls the kernels between
    its graphs."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class LooksOn(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    x, y, f = _positions(dev)
    want = crukx_sync.token_logprobs(x, y)
    leaf = x.clone().requires_grad_()
    with LooksOn():
        assert torch.equal(crukx_sync.token_logprobs(x, y), want)
        grad, = torch.autograd.grad(crukx_sync.policy_loss(leaf, y, f, f + 1).loss, leaf)
    assert torch.equal(grad, crukx_sync.policy_loss_grad(x, y, f, f + 1)[1])
    compiled = torch.compile(lambda t: crukx_sync.token_logprobs(t * 2.0, y) + 1.0, backend="eager")
    for t in (x, -x):
        assert torch.equal(compiled(t), crukx_sync.token_logprobs(t * 2.0, y) + 1.0)


@edge
def lazily_negated_tensors_are_negated(dev):
    """torch keeps some negations as a flag (the imaginary part of a conjugate), which the data do not show."""
    x, y, f = _positions(dev, (2, 5))
    g = _generator(3)
    old, adv, rf = (torch.randn((2, 5), generator=g).to(dev) for _ in range(3))
    neg = torch._neg_view
    assert neg(x).is_neg() and torch.equal(neg(x), -x)
    lp, h = crukx_sync.token_logprobs(neg(x), neg(-y), entropy=True)
    assert all(torch.equal(a, b) for a, b in zip((lp, h), crukx_sync.token_logprobs(-x, y, entropy=True)))
    opts = {"kl_coef": 0.1, "reduction": "sequence"}
    want, want_grad = crukx_sync.policy_loss_grad(-x, y, old, adv, None, rf, **opts)
    got, grad = crukx_sync.policy_loss_grad(neg(x), y, neg(-old), neg(-adv), None, neg(-rf), **opts)
    assert torch.equal(got.loss, want.loss) and torch.equal(got.kl, want.kl) and torch.equal(grad, want_grad)
    leaf = x.clone().requires_grad_()
    loss = crukx_sync.policy_loss(neg(leaf), y, neg(-old), adv, None, rf, **opts).loss
    assert torch.equal(torch.autograd.grad(loss, leaf)[0], -want_grad)
    up = torch.randn((2, 5), generator=g).to(dev)  # upstream gradients
    a, b = (torch.autograd.grad(crukx_sync.token_logprobs(leaf, y), leaf, u)[0] for u in (neg(up), -up))
    assert torch.equal(a, b)
    one = torch.ones((), device=dev)
    a, b = (torch.autograd.grad(crukx_sync.policy_loss(leaf, y, old, adv).loss, leaf, u)[0] for u in (neg(-one * 3), one * 3))
    assert torch.equal(a, b)
    # lists: the norm does not see signs and clipping keeps them; a step would take them the wrong way round
    t = up.clone()
    assert torch.equal(crukx_sync.grad_norm([neg(t)]), crukx_sync.grad_norm([t]))
    view = neg(t)
    norm = crukx_sync.clip_grad_norm([view], 0.5)
    ref.same(view, -up.double() * ref.factor(float(norm), 0.5), 4 * ref.U * up.abs().double())
    s = [{"p": t.clone().abs()} for _ in range(5)]
    for k in range(5):
        with pytest.raises(ValueError, match="negat"):
            crukx_sync.adamw_step(*({"p": neg(d["p"])} if i == k else d for i, d in enumerate(s)), step=1, lr=1e-3)
        assert torch.equal(s[k]["p"], t.abs())
    n = crukx_sync.grad_norm([t])
    one, two = ([{"p": d["p"].clone()} for d in s] for _ in range(2))
    crukx_sync.adamw_step(*one, step=1, lr=1e-3, grad_norm=n, max_norm=0.1)
    crukx_sync.adamw_step(*two, step=1, lr=1e-3, grad_norm=neg(-n), max_norm=0.1)
    assert all(torch.equal(a["p"], b["p"]) for a, b in zip(one, two))


class _Wrapped(torch.Tensor):
    """A tensor without storage of its own, as distributed and fake tensors are."""

    @staticmethod
    def __new__(cls, held):
        t = torch.Tensor._make_wrapper_subclass(cls, held.shape, dtype=held.dtype, device=held.device, strides=held.stride())
        t.held = held
        return t

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        return func(*(a.held if isinstance(a, cls) else a for a in args), **(kwargs or {}))


@edge
def tensors_without_storage_are_refused(dev):
    """A mask or reference policy without data to read is refused, not left out."""
    x, y, f = _positions(dev)
    mask = torch.tensor([True, False, True], device=dev)
    wrap = [_Wrapped, lambda t: torch._efficientzerotensor(t.shape, dtype=t.dtype, device=t.device)]
    for w in wrap:
        for call in (lambda t: crukx_sync.token_logprobs(x, y, t), lambda t: crukx_sync.policy_loss(x, y, f, f, t)):
            call(mask)
            with pytest.raises(ValueError, match="storage"):
                call(w(mask))
        with pytest.raises(ValueError, match="storage"):
            crukx_sync.token_logprobs(x, w(y))
        for name, (call, at) in _calls(x, y, f).items():
            with pytest.raises(ValueError, match="storage"):
                call(w(at))
        with pytest.raises(ValueError, match="storage"):
            crukx_sync.adamw_step(*({"p": f.clone()} for _ in range(5)), step=1, lr=1e-3, grad_norm=w(f[0]), max_norm=1.0)
    # an upstream gradient of nothing is zeros
    leaf = x.clone().requires_grad_()
    zero = wrap[1]
    for r, up in ((crukx_sync.token_logprobs(leaf, y), zero(f)), (crukx_sync.policy_loss(leaf, y, f, f + 1).loss, zero(f[0]))):
        assert not torch.autograd.grad(r, leaf, up)[0].any()
    empty = x[:0].clone().requires_grad_()  # no elements: nothing to read either
    crukx_sync.policy_loss(empty, y[:0], f[:0], f[:0], mask[:0], f[:0]).loss.backward()
    assert crukx_sync.token_logprobs(empty, y[:0], mask[:0]).shape == (0,) and empty.grad.shape == (0, 9)


# ------------------------------------------------------------------ values

@edge
def kl_terms_of_every_size(dev):
    """exp(d) - 1 - d, position by position.  One id in the vocabulary: its log probability is exactly 0, so d is the
    reference's value itself, and with an advantage of 0 the loss is the KL term alone.

    The term is a product of d^2 and a sum whose parts add up to at least a third of their absolute sum (|d| < 1), or a
    difference that leaves at least a third of what is subtracted (beyond), each from operations of one or two roundings:
    16 u bound it."""
    x, y = torch.zeros((1, 1), device=dev), torch.zeros(1, dtype=torch.int64, device=dev)
    zero = torch.zeros(1, device=dev)
    sizes = [1e-30, 1e-12, 1e-6, 1e-3, 0.03, 0.0624, 0.0626, 0.07, 0.09, 0.12, 0.2, 0.249, 0.251, 0.4, 0.49, 0.51, 0.7, 0.99, 1.01, 1.5, 3.0, 20.0, 80.0]
    for d in [s * a for a in sizes for s in (1, -1)] + [0.0]:
        at = torch.tensor([d], device=dev)
        out, _ = crukx_sync.policy_loss_grad(x, y, zero, zero, None, at, kl_coef=1.0, reduction="sum")
        v = at.cpu().double()
        want = (v * v / 2 * (1 + v / 3) if abs(d) < 1e-3 else torch.special.expm1(v) - v).sum()
        tol = 16 * ref.U * float(want) + 2.0 ** -149
        assert abs(float(out.kl) - float(want)) <= tol and abs(float(out.loss) - float(want)) <= tol, (d, float(out.kl), float(want))


@edge
def entropy_gradients_of_any_size_pass_impossible_ids_by(dev):
    """An id without probability has no gradient, however large the upstream one (a loss scale): 0, not NaN."""
    g = _generator(5)
    for dtype, rows, vocab in ((torch.float32, 2, 515), (torch.bfloat16, 300, 515)):
        x = (torch.randn((rows, vocab), generator=g) * 2).to(dtype).to(dev)
        x[:, 400:] = -float("inf")
        x[0, 17] = torch.finfo(dtype).min
        y = torch.randint(0, 400, (rows,), generator=g).to(dev)
        for up in (1.0, 1e12, 1e30):
            leaf = x.clone().requires_grad_()
            lp, h = crukx_sync.token_logprobs(leaf, y, entropy=True)
            u = torch.full((rows,), up, device=dev)
            for outs, ups, a in (([h], [u], None), ([lp, h], [u, u], u)):
                got, = torch.autograd.grad(outs, leaf, ups, retain_graph=True)
                assert not got[:, 400:].any() and not got[0, 17].any()
                want = ref.scores_grad(x, y, a, u)
                ref.check_grad(got, want, u.double() * (2 + 2 * 8), vocab)


@edge
def temperatures_up_to_the_largest(dev):
    """The distribution becomes uniform over the ids that have a probability, and stays one."""
    x, y, f = _positions(dev, (4,), 20)
    x[:, 13:] = -float("inf")
    y %= 13
    for t in (1e6, 1e30, 1e38, 1e44, 1e46, 1e300, 1.7e308):
        lp, h = crukx_sync.token_logprobs(x, y, temperature=t, entropy=True)
        ref.check_scores(x, y, None, t, lp, h)
        out, grad = crukx_sync.policy_loss_grad(x, y, f - 2, f + 1, temperature=t)
        ref.check_policy(x, y, f - 2, f + 1, None, None, {"temperature": t}, out, grad if t <= 1e38 else None)
        if t > 1e38:  # smaller than any 32-bit number says to a place
            assert grad.isfinite().all() and float(grad.abs().max()) <= 1e-43


# ------------------------------------------------------------------ gradients, element by element

def _shapes(dev):
    """Rows cut into parts, rows of a wavefront, of 256 threads, of 1024 that share a CU and of 1024 that have one."""
    if dev == "cpu":
        return [((3, 4, 9), 1.0), ((3, 4, 130), 1.0), ((2, 2, 4099), 1.0), ((260, 515), 0.7), ((257, 8200), 0.03), ((256, 40007), 0.01)]
    return [((3, 4, v), 0.8) for v in (1, 2, 7, 8, 9, 63, 257, 1000, 4096, 4097, 20011, 65537, 151936)] + \
        [((300, 515), 0.8), ((20, 15, 4099), 0.8), ((270, 8200), 0.8), ((260, 40007), 0.5), ((260, 115_003), 0.4), ((2, 130, 152_064), 0.3)]


def _row_cases(dev, dtype, seed):
    for shape, share in _shapes(dev):
        x, y = cases.logits(shape, dtype, seed + shape[-1], dev)
        old, rf, adv = cases.policies(x, y, seed, device=dev)
        mask = cases.mask_of(shape[:-1], seed, dev, share)
        mask.view(-1)[0] = True
        yield x, y, old, rf, adv, mask
        if shape[-1] in (130, 257, 8200, 115_003):  # the same at other alignments than the gradient's
            wide = torch.full((*shape[:-1], shape[-1] + 6), float("nan"), dtype=x.dtype, device=dev)
            wide[..., 5:shape[-1] + 5] = x
            yield wide[..., 5:shape[-1] + 5], y, old, rf, adv, mask


def _loss_scale(dtype):
    return 1024.0 if dtype == "fp16" else 1.0  # without one fp16 holds little of a small gradient


def _policy_rows(dev, dtype):
    for k, (x, y, old, rf, adv, mask) in enumerate(_row_cases(dev, dtype, 3)):
        opts = {"clip": (0.2, 0.28), "kl_coef": 0.05, "reduction": ("sequence", "token", "sum")[k % 3], "scale": _loss_scale(dtype)}
        _, grad = crukx_sync.policy_loss_grad(x, y, old, adv, mask, rf, **opts)
        rows.check_policy_gradient(grad, x, y, old, adv, mask, rf, **opts)


def _score_rows(dev, dtype):
    g = _generator(4)
    for k, (x, y, _, _, _, mask) in enumerate(_row_cases(dev, dtype, 5)):
        if dev == "cpu" and x.shape[-1] > 8200:  # (one kernel for rows of any length)
            continue
        up, uh = ((torch.randn(y.shape, generator=g) * _loss_scale(dtype)).to(dev) for _ in range(2))
        leaf = x.detach().requires_grad_()
        if k % 2:
            lp, h = crukx_sync.token_logprobs(leaf, y, mask, temperature=0.8, entropy=True)
            got, = torch.autograd.grad([lp, h], leaf, [up, uh])
        else:
            uh = None
            got, = torch.autograd.grad(crukx_sync.token_logprobs(leaf, y, mask, temperature=0.8), leaf, up)
        rows.check_score_gradient(got, x, y, up, uh, mask, 0.8)


for _dtype in sorted(cases.TYPES):
    EDGES[f"policy_gradients_row_by_row_{_dtype}"] = lambda dev, t=_dtype: _policy_rows(dev, t)
    EDGES[f"score_gradients_row_by_row_{_dtype}"] = lambda dev, t=_dtype: _score_rows(dev, t)


@edge
def upstream_factors_over_many_parts(dev):
    """A loss divided by a number of accumulations: the first backward pass writes the gradient anew, its workgroups each for
    several parts of rows (more parts than workgroups are launched), and equals the loss made with that scale."""
    rows_, vocab, share = (700, 40_007, 0.9) if dev != "cpu" else (2100, 40, 0.9)  # 700 x 5 parts, 2100 x 1; 2048 workgroups
    x, y = cases.logits((rows_, vocab), "bf16", 9, dev)
    old, rf, adv = cases.policies(x, y, 9, device=dev)
    mask = cases.mask_of((rows_,), 9, dev, share)
    opts = {"clip": (0.2, 0.28), "kl_coef": 0.05}
    for factor in (0.5, -3.0):
        leaf = x.detach().requires_grad_()
        loss = crukx_sync.policy_loss(leaf, y, old, adv, mask, rf, **opts).loss * factor
        got, = torch.autograd.grad(loss, leaf)
        rows.check_policy_gradient(got, x, y, old, adv, mask, rf, scale=factor, **opts)


@edge
def gradients_with_a_graph_have_the_same_values(dev):
    """create_graph hands out the same gradient, once from the loss's forward call and anew after that."""
    x, y, f = _positions(dev, (2, 5), 33)
    leaf = x.clone().requires_grad_()
    want = crukx_sync.policy_loss_grad(x, y, f - 2, f + 1)[1]
    loss = crukx_sync.policy_loss(leaf, y, f - 2, f + 1).loss
    for _ in range(2):
        got, = torch.autograd.grad(loss, leaf, create_graph=True)
        assert got.requires_grad and torch.equal(got.detach(), want) and bool(want.any())
    scores = crukx_sync.token_logprobs(leaf, y).sum()
    plain, = torch.autograd.grad(scores, leaf, retain_graph=True)
    got, = torch.autograd.grad(scores, leaf, create_graph=True)
    assert got.requires_grad and torch.equal(got.detach(), plain) and bool(plain.any())


PAIRS = [(w, g) for w in sorted(cases.TYPES) for g in sorted(cases.TYPES)]


def _check_step(before, after, k, c, step=5, lr=1e-3, wd=0.1):
    w0, m0, v0, g0 = (d[k] for d in before[1:])
    a, b, d = ref.adamw(w0, m0, v0, g0, step, lr, (0.9, 0.999), 1e-8, wd, c)
    g = g0.double().abs() * c
    ref.same(after[2][k], b, 8 * ref.U * (m0.abs().double() + g), "exp_avg")
    ref.same(after[3][k], d, 8 * ref.U * (v0.double() + g * g), "exp_avg_sq")
    size = lr / (1 - 0.9 ** step) / ((d / (1 - 0.999 ** step)).sqrt() + 1e-8) * (m0.abs().double() + g)
    ref.same(after[1][k], a, 4 * ref.U * w0.abs().double() + 32 * ref.U * size, "masters")
    assert torch.equal(after[0][k], after[1][k].to(after[0][k].dtype)), "weights"
    assert torch.equal(after[4][k], before[4][k]), "gradients"


@edge
def adamw_of_every_pair_of_types_and_of_all_in_one_call(dev):
    """Nine pairs of weight and gradient types alone; and one call with all of them, in an order that changes the pair from
    tensor to tensor, over flat buffers where the neighbours of a tensor have another pair (and some the same)."""
    sizes = [5, 1024, 1, 2049, 7, 300, 0, 4099, 64]
    g = _generator(8)

    def flat(types, scale, positive=False):
        """Tensors of `sizes`, type by type, those of one type one behind another in one buffer."""
        bufs = {t: (torch.randn(sum(sizes), generator=g) * scale).abs_() if positive else torch.randn(sum(sizes), generator=g) * scale
                for t in cases.TYPES}
        bufs = {t: b.to(cases.TYPES[t]).to(dev) for t, b in bufs.items()}
        out, at = {}, dict.fromkeys(bufs, 0)
        for k, (n, t) in enumerate(zip(sizes, types)):
            out[f"p{k}"] = bufs[t][at[t]:at[t] + n]
            at[t] += n
        return out

    lists = [([w] * 9, [q] * 9) for w, q in PAIRS]
    lists.append(([w for w, _ in PAIRS], [q for _, q in PAIRS]))
    lists.append((["bf16", "bf16", "fp32", "bf16", "bf16", "fp16", "bf16", "bf16", "fp32"],
                  ["bf16", "bf16", "bf16", "fp32", "bf16", "bf16", "bf16", "bf16", "fp16"]))
    for wtypes, gtypes in lists:
        floats = ["fp32"] * 9
        s = [flat(wtypes, 1.0), flat(floats, 1e-2), flat(floats, 1e-2), flat(floats, 1e-4, True), flat(gtypes, 1.0)]
        before = [{k: t.clone() for k, t in d.items()} for d in s]
        norm = crukx_sync.grad_norm(s[4])
        ref.same(norm, ref.norm(list(s[4].values())), 2 * ref.U * float(norm), "norm")
        crukx_sync.adamw_step(*s, step=5, lr=1e-3, weight_decay=0.1, grad_norm=norm, max_norm=1.0)
        for k in s[0]:
            _check_step(before, s, k, ref.factor(float(norm), 1.0))


@edge
def too_many_positions_are_refused_before_anything_is_allocated(dev):
    """2^48 positions, as views without memory of their own; the results would take a petabyte."""
    x, y, f = (t[:1].expand(1 << 24, 1 << 24, *t.shape[1:]) for t in _positions(dev))
    for call in (lambda: crukx_sync.token_logprobs(x, y, entropy=True), lambda: crukx_sync.policy_loss(x, y, f, f),
                 lambda: crukx_sync.policy_loss_grad(x, y, f, f), lambda: crukx_sync.token_logprobs(x.detach().requires_grad_(), y)):
        with pytest.raises(ValueError, match="2\\^31"):
            call()

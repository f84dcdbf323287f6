"""The losses over rows of class scores (opencl_tf.losses) where an ordinary call does not reach: log-probabilities
far from the reference network's or the old ones, excluded tokens, edits of results and inputs before the backward
pass, derivatives of derivatives, forward-mode tangents, targets of another form than a captured step's, and the
policy loss from the scores of many rows against its definition.

u = 2^-24 is half a step of fp32; sums over tokens are in 64 bits, so what is left of a mean is its terms' errors
and the store's half step."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def cuda(*values, **kw):
    return torch.tensor(values, device="cuda", **kw)


def policy_definition(lp, old, adv, ref=None, low=0.2, high=0.2, kl_coef=0.0):
    """loss, mean KL, clipped share and the slopes d loss / d lp of the unweighted policy loss, in 64 bits."""
    lp, old, adv = lp.double(), old.double(), adv.double()
    n = lp.numel()
    r = torch.exp(lp - old)
    cut = ((adv > 0) & (r > 1 + high)) | ((adv < 0) & (r < 1 - low))
    value = -torch.where(cut, r.clamp(1 - low, 1 + high), r) * adv
    slope = torch.where(cut, torch.zeros_like(r), -r * adv)
    kl = torch.zeros_like(r)
    if ref is not None:
        d = ref.double() - lp
        kl = torch.expm1(d) - d
        if kl_coef != 0.0:
            value, slope = value + kl_coef * kl, slope - kl_coef * torch.expm1(d)
    return value.sum() / n, kl.sum() / n, cut.double().sum() / n, slope / n


def near(got, want, rel, absolute=0.0):
    got, want = got.detach().double().cpu(), want.double().cpu()
    off = torch.where(got == want, torch.zeros_like(want), (got - want).abs())
    assert bool((off <= rel * want.abs() + absolute).all()), (got, want, float((off / want.abs()).max()))


def uniform_scores(rows, classes):
    """Equal scores: each exponential and the sums of them are exact however a row is shared, so the
    log-probability of every call is the same fp32 number."""
    return torch.zeros(rows, classes, device="cuda"), torch.arange(rows, device="cuda") % classes


class _Head(torch.nn.Module):
    def __init__(self):
        super().__init__()
        from opencl_tf.layers import OpenCLDense
        self.out = OpenCLDense(33)
        self.out.build((1, 12))

    def forward(self, x, training=None):
        return self.out(x)


def test_targets_of_another_form_than_the_captured(otf):
    """A captured step refuses targets that are not what it was captured with, before it copies any: the steps around
    the refused calls are the eager ones, bit for bit."""
    from opencl_tf import errors
    from opencl_tf.train import TrainStep

    def batch(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        top = torch.randn(16, 33, generator=g, device="cuda").topk(4, 1)
        return torch.randn(16, 12, generator=g, device="cuda"), (top.indices, top.values)

    def loss(output, y):
        return otf.losses.distillation_loss(output, *y, temperature=2.0)

    def run(graphed):
        torch.manual_seed(3)
        model = _Head().cuda()
        step = TrainStep(model, graphed=graphed, warmup=0, loss=loss)
        losses = [step(*batch(0)).clone()]
        if graphed:
            x, (ids, y) = batch(7)
            for bad in ((ids,), ids, y, (y, ids), (ids, y[:1]), (ids[:8], y[:8]), (ids, y, y), (ids, y.half()), [ids, y],
                        (ids, None), None):
                with pytest.raises(errors.InvalidArgumentError, match="captured"):
                    step(x, bad)
            for bad in (x[:1], x[:, :1], x[0], x.unsqueeze(0), x.long()[:8]):
                with pytest.raises(errors.InvalidArgumentError, match="captured"):
                    step(bad, (ids, y))
        losses += [step(*batch(s)).clone() for s in (1, 2)]
        return losses, [p.detach().clone() for p in model.parameters()]

    b, a = run(False), run(True)
    for x, y in zip((*a[0], *a[1]), (*b[0], *b[1])):
        assert torch.equal(x, y)


def _policy_forms(otf, x, t, old, adv, ref, **kw):
    """(loss, mean KL, share, gradient of the log-probabilities) of the loss from log-probabilities, then (loss, mean KL,
    share, gradient of the scores) of the one from the scores."""
    leaf = otf.losses.token_log_probs(x, t).requires_grad_()
    out = otf.losses.policy_loss(leaf, old, adv, ref_log_probs=ref, **kw)
    grad, = torch.autograd.grad(out[0], leaf)
    return leaf.detach(), (*[o.detach() for o in out], grad), otf.losses.policy_loss_with_grad(x, t, old, adv,
                                                                                               ref_log_probs=ref, **kw)


@pytest.mark.parametrize("classes", [16, 32768])
def test_kl_of_tokens_far_from_the_reference(otf, classes):
    """exp(d) past fp32's range: where kl_coef is 0, loss and gradient are those of no KL term, and the mean KL, which
    fp32 holds, is right; where it is not, the term is its 64-bit value."""
    n = 128
    x, t = uniform_scores(n, classes)
    lp = otf.losses.token_log_probs(x, t)
    old, adv = lp + 0.1, torch.linspace(-1, 1, n, device="cuda")
    ref = lp.clone()
    ref[5] += 90.0  # exp(90) is 1.2e39, the mean of 128 such terms and zeros 9.5e36
    for kl_coef in (0.0, 1e-30):
        lp, parts, fused = _policy_forms(otf, x, t, old, adv, ref, kl_coef=kl_coef)
        want = policy_definition(lp, old, adv, ref, kl_coef=kl_coef)
        # terms in 64 bits (their series to 1e-8), the store's half step; the gradient: slope, 1 / sum and product.
        # The advantages add up to 0, so without a KL term the loss is 0 but for its terms' roundings, each 8 * 2^-53
        # of less than 1 in both sides
        for got in (parts, fused):
            for g, w in zip(got[:3], want):
                near(g, w, 2 * U, 8 * 2.0 ** -53)
        near(parts[3], want[3], 4 * U)
        assert bool(fused[3].isfinite().all())
        # of the scores: factor * (p - q) with p = 1 / classes exact but for its quotient
        p = torch.full((n, classes), 1.0 / classes, device="cuda", dtype=torch.float64)
        p.scatter_add_(1, t[:, None], torch.full((n, 1), -1.0, device="cuda", dtype=torch.float64))
        near(fused[3], -want[3][:, None] * p, 8 * U)


@pytest.mark.parametrize("classes", [40, 20001])
def test_kl_of_an_excluded_token(otf, classes):
    """A token that the scores exclude (log-probability -inf) has an infinite KL, which is only reported where kl_coef
    is 0; one that the reference excludes has a finite slope."""
    x = torch.randn(6, classes, device="cuda")
    t = torch.arange(6, device="cuda")
    x[1, 1] = -math.inf
    old, adv, ref = torch.full((6,), -3.0, device="cuda"), torch.ones(6, device="cuda"), torch.full((6,), -3.0, device="cuda")
    lp, with_ref, fused = _policy_forms(otf, x, t, old, adv, ref)
    _, without, fused_without = _policy_forms(otf, x, t, old, adv, None)
    assert float(lp[1]) == -math.inf and float(with_ref[1]) == math.inf and float(fused[1]) == math.inf
    for a, b in ((with_ref, without), (fused, fused_without)):
        for i in (0, 2, 3):
            assert torch.equal(a[i], b[i]) and bool(a[i].isfinite().all())
    x = torch.randn(6, classes, device="cuda")
    ref[2] = -math.inf
    lp, parts, fused = _policy_forms(otf, x, t, old, adv, ref, kl_coef=0.5)
    assert float(parts[0]) == math.inf and float(fused[0]) == math.inf
    near(parts[3], policy_definition(lp, old, adv, ref, kl_coef=0.5)[3], 4 * U)
    assert bool(fused[3].isfinite().all())


def test_kl_slopes_are_exact_to_their_store(otf):
    """Slopes kl_coef (1 - exp(d)) for d from 1e-6 to 20 either way: the slope's, 1 / sum's and the product's half
    step, and the last one; the mean of the terms: its store alone."""
    d = torch.logspace(-6, math.log10(20.0), 4001, dtype=torch.float64)
    d = torch.cat([d, -d]).cuda()
    lp = -torch.rand(d.numel(), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) * 5
    ref, zero = (lp.double() + d).float(), torch.zeros_like(lp)
    leaf = lp.clone().requires_grad_()
    loss, kl, _ = otf.losses.policy_loss(leaf, lp, zero, ref_log_probs=ref, kl_coef=0.25)
    grad, = torch.autograd.grad(loss, leaf)
    want = policy_definition(lp, lp, zero, ref, kl_coef=0.25)
    near(kl, want[1], U + 2e-8)
    near(loss, want[0], U + 2e-8)
    near(grad, want[3], 4 * U + 2e-8)


@pytest.mark.parametrize("rows,classes", [(40001, 32), (300, 16384), (70, 131072)])
def test_policy_loss_with_grad_of_cancelling_terms(otf, rows, classes):
    """The mean of terms of both signs, clipped ones among them, that nearly cancel: from the scores it is as exact as
    from log-probabilities."""
    x, t = uniform_scores(rows, classes)
    lp = otf.losses.token_log_probs(x, t)
    g = torch.Generator(device="cuda").manual_seed(rows)
    old = lp + 0.3 * torch.randn(rows, generator=g, device="cuda")
    adv = torch.randn(rows, generator=g, device="cuda")
    old[-1], adv[-1] = lp[-1], 0.0
    total = policy_definition(lp, old, adv, high=0.28)[0] * rows
    adv[-1] = total  # its ratio is 1
    want = policy_definition(lp, old, adv, high=0.28)
    assert abs(float(want[0])) < 1e-5 and float(want[2]) > 0.1
    loss, _, share, grad = otf.losses.policy_loss_with_grad(x, t, old, adv, clip_low=0.2, clip_high=0.28)
    # the result's half step, and per term the few 2^-53 of its exponential
    near(loss, want[0], U, 8 * 2.0 ** -53 * float(adv.abs().sum()) / rows * 1.28)
    near(share, want[2], U)
    assert torch.equal(loss, otf.losses.policy_loss(lp, old, adv, clip_low=0.2, clip_high=0.28)[0])


@pytest.mark.parametrize("classes", [16, 32768])
def test_an_advantage_of_zero_has_no_gradient(otf, classes):
    """Whatever finite ratio the token has: exp(100) is past fp32's range, and 0 times it is 0."""
    x, t = uniform_scores(64, classes)
    old, adv = otf.losses.token_log_probs(x, t), torch.ones(64, device="cuda")
    adv[::4] = 0.0
    old[4] -= 100.0  # among those with advantage 0
    lp, parts, fused = _policy_forms(otf, x, t, old, adv, None)
    want = policy_definition(lp, old, adv)
    for got in (parts, fused):
        near(got[0], want[0], 2 * U)
    near(parts[3], want[3], 4 * U)
    assert not parts[3][::4].any() and not fused[3][::4].any() and bool(fused[3].isfinite().all())


def test_policy_metrics_may_be_edited_before_the_backward_pass(otf):
    lp = (-torch.rand(300, device="cuda")).requires_grad_()
    old, adv = lp.detach() + 0.1, torch.randn(300, device="cuda")

    def loss(edit):
        out, kl, share = otf.losses.policy_loss(lp, old, adv, ref_log_probs=old, kl_coef=0.1)
        if edit:
            kl /= 7
            share.zero_()
        return torch.autograd.grad(out, lp)[0]

    assert torch.equal(loss(True), loss(False))


def test_log_probabilities_are_not_needed_after_the_loss(otf):
    """The gradients of the token losses do not depend on them: they may be edited, and are not kept."""
    n = 1 << 20
    base = (-torch.rand(n, device="cuda")).requires_grad_()
    off = cuda(0, n // 2, n)
    adv = torch.randn(n, device="cuda")

    def policy(lp):
        return otf.losses.policy_loss(lp, adv, adv)[0]

    def preference(lp):
        return otf.losses.preference_loss(lp, off)[0]

    for f in (policy, preference):
        want, = torch.autograd.grad(f(base * 1), base)
        lp = base.clone()
        loss = f(lp)
        lp.detach().zero_()
        before = torch.cuda.memory_allocated()
        del lp
        assert torch.cuda.memory_allocated() <= before - 4 * n
        assert torch.equal(torch.autograd.grad(loss, base)[0], want)


def test_second_derivatives_are_refused(otf):
    """Every gradient of a loss says so where it is differentiated again by its scores or log-probabilities."""
    x = torch.randn(8, 40, device="cuda", requires_grad=True)
    t = torch.arange(8, device="cuda")
    off, adv = cuda(0, 4, 8), torch.randn(8, device="cuda")
    lp = (-torch.rand(8, device="cuda")).requires_grad_()
    for leaf, loss in ((x, lambda: otf.losses.token_log_probs(x, t).sum()),
                       (x, lambda: otf.losses.distillation_loss(x, t[:, None], adv[:, None])),
                       (lp, lambda: otf.losses.preference_loss(lp, off)[0]),
                       (lp, lambda: otf.losses.policy_loss(lp, adv, adv)[0])):
        g, = torch.autograd.grad(loss(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad((g * g).sum() + leaf.sum(), leaf)
        g, = torch.autograd.grad((2 * loss()).exp(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(g.sum() + leaf.sum(), leaf)


def test_second_derivatives_by_what_scales_a_loss_are_refused(otf):
    """A gradient depends on its upstream gradient too; a derivative by that must not come out without this part."""
    x = torch.randn(8, 40, device="cuda", requires_grad=True)
    t = torch.arange(8, device="cuda")
    off, adv = cuda(0, 4, 8), torch.randn(8, device="cuda")
    lp = (-torch.rand(8, device="cuda")).requires_grad_()
    for leaf, loss in ((x, lambda: otf.losses.token_log_probs(x, t)),
                       (x, lambda: otf.losses.distillation_loss(x, t[:, None], adv[:, None])),
                       (lp, lambda: otf.losses.preference_loss(lp, off)[0]),
                       (lp, lambda: otf.losses.policy_loss(lp, adv, adv)[0])):
        scale = cuda(2.0, requires_grad=True)
        g, = torch.autograd.grad((loss() * scale).sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(g.sum() + scale.sum(), scale)


def test_forward_mode_tangents_are_refused(otf):
    """The losses have no forward-mode derivative: a tangent is not dropped in silence."""
    import torch.autograd.forward_ad as fwd
    from opencl_tf import errors
    x, lp = torch.randn(4, 10, device="cuda"), -torch.rand(4, device="cuda")
    t, off = torch.arange(4, device="cuda"), cuda(0, 2, 4)
    calls = {"token_log_probs": (x, lambda a: otf.losses.token_log_probs(a, t)),
             "distillation_loss": (x, lambda a: otf.losses.distillation_loss(a, t[:, None], lp[:, None])),
             "distillation_loss_with_grad":
                 (x, lambda a: otf.losses.distillation_loss_with_grad(a, t[:, None], lp[:, None])),
             "preference_loss": (lp, lambda a: otf.losses.preference_loss(a, off)),
             "policy_loss": (lp, lambda a: otf.losses.policy_loss(a, lp, lp)),
             "policy_loss_with_grad": (x, lambda a: otf.losses.policy_loss_with_grad(a, t, lp, lp))}
    for name, (primal, call) in calls.items():
        for requires_grad in (False, True):
            with fwd.dual_level():
                primal = primal.detach().requires_grad_(requires_grad)
                dual = fwd.make_dual(primal, torch.ones_like(primal))
                with pytest.raises(errors.InvalidArgumentError, match="forward-mode"):
                    call(dual)
        call(primal.detach())


@pytest.mark.parametrize("pairs", [2, 40])  # one launch, and several
def test_a_rejected_answer_that_the_scores_exclude(otf, pairs):
    """Without smoothing an infinitely preferred answer costs nothing and moves nothing."""
    lp = torch.full((2 * pairs,), -1.0, device="cuda")
    lp[pairs] = -math.inf
    off = torch.arange(2 * pairs + 1, device="cuda")
    leaf = lp.clone().requires_grad_()
    loss, chosen, rejected = otf.losses.preference_loss(leaf, off, beta=1.0)
    near(loss, cuda((pairs - 1) * math.log(2.0) / pairs, dtype=torch.float64)[0], 2 * U)
    assert float(rejected[0]) == -math.inf
    grad, = torch.autograd.grad(loss, leaf)
    want = torch.full((2 * pairs,), 0.5 / pairs, device="cuda")
    want[:pairs] *= -1
    want[0] = want[pairs] = 0.0
    near(grad, want, 2 * U)
    # with smoothing the loss is infinite, and its gradient is not
    loss = otf.losses.preference_loss(leaf, off, beta=1.0, label_smoothing=0.1)[0]
    assert float(loss) == math.inf and bool(torch.autograd.grad(loss, leaf)[0].isfinite().all())
    # a chosen answer that the scores exclude: infinite, and its gradient finite
    loss = otf.losses.preference_loss(-leaf, off, beta=1.0)[0]
    assert float(loss) == math.inf and bool(torch.autograd.grad(loss, leaf)[0].isfinite().all())


def test_the_first_call_of_a_process_may_be_captured():
    """In a process of its own, whose first calls of the library are captured ones: they replay as they run."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import torch
from opencl_tf import losses
torch.manual_seed(0)
x = torch.randn(50, 6000, device="cuda")
t = torch.arange(50, device="cuda")
old, adv = torch.full((50,), -9.0, device="cuda"), torch.randn(50, device="cuda")
def step():
    return (losses.token_log_probs(x, t), *losses.policy_loss_with_grad(x, t, old, adv, mask=t > 3))
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, step()))
print("captured first")
"""
    package = Path(__file__).resolve().parent.parent / "opencl-tensorflow_b200"
    done = subprocess.run([sys.executable, "-c", code], cwd=package, capture_output=True, text=True, timeout=300)
    assert "captured first" in done.stdout, done.stderr[-2000:]


def test_the_losses_as_they_are_called_in_a_program(otf):
    """Log-probabilities of a view to a preference loss, a policy step in one call with ignored targets, a captured
    distillation step: what each returns."""
    from opencl_tf import losses
    from opencl_tf.train import TrainStep
    torch.manual_seed(5)
    scores = torch.randn(4, 9, 50, device="cuda", requires_grad=True)
    tokens = torch.randint(0, 50, (4, 9), device="cuda")
    answer = torch.rand(4, 8, device="cuda") > 0.2
    offsets, ref = cuda(0, 8, 16, 24, 32), -torch.rand(32, device="cuda")
    lp = losses.token_log_probs(scores[:, :-1], tokens[:, 1:])
    loss, chosen, rejected = losses.preference_loss(lp.flatten(), offsets, ref_log_probs=ref, mask=answer.flatten())
    loss.backward()
    assert chosen.shape == rejected.shape == (2,) and bool(scores.grad.isfinite().all()) and bool(scores.grad.any())
    scores.grad = None
    tokens[:, 0] = -100
    old, advantages = -torch.rand(4, 9, device="cuda"), torch.randn(4, 9, device="cuda")
    loss, kl, clipped, grad = losses.policy_loss_with_grad(scores, tokens, old, advantages, ref_log_probs=old,
                                                           mask=tokens >= 0, kl_coef=0.02)
    scores.backward(grad)
    assert loss.shape == kl.shape == clipped.shape == () and torch.equal(scores.grad, grad)
    assert not grad[:, 0].any() and bool(grad[:, 1:].any(-1).all())
    # without the mask the ignored targets count, with log-probability 0
    lp = losses.token_log_probs(scores.detach(), tokens)
    assert not lp[:, 0].any()
    for mask in (None, tokens >= 0):
        got = losses.policy_loss_with_grad(scores, tokens, old, advantages, ref_log_probs=old, mask=mask, kl_coef=0.02)
        keep = slice(0 if mask is None else 1, None)
        want = policy_definition(lp[:, keep].flatten(), old[:, keep].flatten(), advantages[:, keep].flatten(),
                                 old[:, keep].flatten(), kl_coef=0.02)
        # the log-probability of the fused pass may be two roundings off: 4 U of at most |lp| < 16, moving a term by
        # at most its ratio times its advantage and the KL's slope
        near(got[0], want[0], 2 * U, 64 * U * float(want[3].abs().sum() + want[2] * advantages.abs().max()))
        near(got[1], want[1], 2 * U, 64 * U * float(torch.expm1(old.double() - lp.double()).abs().max()))
        near(got[2], want[2], 2 * U)
    torch.manual_seed(0)
    model = _Head().cuda()
    step = TrainStep(model, lr=1e-3, loss=lambda out, t: losses.distillation_loss(out, t[0], t[1], temperature=2.0))
    top = torch.randn(16, 33, device="cuda").topk(4, 1)
    loss = step(torch.randn(16, 12, device="cuda"), (top.indices, top.values))
    assert math.isfinite(float(loss))


# 8 lanes a row, a warp, a CTA, a cluster
@pytest.mark.parametrize("rows,classes,dtype", [(30011, 37, "f32"), (29000, 1500, "bf16"), (15000, 5003, "f16"),
                                                (1200, 2100, "f32"), (700, 16000, "bf16"), (160, 60000, "f16"),
                                                (9, 200000, "f32")])
def test_policy_loss_with_grad_of_many_rows(otf, rows, classes, dtype):
    """Loss and gradient against the definition in 64 bits.  The log-probability l that the ratio is taken from is off by
    u (3 D + 4 + c) + 2 u |l| + u: D = sum p |x - m|, c additions and merges that follow one another in a row's sum
    (at most 32, then an eighth of a row's values in batches of 32, then 61 in merging)."""
    dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    eps = torch.finfo(dt).eps / 2
    tiny = {"f32": 2.0 ** -126, "f16": 2.0 ** -25, "bf16": 2.0 ** -126}[dtype]
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = (3 * torch.randn(rows, classes, generator=g, device="cuda")).to(dt)
    t = torch.randint(0, classes, (rows,), generator=g, device="cuda")
    t[::7] = -100  # counted, with log-probability 0 and no gradient
    z = torch.log_softmax(x.double(), 1)
    ignored = t < 0
    at = t.clamp(min=0)[:, None]
    lp = torch.where(ignored, torch.zeros_like(z[:, 0]), z.gather(1, at)[:, 0])
    ratio = torch.rand(rows, generator=g, device="cuda") * 0.15 + torch.where(
        torch.rand(rows, generator=g, device="cuda") < 0.5, 0.9, 1.5)  # away from the borders 0.8 and 1.28
    old = (lp - ratio.double().log()).float()
    ref = (lp + 0.3 * torch.randn(rows, generator=g, device="cuda")).float()
    adv = torch.randn(rows, generator=g, device="cuda")
    w = torch.rand(rows, generator=g, device="cuda") + 0.1
    w[rows // 2] = 0.0
    scale, coef = 4096.0, 0.05
    loss, kl, share, grad = otf.losses.policy_loss_with_grad(
        x, t, old, adv, ref_log_probs=ref, mask=w, clip_low=0.2, clip_high=0.28, kl_coef=coef, grad_loss=cuda(scale)[0])

    r = torch.exp(lp - old.double())
    a, wd = adv.double(), w.double()
    cut = ((a > 0) & (r > 1.28)) | ((a < 0) & (r < 0.8))
    d = ref.double() - lp
    k3 = torch.expm1(d) - d
    value = -torch.where(cut, r.clamp(0.8, 1.28), r) * a + coef * k3
    slope = torch.where(cut, torch.zeros_like(r), -r * a) - coef * torch.expm1(d)
    share_w = wd / wd.sum()
    p = z.exp()
    away = torch.where(p > 0, x.double().amax(1, keepdim=True) - x.double(), torch.zeros_like(p))
    rel_s = U * (3 * (p * away).sum(1) + 4 + 93 + classes / 256)
    lp_off = torch.where(ignored, torch.zeros_like(lp), rel_s + 2 * U * lp.abs() + U)
    # a token's value moves with its log-probability by its slope, which itself moves by at most r |a| + coef exp(d)
    bend = r * a.abs() + coef * torch.exp(d)
    near(loss, (share_w * value).sum(), U, float((share_w * (slope.abs() + bend * lp_off) * lp_off).sum()))
    near(kl, (share_w * k3).sum(), U + 2e-8, float((share_w * (torch.expm1(d).abs() + torch.exp(d) * lp_off) * lp_off).sum()))
    near(share, (share_w * cut).sum(), U)
    factor = torch.where(ignored, torch.zeros_like(slope), scale * share_w * slope)[:, None]
    hot = torch.zeros_like(p).scatter_(1, at, 1.0)
    want = factor * (hot - p)
    moved = (scale * share_w * bend * lp_off * ~ignored)[:, None] * (hot - p).abs()
    # p: 3 u |x - m| and 8 u of its own beside s; the difference, the factor's roundings, the store
    tol = factor.abs() * (p * (rel_s[:, None] + U * (3 * away + 8)) + 2 * U) + want.abs() * (6 * U + eps) + tiny
    off = (grad.double() - want).abs()
    assert bool((off <= tol + moved).all()), float((off - tol - moved).max())
    assert not grad[ignored].any() and not grad[rows // 2].any()


def test_a_loss_node_called_by_itself(otf):
    """The node of a loss, called outside of a backward pass, gives the gradient that a backward pass gives; recorded,
    it refuses to be differentiated again."""
    x = torch.randn(8, 40, device="cuda", requires_grad=True)
    t = torch.arange(8, device="cuda")
    off, adv = cuda(0, 4, 8), torch.randn(8, device="cuda")
    lp = (-torch.rand(8, device="cuda")).requires_grad_()
    for leaf, loss in ((x, lambda: otf.losses.token_log_probs(x, t)),
                       (x, lambda: otf.losses.distillation_loss(x, t[:, None], adv[:, None])),
                       (lp, lambda: otf.losses.preference_loss(lp, off)[0]),
                       (lp, lambda: otf.losses.policy_loss(lp, adv, adv)[0])):
        out = loss()
        up = torch.ones_like(out)
        want, = torch.autograd.grad(loss(), leaf, up)
        for recorded in (False, True):
            out = loss()
            with torch.set_grad_enabled(recorded):
                got = out.grad_fn(*(up, None)[:len(out.grad_fn._input_metadata)])  # a second result has no gradient
            got = got[0] if isinstance(got, tuple) else got
            assert torch.equal(got, want) and got.requires_grad == recorded
            if recorded:
                with pytest.raises(RuntimeError, match="once"):
                    torch.autograd.grad(got.sum() + leaf.sum(), leaf)

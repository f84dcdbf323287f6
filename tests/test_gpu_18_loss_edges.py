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
    value = -torch.where(cut, torch.where(adv > 0, 1 + high, 1 - low), r) * adv
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

"""The losses over rows of class scores without a GPU: the names a user has,
what the Python package refuses before any launch, and what the C entries
refuse before they look for a device."""
from __future__ import annotations

import ctypes

import pytest
import torch

import opencl_tf
from opencl_tf import _library as L
from opencl_tf import errors

NAMES = ["token_log_probs", "distillation_loss", "distillation_loss_with_grad", "preference_loss", "policy_loss",
         "policy_loss_with_grad"]


def test_names():
    for n in NAMES:
        assert callable(getattr(opencl_tf.losses, n)), n
        assert callable(getattr(opencl_tf.step_ops, "opencl_" + n)), n


def test_cpu_tensors_are_refused():
    x, t, lp, off = torch.zeros(2, 5), torch.zeros(2, dtype=torch.long), torch.zeros(2), torch.tensor([0, 1, 2])
    f = opencl_tf.losses
    for call in (lambda: f.token_log_probs(x, t), lambda: f.distillation_loss(x, t[:, None], x[:, :1]),
                 lambda: f.distillation_loss_with_grad(x, t[:, None], x[:, :1]),
                 lambda: f.preference_loss(lp, off), lambda: f.policy_loss(lp, lp, lp),
                 lambda: f.policy_loss_with_grad(x, t, lp, lp), lambda: f.token_log_probs([1.0], t)):
        with pytest.raises(errors.InvalidArgumentError, match="CUDA device"):
            call()


P = ctypes.c_void_p(64)  # never looked at: every call below is refused first


def scores(**over):
    v = dict(data=64, dtype=0, outer=1, inner=4, classes=10, outer_stride=0, inner_stride=10)
    return ctypes.byref(L.Logits(**{**v, **over}))


def refused(rc, *words):
    msg = L._lib.b2_last_error().decode()
    assert rc == 1, (rc, msg)
    for w in words:
        assert w in msg, msg


BAD_SCORES = [(dict(dtype=3), "bfloat16"), (dict(dtype=-1), "bfloat16"), (dict(classes=0), "classes"),
              (dict(classes=2 ** 30 + 1), "classes"), (dict(inner=-1), "negative"), (dict(outer=-1), "negative"),
              (dict(outer=2 ** 20, inner=2 ** 20), "too many rows"), (dict(data=None), "null")]


@pytest.mark.parametrize("over,word", BAD_SCORES)
def test_bad_scores(over, word):
    lib, x = L._lib, scores(**over)
    refused(lib.b2_token_log_probs(None, x, P, 8, P, None), word)
    refused(lib.b2_token_log_probs_grad(None, x, P, 8, P, P, P), word)
    refused(lib.b2_distillation_loss(None, x, P, 8, P, 0, 4, None, 0, 1.0, P, None, None, None), word)
    refused(lib.b2_distillation_loss_grad(None, x, P, 8, P, 0, 4, None, 0, 1.0, P, P, P), word)
    refused(lib.b2_policy_loss_with_grad(None, x, P, 8, P, P, None, None, 0, 0.2, 0.2, 0.0, None, P, P, P), word)


def test_bad_arguments():
    lib, x = L._lib, scores()
    assert lib.b2_token_log_probs(None, scores(inner=0, data=None), None, 8, None, None) == 0  # no rows: nothing to do
    assert lib.b2_token_log_probs_grad(None, scores(outer=0), None, 8, None, None, None) == 0
    refused(lib.b2_token_log_probs(None, None, P, 8, P, None), "null logits")
    refused(lib.b2_token_log_probs(None, x, P, 2, P, None), "targets", "32- or 64-bit")
    refused(lib.b2_token_log_probs(None, x, None, 8, P, None), "null")
    refused(lib.b2_token_log_probs(None, x, P, 8, None, None), "null")
    refused(lib.b2_token_log_probs_grad(None, x, P, 8, None, P, P), "null")

    def distill(ids=P, ids_bytes=8, y=P, y_dtype=0, top=4, w=None, w_bytes=0, t=1.0, loss=P, rows=4):
        return lib.b2_distillation_loss(None, scores(inner=rows), ids, ids_bytes, y, y_dtype, top, w, w_bytes, t, loss,
                                        None, None, None)
    refused(distill(rows=0), "no rows")
    refused(distill(ids=None), "null")
    refused(distill(y=None), "null")
    refused(distill(loss=None), "null")
    refused(distill(ids_bytes=1), "teacher_ids")
    refused(distill(y_dtype=9), "teacher_logits")
    refused(distill(w=P, w_bytes=2), "weights")
    for top in (0, -1, 1025):
        refused(distill(top=top), "[1, 1024]")
    for t in (0.0, -1.0, 1e-31, 1e31, float("inf"), float("nan")):
        refused(distill(t=t), "temperature")

    def preference(off=P, off_bytes=8, pairs=2, beta=0.1, eps=0.0, n=5, lp=P, loss=P, w=None, w_bytes=0):
        return lib.b2_preference_loss(None, lp, None, w, w_bytes, n, off, off_bytes, pairs, beta, eps, loss, P, P)
    refused(preference(pairs=0), "no pairs")
    refused(preference(pairs=2 ** 30), "pairs")
    refused(preference(n=-1), "negative")
    refused(preference(off=None), "null")
    refused(preference(lp=None), "null")
    refused(preference(off_bytes=3), "offsets")
    refused(preference(w=P, w_bytes=8), "weights")
    refused(preference(beta=float("nan")), "beta")
    for eps in (-0.1, 0.6, float("nan")):
        refused(preference(eps=eps), "label_smoothing")
    refused(lib.b2_preference_loss_grad(None, None, P, None, 0, 5, P, 8, 2, P), "null")

    def policy(n=5, low=0.2, high=0.2, kl=0.0, old=P, w=None, w_bytes=0):
        return lib.b2_policy_loss(None, P, old, P, None, w, w_bytes, n, low, high, kl, P, P, None)
    refused(policy(n=0), "no tokens")
    refused(policy(n=-3), "no tokens")
    refused(policy(old=None), "null")
    refused(policy(w=P, w_bytes=3), "weights")
    for bad in (-0.1, float("nan")):
        refused(policy(low=bad), "clip")
        refused(policy(high=bad), "clip")
    refused(policy(kl=float("inf")), "kl_coef")
    refused(lib.b2_policy_loss_grad(None, P, P, P, 0, P), "no tokens")
    refused(lib.b2_policy_loss_grad(None, P, None, P, 5, P), "null")


def test_folding_of_leading_axes():
    """The strides that the C entries get for a view, and when a copy is made."""
    base = torch.arange(3 * 6 * 20, dtype=torch.float32).view(3, 6, 20)

    def folded(t):
        v = L._class_scores.fold(t)
        if v is None:
            return False
        outer, inner, classes, so, si = v
        rows = [torch.as_strided(t, (classes,), (1,), t.storage_offset() + i * so + j * si) for i in range(outer)
                for j in range(inner)]
        assert torch.equal(torch.stack(rows), t.reshape(-1, t.shape[-1]))
        return True
    assert folded(base) and folded(base[:, :-1]) and folded(base[:, :, :13]) and folded(base[:, 1:, 2:])
    assert folded(base.transpose(0, 1)) and folded(base[1, 2]) and folded(base[0, 0].expand(4, -1))
    assert folded(base.view(18, 20)[::3]) and folded(base[:, :1]) and folded(base[::2, ::2, :1])
    assert not folded(base.transpose(1, 2)) and not folded(base[None].expand(2, -1, -1, -1)[:, :, ::5])

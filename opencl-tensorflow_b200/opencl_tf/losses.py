"""Losses over rows of class scores ("logits"): what a network that ends in
scores over many classes is trained with on chosen classes, on a teacher's
top answers, on pairs of answers, or on rewards.

Beside the mean squared error of the reference's recipe (``train.mse``); none of
these is an op of the reference.

Scores are float32, float16 or bfloat16 CUDA tensors [..., classes]; the
leading axes are rows.  A view whose classes are adjacent is read in place when
its leading axes fold into two strides (``scores[:, :-1]``), else copied.
Log-probabilities, weights and losses are float32 (a mask may be bool or
uint8).  Integers are int32 or int64.  What a weight of 0 belongs to is not looked
at: whatever it holds, it adds nothing and its gradient is 0.  Scores that are NaN or
+inf, or a row of -inf only, have no softmax, so a row that counts gives NaN.

Gradients go to the scores (or log-probabilities) only: the teacher, the
reference and old log-probabilities, advantages and weights are constants.  They are
differentiable once, and backward only.  All results are deterministic, and every call may be
captured in a CUDA graph (a backward pass as torch captures any: with no eager graph
of the same leaves alive).

A weighted mean divides by the sum of the call's weights.  Where ranks average their
gradients (``TrainStep``), that is the mean over the whole batch only if the ranks' sums
are equal; else multiply a rank's loss by its sum times the ranks over the sum of all.

The ``_with_grad`` forms return the gradient of the scores with the loss, from one
pass over the scores: ``scores.backward(grad)`` then continues the backward
pass.  ``grad_loss`` is the upstream gradient (a loss scale, say): a float32
scalar on the device, 1 by default.
"""
from __future__ import annotations

from ._library import step_ops


def token_log_probs(logits, targets):
    """log softmax(logits)[..., targets], float32 with the shape of ``targets``
    (the leading axes of ``logits``).  A target outside [0, classes) is ignored:
    0, and no gradient.  A row whose upstream gradient is 0 gets a zero gradient
    whatever its scores hold."""
    return step_ops.opencl_token_log_probs(logits, targets)


def distillation_loss(logits, teacher_ids, teacher_logits, weights=None, temperature=1.0):
    """temperature^2 KL(q || softmax(logits / temperature)), the weighted mean over
    the rows, where q is the softmax of the row's ``teacher_logits`` /
    temperature over the classes ``teacher_ids`` (both [..., entries], 1 to 1024
    entries) -- a teacher's top logits.

    Entries whose class lies outside [0, classes) or whose logit is -inf are left
    out; a row without entries has loss 0 and no gradient.  A class may be repeated:
    its entries' q add up in the gradient, and in the loss each has its own term
    q (log q - log P), together less than that of the summed q.  ``weights``: one per
    row.  0 when the weights sum to 0."""
    return step_ops.opencl_distillation_loss(logits, teacher_ids, teacher_logits, weights, temperature)


def distillation_loss_with_grad(logits, teacher_ids, teacher_logits, weights=None, temperature=1.0, grad_loss=None):
    """(``distillation_loss``, its gradient with respect to ``logits`` times
    ``grad_loss``) in one pass over the scores."""
    return step_ops.opencl_distillation_loss_with_grad(logits, teacher_ids, teacher_logits, weights, temperature,
                                                       grad_loss)


def preference_loss(log_probs, offsets, ref_log_probs=None, mask=None, beta=0.1, label_smoothing=0.0):
    """Preference loss of pairs of answers: with the reward of a sequence
    beta * sum(mask * (log_probs - ref_log_probs)) over its tokens and h the
    chosen answer's reward less the rejected one's,

        mean over pairs of -(1 - e) log sigma(h) - e log sigma(-h),  e = label_smoothing.

    ``offsets`` [2 * pairs + 1], non-decreasing: sequence i is the (flattened)
    tokens offsets[i] .. offsets[i + 1] - 1; the first ``pairs`` sequences are the
    chosen answers, the others the rejected ones in the same order.  Tokens outside
    the sequences do not count.  ``mask``: which tokens count, or their weights.

    Returns (loss, rewards of the chosen answers, rewards of the rejected ones);
    the rewards carry no gradient."""
    loss, rewards = step_ops.opencl_preference_loss(log_probs, offsets, ref_log_probs, mask, beta, label_smoothing)
    pairs = rewards.shape[0] // 2
    return loss, rewards[:pairs], rewards[pairs:]


def policy_loss(log_probs, old_log_probs, advantages, ref_log_probs=None, mask=None, clip_low=0.2, clip_high=None,
                kl_coef=0.0):
    """Clipped policy loss with a KL term, the weighted mean over the tokens of

        max(-r A, -clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(d) - d - 1)

    with A = advantages, r = exp(log_probs - old_log_probs) and d =
    ref_log_probs - log_probs (no KL term without ``ref_log_probs``).
    ``clip_high`` is ``clip_low`` by default; ``mask``: which tokens count, or their
    weights.  With ``kl_coef`` 0 the KL is only reported, and may be infinite.

    Returns (loss, mean of exp(d) - d - 1, share of the weight whose ratio is
    clipped); the last two carry no gradient.  All 0 when the weights sum to 0."""
    loss, stats = step_ops.opencl_policy_loss(log_probs, old_log_probs, advantages, ref_log_probs, mask, clip_low,
                                              clip_low if clip_high is None else clip_high, kl_coef)
    # The backward pass needs 1 / sum of the weights behind them: with a version counter of their own the two may be
    # edited before it.
    metrics = stats.data
    return loss, metrics[0], metrics[1]


def policy_loss_with_grad(logits, targets, old_log_probs, advantages, ref_log_probs=None, mask=None, clip_low=0.2,
                          clip_high=None, kl_coef=0.0, grad_loss=None):
    """(the results of ``policy_loss`` for ``token_log_probs(logits, targets)``, the
    loss's gradient with respect to ``logits`` times ``grad_loss``) in one pass over
    the scores: (loss, mean KL, clipped share, gradient).

    A target outside [0, classes) is a token of log-probability 0 without gradient:
    unless ``mask`` leaves it out, its ratio exp(-old_log_probs) counts in the means."""
    loss, stats, grad = step_ops.opencl_policy_loss_with_grad(
        logits, targets, old_log_probs, advantages, ref_log_probs, mask, clip_low,
        clip_low if clip_high is None else clip_high, kl_coef, grad_loss)
    return loss, stats[0], stats[1], grad

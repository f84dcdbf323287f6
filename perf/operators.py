"""The log-probability losses as they are used: cases, inputs, plain forms and values in 64 bits.

Four operators over scores of many classes: the log-probability of a chosen
class (``token_log_probs``), the distillation loss from a teacher's top logits,
the preference loss over pairs of sequences and the clipped policy loss with a
KL term.  ``run`` computes them with elementary torch operations, or through
``opencl_tf.losses`` where ``own`` is true.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = Path(__file__).resolve().parent.parent / "opencl-tensorflow_b200"
_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_IGNORED = -100

# Of every large case: 4096 rows of 128000 bf16 scores, read and written.
_MOST_VALUES = 4096 * 128000


def _losses():
    if str(_PACKAGE) not in sys.path:
        sys.path.insert(0, str(_PACKAGE))
    from opencl_tf import losses
    return losses


# ------------------------------------------------------------------- cases

def listed():
    return [
        # the score of one sampled token: one row, an odd vocabulary
        {"name": "score_one_token", "op": "logp", "rows": 1, "classes": 50257, "dtype": "f32", "dead": 0},
        # scoring prompts with a reference network: forward only
        {"name": "score_prompts", "op": "logp", "rows": 8192, "classes": 32000, "dtype": "bf16", "dead": 0},
        # log-likelihood training on an odd vocabulary: rows that start on no vector's border
        {"name": "likelihood_step_odd", "op": "logp_train", "rows": 1531, "classes": 50257, "dtype": "bf16", "dead": 0},
        # two pairs of short answers: latency
        {"name": "preference_two_pairs", "op": "pref", "pairs": 2, "mean_len": 24, "smoothing": 0.0},
        # many pairs of long answers, their log-probabilities in hand
        {"name": "preference_many_pairs", "op": "pref", "pairs": 256, "mean_len": 2048, "smoothing": 0.1},
        # a preference step from the scores to their gradient
        {"name": "preference_from_scores", "op": "pref_logits", "pairs": 4, "mean_len": 192, "smoothing": 0.0,
         "classes": 32000, "dtype": "f16", "dead": 0},
        # a policy update of one short answer
        {"name": "policy_64_tokens", "op": "policy", "rows": 64, "kl": 0.05},
        # a rollout batch of a million tokens, their log-probabilities in hand
        {"name": "policy_million_tokens", "op": "policy", "rows": 1000003, "kl": 0.02},
        # a policy step from the scores to their gradient in one call
        {"name": "policy_from_scores", "op": "policy_logits", "rows": 4099, "classes": 64000, "dtype": "bf16",
         "kl": 0.04, "dead": 0},
        # a small network's head: a batch of 256 samples with 128 classes
        {"name": "distill_dense_head", "op": "distill", "rows": 256, "classes": 128, "dtype": "f32", "top": 8,
         "temperature": 2.0, "dead": 0},
        # odd sizes everywhere, a padded vocabulary whose last columns are -inf
        {"name": "distill_step_odd", "op": "distill", "rows": 1021, "classes": 32003, "dtype": "f16", "top": 100,
         "temperature": 2.0, "dead": 3},
        # the largest: a distillation step over a wide vocabulary, loss and gradient in one call
        {"name": "distill_wide_step", "op": "distill_grad", "rows": 4096, "classes": 128000, "dtype": "bf16",
         "top": 64, "temperature": 1.0, "dead": 0},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["logp", "logp_train", "pref", "pref_logits", "policy", "policy_logits", "distill", "distill_grad"])
    if op == "pref":
        pairs = _log_int(rng, 1, 1024)
        return {"op": op, "pairs": pairs, "mean_len": _log_int(rng, 1, max(1, (1 << 20) // (2 * pairs))),
                "smoothing": rng.choice([0.0, 0.1])}
    if op == "policy":
        return {"op": op, "rows": _log_int(rng, 1, 1 << 20), "kl": rng.choice([0.0, 0.03])}
    dtype = rng.choice(["f32", "f16", "bf16"])
    most = _MOST_VALUES * 15 // 16 // (2 if dtype == "f32" else 1)
    classes = _log_int(rng, 8, 160000)
    case = {"op": op, "classes": classes, "dtype": dtype, "dead": rng.choice([0, 0, rng.randrange(1, 1 + classes // 8)])}
    if op == "pref_logits":
        pairs = _log_int(rng, 1, 16)
        longest = max(1, min(2048, most // 2 // classes // (2 * pairs)))
        return {**case, "pairs": pairs, "mean_len": _log_int(rng, 1, longest), "smoothing": rng.choice([0.0, 0.1])}
    case["rows"] = _log_int(rng, 1, max(1, min(1 << 17, most // classes)))
    if op == "policy_logits":
        case["kl"] = rng.choice([0.0, 0.03])
    if op in ("distill", "distill_grad"):
        live = classes - case["dead"]
        case |= {"top": _log_int(rng, 1, min(128, live)), "temperature": rng.choice([1.0, 1.5, 2.0])}
    return case


# ------------------------------------------------------------------ inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _scores(case, rows, g):
    """[rows, classes] scores as a network gives them, and one class a row that is mostly among the likely ones."""
    classes, dead = case["classes"], case["dead"]
    x = torch.randn(rows, classes, generator=g, device="cuda").mul_(2.0)
    targets = torch.randint(0, classes - dead, (rows,), generator=g, device="cuda")
    lift = torch.rand(rows, 1, generator=g, device="cuda").mul_(12.0)
    x.scatter_add_(1, targets[:, None], lift)
    if dead:
        x[:, classes - dead:] = -math.inf
    return x.to(_DTYPES[case["dtype"]]), targets


def _row_log_probs(x, targets):
    x = x.float()
    return (x.gather(1, targets[:, None])[:, 0] - torch.logsumexp(x, 1)).float()


def _sequences(case, g):
    """Offsets of the 2 * pairs sequences, of 1 to 2 * mean_len - 1 tokens each, and the number of tokens: a
    few lie behind the last sequence.  The lengths are the case's, their order the seed's."""
    pairs, mean = case["pairs"], case["mean_len"]
    lengths = torch.randint(1, 2 * mean, (2 * pairs,), generator=torch.Generator().manual_seed(11))
    order = torch.randperm(2 * pairs, generator=torch.Generator().manual_seed(int(g.initial_seed())))
    ends = lengths[order].cumsum(0)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), ends]).to(torch.int64)
    return offsets.cuda(), int(ends[-1]) + 3


def prepare(case, seed):
    g = _generator(seed)
    op, s = case["op"], {"case": dict(case)}

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if op in ("pref", "pref_logits"):
        s["offsets"], rows = _sequences(case, g)
        s["mask"] = rand(rows) > 0.2  # the prompt's tokens do not count
    else:
        rows = case["rows"]
    if "classes" in case:
        s["x"], targets = _scores(case, rows, g)
        s["targets"] = targets
        # fp16 gradients carry a loss scale, or most of them would be under the type's smallest values
        scale = 4096.0 * (1 << max(0, (rows // 1024).bit_length() - 1)) if case["dtype"] == "f16" else 1.0
        s["scale"] = torch.tensor(scale, device="cuda")
        if op in ("logp", "logp_train"):
            s["targets"] = torch.where(rand(rows) < 0.08, torch.full_like(targets, _IGNORED), targets)
            s["upstream"] = randn(rows)
        elif op in ("pref_logits", "policy_logits"):
            lp = _row_log_probs(s["x"], targets)
    else:
        lp = -torch.empty(rows, device="cuda").exponential_(0.7, generator=g)
        s["lp"] = lp
    if op in ("pref", "pref_logits"):
        # the chosen answers have become likelier than under the reference network, the rejected ones less likely
        mean = case["mean_len"]
        sign = torch.where(torch.arange(rows, device="cuda") < s["offsets"][case["pairs"]], 1.0, -1.0)
        s["ref"] = lp - min(0.25, 8.0 / mean) * sign + min(0.3, 4.0 / math.sqrt(mean)) * randn(rows)
    if op in ("policy", "policy_logits"):
        s["old"] = lp + 0.15 * randn(rows)
        s["ref"] = lp + 0.25 * randn(rows) if case["kl"] else None
        s["advantages"] = randn(-(-rows // 128)).repeat_interleave(128)[:rows].contiguous()
        s["mask"] = rand(rows) > 0.1
    if op in ("distill", "distill_grad"):
        noisy = s["x"].float().add_(0.7 * randn(rows, case["classes"]))
        top = noisy.topk(case["top"], dim=1)
        wide = case["dtype"] == "f32"
        s["teacher"] = top.values.to(_DTYPES[case["dtype"]])
        ids = top.indices if wide else top.indices.to(torch.int32)
        # some teachers gave fewer answers than the others
        keep = torch.arange(case["top"], device="cuda")[None] < torch.where(rand(rows) < 0.1, 1 + case["top"] // 2, case["top"])[:, None]
        s["ids"] = torch.where(keep, ids, torch.full_like(ids, -1))
        w = 0.5 + rand(rows)
        s["weights"] = torch.where(rand(rows) < 0.15, torch.zeros_like(w), w)
    return s


# --------------------------------------------------------------- plain form

def _softmax_parts(x):
    x = x.float()
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    return x, m, e, e.sum(1, keepdim=True)


def _plain_log_probs(x, targets, classes):
    """(log-probabilities, their gradient's parts) of the chosen classes."""
    valid = (targets >= 0) & (targets < classes)
    at = targets.clamp(0, classes - 1)[:, None]
    f, m, e, total = _softmax_parts(x)
    lp = f.gather(1, at) - m - torch.log(total)
    return torch.where(valid, lp[:, 0], torch.zeros_like(lp[:, 0])), (e, total, at, valid)


def _plain_log_probs_grad(upstream, parts, dtype):
    e, total, at, valid = parts
    g = torch.where(valid, upstream.float(), torch.zeros_like(upstream, dtype=torch.float32))[:, None]
    return (e * (-g / total)).scatter_add_(1, at, g).to(dtype)


def _plain_preference(lp, ref, mask, offsets, beta, smoothing):
    d = torch.where(mask, (lp.double() - ref.double()), torch.zeros_like(lp, dtype=torch.float64))
    sums = torch.cat([torch.zeros_like(d[:1]), d.cumsum(0)])
    per = beta * (sums[offsets[1:]] - sums[offsets[:-1]])
    pairs = per.numel() // 2
    chosen, rejected = per[:pairs], per[pairs:]
    h = chosen - rejected
    tail = torch.log1p(torch.exp(-h.abs()))
    like, unlike = torch.clamp(h, max=0) - tail, torch.clamp(-h, max=0) - tail  # log sigma(h), log sigma(-h)
    loss = -((1 - smoothing) * like + smoothing * unlike).mean()
    slope = (-(1 - smoothing) * torch.exp(unlike) + smoothing * torch.exp(like)) * (beta / pairs)
    per_seq = torch.cat([slope, -slope, torch.zeros_like(slope[:1])])
    token = torch.arange(lp.numel(), device=lp.device)
    seq = torch.searchsorted(offsets, token, right=True) - 1  # 2 * pairs for those behind the last sequence
    grad = torch.where(mask, per_seq[seq], torch.zeros_like(d))
    return loss.float(), chosen.float(), rejected.float(), grad.float()


def _plain_policy(lp, s, low, high, kl):
    lp, old, adv = lp.double(), s["old"].double(), s["advantages"].double()
    w = s["mask"].double()
    count = w.sum()
    r = torch.exp(lp - old)
    cut = ((adv > 0) & (r > 1 + high)) | ((adv < 0) & (r < 1 - low))
    value = torch.maximum(-r * adv, -r.clamp(1 - low, 1 + high) * adv)
    slope = torch.where(cut, torch.zeros_like(r), -adv * r)
    mean_kl = torch.zeros_like(count)
    if s["ref"] is not None:
        d = s["ref"].double() - lp
        k3 = torch.exp(d) - d - 1
        mean_kl = (w * k3).sum() / count.clamp(min=1)
        value = value + kl * k3
        slope = slope + kl * (1 - torch.exp(d))
    scale = w / count.clamp(min=1)
    return (scale * value).sum().float(), mean_kl.float(), (scale * cut).sum().float(), (scale * slope).float()


def _plain_distill(s, case):
    t, classes = case["temperature"], case["classes"]
    x = s["x"].float() / t
    f, m, e, total = _softmax_parts(x)
    valid = (s["ids"] >= 0) & (s["ids"] < classes)
    at = s["ids"].long().clamp(0, classes - 1)
    y = torch.where(valid, s["teacher"].double() / t, torch.full_like(at, -math.inf, dtype=torch.float64))
    y = y - y.amax(1, keepdim=True)
    q = torch.exp(y)
    mass = q.sum(1, keepdim=True)
    q = q / mass
    log_p = f.gather(1, at).double() - m.double() - torch.log(total.double())
    terms = torch.where(q > 0, q * (y - torch.log(mass) - log_p), torch.zeros_like(q))
    w = s["weights"].double()
    whole = w.sum()
    scale = torch.where(whole > 0, w / whole, torch.zeros_like(w))
    loss = (scale * terms.sum(1)).sum() * t * t
    coefficient = (scale * t * s["scale"]).float()[:, None]
    grad = e * (coefficient / total)
    grad.scatter_add_(1, at, torch.where(valid, -coefficient * q.float(), torch.zeros_like(coefficient)))
    return loss.float(), grad.to(s["x"].dtype)


_BETA, _LOW, _HIGH = 0.1, 0.2, 0.28


def _run_plain(s, case):
    op = case["op"]
    if op == "logp":
        return _plain_log_probs(s["x"], s["targets"], case["classes"])[0]
    if op == "logp_train":
        lp, parts = _plain_log_probs(s["x"], s["targets"], case["classes"])
        return lp, _plain_log_probs_grad(s["upstream"], parts, s["x"].dtype)
    if op == "pref":
        return _plain_preference(s["lp"], s["ref"], s["mask"], s["offsets"], _BETA, case["smoothing"])
    if op == "pref_logits":
        lp, parts = _plain_log_probs(s["x"], s["targets"], case["classes"])
        loss, chosen, rejected, g = _plain_preference(lp, s["ref"], s["mask"], s["offsets"], _BETA, case["smoothing"])
        return loss, chosen, rejected, _plain_log_probs_grad(g * s["scale"], parts, s["x"].dtype)
    if op == "policy":
        return _plain_policy(s["lp"], s, _LOW, _HIGH, case["kl"])
    if op == "policy_logits":
        lp, parts = _plain_log_probs(s["x"], s["targets"], case["classes"])
        loss, kl, cut, g = _plain_policy(lp, s, _LOW, _HIGH, case["kl"])
        return loss, kl, cut, _plain_log_probs_grad(g * s["scale"], parts, s["x"].dtype)
    return _plain_distill(s, case)


# ------------------------------------------------------- the framework's own

def _run_own(s, case):
    losses = _losses()
    op = case["op"]
    if op == "logp":
        return losses.token_log_probs(s["x"], s["targets"])
    if op == "policy_logits":
        return losses.policy_loss_with_grad(s["x"], s["targets"], s["old"], s["advantages"], ref_log_probs=s["ref"],
                                            mask=s["mask"], clip_low=_LOW, clip_high=_HIGH, kl_coef=case["kl"],
                                            grad_loss=s["scale"])
    if op == "distill_grad":
        return losses.distillation_loss_with_grad(s["x"], s["ids"], s["teacher"], weights=s["weights"],
                                                  temperature=case["temperature"], grad_loss=s["scale"])
    leaf = s["lp" if op in ("pref", "policy") else "x"].detach().requires_grad_()
    if op == "logp_train":
        lp = losses.token_log_probs(leaf, s["targets"])
        return lp.detach(), torch.autograd.grad(lp, leaf, s["upstream"])[0]
    if op == "distill":
        out = (losses.distillation_loss(leaf, s["ids"], s["teacher"], weights=s["weights"],
                                        temperature=case["temperature"]),)
    elif op == "policy":
        out = losses.policy_loss(leaf, s["old"], s["advantages"], ref_log_probs=s["ref"], mask=s["mask"],
                                 clip_low=_LOW, clip_high=_HIGH, kl_coef=case["kl"])
    else:
        lp = leaf if op == "pref" else losses.token_log_probs(leaf, s["targets"])
        out = losses.preference_loss(lp, s["offsets"], ref_log_probs=s["ref"], mask=s["mask"], beta=_BETA,
                                     label_smoothing=case["smoothing"])
    grad = torch.autograd.grad(out[0], leaf, s.get("scale"))[0]
    return (*(o.detach() for o in out), grad)


def run(state):
    return _run_own(state, state["case"]) if own else _run_plain(state, state["case"])


# ------------------------------------------------------------ bytes and flops

def _tokens(case):
    """Tokens of the mean draw: sequences of 1 to 2 * mean_len - 1 tokens are mean_len long on average."""
    return 2 * case["pairs"] * case["mean_len"] + 3 if "pairs" in case else case["rows"]


def work(case):
    op, n = case["op"], _tokens(case)
    nbytes = flops = 0
    if "classes" in case:
        values = n * case["classes"]
        size = 4 if case["dtype"] == "f32" else 2
        grad = op != "logp"
        nbytes += values * size * (2 if grad else 1)
        flops += values * (6 if grad else 4)  # maximum, difference, exponential, sum; difference or product, rounding
        nbytes += 8 * n if not op.startswith("distill") else 0
    if op in ("logp", "logp_train"):
        nbytes += (4 if op == "logp" else 8) * n
    if op in ("pref", "pref_logits"):
        nbytes += (4 + 1) * n + 8 * (2 * case["pairs"] + 1) + (8 * n if op == "pref" else 0) + 8 * case["pairs"]
        flops += 4 * n
    if op in ("policy", "policy_logits"):
        nbytes += (4 + 4 + 1 + (4 if case["kl"] else 0)) * n + (8 * n if op == "policy" else 0)
        flops += 20 * n
    if op in ("distill", "distill_grad"):
        nbytes += n * (case["top"] * (8 if case["dtype"] == "f32" else 6) + 4)
        flops += 10 * n * case["top"]
    return {"bytes": int(nbytes), "flops": int(flops)}


# --------------------------------------------------------------- in 64 bits

def _chunks(rows, classes):
    step = max(1, (1 << 26) // classes)
    return [(i, min(rows, i + step)) for i in range(0, rows, step)]


def _exact_log_probs(x, targets):
    out = torch.zeros(x.shape[0], dtype=torch.float64, device=x.device)
    for a, b in _chunks(*x.shape):
        lse = torch.logsumexp(x[a:b].double(), 1)
        for_row = x[a:b].double().gather(1, targets[a:b].clamp(0, x.shape[1] - 1)[:, None])[:, 0] - lse
        out[a:b] = for_row.masked_fill((targets[a:b] < 0) | (targets[a:b] >= x.shape[1]), 0.0)
    return out


def _exact_log_probs_grad(x, targets, upstream):
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for a, b in _chunks(*x.shape):
        out[a:b] = -torch.softmax(x[a:b].double(), 1)
        real = ((targets[a:b] >= 0) & (targets[a:b] < x.shape[1])).nonzero()[:, 0]
        out[a:b][real, targets[a:b][real]] += 1.0
        use = torch.zeros(b - a, dtype=torch.float64, device=x.device)
        use[real] = upstream[a:b].double()[real]
        out[a:b] *= use[:, None]
    return out


def _exact_preference(lp, s, case):
    offsets, pairs = s["offsets"].tolist(), case["pairs"]
    ratio = (lp.double() - s["ref"].double()).cpu()
    mask = s["mask"].cpu()
    rewards = [_BETA * float(ratio[a:b][mask[a:b]].sum()) for a, b in zip(offsets, offsets[1:])]
    loss, grad = 0.0, torch.zeros(ratio.numel(), dtype=torch.float64)
    eps = case["smoothing"]
    for p in range(pairs):
        h = rewards[p] - rewards[pairs + p]
        up = 1.0 / (1.0 + math.exp(-h)) if h > -700 else 0.0
        down = 1.0 / (1.0 + math.exp(h)) if h < 700 else 0.0
        softplus = max(-h, 0.0) + math.log1p(math.exp(-abs(h)))  # -log sigma(h)
        loss += ((1 - eps) * softplus + eps * (softplus + h)) / pairs
        slope = _BETA / pairs * (eps * up - (1 - eps) * down)
        for seq, sign in ((p, 1.0), (pairs + p, -1.0)):
            a, b = offsets[seq], offsets[seq + 1]
            grad[a:b] = mask[a:b].double() * (sign * slope)
    per = torch.tensor(rewards, dtype=torch.float64)
    return torch.tensor(loss, dtype=torch.float64), per[:pairs], per[pairs:], grad.to(lp.device)


def _exact_policy(lp, s, case):
    keep = s["mask"]
    lp, old, adv = lp.double()[keep], s["old"].double()[keep], s["advantages"].double()[keep]
    count = max(1, int(keep.sum()))
    ratio = (lp - old).exp()
    bound = torch.where(adv >= 0, torch.clamp(ratio, max=1 + _HIGH), torch.clamp(ratio, min=1 - _LOW))
    kept = bound == ratio
    value, slope = -(bound * adv), torch.where(kept, -(ratio * adv), torch.zeros_like(adv))
    kl = torch.zeros((), dtype=torch.float64)
    if s["ref"] is not None:
        gap = s["ref"].double()[keep] - lp
        k3 = torch.expm1(gap) - gap
        kl = k3.sum() / count
        value, slope = value + case["kl"] * k3, slope - case["kl"] * torch.expm1(gap)
    grad = torch.zeros(keep.numel(), dtype=torch.float64, device=lp.device)
    grad[keep] = slope / count
    return value.sum() / count, kl, (~kept).sum() / torch.tensor(float(count), dtype=torch.float64), grad


def _exact_distill(s, case):
    x, ids, t = s["x"], s["ids"].long(), case["temperature"]
    w = s["weights"].double()
    whole = float(w.sum())
    w = w / whole if whole > 0 else w * 0
    loss, scale = 0.0, float(s["scale"])
    grad = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for a, b in _chunks(*x.shape):
        real = (ids[a:b] >= 0) & (ids[a:b] < case["classes"])
        log_p = torch.log_softmax(x[a:b].double() / t, 1)
        log_q = torch.log_softmax((s["teacher"][a:b].double() / t).masked_fill(~real, -math.inf), 1)
        q = log_q.exp()
        at = ids[a:b].clamp(0, case["classes"] - 1)
        gap = (log_q - log_p.gather(1, at)).masked_fill(~real, 0.0)
        loss += float((w[a:b, None] * q * gap).sum()) * t * t
        grad[a:b] = log_p.exp().scatter_add_(1, at, -q.masked_fill(~real, 0.0)) * (t * scale * w[a:b, None])
    return torch.tensor(loss, dtype=torch.float64), grad


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("logp", "logp_train"):
        lp = _exact_log_probs(s["x"], s["targets"])
        return lp if op == "logp" else (lp, _exact_log_probs_grad(s["x"], s["targets"], s["upstream"]))
    if op in ("distill", "distill_grad"):
        return _exact_distill(s, case)
    lp = s["lp"] if op in ("pref", "policy") else _exact_log_probs(s["x"], s["targets"])
    out = (_exact_preference if op in ("pref", "pref_logits") else _exact_policy)(lp, s, case)
    if op in ("pref", "policy"):
        return out
    return (*out[:3], _exact_log_probs_grad(s["x"], s["targets"], out[3] * s["scale"].double()))

"""The losses over rows of class scores (opencl_tf.losses) against their
definitions in float64: sizes from one class and one token to rows of several
CTAs and tensors past 2^31 values, ragged and strided rows, ignored and
masked entries, rows without a softmax, repeated teacher classes, empty
sequences, graph capture, streams.

Tolerances.  u = 2^-24 is half a step of fp32.  A row's exponent (x - m) * c has
relative error 3u (difference, product, the constant c), so 2^that is off by
3u |x - m| / T; ex2 adds 4u (2 ulp).  s is a sum of positive terms: at most
``chain`` additions follow one another, each u.  With
D = sum_j p_j |x_j - m| / T the relative error of s is <= u (3 D + 4 + chain),
and that of p_j <= u (3 |x_j - m| / T + 8) more.  A stored value adds half a step of its type."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# half of the smallest value that the type tells from 0
TINY = {torch.float64: 0.0, torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}


def chain(classes):
    """Additions that follow one another in a row's sum: a thread's values
    (batches of at most 32, then the batches), the warp's 5 + the CTA's 5 + the
    cluster's 5 merges of one addition and two products each.  A thread has an eighth of a row of up to
    4096 values at most, a 32nd of one of up to 16384, a 256th of a longer one."""
    per_thread = -(-classes // (8 if classes <= 4096 else 32 if classes <= 16384 else 256))
    return 32 + per_thread // 32 + 16 + 45


def parts(x, temperature=1.0):
    """m, s, p, and the relative error that p may have, all float64."""
    z = x.double()
    m = z.amax(-1, keepdim=True)
    d = (z - m) / temperature
    p = torch.softmax(z / temperature, -1)
    away = torch.where(p > 0, -d, torch.zeros_like(d))
    big_d = (p * away).sum(-1, keepdim=True)
    rel_s = U * (3 * big_d + 4 + chain(x.shape[-1]))
    return p, rel_s, rel_s + U * (3 * away + 8)


def close(got, want, tol, what=""):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    off = (got - want).abs()
    off = torch.where(want.isnan() | (got == want), torch.zeros_like(off), off)
    over = off - tol
    assert bool((over <= 0).all()), f"{what}: off by {float(off.max()):.3e}, {float(over.max()):.3e} more than allowed"


def grad_tol(factor, p, rel_p, want, dtype):
    """Of factor * (p - q): p's error, the difference and the factor's three roundings, the store."""
    eps = torch.finfo(dtype).eps / 2
    return factor.abs() * (p * rel_p + 2 * U) + want.abs() * (6 * U + eps) + TINY[dtype]


def scores(rows, classes, dtype, seed, dead=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = 3 * torch.randn(rows, classes, generator=g, device="cuda")
    t = torch.randint(0, classes, (rows,), generator=g, device="cuda")
    x.scatter_add_(1, t[:, None], 8 * torch.rand(rows, 1, generator=g, device="cuda"))
    if dead and classes > 4:  # excluded classes, by -inf and by the type's lowest value
        off = torch.rand(rows, classes, generator=g, device="cuda") < 0.05
        off.scatter_(1, t[:, None], False)
        x = x.masked_fill(off, -math.inf)
        x[:, classes // 2] = torch.where(t == classes // 2, x[:, classes // 2], torch.finfo(DTYPES[dtype]).min)
    return x.to(DTYPES[dtype]), t


def ref_log_probs(x, t):
    z = x.double()
    valid = (t >= 0) & (t < x.shape[-1])
    lp = torch.log_softmax(z, -1).gather(-1, t.clamp(0, x.shape[-1] - 1).long()[..., None])[..., 0]
    return torch.where(valid, lp, torch.zeros_like(lp)), valid


def ref_log_probs_grad(x, t, g, dtype):
    lp, valid = ref_log_probs(x, t)
    p, _, rel_p = parts(x)
    f = torch.where(valid, g.double(), torch.zeros_like(lp))[..., None]
    want = -f * p
    want.scatter_add_(-1, t.clamp(0, x.shape[-1] - 1).long()[..., None], f)
    off = (f == 0).expand_as(want)
    return want.masked_fill(off, 0.0), grad_tol(f, p, rel_p, want, dtype).masked_fill(off, 0.0)


SIZES = [(1, 1), (1, 2), (3, 7), (70, 33), (9, 1023), (8, 1024), (2, 1025), (1, 4096), (5, 8191), (300, 4099),
         (1, 50257), (40, 32000), (2, 131075)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,classes", SIZES)
def test_token_log_probs(otf, rows, classes, dtype):
    x, t = scores(rows, classes, dtype, rows * 7 + classes)
    t[::3] = torch.tensor([-100, classes, -1, classes + 7], device="cuda").repeat(rows)[:len(t[::3])]
    if rows == 1:
        t[0] = classes - 1
    g = torch.randn(rows, device="cuda")
    g[rows // 2:rows // 2 + 1] = 0.0 if rows > 1 else 1.5
    leaf = x.clone().requires_grad_()
    lp = otf.losses.token_log_probs(leaf, t)
    assert lp.dtype == torch.float32 and lp.shape == t.shape
    want, valid = ref_log_probs(x, t)
    _, rel_s, _ = parts(x)
    close(lp.detach(), want, rel_s[:, 0] + 2 * U * want.abs() + U, "log-probabilities")
    assert torch.equal(lp.detach(), otf.losses.token_log_probs(x, t.to(torch.int32)))  # no gradient, 32-bit targets
    grad, = torch.autograd.grad(lp, leaf, g)
    assert grad.dtype == x.dtype and grad.is_contiguous()
    close(grad, *ref_log_probs_grad(x, t, g, x.dtype), "gradient")


@pytest.mark.parametrize("classes", [6, 5000, 40000])
def test_rows_without_a_softmax(otf, classes):
    """NaN, +inf and -inf-only rows give NaN there and nowhere else; nothing where they do not count."""
    x, t = scores(8, classes, "f32", 3, dead=False)
    x[0] = -math.inf
    x[1, classes // 3] = math.nan
    x[2, classes - 1] = math.inf
    x[3] = math.nan
    x[4] = torch.finfo(torch.float32).min  # a uniform row all the same
    x[5] = math.nan
    t[5] = -100
    x[6] = math.nan
    g = torch.ones(8, device="cuda")
    g[6] = 0.0
    leaf = x.clone().requires_grad_()
    lp = otf.losses.token_log_probs(leaf, t)
    assert lp[:4].isnan().all() and lp[6].isnan() and float(lp[5]) == 0.0
    assert abs(float(lp[4]) + math.log(classes)) <= (chain(classes) + 8) * U * max(1.0, math.log(classes))
    grad, = torch.autograd.grad(lp, leaf, g)
    assert grad[:4].isnan().all() and not grad[4:].isnan().any()
    assert not grad[5].any() and not grad[6].any()
    want, tol = ref_log_probs_grad(x[7:], t[7:], g[7:], torch.float32)
    close(grad[7:], want, tol)
    # a target excluded by -inf: -inf, and a finite gradient
    y, t = scores(2, classes, "f32", 4, dead=False)
    y[0, t[0]] = -math.inf
    leaf = y.clone().requires_grad_()
    lp = otf.losses.token_log_probs(leaf, t)
    assert float(lp[0]) == -math.inf and math.isfinite(float(lp[1]))
    grad, = torch.autograd.grad(lp, leaf, torch.ones(2, device="cuda"))
    assert float(grad[0, t[0]]) == 1.0 and bool(grad.isfinite().all())


def _views(classes):
    big = 2 * torch.randn(3, 6, classes + 5, device="cuda")
    return {
        "all but the last position": big[:, :-1],
        "a padded vocabulary": big[:, :, :classes],
        "a padded vocabulary, shifted": big[:, 1:, 3:classes + 3],
        "every other row": big.view(18, -1)[::2],
        "swapped leading axes": big.transpose(0, 1),
        "one row for all": big[0, 0].expand(4, -1),
        "classes not adjacent": big.transpose(1, 2)[:, :, :6],
        "three loose axes": big[None].expand(2, -1, -1, -1)[:, :, ::5],
        "one row": big[1, 2],
    }


@pytest.mark.parametrize("classes", [40, 2501])
@pytest.mark.parametrize("view", list(_views(2)) if torch.cuda.is_available() else ["all"])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_strided_scores(otf, view, classes, dtype):
    torch.manual_seed(classes)
    x = _views(classes)[view]
    if dtype != "f32":  # the view's strides, in the other type
        base = torch.empty(x.untyped_storage().size() // 4, device="cuda", dtype=DTYPES[dtype])
        base.copy_(torch.as_strided(x, (base.numel(),), (1,), 0))
        x = base.as_strided(x.shape, x.stride(), x.storage_offset())
    t = torch.randint(0, x.shape[-1], x.shape[:-1], device="cuda")
    g = torch.randn(t.shape, device="cuda")
    leaf = x.detach().requires_grad_()
    lp = otf.losses.token_log_probs(leaf, t)
    want, _ = ref_log_probs(x, t)
    _, rel_s, _ = parts(x)
    close(lp.detach(), want, rel_s[..., 0] + 2 * U * want.abs() + U, view)
    grad, = torch.autograd.grad(lp, leaf, g)
    close(grad, *ref_log_probs_grad(x, t, g, x.dtype), view)


def test_more_than_2_31_values(otf):
    rows, classes = 70001, 32003  # 2.2e9 scores, 4.5 GB
    x = torch.empty(rows, classes, device="cuda", dtype=torch.bfloat16)
    x.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    t = torch.arange(rows, device="cuda") % classes
    g = torch.randn(rows, device="cuda")
    leaf = x.requires_grad_()
    lp = otf.losses.token_log_probs(leaf, t)
    grad, = torch.autograd.grad(lp, leaf, g)
    pick = torch.cat([torch.arange(4), torch.arange(67100, 67110), torch.arange(rows - 4, rows)]).cuda()
    x = x.detach()[pick]
    want, _ = ref_log_probs(x, t[pick])
    _, rel_s, _ = parts(x)
    close(lp.detach()[pick], want, rel_s[:, 0] + 2 * U * want.abs() + U)
    close(grad[pick], *ref_log_probs_grad(x, t[pick], g[pick], torch.bfloat16))


# ------------------------------------------------------------ distillation

def ref_distill(x, ids, y, w, T, gl=1.0):
    """loss, gradient, and their tolerances"""
    classes = x.shape[-1]
    z = x.double().reshape(-1, classes)
    ids, y = ids.long().reshape(z.shape[0], -1), y.double().reshape(z.shape[0], -1)
    w = torch.ones(z.shape[0], dtype=torch.float64, device=x.device) if w is None else w.double().reshape(-1)
    real = (ids >= 0) & (ids < classes) & (y != -math.inf)
    some = real.any(1) & (w != 0)
    log_q = torch.log_softmax((y / T).masked_fill(~real, -math.inf), 1).masked_fill(~real, -math.inf)
    q = log_q.exp().masked_fill(~real, 0.0)
    log_p = torch.log_softmax(z / T, 1)
    at = ids.clamp(0, classes - 1)
    gap = torch.where(q > 0, log_q - log_p.gather(1, at), torch.zeros_like(q))
    rows = T * T * (q * gap).sum(1)
    total = float(w.sum())
    share = w / total if total != 0 else torch.zeros_like(w)
    counted = torch.where(some, share * rows, torch.zeros_like(rows))
    p, rel_s, rel_p = parts(z, T)
    f = (gl * T * share * some)[:, None]
    want = f * p
    want.scatter_add_(1, at, -f * q)
    dropped = (~some)[:, None].expand_as(want)
    want = want.masked_fill(dropped, 0.0)
    # q: exponent 3u |y - max| / T, expf 2u, the sum over K entries in 32 lanes, the quotient
    k = ids.shape[1]
    rel_q = U * (3 * torch.where(real, (y.masked_fill(~real, -math.inf).amax(1, keepdim=True) - y) / T,
                                 torch.zeros_like(y)).nan_to_num() + 6 + k / 32 + 5)
    q_tol = torch.zeros_like(want).scatter_add_(1, at, f.abs() * q * (rel_q + U * k))
    tol = grad_tol(f, p, rel_p, want, x.dtype) + q_tol
    # the loss: q's error times the gap, log s and log sum q in 32 bits
    log_err = rel_s[:, 0] + U * (2 * torch.log(torch.tensor(float(max(classes, k)))) + 4 + k / 32 + 8)
    row_tol = T * T * ((q * rel_q * gap.abs()).sum(1) + log_err)
    loss_tol = (share.abs() * torch.where(some, row_tol, torch.zeros_like(row_tol))).sum() + 2 * U * counted.sum().abs()
    return counted.sum(), want.reshape(x.shape), loss_tol, tol.masked_fill(dropped, 0.0).reshape(x.shape)


def teacher(x, k, seed, dtype=torch.float32):
    """k entries a row: real classes, some repeated, some out of range, some of -inf."""
    rows, classes = x.shape
    g = torch.Generator(device="cuda").manual_seed(seed)
    alive = x.float().masked_fill(x == torch.finfo(x.dtype).min, -math.inf)
    ids = (alive + torch.randn(x.shape, generator=g, device="cuda")).topk(min(k, classes), 1).indices
    ids = ids.repeat(1, -(-k // ids.shape[1]))[:, :k].contiguous()
    y = x.float().gather(1, ids) + torch.randn(rows, k, generator=g, device="cuda")
    y = y.masked_fill(~y.isfinite(), -math.inf).masked_fill(y < -1e4, -math.inf)
    if k > 2:
        ids[:, k - 1] = ids[:, 0]  # repeated
        ids[::2, k // 2] = -1
        ids[1::4, 1] = classes
        y[1::3, 2] = -math.inf
    return ids, y.to(dtype)


DISTILL = [(1, 1, 1), (4, 2, 3), (33, 70, 8), (5, 1000, 1024), (7, 1025, 1), (3, 5000, 64), (1, 32003, 100),
           (300, 2050, 17), (2, 131075, 128), (200, 4003, 600), (30, 129, 257)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,classes,k", DISTILL)
def test_distillation(otf, rows, classes, k, dtype):
    x, _ = scores(rows, classes, dtype, rows + classes + k)
    ids, y = teacher(x, k, rows + k, torch.bfloat16 if dtype == "bf16" else torch.float32)
    if rows > 3:
        ids[2] = -1  # a row without entries
    w = None
    if rows > 1:
        w = torch.rand(rows, device="cuda") + 0.1
        w[rows - 1] = 0.0
        x[rows - 1] = math.nan  # not looked at
    T = 2.0 if classes % 2 else 1.0
    gl = torch.tensor(64.0, device="cuda")
    loss, grad, loss_tol, tol = ref_distill(x, ids, y, w, T, 64.0)
    leaf = x.clone().requires_grad_()
    got = otf.losses.distillation_loss(leaf, ids, y, weights=w, temperature=T)
    close(got.detach(), loss, loss_tol, "loss")
    d, = torch.autograd.grad(got, leaf, gl)
    close(d, grad, tol, "gradient")
    with_grad = otf.losses.distillation_loss_with_grad(x, ids.to(torch.int32), y, weights=w, temperature=T, grad_loss=gl)
    assert torch.equal(with_grad[0], got.detach()) and torch.equal(with_grad[1], d)
    assert torch.equal(otf.losses.distillation_loss(x, ids, y, weights=w, temperature=T), got.detach())


def test_distillation_weights(otf):
    x, _ = scores(6, 3000, "f32", 1, dead=False)
    ids, y = teacher(x, 20, 2)
    # bytes as weights; a sum of 0; no weights
    keep = torch.tensor([1, 0, 1, 1, 0, 1], device="cuda", dtype=torch.bool)
    a = otf.losses.distillation_loss_with_grad(x, ids, y, weights=keep)
    b = otf.losses.distillation_loss_with_grad(x, ids, y, weights=keep.float())
    c = otf.losses.distillation_loss_with_grad(x, ids, y, weights=keep.to(torch.uint8) * 7)
    for o in (b, c):
        assert torch.equal(a[0], o[0]) and torch.equal(a[1], o[1])
    for w in (torch.zeros(6, device="cuda"), torch.tensor([1.0, -1.0, 2.0, -2.0, 0.0, 0.0], device="cuda")):
        loss, grad = otf.losses.distillation_loss_with_grad(x, ids, y, weights=w)
        assert float(loss) == 0.0 and not grad.any()
    # a teacher class that the scores exclude: an infinite loss, a finite gradient
    x[0, ids[0, 0]] = -math.inf
    loss, grad = otf.losses.distillation_loss_with_grad(x, ids, y)
    assert float(loss) == math.inf and bool(grad.isfinite().all())


# -------------------------------------------------------------- preference

def ref_preference(lp, off, ref, mask, beta, eps):
    """loss, chosen, rejected as float64, differentiable in lp"""
    off = [min(max(int(o), 0), lp.numel()) for o in off.tolist()]
    w = torch.ones_like(lp) if mask is None else mask.reshape(-1).double()
    d = lp if ref is None else lp - ref.reshape(-1).double()
    d = torch.where(w != 0, w * torch.where(w != 0, d, torch.zeros_like(d)), torch.zeros_like(d))
    sums = torch.stack([beta * d[a:b].sum() for a, b in zip(off, off[1:])])
    p = sums.numel() // 2
    h = sums[:p] - sums[p:]
    ls = torch.nn.functional.logsigmoid
    return (-(1 - eps) * ls(h) - eps * ls(-h)).mean(), sums[:p], sums[p:]


@pytest.mark.parametrize("pairs,longest,mask,has_ref,eps", [
    (1, 1, None, True, 0.0), (1, 5000, "bool", True, 0.1), (3, 40, "float", True, 0.5), (64, 300, "uint8", False, 0.0),
    (700, 9, "bool", True, 0.2), (2, 200000, None, True, 0.0)])
def test_preference_loss(otf, pairs, longest, mask, has_ref, eps):
    g = torch.Generator().manual_seed(pairs + longest)
    lengths = torch.randint(0 if longest > 1 else 1, longest + 1, (2 * pairs,), generator=g)  # empty ones among them
    if pairs > 1:
        lengths[1] = lengths[pairs] = 0
    off = torch.cat([torch.zeros(1, dtype=torch.long), lengths.cumsum(0)]) + 2
    n = int(off[-1]) + 5  # tokens before the first and behind the last sequence
    lp = -torch.rand(n, generator=g) * 4
    ref = lp + 0.2 * torch.randn(n, generator=g) if has_ref else None
    w = {None: None, "bool": torch.rand(n, generator=g) > 0.3, "uint8": (torch.rand(n, generator=g) > 0.3).to(torch.uint8),
         "float": torch.rand(n, generator=g).floor_divide(0.25) / 4}[mask]
    if w is not None:
        lp = lp.masked_fill(w == 0, math.nan)  # not looked at
    lp[:2] = math.nan
    lp[-5:] = math.inf
    z = lp.double().requires_grad_()
    loss, chosen, rejected = ref_preference(z, off, ref, w, 0.3, eps)
    want, = torch.autograd.grad(loss, z)
    cuda = [None if a is None else a.cuda() for a in (off, ref, w)]
    leaf = lp.cuda().requires_grad_()
    got = otf.losses.preference_loss(leaf, cuda[0], cuda[1], cuda[2], beta=0.3, label_smoothing=eps)
    grad, = torch.autograd.grad(got[0], leaf)
    # sums in 64 bits: what is left is the store's half step, and the slope's and the products' for the gradient
    close(got[0].detach().cpu(), loss.detach(), U * loss.detach().abs() * 2 + 1e-12, "loss")
    close(got[1].cpu(), chosen.detach(), U * chosen.detach().abs() * 2 + 1e-12, "chosen")
    close(got[2].cpu(), rejected.detach(), U * rejected.detach().abs() * 2 + 1e-12, "rejected")
    assert not got[1].requires_grad and not got[2].requires_grad
    close(grad.cpu(), want, 4 * U * want.abs() + 1e-12 * want.abs().max(), "gradient")
    twice, = torch.autograd.grad(otf.losses.preference_loss(leaf, cuda[0].to(torch.int32), cuda[1], cuda[2], beta=0.3,
                                                            label_smoothing=eps)[0], leaf)
    assert torch.equal(grad, twice)


def test_preference_extremes_and_bad_offsets(otf):
    lp = torch.tensor([-1.0, -900.0, -1.0, -2.0], device="cuda")
    off = torch.tensor([0, 1, 2, 3, 4], device="cuda")
    loss, c, r = otf.losses.preference_loss(lp, off, beta=1.0)
    want = (math.log1p(math.exp(0.0)) + 898.0) / 2  # h = 0 and h = -898
    assert abs(float(loss) - want) <= 2 * U * want
    leaf = lp.clone().requires_grad_()
    g, = torch.autograd.grad(otf.losses.preference_loss(leaf, off, beta=1.0)[0], leaf)
    assert g.tolist() == [-0.25, -0.5, 0.25, 0.5]
    # offsets beyond the tokens end at the tokens; falling ones give empty sequences: nothing outside is read
    far = torch.tensor([-7, 1, 2, 3, 1 << 40], device="cuda")
    assert torch.equal(otf.losses.preference_loss(lp, far, beta=1.0)[0], loss)
    loss, c, r = otf.losses.preference_loss(lp, torch.tensor([4, 3, 2, 1, 0], device="cuda"))
    assert float(loss) == pytest.approx(math.log(2.0), rel=2 * U) and not c.any() and not r.any()
    # no tokens at all
    loss, _, _ = otf.losses.preference_loss(lp[:0], torch.zeros(3, device="cuda", dtype=torch.int64))
    assert float(loss) == pytest.approx(math.log(2.0), rel=2 * U)


# ------------------------------------------------------------------ policy

def ref_policy(lp, old, adv, ref, mask, low, high, kl_coef):
    """loss, kl, clipped share as float64, differentiable in lp; only the tokens that count"""
    w = torch.ones(lp.shape, dtype=torch.float64) if mask is None else mask.double()
    keep = w != 0
    w, lp, old, adv = w[keep], lp[keep], old.double()[keep], adv.double()[keep]
    r = torch.exp(lp - old)
    cut = ((adv > 0) & (r > 1 + high)) | ((adv < 0) & (r < 1 - low))
    held = torch.where(adv > 0, r.clamp(max=1 + high), r.clamp(min=1 - low))
    value = -torch.where(cut, held.detach(), r) * adv
    kl = torch.zeros_like(r)
    if ref is not None:
        d = ref.double()[keep] - lp
        kl = torch.expm1(d) - d
        value = value + kl_coef * kl
    total = w.sum() if float(w.sum()) != 0 else torch.tensor(math.inf, dtype=torch.float64)
    return (w * value).sum() / total, (w * kl).sum() / total, (w * cut).sum() / total


def policy_tol(lp, old, adv, ref, mask, kl_coef):
    """How far a token's term and slope may be off, computed in 32 bits: the ratio by its exponent's rounding
    (u |lp - old|), expf's ulp (2u) and one product; exp(d) - d - 1 by d's rounding, whose relative effect is at most
    2 + |d| times u |d| / |d|, ten roundings of its series (each below u of the result) or of the subtraction at |d| > 1
    (4u); one fused multiply-add.  -> (sum of the terms' errors / total weight, slopes' errors / total weight)"""
    w = torch.ones(lp.shape, dtype=torch.float64) if mask is None else mask.double()
    keep = w != 0
    lp, old, adv = (torch.where(keep, a.double(), torch.zeros_like(w)) for a in (lp, old, adv))
    ra = (torch.exp(lp - old) * adv).abs()
    value = U * ((lp - old).abs() + 6) * ra
    slope = value.clone()
    if ref is not None:
        d = torch.where(keep, ref.double(), torch.zeros_like(w)) - lp
        kl = torch.expm1(d) - d
        value = value + kl_coef * U * (2 + d.abs() + 12) * kl
        slope = slope + kl_coef * U * ((2 + d.abs() + 12) * kl + 3 * d.abs() + 2 * torch.expm1(d).abs())
    total = max(float(w.sum()), 1e-300)
    return float((w.abs() * value).sum() / total), 2 * w.abs() * slope / total


POLICY = [(1, None, True, 0.0), (64, "bool", True, 0.05), (4097, "float", True, 0.02), (333, "uint8", False, 0.0),
          (1000003, "bool", True, 0.1), (50, "none counts", True, 0.1)]


def policy_inputs(n, mask, has_ref, seed):
    g = torch.Generator().manual_seed(seed)
    lp = -3 * torch.rand(n, generator=g)
    old = lp + 0.3 * torch.randn(n, generator=g)
    adv = torch.randn(n, generator=g)
    adv[::5] = 0.0
    ref = lp + 0.3 * torch.randn(n, generator=g) if has_ref else None
    w = {None: None, "bool": torch.rand(n, generator=g) > 0.3, "uint8": (torch.rand(n, generator=g) > 0.3).to(torch.uint8),
         "float": torch.rand(n, generator=g).floor_divide(0.25) / 4, "none counts": torch.zeros(n, dtype=torch.bool)}[mask]
    return lp, old, adv, ref, w


@pytest.mark.parametrize("n,mask,has_ref,kl", POLICY)
def test_policy_loss(otf, n, mask, has_ref, kl):
    lp, old, adv, ref, w = policy_inputs(n, mask, has_ref, n)
    if w is not None:
        lp, old = lp.masked_fill(w == 0, math.nan), old.masked_fill(w == 0, math.inf)
    z = lp.double().requires_grad_()
    loss, mean_kl, share = ref_policy(z, old, adv, ref, w, 0.2, 0.28, kl)
    want = torch.autograd.grad(loss, z)[0].nan_to_num()
    leaf = lp.cuda().requires_grad_()
    cuda = [None if a is None else a.cuda() for a in (old, adv, ref, w)]
    got = otf.losses.policy_loss(leaf, *cuda, clip_low=0.2, clip_high=0.28, kl_coef=kl)
    # the terms' errors, added in 64 bits, and the store's half step
    off, slope_off = policy_tol(lp, old, adv, ref, w, kl)
    for a, b, o in zip(got, (loss, mean_kl, share), (off, off / kl if kl else 0.0, 0.0)):
        close(a.detach().cpu(), b.detach(), o + 2 * U * b.detach().abs() + 1e-12)
    grad, = torch.autograd.grad(got[0], leaf, torch.tensor(3.0, device="cuda"))
    close(grad.cpu(), 3 * want, 3 * slope_off + 6 * U * 3 * want.abs(), "gradient")


@pytest.mark.parametrize("n", [500, 40001])
def test_policy_loss_of_cancelling_terms(otf, n):
    """The mean of terms of both signs, clipped ones among them, that nearly cancel: it is exact to its own size."""
    lp, old, adv, _, _ = policy_inputs(n, None, False, n + 1)
    old[-1], lp[-1], adv[-1] = -1.0, -1.0, 0.0
    total = ref_policy(lp.double(), old, adv, None, None, 0.2, 0.28, 0.0)[0] * n
    adv[-1] = total  # its ratio is 1
    want, _, share = ref_policy(lp.double(), old, adv, None, None, 0.2, 0.28, 0.0)
    assert abs(want) < 1e-5 and share > 0.1
    loss = otf.losses.policy_loss(*[a.cuda() for a in (lp, old, adv)], clip_low=0.2, clip_high=0.28)[0]
    # the result's half step, and per term the few 2^-53 of its exponential
    close(loss.cpu(), want, U * want.abs() + 8 * 2.0 ** -53 * adv.abs().sum() / n * 1.28)


def test_policy_borders(otf):
    """At the border itself a ratio is not clipped; beyond it on the other side of the advantage neither."""
    one = torch.zeros(5, device="cuda")
    old = torch.log(torch.tensor([1.0, 2.0, 0.5, 0.5, 2.0], device="cuda", dtype=torch.float64)).float().neg()
    adv = torch.tensor([1.0, 1.0, -1.0, 1.0, -1.0], device="cuda")  # ratios 1, 2 (cut), 0.5 (cut), 0.5, 2
    leaf = one.clone().requires_grad_()
    loss, _, share = otf.losses.policy_loss(leaf, old, adv, clip_low=0.2, clip_high=0.2)
    grad, = torch.autograd.grad(loss, leaf)
    assert float(share) == pytest.approx(0.4)
    assert grad[1] == 0 and grad[2] == 0
    close(grad * 5, torch.tensor([-1.0, 0.0, 0.0, -0.5, 2.0], device="cuda"), 8 * U)
    close(loss.detach() * 5, torch.tensor(-1.0 - 1.2 + 0.8 - 0.5 + 2.0, device="cuda"), 16 * U)
    # no range at all: a ratio of exactly 1 still moves
    leaf = one.clone().requires_grad_()
    loss, _, share = otf.losses.policy_loss(leaf, one, adv, clip_low=0.0, clip_high=0.0)
    grad, = torch.autograd.grad(loss, leaf)
    assert float(share) == 0.0
    close(grad * 5, -adv, 4 * U)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,classes", [(1, 5), (40, 300), (6, 5003), (700, 2048), (1, 50257)])
def test_policy_loss_with_grad(otf, rows, classes, dtype):
    x, t = scores(rows, classes, dtype, rows + classes)
    if rows > 4:
        t[1] = -100
        t[2] = classes
    exact, valid = ref_log_probs(x, t)
    _, old, adv, ref, w = policy_inputs(rows, "bool", True, rows)
    w[0] = True
    if rows > 4:
        w[3] = False
    old, ref = (exact.cpu() + 0.15).float(), (exact.cpu() - 0.2).float()
    if rows > 4:
        x[3] = math.nan
    exact = exact.masked_fill(~w.cuda(), 0.0)
    z = exact.cpu().requires_grad_()
    loss, kl, share = ref_policy(z, old, adv, ref, w, 0.2, 0.28, 0.04)
    up = torch.autograd.grad(loss, z)[0].cuda()
    gl = torch.tensor(32.0, device="cuda")
    got = otf.losses.policy_loss_with_grad(x, t.to(torch.int32), old.cuda(), adv.cuda(), ref.cuda(), w.cuda(),
                                           clip_low=0.2, clip_high=0.28, kl_coef=0.04, grad_loss=gl)
    keep = w.cuda()
    counted = torch.where(keep[:, None], x, torch.zeros_like(x))
    _, rel_s, _ = parts(counted)
    lp_tol = float((rel_s[:, 0] + 2 * U * exact.abs() + U).max())
    slope = float(adv.abs().max()) * 1.5 + 0.1  # how fast a token's loss moves with its log-probability
    term_off, slope_off = policy_tol(exact.cpu(), old, adv, ref, w, 0.04)
    loss_off = slope * lp_tol + term_off + 2 * U * float(loss.detach().abs())
    kl_off = lp_tol + term_off / 0.04 + 2 * U * float(kl.detach().abs())
    for a, b, o in zip(got[:2], (loss, kl), (loss_off, kl_off)):
        close(a.cpu(), b.detach(), o)
    close(got[2].cpu(), share, 2 * U * share)
    want, tol = ref_log_probs_grad(counted, t, 32 * up * keep, x.dtype)
    p = parts(counted)[0]
    onehot = torch.zeros_like(p).scatter_(1, t.clamp(0, classes - 1)[:, None], 1.0)
    moved = (32 * (lp_tol * slope / max(1, int(w.sum())) + slope_off.cuda()) * (valid & keep))[:, None] * (p - onehot).abs()
    close(got[3], want, tol + moved, "gradient")
    # the same as its parts, one after the other
    leaf = counted.clone().requires_grad_()
    whole = otf.losses.policy_loss(otf.losses.token_log_probs(leaf, t), old.cuda(), adv.cuda(), ref.cuda(), w.cuda(),
                                   clip_low=0.2, clip_high=0.28, kl_coef=0.04)
    for a, b, o in zip(got[:3], whole, (2 * loss_off, 2 * kl_off, 0.0)):  # each is that near to the definition
        close(a, b.detach(), o + 4 * U * b.detach().abs())
    d, = torch.autograd.grad(whole[0], leaf, gl)
    close(got[3], d, 2 * (tol + moved), "gradient by parts")


# --------------------------------------------------- every way a row is shared

# 8 lanes a row, a warp, a CTA, a cluster; forward alone, gradient alone, both in one call; rows that start on a 16-byte
# border and rows that do not
MANY = [(30011, 37, "f32"), (30000, 64, "bf16"), (29000, 1500, "bf16"), (29000, 3001, "f16"), (15000, 5003, "bf16"),
        (15000, 9001, "f16"), (1200, 2100, "f32"), (700, 16000, "bf16"), (400, 30001, "f16"), (160, 60000, "bf16"),
        (151, 131075, "f32"), (9, 400000, "bf16"), (1, 700001, "f32")]


@pytest.mark.parametrize("rows,classes,dtype", MANY)
def test_many_rows(otf, rows, classes, dtype):
    x, t = scores(rows, classes, dtype, rows)
    t[::5] = -100
    g = torch.randn(rows, device="cuda")
    ids, y = teacher(x, min(9, classes), 3)
    w = torch.rand(rows, device="cuda") + 0.5
    if rows > 1:
        w[rows // 2] = 0.0
        x[rows // 2] = math.nan
        t[rows // 2] = -1
    leaf = x.clone().requires_grad_()
    lp = otf.losses.token_log_probs(leaf, t)
    lp_grad, = torch.autograd.grad(lp, leaf, g)
    scale = torch.tensor(float(rows), device="cuda")
    loss, grad = otf.losses.distillation_loss_with_grad(x, ids, y, weights=w, temperature=1.5, grad_loss=scale)
    two = otf.losses.distillation_loss(leaf, ids, y, weights=w, temperature=1.5)
    two_grad, = torch.autograd.grad(two, leaf, scale)
    adv = torch.randn(rows, device="cuda")
    old = lp.detach() + 0.1 * torch.randn(rows, device="cuda")
    pol = otf.losses.policy_loss_with_grad(x, t, old, adv, mask=w, grad_loss=scale)
    pol_grad, = torch.autograd.grad(otf.losses.policy_loss(otf.losses.token_log_probs(leaf, t), old, adv, mask=w)[0], leaf,
                                    scale)
    total, loss_sum, loss_off = float(w.double().sum()), 0.0, 0.0
    step = max(1, (1 << 25) // classes)
    for a in range(0, rows, step):
        r = slice(a, min(rows, a + step))
        want, valid = ref_log_probs(x[r], t[r])
        want = want.masked_fill(~valid, 0.0)
        _, rel_s, _ = parts(x[r].nan_to_num() if rows > 1 else x[r])
        close(lp.detach()[r], want, rel_s[:, 0] + 2 * U * want.abs() + U, "log-probabilities")
        want, tol = ref_log_probs_grad(x[r].nan_to_num(nan=0.0, neginf=-math.inf), t[r], g[r], x.dtype)
        close(lp_grad[r], want, tol, "their gradient")
        part = float(w[r].double().sum())
        if part == 0.0:
            assert not grad[r].any()
            continue
        l, d, l_off, tol = ref_distill(x[r].nan_to_num(nan=0.0, neginf=-math.inf), ids[r], y[r], w[r], 1.5, rows * part / total)
        loss_sum += float(l) * part / total
        loss_off += float(l_off) * part / total
        close(grad[r], d, tol, "gradient in one call")
        close(two_grad[r], d, tol, "gradient")
        # both forms of the policy loss are within their tolerance of the same value: the log-probability's error
        # times how fast the slope moves with it, and the gradient's own
        p = parts(x[r].nan_to_num(nan=0.0, neginf=-math.inf))[2]
        near = (w[r, None] * adv[r, None].abs() * 2 * rows / total).double()
        close(pol[3][r], pol_grad[r], 2 * near * (p + 8 * rel_s + 20 * U) + 2 * torch.finfo(x.dtype).eps * pol_grad[r].double().abs()
              + 2 * TINY[x.dtype], "policy gradient")
    for got in (loss, two.detach()):
        assert abs(float(got) - loss_sum) <= loss_off + 2 * U * abs(loss_sum)


def test_no_token_counts(otf):
    x, t = scores(40, 300, "f32", 1)
    none = torch.zeros(40, dtype=torch.bool, device="cuda")
    lp = torch.zeros(40, device="cuda")
    got = otf.losses.policy_loss_with_grad(x, t, lp, lp + 1, ref_log_probs=lp, mask=none, kl_coef=1.0)
    assert all(not o.any() for o in got)


REFUSED = {
    "token_log_probs": [(dict(logits=lambda a: a.double()), "logits must be float32"),
                        (dict(logits=lambda a: a[:, :0]), "at least one class"),
                        (dict(logits=lambda a: a.sum()), "classes"),
                        (dict(logits=lambda a: a.cpu()), "CUDA device"),
                        (dict(targets=lambda a: a.float()), "targets must be int32, int64"),
                        (dict(targets=lambda a: a[:3]), "targets must have shape"),
                        (dict(targets=lambda a: a.cpu()), "CUDA device")],
    "distillation_loss": [(dict(teacher_ids=lambda a: a[:3]), "teacher_ids must be"),
                          (dict(teacher_ids=lambda a: a.float()), "teacher_ids must be int32, int64"),
                          (dict(teacher_logits=lambda a: a[:, :2]), "teacher_logits must have shape"),
                          (dict(teacher_logits=lambda a: a.double()), "teacher_logits must be float32"),
                          (dict(teacher_ids=lambda a: a[:, :0], teacher_logits=lambda a: a[:, :0]), "entries"),
                          (dict(teacher_ids=lambda a: a.repeat(1, 342), teacher_logits=lambda a: a.repeat(1, 342)),
                           "entries"),
                          (dict(weights=lambda a: torch.ones(3, device="cuda")), "weights must have shape"),
                          (dict(weights=lambda a: torch.ones(4, device="cuda").long()), "weights must be float32, bool"),
                          (dict(temperature=lambda a: 0.0), "temperature"),
                          (dict(temperature=lambda a: math.nan), "temperature"),
                          (dict(logits=lambda a: a[:0], teacher_ids=lambda a: a[:0], teacher_logits=lambda a: a[:0]),
                           "no rows")],
    "distillation_loss_with_grad": [(dict(grad_loss=lambda a: torch.ones(2, device="cuda")), "grad_loss must be"),
                                    (dict(grad_loss=lambda a: 2.0), "grad_loss must be")],
    "preference_loss": [(dict(log_probs=lambda a: a.half()), "log_probs must be float32"),
                        (dict(offsets=lambda a: a[:4]), "offsets"), (dict(offsets=lambda a: a[:1]), "offsets"),
                        (dict(offsets=lambda a: a[None]), "offsets"), (dict(offsets=lambda a: a.float()), "offsets"),
                        (dict(ref_log_probs=lambda a: torch.ones(5, device="cuda")), "ref_log_probs must have shape"),
                        (dict(mask=lambda a: torch.ones(4)), "CUDA device"),
                        (dict(beta=lambda a: math.inf), "beta"),
                        (dict(label_smoothing=lambda a: 0.6), "label_smoothing")],
    "policy_loss": [(dict(old_log_probs=lambda a: a[:2]), "old_log_probs must have shape"),
                    (dict(advantages=lambda a: a.half()), "advantages must be float32"),
                    (dict(clip_low=lambda a: -0.1), "clip"), (dict(clip_high=lambda a: math.nan), "clip"),
                    (dict(kl_coef=lambda a: math.inf), "kl_coef")],
    "policy_loss_with_grad": [(dict(targets=lambda a: a[:, None]), "targets must have shape"),
                              (dict(grad_loss=lambda a: torch.ones((), device="cuda").half()), "grad_loss must be")],
}


@pytest.mark.parametrize("name,change,words", [(n, *c) for n, l in REFUSED.items() for c in l])
def test_refusals(otf, name, change, words):
    """Wrong types, shapes and values are refused before anything runs."""
    from opencl_tf import errors
    x, t, lp = torch.zeros(4, 10, device="cuda"), torch.zeros(4, device="cuda").long(), torch.zeros(4, device="cuda")
    calls = {
        "token_log_probs": dict(logits=x, targets=t),
        "distillation_loss": dict(logits=x, teacher_ids=t[:, None].repeat(1, 3), teacher_logits=x[:, :3]),
        "preference_loss": dict(log_probs=lp, offsets=torch.arange(5, device="cuda")),
        "policy_loss": dict(log_probs=lp, old_log_probs=lp, advantages=lp),
        "policy_loss_with_grad": dict(logits=x, targets=t, old_log_probs=lp, advantages=lp),
    }
    args = dict(calls.get(name, calls["distillation_loss"]))
    getattr(otf.losses, name)(**args)
    for k, f in change.items():
        args[k] = f(args.get(k))
    with pytest.raises(errors.InvalidArgumentError, match=words):
        getattr(otf.losses, name)(**args)


# ---------------------------------------------------------------- together

def test_gradients_against_differences(otf):
    """Central differences of the definitions in 64 bits: step 1e-5, so their own error is about 1e-10."""
    x, t = scores(4, 37, "f32", 8, dead=False)
    ids, y = teacher(x, 6, 9)
    w = torch.tensor([1.0, 0.5, 0.0, 2.0], device="cuda")
    off = torch.tensor([0, 1, 2, 3, 4], device="cuda")
    old, adv = torch.randn(4, device="cuda") * 0.1 - 2, torch.randn(4, device="cuda")
    lp = ref_log_probs(x, t)[0]
    old = (lp + 0.05 * old).float()
    ref = (lp + 0.3).float()

    def distill(z):
        return ref_distill(z, ids, y, w, 1.5)[0]

    def preference(z):
        return ref_preference(ref_log_probs(z, t)[0].cpu(), off.cpu(), ref.cpu(), None, 0.7, 0.1)[0]

    def policy(z):
        return ref_policy(ref_log_probs(z, t)[0].cpu(), old.cpu(), adv.cpu(), ref.cpu(), None, 0.2, 0.2, 0.1)[0]

    leaf = x.clone().requires_grad_()
    kernels = {
        distill: otf.losses.distillation_loss(leaf, ids, y, weights=w, temperature=1.5),
        preference: otf.losses.preference_loss(otf.losses.token_log_probs(leaf, t), off, ref, beta=0.7,
                                               label_smoothing=0.1)[0],
        policy: otf.losses.policy_loss(otf.losses.token_log_probs(leaf, t), old, adv, ref, kl_coef=0.1)[0],
    }
    for formula, loss in kernels.items():
        grad, = torch.autograd.grad(loss, leaf)
        for seed in range(3):
            v = torch.randn(x.shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").double()
            h = 1e-5
            slope = (float(formula(x.double() + h * v)) - float(formula(x.double() - h * v))) / (2 * h)
            mine = float((grad.double() * v).sum())
            # every gradient value is off by at most 300u of the largest
            assert abs(mine - slope) <= 1e-8 + 300 * U * float((grad.abs().max() * v.abs()).sum()), formula


def test_preference_step_in_a_graph(otf):
    """scores -> log-probabilities -> preference loss -> gradient, captured and replayed on new inputs, as the
    eager calls on them; two graphs do not share their workspaces."""
    off = torch.tensor([0, 3, 9, 14, 20], device="cuda")

    def inputs(seed):
        x, t = scores(21, 5001, "bf16", seed)
        t[::4] = -100
        return x, t, -3 * torch.rand(21, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))

    def step(x, t, ref):
        leaf = x.detach().requires_grad_()
        lp = otf.losses.token_log_probs(leaf, t)
        loss, c, r = otf.losses.preference_loss(lp, off, ref, mask=t >= 0)
        ids = t.clamp(min=0)[:, None].expand(-1, 3).contiguous()
        both, dx = otf.losses.distillation_loss_with_grad(x, ids, torch.ones(21, 3, device="cuda"), weights=t >= 0)
        pl = otf.losses.policy_loss(lp, ref, ref, ref, kl_coef=0.1)
        fused = otf.losses.policy_loss_with_grad(x, t, ref, ref, ref, mask=t >= 0, kl_coef=0.1)
        return loss, c, r, both, dx, *fused, *torch.autograd.grad(loss + pl[0], leaf)

    eager = [[o.clone() for o in step(*inputs(s))] for s in (1, 2, 3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    statics, graphs, outs = [], [], []
    with torch.cuda.stream(side):
        for s in (1, 2):
            st = [a.clone() for a in inputs(s)]
            step(*st)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(step(*st))
            statics.append(st)
            graphs.append(graph)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    for _ in range(3):  # both at once, on two streams
        graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
    torch.cuda.synchronize()
    for k in (0, 1):
        for a, b in zip(outs[k], eager[k]):
            assert torch.equal(a, b)
    for a, b in zip(statics[0], inputs(3)):
        a.copy_(b)
    graphs[0].replay()
    torch.cuda.synchronize()
    for a, b in zip(outs[0], eager[2]):
        assert torch.equal(a, b)


def test_calls_on_two_streams_and_twice(otf):
    """The same calls at once on two streams, and again: the same bits."""
    x, t = scores(200, 6007, "f16", 5)
    ids, y = teacher(x, 40, 6)
    w = torch.rand(200, device="cuda")
    want = otf.losses.distillation_loss_with_grad(x, ids, y, weights=w, temperature=1.5)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(otf.losses.distillation_loss_with_grad(x, ids, y, weights=w, temperature=1.5))
    torch.cuda.synchronize()
    for loss, grad in got:
        assert torch.equal(loss, want[0]) and torch.equal(grad, want[1])


def test_gradient_is_once_differentiable_and_sums_over_uses(otf):
    x, t = scores(3, 50, "f32", 2)
    leaf = x.clone().requires_grad_()
    lp = otf.losses.token_log_probs(leaf, t)
    a, = torch.autograd.grad(lp.sum(), leaf, retain_graph=True)
    b, = torch.autograd.grad((lp * 2).sum() + lp.sum(), leaf, retain_graph=True)
    assert torch.allclose(b, 3 * a, rtol=8 * U, atol=1e-30)
    g, = torch.autograd.grad(lp.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), leaf)
    rewards = otf.losses.preference_loss(otf.losses.token_log_probs(leaf, t), torch.tensor([0, 1, 2], device="cuda"))[1]
    assert not rewards.requires_grad


def test_dense_head_distilled(otf):
    """A Dense layer's scores distilled from another's top answers: the layer's own gradient, from the definition."""
    torch.manual_seed(0)
    x = torch.randn(24, 40, device="cuda")
    w = (0.3 * torch.randn(40, 90, device="cuda")).requires_grad_()
    b = torch.zeros(90, device="cuda", requires_grad=True)
    top = torch.randn(24, 90, device="cuda").topk(7, 1)
    loss = otf.losses.distillation_loss(otf.dense(x, w, b), top.indices, top.values, temperature=2.0)
    loss.backward()
    w64, b64 = w.detach().double().requires_grad_(), b.detach().double().requires_grad_()
    ref = ref_distill(x.double() @ w64 + b64, top.indices, top.values, None, 2.0)[0]
    ref.backward()
    # the product's fp32-tolerance (5e-6 of the largest score here) moves every softmax value by that much
    assert abs(float(loss) - float(ref)) <= 1e-5 * abs(float(ref))
    for got, want in ((w.grad, w64.grad), (b.grad, b64.grad)):
        assert float((got - want).norm() / want.norm()) <= 2e-5


class _Classifier(torch.nn.Module):
    def __init__(self):
        super().__init__()
        from opencl_tf.layers import OpenCLDense
        self.hidden, self.out = OpenCLDense(48), OpenCLDense(1021)
        self.hidden.build((1, 30))
        self.out.build((1, 48))

    def forward(self, x, training=None):
        return self.out(self.hidden.forward_relu(x))


@pytest.mark.parametrize("kind", ["distillation", "likelihood"])
def test_train_step_with_a_loss(otf, kind):
    """TrainStep on one of the losses: captured in a graph it does what it does eagerly, bit for bit, over steps with
    new inputs; and the first step's gradients are the definition's."""
    from opencl_tf.train import TrainStep

    def batch(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x = torch.randn(64, 30, generator=g, device="cuda")
        if kind == "likelihood":
            return x, torch.randint(0, 1021, (64,), generator=g, device="cuda")
        top = torch.randn(64, 1021, generator=g, device="cuda").topk(8, 1)
        return x, (top.indices, top.values)

    def loss(output, y):
        if kind == "likelihood":
            return -otf.losses.token_log_probs(output, y).mean()
        return otf.losses.distillation_loss(output, *y, temperature=2.0)

    def run(graphed):
        torch.manual_seed(3)
        model = _Classifier().cuda()
        first = [p.detach().clone() for p in model.parameters()]
        step = TrainStep(model, graphed=graphed, warmup=1, loss=loss)
        if graphed:  # the capture's warm-up takes steps of its own: back to the start
            step(*batch(0))
            with torch.no_grad():
                for p, f in zip(model.parameters(), first):
                    p.copy_(f)
                for o in step.opts:
                    o.iterations.zero_()
                    for slot in (*o.m, *o.v):
                        slot.zero_()
        losses = [step(*batch(s)).clone() for s in (1, 2, 3)]
        return losses, [p.detach().clone() for p in model.parameters()]

    a, b = run(True), run(False)
    for x, y in zip((*a[0], *a[1]), (*b[0], *b[1])):
        assert torch.equal(x, y)
    torch.manual_seed(3)
    model = _Classifier().cuda()
    x, y = batch(1)
    loss(model(x), y).backward()
    params = [p.detach().double().requires_grad_() for p in model.parameters()]
    h = torch.relu(x.double() @ params[0] + params[1]) @ params[2] + params[3]
    if kind == "likelihood":
        ref = -torch.log_softmax(h, 1).gather(1, y[:, None]).mean()
    else:
        ref = ref_distill(h, *y, None, 2.0)[0]
    for got, want in zip(model.parameters(), torch.autograd.grad(ref, params)):
        # the products' fp32 tolerance, 5e-6 of the largest value each way
        assert float((got.grad - want).norm() / want.norm()) <= 2e-5


def test_errors_of_a_backward_pass(otf):
    """What fails in the backward pass, on autograd's own thread, is raised where the gradient was asked for: scores
    changed since the forward pass, and a wait of another op that ran out (a matrix product given 1 ns; it gives up)."""
    from opencl_tf import errors, raw_ops
    x = torch.randn(40, 5000, device="cuda", requires_grad=True)
    t = torch.randint(0, 5000, (40,), device="cuda")
    y = x * 1
    lp = otf.losses.token_log_probs(y, t).sum()
    y.detach().add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(lp, x)

    lp = otf.losses.token_log_probs(x, t).sum()
    want, = torch.autograd.grad(lp, x, retain_graph=True)
    a, w, b = torch.randn(512, 4096, device="cuda"), torch.randn(4096, 96, device="cuda"), torch.zeros(96, device="cuda")
    before = otf.device_timeouts()
    try:
        otf.set_wait_limit_ns(1)
        for _ in range(5):
            try:
                raw_ops.opencl_dense(a, w, b)
            except errors.DeadlineExceededError:
                pass
            torch.cuda.synchronize()
            if otf.device_timeouts() > before:
                break
    finally:
        otf.set_wait_limit_ns(0)
    with pytest.raises(errors.DeadlineExceededError):
        torch.autograd.grad(lp, x, retain_graph=True)
    with pytest.raises(errors.DeadlineExceededError):
        otf.losses.token_log_probs(x, t)
    with pytest.raises(errors.DeadlineExceededError):
        otf.stream_status()
    again, = torch.autograd.grad(lp, x)
    assert torch.equal(again, want)


def test_calls_of_two_threads(otf):
    """Losses and gradients of two threads, each on a stream of its own, and a backward pass on the calling thread."""
    import threading
    inputs = [scores(60, 7001 + 100 * i, "bf16", i, dead=False) for i in range(2)]
    old, adv = torch.zeros(60, device="cuda") - 9, torch.randn(60, device="cuda")

    def step(x, t):
        leaf = x.clone().requires_grad_()
        loss = otf.losses.policy_loss(otf.losses.token_log_probs(leaf, t), old, adv)[0]
        return loss.detach(), *torch.autograd.grad(loss, leaf)

    want = [step(*a) for a in inputs]
    torch.cuda.synchronize()
    got, failed = [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    got[i].append(step(*inputs[i]))
            torch.cuda.synchronize()
        except BaseException as e:
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failed, failed
    with torch.autograd.set_multithreading_enabled(False):
        got[0].append(step(*inputs[0]))
    for w, g in zip(want, got):
        assert len(g) >= 30 and all(torch.equal(a, b) for one in g for a, b in zip(w, one))

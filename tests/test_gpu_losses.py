"""Token log-probabilities, the policy loss and the preference loss against
plain 64-bit implementations.

Tolerances. The kernels form each term 2^t, t = (l - M) * log2(e) / T, in fp32:
the subtraction, the rounded factor and the product are off by at most 2^-24
each relative to t, ex2.approx by 2^-22 relative. A log-sum of such terms is off
by the terms' mean error, (4 + 3 E|t|) 2^-24 with E|t| <= log2 V + 4 < 24, by at
most 2 + V / (256 * 4) additions within a thread (V <= 2^18 here on one CTA:
under 260 steps of half a unit, 2^-24 each) and by two rebasings (4 each): under
350 * 2^-24 = 2.1e-5 at the worst and a twentieth of that as errors of random
sign; the target's own t adds 3 |t| 2^-24 and the output's rounding |lp| 2^-24.
The bounds below are the worst case. A probability inherits the log-sum's error
and its own t's: (350 + 4 + 3 |t|) 2^-24 relative."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def q():
    import quasar_b200
    return quasar_b200


def rows_of(rows, V, dtype, seed, pad=0, offset=0, scale=3.0):
    """[rows, V] logits in a storage with `pad` columns behind and `offset` elements before."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    flat = torch.randn(offset + rows * (V + pad), generator=g, device="cuda").mul_(scale).to(dtype)
    logits = flat[offset:].as_strided((rows, V), (V + pad, 1), offset)
    targets = torch.randint(0, V, (rows,), generator=g, device="cuda", dtype=torch.int32)
    return logits, targets, g


def softmax64(logits, T):
    """(ln p, p, t) in 64 bits; a row without a finite logit has p = 0."""
    z = logits.double() / T
    m = z.amax(1, keepdim=True)
    m0 = torch.where(torch.isinf(m) & (m < 0), torch.zeros_like(m), m)
    e = (z - m0).exp()
    lnp = z - m0 - e.sum(1, keepdim=True).log()
    empty = (m == -math.inf).expand_as(z)
    lnp = torch.where(empty, torch.full_like(z, -math.inf), lnp)
    return lnp, lnp.exp(), (z - m0) / math.log(2)


def reference(logits, targets, T):
    lnp, p, t = softmax64(logits, T)
    on = targets >= 0
    lp = lnp.gather(1, targets.clamp(min=0).long()[:, None])[:, 0]
    h = -torch.where(p > 0, p * lnp, torch.zeros_like(p)).sum(1)
    zero = torch.zeros_like(lp)
    return torch.where(on, lp, zero), torch.where(on, h, zero)


def reference_grad(logits, targets, T, c, gh=None):
    """The gradient in 64 bits and a bound on the kernel's error: relative errors of p (2e-5 + 3 |t| eps),
    of the coefficients (rounded to fp32: 4 eps) and half a step of the output type."""
    lnp, p, t = softmax64(logits, T)
    on = (targets >= 0)[:, None]
    c = c.double()[:, None]
    hot = torch.zeros_like(p)
    hot.scatter_(1, targets.clamp(min=0).long()[:, None], 1.0)
    alive = (logits.double().amax(1, keepdim=True) > -math.inf)
    lnp0 = torch.where(p > 0, lnp, torch.zeros_like(lnp))
    h = -(p * lnp0).sum(1, keepdim=True)
    g = torch.zeros_like(c) if gh is None else gh.double()[:, None]
    d = (c * (hot - p) - g * p * (lnp0 + h)) / T
    big = (c.abs() * p + g.abs() * p * (lnp0.abs() + h + 24 * math.log(2))) / T
    rel = 2e-5 + 3 * t.abs().clamp(max=200) * EPS
    fi = torch.finfo(logits.dtype)
    # below the smallest normal number: half a step of the type's, or flushed to zero by an fp32 product
    bound = big * rel + (c.abs() * hot / T) * 4 * EPS + d.abs() * (fi.eps / 2 + 2 * EPS) + fi.tiny * (fi.eps / 2 if logits.dtype != torch.float32 else 1)
    keep = on & alive
    return torch.where(keep, d, torch.zeros_like(d)), torch.where(keep, bound, torch.zeros_like(bound))


def close(x, ref, atol, what=""):
    """Equal where ref is not finite, else within atol (a number or a tensor) and half a step of fp32."""
    x, ref = x.double(), ref.double()
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isnan(x), torch.isnan(ref)), f"{what}: NaN in other places"
    inf = torch.isinf(ref)
    assert torch.equal(x[inf], ref[inf]), f"{what}: infinities"
    err = (x - ref)[fin].abs()
    lim = atol[fin] if isinstance(atol, torch.Tensor) else atol + 0 * err
    lim = lim + ref[fin].abs() * EPS
    worst = (err - lim).max().item() if err.numel() else -1.0
    assert worst <= 0, f"{what}: off by {err.max().item():.3g}, {worst:.3g} over the bound"


LP_ATOL = 2.1e-5 + 3 * 60 * EPS          # |t| of a target up to 60
H_ATOL = 2.1e-5 + 24 * 2.1e-5            # the mean of t (< 24) with the terms' relative error


SHAPES = [  # rows, V, pad, offset
    (1, 1, 0, 0), (2, 2, 0, 0), (3, 5, 1, 1), (5, 31, 0, 3), (4, 260, 4, 0), (7, 1023, 0, 0), (3, 4096, 0, 0),
    (6, 4099, 9, 5), (33, 18992, 0, 0), (2, 50021, 0, 1), (3, 151936, 0, 0), (2, 151936, 7, 0), (300, 777, 0, 0),
    (1, 262144, 0, 0),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_logprobs(dtype, shape):
    rows, V, pad, offset = shape
    for T in (1.0, 0.6):
        logits, targets, g = rows_of(rows, V, dtype, 11, pad, offset)
        if rows > 2:
            targets[1] = -1
        lp, h = reference(logits, targets, T)
        for entropy in (False, True):
            out = q().token_logprobs(logits, targets, temperature=T, entropy=entropy)
            close(out.logprob, lp, LP_ATOL, "logprob")
            assert (out.entropy is not None) == entropy
            if entropy:
                close(out.entropy, h, H_ATOL, "entropy")
        on = targets >= 0
        assert torch.equal(out.stats[on, 0], logits.float().amax(1)[on])
        s = ((logits.double() - logits.double().amax(1, keepdim=True)) / T).exp().sum(1)
        close(out.stats[on, 1] / s[on], torch.ones_like(s[on]), 2.1e-5, "sum")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_logprobs_gradient(dtype, shape):
    rows, V, pad, offset = shape
    T = 0.8
    logits, targets, g = rows_of(rows, V, dtype, 12, pad, offset)
    if rows > 2:
        targets[0] = -1
    c, gh = torch.randn(rows, generator=g, device="cuda"), torch.randn(rows, generator=g, device="cuda")
    fwd = q().token_logprobs(logits, targets, temperature=T, entropy=True)
    for with_h in (False, True):
        kw = dict(entropy=fwd.entropy, grad_entropy=gh) if with_h else {}
        ref, bound = reference_grad(logits, targets, T, c, gh if with_h else None)
        out = q().token_logprobs_grad(logits, targets, fwd.stats, c, temperature=T, **kw)
        close(out, ref, bound, "grad")
        # into a buffer of another alignment, columns behind it untouched
        store = torch.full((rows, V + 3), 7.0, dtype=dtype, device="cuda")
        into = store[:, 1:V + 1]
        q().token_logprobs_grad(logits, targets, fwd.stats, c, temperature=T, out=into, **kw)
        assert torch.equal(into, out)
        assert (store[:, 0] == 7).all() and (store[:, V + 1:] == 7).all()
        # in place
        again = torch.empty(0, dtype=dtype, device="cuda").set_(logits.untyped_storage().clone(), offset, (rows, V), (V + pad, 1))
        q().token_logprobs_grad(again, targets, fwd.stats, c, temperature=T, out=again, **kw)
        assert torch.equal(again, out)


@pytest.mark.parametrize("dtype", DTYPES)
def test_logprobs_are_not_biased(dtype):
    """The mean error over many rows, which a loss that averages rows of either sign sees: that of ex2.approx on the
    terms (5e-8 low on average, so at most 5e-8 high in the log-probability), once and not with every join of sums,
    and four standard errors of the rows' own."""
    rows, V = 4000, 4099
    logits, _, g = rows_of(rows, V, dtype, 18)
    targets = (logits.float() - torch.empty(rows, V, device="cuda").exponential_(generator=g).log()).argmax(1).to(torch.int32)
    lp, _ = reference(logits, targets, 1.0)
    err = q().token_logprobs(logits, targets).logprob.double() - lp
    assert err.mean().abs().item() <= 5e-8 + 4 * err.std().item() / math.sqrt(rows)


def test_gradient_against_differences():
    """Central differences of the kernel's own forward pass: error h^2/6 |f'''| (f''' <= 2 |g| for the
    log-probability, and under 8 for the entropies of these rows) plus the forward's 2.1e-5 / h; in fact the
    forward of 40 columns is good to 1e-6, of which a difference takes 1e-6 / h."""
    rows, V, T, h = 3, 40, 1.0, 0.03
    logits, targets, g = rows_of(rows, V, torch.float32, 13, scale=1.0)
    c, gh = torch.randn(rows, generator=g, device="cuda"), torch.randn(rows, generator=g, device="cuda")
    fwd = q().token_logprobs(logits, targets, entropy=True)
    grad = q().token_logprobs_grad(logits, targets, fwd.stats, c, entropy=fwd.entropy, grad_entropy=gh)
    up, down = (logits.repeat_interleave(V, 0) + s * h * torch.eye(V, device="cuda").repeat(rows, 1) for s in (1, -1))
    t = targets.repeat_interleave(V).contiguous()
    a, b = (q().token_logprobs(x.contiguous(), t, entropy=True) for x in (up, down))
    num = ((a.logprob - b.logprob).double().view(rows, V) * c[:, None] + (a.entropy - b.entropy).double().view(rows, V) * gh[:, None]) / (2 * h)
    tol = h * h / 6 * (2 * c.abs().max() + 8 * gh.abs().max()).item() + 2e-6 / h * 3
    assert (num - grad.double()).abs().max().item() < tol


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [9, 4099, 151936])
def test_rows_of_masks(dtype, V):
    """-inf, the type's lowest value, NaN and infinities, in rows that take part and in rows that do not."""
    rows = 12
    low = torch.finfo(dtype).min
    logits, targets, g = rows_of(rows, V, dtype, 14)
    targets[:] = V - 1
    logits[0] = -math.inf                     # no distribution at all
    logits[1] = low                           # masked by the lowest value throughout: uniform
    logits[2] = -math.inf
    logits[2, V - 1] = 2.0                    # one token left: probability 1
    logits[3, V - 1] = -math.inf              # the target itself is banned
    logits[4, :V - 1] = low                   # one token above the lowest value
    logits[5] = math.nan
    targets[5] = -1                           # a row that takes no part may hold anything
    logits[6, 0] = math.nan
    logits[7, 0] = math.inf
    targets[8] = V                            # behind the vocabulary
    logits[9, ::2] = -math.inf
    logits[9, V - 1] = 0.5
    logits[10] = 0.0                          # all equal
    logits[11] = torch.finfo(dtype).max       # all at the largest value
    out = q().token_logprobs(logits, targets, entropy=True)
    lp, h = out.logprob.double().cpu(), out.entropy.double().cpu()
    assert lp[0] == -math.inf and h[0] == 0
    for r in (1, 10, 11):
        assert abs(lp[r] + math.log(V)) < LP_ATOL and abs(h[r] - math.log(V)) < H_ATOL
    assert -LP_ATOL < lp[2] <= 0 and 0 <= h[2] < H_ATOL
    assert lp[3] == -math.inf and torch.isfinite(h[3])
    assert abs(lp[4]) < LP_ATOL and abs(h[4]) < H_ATOL
    assert lp[5] == 0 and h[5] == 0
    for r in (6, 7, 8):
        assert torch.isnan(lp[r]) and torch.isnan(h[r])
    ref, _ = reference(logits[9:10], targets[9:10], 1.0)
    close(out.logprob[9:10], ref, LP_ATOL)

    c, gh = torch.ones(rows, device="cuda"), torch.full((rows,), 0.5, device="cuda")
    grad = q().token_logprobs_grad(logits, targets, out.stats, c, entropy=out.entropy, grad_entropy=gh)
    fine = [1, 2, 3, 4, 9, 10, 11]
    ref, bound = reference_grad(logits[fine], targets[fine], 1.0, c[fine], gh[fine])
    if V > 9:
        ref_lo = logits[fine] == low  # (l - M) overflows to -inf there: p = 0 either way
        ref[ref_lo & (ref.abs() < 1e-300)] = 0
    close(grad[fine], ref, bound + 1e-30, "grad")
    assert (grad[0] == 0).all() and (grad[5] == 0).all()
    for r in (6, 7, 8):
        assert torch.isnan(grad[r]).all()

    one = torch.ones(rows, device="cuda")
    pol = q().policy_loss(logits, targets, torch.full((rows,), -2.0, device="cuda"), one, entropy_coef=0.1)
    assert torch.equal(torch.isnan(pol.row_loss).cpu(), torch.tensor([r in (6, 7, 8) for r in range(rows)]))
    assert (pol.grad[0] == 0).all() and (pol.grad[5] == 0).all()
    for r in (6, 7, 8):
        assert torch.isnan(pol.grad[r]).all()
    assert torch.isnan(pol.loss)
    w = one.clone()
    w[6:9] = 0                                # left out, whatever they hold
    pol = q().policy_loss(logits, targets, torch.full((rows,), -2.0, device="cuda"), one, weight=w, entropy_coef=0.1)
    assert torch.isfinite(pol.loss) and torch.isfinite(pol.grad.float()).all()
    assert (pol.grad[6:9] == 0).all() and (pol.logprob[6:9] == 0).all() and (pol.row_loss[6:9] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1000, 40001])
def test_rows_of_large_values(dtype, V):
    """Masks of every size (-1e4 to -1e30) over parts of a row, over all of it, and large positive rows: the same
    probabilities as with the row's maximum taken off first. t is formed from l - M, rounded like l itself."""
    fills = [-1e4, -1e7, -1e9, -1e12, -1e20, -1e30, 1e6, 1e9, 1e20, 1e30]
    rows = 4 * len(fills)
    logits, targets, g = rows_of(rows, V, dtype, 19)
    keep = torch.rand(V, generator=g, device="cuda") < 0.5
    for i, f in enumerate(fills):
        logits[4 * i] = f                                                      # the whole row
        logits[4 * i + 1] = torch.where(keep, logits[4 * i + 1], torch.full_like(logits[0], f))  # half of it
        logits[4 * i + 2, :V - 3] = f                                          # all but three
        logits[4 * i + 3, V // 2] = f                                          # one
        targets[4 * i + 1] = int(keep.nonzero()[7])
        targets[4 * i + 2] = V - 2
    lp, h = reference(logits, targets, 1.0)
    out = q().token_logprobs(logits, targets, entropy=True)
    close(out.logprob, lp, LP_ATOL + lp.abs() * 4 * EPS, "logprob")
    close(out.entropy, h, H_ATOL, "entropy")
    c, gh = torch.randn(rows, generator=g, device="cuda"), torch.randn(rows, generator=g, device="cuda")
    ref, bound = reference_grad(logits, targets, 1.0, c, gh)
    close(q().token_logprobs_grad(logits, targets, out.stats, c, entropy=out.entropy, grad_entropy=gh), ref, bound + 1e-30, "grad")
    few = q().policy_loss(logits, targets, torch.full((rows,), -3.0, device="cuda"), c, entropy_coef=0.1)
    many = [t.repeat(8, *[1] * (t.dim() - 1)) for t in (logits, targets, c)]   # 320 rows: the kernels of many rows
    out = q().policy_loss(many[0], many[1], torch.full((8 * rows,), -3.0, device="cuda"), many[2], entropy_coef=0.1,
                          weight=torch.full((8 * rows,), 1.0 / rows, device="cuda"))
    fi = torch.finfo(dtype)
    for j in range(0, 8 * rows, rows):
        close(out.logprob[j:j + rows], few.logprob, 2 * LP_ATOL + lp.abs() * 8 * EPS)
        close(out.grad[j:j + rows], few.grad, few.grad.double().abs() * (2 * fi.eps + 2e-4) + 1e-8)


def policy64(lp, h, old, adv, ref, lo, hi, kl, ec):
    r = (lp - old.double()).exp()
    loss = -torch.minimum(r * adv.double(), r.clamp(1 - lo, 1 + hi) * adv.double())
    if kl:
        u = ref.double() - lp
        loss = loss + kl * (u.exp() - u - 1)
    return loss - ec * h


POLICY = [  # rows, V, pad, offset, T, clip_low, clip_high, kl, entropy_coef, weighted
    (1, 1, 0, 0, 1.0, 0.2, 0.2, 0.0, 0.0, False), (5, 31, 0, 3, 1.0, 0.2, 0.28, 0.05, 0.0, True),
    (64, 260, 0, 0, 0.7, 0.1, 0.3, 0.0, 0.02, True), (9, 4099, 5, 1, 1.0, 0.2, 0.2, 0.1, 0.01, True),
    (40, 18992, 0, 0, 1.0, 0.0, 0.0, 0.05, 0.0, False), (3, 50021, 0, 0, 1.3, 0.2, 0.2, 0.05, 0.01, True),
    (4, 151936, 0, 0, 1.0, 0.2, 0.28, 0.05, 0.01, True), (700, 4096, 0, 0, 1.0, 0.2, 0.2, 0.0, 0.0, False),
    # many long rows: the streaming kernel, for rows of 100 to 200 KB and longer ones
    (600, 30001, 0, 3, 0.9, 0.2, 0.2, 0.05, 0.01, True), (150, 75000, 4, 0, 1.0, 0.2, 0.2, 0.0, 0.0, False),
    (149, 151936, 0, 0, 1.0, 0.2, 0.28, 0.05, 0.0, True),
]


def policy_inputs(rows, V, pad, offset, T, lo, hi, dtype, seed, weighted):
    logits, targets, g = rows_of(rows, V, dtype, seed, pad, offset)
    lp, h = reference(logits, targets, T)
    d = torch.randn(rows, generator=g, device="cuda").double() * 0.3
    for b in (1 - lo, 1 + hi):  # not at a border, where rounding decides
        d = torch.where((d - math.log(b)).abs() < 1e-3, math.log(b) + 2e-3, d)
    old = (lp - d).float()
    adv = torch.randn(rows, generator=g, device="cuda")
    ref = (lp + 0.3 * torch.randn(rows, generator=g, device="cuda").double()).float()
    w = None
    if weighted:
        w = torch.rand(rows, generator=g, device="cuda")
        w[rows // 2] = 0
        targets[0] = -1
    return logits, targets, old, adv, ref, w


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", POLICY, ids=str)
def test_policy_loss(dtype, case):
    rows, V, pad, offset, T, lo, hi, kl, ec, weighted = case
    logits, targets, old, adv, ref, w = policy_inputs(rows, V, pad, offset, T, lo, hi, dtype, 21, weighted)
    kw = dict(ref_logprob=ref if kl else None, weight=w, temperature=T, clip_low=lo, clip_high=hi, kl_coef=kl,
              entropy_coef=ec, grad_scale=64.0)
    out = q().policy_loss(logits, targets, old, adv, **kw)
    live = targets >= 0
    wd = torch.full((rows,), 1.0 / rows, device="cuda", dtype=torch.float64) if w is None else w.double()
    live &= wd != 0
    lp, h = reference(logits, targets, T)
    zero = torch.zeros_like(lp)
    lp, h = torch.where(live, lp, zero), torch.where(live, h, zero)
    x = lp.clone().requires_grad_(True)
    row = torch.where(live, policy64(x, h, old, adv, ref, lo, hi, kl, ec), zero)
    loss = (wd * row).sum()
    c, = torch.autograd.grad(loss, x)
    row, loss = row.detach(), loss.detach()
    # ratio and exp(u) carry the log-probability's error
    slope = (lp - old.double()).exp() * adv.double().abs() + kl * ((ref.double() - lp).exp() + 1) + 1e-30
    tol = torch.where(live, slope * LP_ATOL * 1.1 + ec * H_ATOL, zero)
    close(out.logprob, lp, LP_ATOL, "logprob")
    close(out.row_loss, row, tol, "row_loss")
    close(out.loss, loss, (wd * tol).sum().item() + (wd * row.abs()).sum().item() * EPS, "loss")
    gh = -ec * wd * 64 if ec else None
    if ec:
        close(out.entropy, h, H_ATOL, "entropy")
    else:
        assert out.entropy is None
    gref, bound = reference_grad(logits, torch.where(live, targets, -torch.ones_like(targets)), T, c * 64, gh)
    _, p, _ = softmax64(logits, T)
    hot = torch.zeros_like(p).scatter_(1, targets.clamp(min=0).long()[:, None], 1.0)
    dc = torch.where(live, wd * 64 * slope * LP_ATOL * 1.1, zero)[:, None] * (hot + p) / T  # the coefficient's own error
    close(out.grad, gref, bound + dc, "grad")
    # without the gradient; in place: the same gradient
    none = q().policy_loss(logits, targets, old, adv, grad=False, **kw)
    assert none.grad is None  # many long rows take another kernel then, with another order of sums: the same bounds
    close(none.row_loss, row, tol, "row_loss without gradient")
    close(none.loss, loss, (wd * tol).sum().item() + (wd * row.abs()).sum().item() * EPS, "loss without gradient")
    again = torch.empty(0, dtype=dtype, device="cuda").set_(logits.untyped_storage().clone(), offset, (rows, V), (V + pad, 1))
    over = q().policy_loss(again, targets, old, adv, grad=again, **kw)
    assert over.grad is again and torch.equal(again, out.grad)
    # into a buffer of another alignment
    into = torch.empty(rows, V + 3, dtype=dtype, device="cuda")[:, 1:V + 1]
    q().policy_loss(logits, targets, old, adv, grad=into, out=out, **kw)
    assert torch.equal(into, out.grad)


def special_rows(logits, targets):
    """Masks of every kind in the first rows of a batch; returns the rows whose outputs are NaN."""
    low, V = torch.finfo(logits.dtype).min, logits.shape[1]
    targets[:14] = V // 2
    logits[0] = -math.inf
    logits[1] = low
    logits[2] = -math.inf
    logits[2, V // 2] = 2.0
    logits[3, V // 2] = -math.inf
    logits[4, :V // 2] = low
    logits[5] = math.nan
    targets[5] = -1
    logits[6, V - 1] = math.nan
    logits[7, 0] = math.inf
    targets[8] = V
    logits[9, ::2] = -math.inf
    logits[9, V // 2] = 0.5
    logits[10] = 0.0
    logits[11] = torch.finfo(logits.dtype).max
    targets[12], targets[13] = 0, V - 1
    return [6, 7, 8]


@pytest.mark.parametrize("shape", [(600, 50021, torch.float16), (160, 40001, torch.float32), (300, 151936, torch.bfloat16),
                                   (321, 1001, torch.float32), (403, 3001, torch.bfloat16), (330, 9001, torch.float16)], ids=str)
def test_many_rows_against_few(shape):
    """The streaming kernel takes many long rows, a warp or a small CTA each of many short ones, a cluster each of
    few: the same rows either way, masks of every kind and rows that take no part among them. Both are within the bounds above of the exact values, and so within
    twice of each other; coefficients are rounded from sums that differ by those bounds, not more."""
    rows, V, dtype = shape
    logits, targets, old, adv, ref, w = policy_inputs(rows, V, 0, 0, 1.0, 0.2, 0.2, dtype, 60, True)
    targets[torch.rand(rows, device="cuda") < 0.3] = -1
    nans = special_rows(logits, targets)
    old[:14], ref[:14] = -3.0, -2.5
    kw = dict(clip_low=0.2, clip_high=0.2, entropy_coef=0.01)
    for kl in (0.0, 0.05):
        if kl:  # a KL term of a probability of 0 is infinite
            targets[0] = targets[3] = -1
        out = q().policy_loss(logits, targets, old, adv, ref_logprob=ref, weight=w, kl_coef=kl, grad_scale=64.0, **kw)
        for a in range(0, rows, 60):
            b = min(rows, a + 60)
            one = q().policy_loss(logits[a:b], targets[a:b], old[a:b], adv[a:b], ref_logprob=ref[a:b], weight=w[a:b], kl_coef=kl,
                                  grad_scale=64.0, **kw)
            close(out.logprob[a:b], one.logprob, 2 * LP_ATOL, "logprob")
            close(out.entropy[a:b], one.entropy, 2 * H_ATOL, "entropy")
            scale = (one.logprob - old[a:b]).exp() * adv[a:b].abs() + kl * ((ref[a:b] - one.logprob).exp() + 1)
            scale = torch.where(torch.isfinite(scale), scale, torch.zeros_like(scale)).double()
            close(out.row_loss[a:b], one.row_loss, scale * 2.2 * LP_ATOL + 0.02 * H_ATOL, "row_loss")
            g, x = one.grad.double(), out.grad[a:b].double()
            bad = [r - a for r in nans if a <= r < b]
            assert all(torch.isnan(x[r]).all() == bool(w[a + r] != 0) for r in bad)
            keep = [r for r in range(b - a) if r not in bad]
            fi = torch.finfo(dtype)
            lim = g.abs() * (2 * fi.eps + 2e-4) + fi.tiny + (w[a:b].double() * 64 * (scale + 0.01))[:, None] * 1e-6
            close(x[keep], g[keep], lim[keep], "grad")
        dead = (targets < 0) | (w == 0)
        assert (out.grad[dead] == 0).all() and (out.logprob[dead] == 0).all() and (out.row_loss[dead] == 0).all()


@pytest.mark.parametrize("shape", [(6, 300), (600, 30001)], ids=str)
def test_clipped_rows(shape):
    """A clipped ratio without KL term and bonus: a gradient of zeros, the clipped loss."""
    rows, V = shape
    logits, targets, g = rows_of(rows, V, torch.float32, 62)
    lp, _ = reference(logits, targets, 1.0)
    up = torch.arange(rows, device="cuda") % 2 == 0
    old = (lp - torch.where(up, 1.0, -1.0)).float()          # ratios of e and 1/e
    adv = torch.where(up, 1.0, -1.0).float().contiguous()     # out of the range on the side that is clipped
    adv[rows // 2:] *= -1                                     # ... and on the side that is not
    out = q().policy_loss(logits, targets, old, adv, weight=torch.ones(rows, device="cuda"))
    clipped = torch.arange(rows, device="cuda") < rows // 2
    assert (out.grad[clipped] == 0).all()
    assert (out.grad[~clipped].abs().amax(1) > 0).all()
    want = torch.where(up, -1.2, 0.8).float()                 # fp32 borders: half a step each
    assert (out.row_loss[clipped] - want[clipped]).abs().max() <= 2.0 ** -23


def test_two_streamed_calls_at_once():
    """Two calls of the streaming kernel on two streams, each holding SMs that the other waits for."""
    rows, V = 600, 30001
    sets = [policy_inputs(rows, V, 0, 0, 1.0, 0.2, 0.2, torch.float32, 70 + i, True) for i in range(2)]
    call = lambda s, **kw: q().policy_loss(s[0], s[1], s[2], s[3], weight=s[5], entropy_coef=0.01, **kw)  # noqa: E731
    want = [call(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[call(s, stream=st) for s, st in zip(sets, streams)] for _ in range(4)]
    torch.cuda.synchronize()
    for turn in got:
        for a, b in zip(turn, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_gradient_behind_copies_and_other_streams():
    """The gradient's launch may start before the work in front of it has ended, and waits for it: behind a copy, a
    fill, another stream's work, as the first of a graph and within one."""
    rows, V = 64, 50021
    logits, targets, g = rows_of(rows, V, torch.float32, 63)
    c = torch.randn(rows, generator=g, device="cuda")
    fwd = q().token_logprobs(logits, targets)
    want = q().token_logprobs_grad(logits, targets, fwd.stats, c)
    buf, derivative = torch.empty_like(logits), torch.empty_like(c)
    side = torch.cuda.Stream()

    def work():
        buf.zero_()
        derivative.zero_()
        a = q().token_logprobs_grad(buf, targets, fwd.stats, derivative)       # zeros
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            buf.copy_(logits)
            derivative.copy_(c)
        here.wait_stream(side)
        b = q().token_logprobs_grad(buf, targets, fwd.stats, derivative)
        q().token_logprobs_grad(buf, targets, fwd.stats, derivative, out=buf)  # in place, behind its own reading
        d = buf.clone()
        buf.fill_(7.0)
        return a, b, d

    def check(res):
        torch.cuda.synchronize()
        assert (res[0] == 0).all() and torch.equal(res[1], want) and torch.equal(res[2], want)

    for _ in range(5):
        check(work())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = q().token_logprobs_grad(logits, targets, fwd.stats, c)
        res = work()
    for _ in range(5):
        graph.replay()
        check(res)
        assert torch.equal(first, want)


def test_first_calls_under_capture():
    """A process whose first calls are captured, without a call before that sets the kernels up."""
    code = """
import torch, quasar_b200 as q
l = torch.randn(600, 30001, device='cuda'); t = torch.zeros(600, dtype=torch.int32, device='cuda'); f = torch.full((600,), -9.0, device='cuda')
cu = torch.tensor([0, 300, 600], dtype=torch.int32, device='cuda')
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    a, b, c = q.policy_loss(l, t, f, f, entropy_coef=0.1), q.preference_loss(l, t, cu), q.token_logprobs(l, t)
g.replay()
torch.cuda.synchronize()
x, y, z = q.policy_loss(l, t, f, f, entropy_coef=0.1), q.preference_loss(l, t, cu), q.token_logprobs(l, t)
same = lambda m, n: all(torch.equal(i, j) for i, j in zip(m, n) if i is not None)
assert same(a, x) and same(b, y) and same(c, z)
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def test_more_rows_than_one_launch_takes():
    """Batches beyond 16384 streamed rows: every row as in a batch of its own half."""
    rows, V = 16500, 50021
    logits, targets, g = rows_of(rows, V, torch.float16, 61)
    old, adv, w = (torch.randn(rows, generator=g, device="cuda") for _ in range(3))
    old = old - 11
    targets[::7] = -1
    out = q().policy_loss(logits, targets, old, adv, weight=w)
    for a, b in ((0, 8000), (8000, 16300), (15800, 16500)):
        part = q().policy_loss(logits[a:b], targets[a:b], old[a:b], adv[a:b], weight=w[a:b])
        for x, y in zip(out[1:], part[1:]):
            assert x is None or torch.equal(x[a:b], y)


PAIRS = [  # lengths, rows behind, V, T, beta, smoothing, mean, with reference
    ([1, 1], 0, 5, 1.0, 0.1, 0.0, False, True), ([3, 2, 1, 4], 2, 31, 1.0, 0.3, 0.1, False, False),
    ([0, 3, 5, 0, 0, 0], 1, 260, 0.7, 0.5, 0.0, True, True), ([17, 9, 200, 150], 0, 4099, 1.0, 0.05, 0.2, False, True),
    ([4, 5, 2, 7], 3, 18992, 1.0, 2.0, 0.0, True, False), ([3, 2], 0, 151936, 1.0, 0.1, 1.0, False, True),
    ([2, 1] * 150, 5, 97, 1.0, 0.2, 0.0, False, True),
    # batches beyond L2, with long, short and empty sequences
    ([100, 90, 400, 300, 0, 5, 250, 255, 1, 1, 600, 100, 0, 0, 3, 2], 7, 30001, 1.0, 0.02, 0.1, False, True),
    ([2, 3] * 420, 0, 30001, 0.9, 0.5, 0.0, True, False),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", PAIRS, ids=lambda c: str(c)[:40])
def test_preference_loss(dtype, case):
    n, behind, V, T, beta, eps, mean, with_ref = case
    rows, pairs = sum(n) + behind, len(n) // 2
    logits, targets, g = rows_of(rows, V, dtype, 31, pad=1)
    targets[torch.rand(rows, generator=g, device="cuda") < 0.2] = -1
    cu = torch.tensor(np.cumsum([0] + n), dtype=torch.int32, device="cuda")
    lp, _ = reference(logits, targets, T)
    x = lp.clone().requires_grad_(True)
    cut = [(x[cu[i]:cu[i + 1]], max(1, int((targets[cu[i]:cu[i + 1]] >= 0).sum()))) for i in range(2 * pairs)]
    seq = torch.stack([a.sum() for a, _ in cut])
    count = torch.tensor([k for _, k in cut], device="cuda", dtype=torch.float64)
    score = seq / count if mean else seq
    ref = None
    if with_ref:
        ref = (score.detach() + torch.randn(2 * pairs, generator=g, device="cuda").double()).float()
        score = score - ref.double()
    m = beta * (score[0::2] - score[1::2])
    pair = -(1 - eps) * torch.nn.functional.logsigmoid(m) - eps * torch.nn.functional.logsigmoid(-m)
    w = torch.rand(pairs, generator=g, device="cuda")
    if pairs > 1:
        w[1] = 0.0
    for weight in (None, w):
        wd = torch.full((pairs,), 1.0 / pairs, device="cuda", dtype=torch.float64) if weight is None else weight.double()
        loss = (wd * pair).sum()
        c, = torch.autograd.grad(loss, x, retain_graph=True)
        c = torch.where(targets >= 0, c, torch.zeros_like(c))  # rows that take no part stand as zeros in the sums
        out = q().preference_loss(logits, targets, cu, ref_logprob=ref, pair_weight=weight, temperature=T, beta=beta,
                                  label_smoothing=eps, length_normalize=mean, grad_scale=32.0)
        # each token's error, and the rounding of its log-probability (|lp| < 40) to fp32
        tok = LP_ATOL + 40 * EPS
        stol = count * tok
        close(out.logprob, lp, LP_ATOL, "logprob")
        close(out.seq_logprob, seq.detach(), stol, "seq_logprob")
        mt = beta * ((stol / count if mean else stol).view(-1, 2).sum(1))  # x's error; d pair/dx <= 1, d2 <= 1/4
        close(out.pair_loss, pair.detach(), mt, "pair_loss")
        close(out.loss, loss.detach(), (wd * mt).sum().item() + (wd * pair.detach().abs()).sum().item() * EPS, "loss")
        per = torch.zeros(rows, dtype=torch.float64, device="cuda")
        for i in range(2 * pairs):
            per[cu[i]:cu[i + 1]] = wd[i // 2] * beta * mt[i // 2] / 4 / (count[i] if mean else 1)
        per = torch.where(targets >= 0, per, torch.zeros_like(per)) * 32
        close(out.row_grad, c * 32, per, "row_grad")
        gref, bound = reference_grad(logits, targets, T, c * 32)
        _, p, _ = softmax64(logits, T)
        hot = torch.zeros_like(p).scatter_(1, targets.clamp(min=0).long()[:, None], 1.0)
        close(out.grad, gref, bound + per[:, None] * (hot + p) / T, "grad")
        assert (out.grad[sum(n):] == 0).all()
        none = q().preference_loss(logits, targets, cu, ref_logprob=ref, pair_weight=weight, temperature=T, beta=beta,
                                   label_smoothing=eps, length_normalize=mean, grad_scale=32.0, grad=False)
        assert none.grad is None and torch.equal(none.loss, out.loss)
    again = torch.empty(0, dtype=dtype, device="cuda").set_(logits.untyped_storage().clone(), 0, (rows, V), (V + 1, 1))
    over = q().preference_loss(again, targets, cu, ref_logprob=ref, pair_weight=w, temperature=T, beta=beta,
                               label_smoothing=eps, length_normalize=mean, grad_scale=32.0, grad=again, out=out)
    assert torch.equal(over.grad, out.grad)


def test_infinite_preferences():
    """A chosen sequence of probability 0: an infinite loss, but with the pair turned round (label_smoothing 1) none;
    the gradient stays finite."""
    logits, targets, g = rows_of(4, 50, torch.float32, 33)
    logits[1, targets[1]] = -math.inf
    cu = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    out = q().preference_loss(logits, targets, cu)
    assert out.loss.item() == math.inf and out.seq_logprob[0].item() == -math.inf
    assert torch.isfinite(out.grad).all()
    assert torch.allclose(out.row_grad, torch.tensor([-0.1, -0.1, 0.1, 0.1], device="cuda"), rtol=1e-6)
    out = q().preference_loss(logits, targets, cu, label_smoothing=1.0)
    assert out.loss.item() == 0 and (out.grad == 0).all()


def test_pairs_of_weight_zero():
    """A pair of weight 0 takes no part: no gradient, and nothing of its loss, NaN among it."""
    for n in (2, 20):                                   # few pairs and more
        logits, targets, g = rows_of(4 * n, 50, torch.float32, 34)
        logits[5] = math.nan
        cu = torch.arange(0, 4 * n + 1, 2, dtype=torch.int32, device="cuda")
        w = torch.ones(n, device="cuda")
        w[1] = 0
        out = q().preference_loss(logits, targets, cu, pair_weight=w)
        assert torch.isfinite(out.loss) and torch.isnan(out.pair_loss[1]) and (out.grad[4:8] == 0).all()
        assert torch.isfinite(out.grad).all()
        rest = torch.arange(n, device="cuda") != 1
        close(out.loss, out.pair_loss[rest].double().sum(), 4 * n * EPS)


def test_preference_offsets_that_leave_the_rows():
    """Offsets that fall or leave the rows: NaN for the pair and the loss, no gradient for its rows, the other pairs as ever."""
    logits, targets, g = rows_of(12, 77, torch.float32, 32)
    good = torch.tensor([0, 2, 5, 7, 9], dtype=torch.int32, device="cuda")
    want = q().preference_loss(logits, targets, good, pair_weight=torch.tensor([1.0, 0.0], device="cuda"))
    for cu in ([0, 2, 5, 3, 9], [0, 2, 5, 7, 13], [0, 2, 5, 2 ** 31 - 1, 9]):
        out = q().preference_loss(logits, targets, torch.tensor(cu, dtype=torch.int32, device="cuda"),
                                  pair_weight=torch.ones(2, device="cuda"))
        assert torch.isnan(out.loss) and torch.isnan(out.pair_loss[1]) and torch.isnan(out.seq_logprob[2:]).all()
        assert torch.equal(out.pair_loss[0], want.pair_loss[0])
        assert torch.equal(out.grad[:5], want.grad[:5]) and (out.grad[5:] == 0).all()
    out = q().preference_loss(logits, targets, torch.tensor([-1, 2, 5], dtype=torch.int32, device="cuda"))
    assert torch.isnan(out.loss) and (out.grad == 0).all()


def test_nothing_to_do():
    e = torch.empty(0, 64, device="cuda")
    t, f = torch.empty(0, dtype=torch.int32, device="cuda"), torch.empty(0, device="cuda")
    assert q().token_logprobs(e, t).logprob.shape == (0,)
    out = q().policy_loss(e, t, f, f)
    assert out.loss.item() == 0 and out.grad.shape == (0, 64)
    out = q().preference_loss(e, t, torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert out.loss.item() == 0
    logits, targets, _ = rows_of(3, 64, torch.float32, 1)
    out = q().preference_loss(logits, targets, torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert out.loss.item() == 0 and (out.grad == 0).all()
    out = q().preference_loss(logits, targets, torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert abs(out.loss.item() - math.log(2)) < 1e-6 and (out.grad == 0).all()


def test_offsets_past_32_bits():
    """Rows more than 2^31 elements apart."""
    rows, V, ld = 3, 4099, (1 << 30) + 77
    store = torch.empty((rows - 1) * ld + V, dtype=torch.bfloat16, device="cuda")
    logits = store.as_strided((rows, V), (ld, 1))
    src, targets, g = rows_of(rows, V, torch.bfloat16, 15)
    logits.copy_(src)
    lp, _ = reference(src, targets, 1.0)
    out = q().token_logprobs(logits, targets)
    close(out.logprob, lp, LP_ATOL)
    c = torch.ones(rows, device="cuda")
    want = q().token_logprobs_grad(src, targets, out.stats, c)
    assert torch.equal(q().token_logprobs_grad(logits, targets, out.stats, c), want)
    assert torch.equal(q().token_logprobs_grad(logits, targets, out.stats, c, out=logits), want)


def test_out_is_written_again():
    logits, targets, g = rows_of(6, 5000, torch.float32, 16)
    out = q().token_logprobs(logits, targets, entropy=True)
    want = [t.clone() for t in out]
    for t in out:
        t.fill_(-5)
    assert q().token_logprobs(logits, targets, entropy=True, out=out) is out
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    with pytest.raises(ValueError, match="entropy"):
        q().token_logprobs(logits, targets, out=out)


@pytest.mark.parametrize("shape", [(3, 97), (6, 60000), (40, 9001), (700, 60001), (200, 151936)])
def test_inputs_from_the_buffers_of_out(shape):
    """Log-probabilities of an earlier call as the old (or reference) ones, whose tensors the call writes again."""
    rows, V = shape
    logits, targets, g = rows_of(rows, V, torch.bfloat16, 18)
    targets[rows // 2] = -1
    adv = torch.randn(rows, generator=g, device="cuda")
    first = q().policy_loss(logits, targets, torch.zeros(rows, device="cuda"), adv)
    old = first.logprob + 0.1 * torch.randn(rows, generator=g, device="cuda")
    want = q().policy_loss(logits, targets, old, adv, ref_logprob=old, kl_coef=0.5)
    for _ in range(3):
        first.logprob.copy_(old)
        got = q().policy_loss(logits, targets, first.logprob, adv, ref_logprob=first.logprob, kl_coef=0.5, out=first)
        assert got.logprob is first.logprob
        assert all(torch.equal(a, b) for a, b in zip(got, want) if a is not None)


@pytest.mark.parametrize("pairs,length", [(3, 5), (40, 3), (2, 400)])
def test_reference_scores_from_the_buffers_of_out(pairs, length):
    logits, targets, g = rows_of(2 * pairs * length, 97, torch.float32, 19)
    cu = torch.arange(0, 2 * pairs * length + 1, length, dtype=torch.int32, device="cuda")
    first = q().preference_loss(logits, targets, cu, grad=False)
    ref = first.seq_logprob + torch.randn(2 * pairs, generator=g, device="cuda")
    want = q().preference_loss(logits, targets, cu, ref_logprob=ref)
    for _ in range(20):
        first.seq_logprob.copy_(ref)
        got = q().preference_loss(logits, targets, cu, ref_logprob=first.seq_logprob, out=first)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    logits, targets, g = rows_of(4, 64, torch.float32, 17)
    f = torch.zeros(4, device="cuda")
    st = torch.zeros(4, 2, device="cuda")
    cases = [
        lambda: q().token_logprobs(logits.t(), targets),
        lambda: q().token_logprobs(logits[:, ::2], targets),
        lambda: q().token_logprobs(logits[:1].expand(4, 64), targets),
        lambda: q().token_logprobs(logits, targets.long()),
        lambda: q().token_logprobs(logits, targets[:3]),
        lambda: q().token_logprobs(logits, targets.cpu()),
        lambda: q().token_logprobs_grad(logits, targets, st, f[:3]),
        lambda: q().token_logprobs_grad(logits, targets, st, f, grad_entropy=f),
        lambda: q().token_logprobs_grad(logits, targets, st, f, out=logits.half()),
        lambda: q().token_logprobs_grad(logits, targets, st, f, out=logits.t()),
        lambda: q().policy_loss(logits, targets, f, f, kl_coef=0.1),
        lambda: q().policy_loss(logits, targets, f, f[:1].expand(4)),
        lambda: q().policy_loss(logits, targets, f, f.double()),
        lambda: q().policy_loss(logits, targets, f, f, grad=None),
        lambda: q().preference_loss(logits, targets, torch.zeros(4, dtype=torch.int32, device="cuda")),
        lambda: q().preference_loss(logits, targets, torch.zeros(3, dtype=torch.int64, device="cuda")),
    ]
    for i, call in enumerate(cases):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"case {i} was taken")
    store = torch.zeros(4 * 64 + 32, device="cuda")
    logits, shifted = store[:256].view(4, 64), store[32:].view(4, 64)  # a gradient that overlaps the logits
    for call in (lambda: q().token_logprobs(logits, targets, temperature=0.0),
                 lambda: q().policy_loss(logits, targets, f, f, clip_low=-0.1),
                 lambda: q().token_logprobs_grad(logits, targets, st, f, out=shifted)):
        with pytest.raises(q().QuasarError):
            call()


def test_streams_and_graphs():
    """The same results on a side stream, from two streams at once, and from a captured graph replayed on new inputs."""
    rows, V = 40, 18992
    sets = [policy_inputs(rows, V, 0, 0, 1.0, 0.2, 0.2, torch.bfloat16, 40 + i, True) for i in range(2)]
    call = lambda s, **kw: q().policy_loss(s[0], s[1], s[2], s[3], ref_logprob=s[4], weight=s[5], kl_coef=0.05,  # noqa: E731
                                           entropy_coef=0.01, **kw)
    want = [call(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[call(s, stream=st) for s, st in zip(sets, streams)] for _ in range(3)]
    torch.cuda.synchronize()
    for turn in got:
        for a, b in zip(turn, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    static = [t.clone() for t in sets[0]]
    warm = torch.cuda.Stream()
    with torch.cuda.stream(warm):
        call(static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(static)
    for i in (1, 0, 1):
        for a, b in zip(static, sets[i]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want[i]))
    # two graphs of the preference loss, replayed at once on two streams
    cus = [torch.tensor(c, dtype=torch.int32, device="cuda") for c in ([0, 9, 18, 30, 40], [0, 20, 21, 22, 37])]
    pwant = [q().preference_loss(s[0], s[1], cu) for s, cu in zip(sets, cus)]
    graphs, outs = [], []
    for s, cu in zip(sets, cus):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(q().preference_loss(s[0], s[1], cu))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, pwant):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sampled_tokens_to_gradient(dtype):
    """Tokens picked by the sampler, their log-probabilities, the policy loss on them and its gradient through an
    LM head, against autograd in 64 bits; then a preference loss over the same rows as two pairs."""
    rows, V, D, T = 24, 18992, 64, 0.9
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(rows, D, generator=g, device="cuda", dtype=torch.float32)
    head = torch.randn(V, D, generator=g, device="cuda", dtype=torch.float32).mul_(0.3).requires_grad_(True)
    rng = torch.arange(1, rows + 1, dtype=torch.int64, device="cuda") * 7919
    logits = (x @ head.t())
    seen = logits.detach()
    ids = q().pick_batch(seen, rng, params=dict(temperature=T))
    assert ids.dtype == torch.int32
    old = q().token_logprobs(seen, ids, temperature=T)
    assert torch.isfinite(old.logprob).all()
    adv = torch.randn(rows, generator=g, device="cuda")
    cast = logits.to(dtype)
    out = q().policy_loss(cast.detach(), ids, old.logprob, adv, ref_logprob=old.logprob, temperature=T, kl_coef=0.1,
                          entropy_coef=0.01)
    cast.backward(out.grad)
    lp, h = reference(cast.detach(), ids, T)
    z = cast.detach().double().requires_grad_(True)
    lnp = torch.log_softmax(z / T, 1)
    lp = lnp.gather(1, ids.long()[:, None])[:, 0]
    h = -(lnp.exp() * lnp).sum(1)
    loss = policy64(lp, h, old.logprob, adv, old.logprob, 0.2, 0.2, 0.1, 0.01).mean()
    loss.backward()
    want = z.grad.t() @ x.double()
    # the head's gradient is a sum over the rows of values rounded to dtype (and of products in fp32 or dtype)
    lim = (z.grad.abs().t() @ x.double().abs()) * (torch.finfo(dtype).eps / 2 + 1e-4) + 1e-9
    assert ((head.grad.double() - want).abs() <= lim).all()
    cu = torch.tensor([0, 5, 12, 20, 24], dtype=torch.int32, device="cuda")
    pref = q().preference_loss(cast.detach(), ids, cu, temperature=T, beta=0.1)
    again = q().token_logprobs(cast.detach(), ids, temperature=T)
    assert torch.equal(pref.logprob, again.logprob) and torch.equal(pref.stats, again.stats)
    assert torch.equal(pref.grad, q().token_logprobs_grad(cast.detach(), ids, pref.stats, pref.row_grad, temperature=T))


def test_runs_repeat():
    """No result depends on the run."""
    logits, targets, old, adv, ref, w = policy_inputs(500, 18992, 0, 0, 1.0, 0.2, 0.2, torch.bfloat16, 50, True)
    a = q().policy_loss(logits, targets, old, adv, ref_logprob=ref, weight=w, kl_coef=0.1, entropy_coef=0.01)
    for _ in range(3):
        b = q().policy_loss(logits, targets, old, adv, ref_logprob=ref, weight=w, kl_coef=0.1, entropy_coef=0.01)
        assert all(torch.equal(x, y) for x, y in zip(a, b))

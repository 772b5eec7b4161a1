"""Token log-probabilities and losses at the ends of their ranges: ratios and derivatives beyond fp32, targets and
offsets out of range, waits that run out, sizes beyond 32 bits, and the accuracy of entropies. Plain 64-bit
implementations and bounds are those of test_gpu_losses.py."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_losses import DTYPES, EPS, H_ATOL, LP_ATOL, close, q, reference, reference_grad, rows_of, softmax64  # noqa: E402

pytestmark = pytest.mark.gpu


# a warp per row, clusters, and the streaming kernel for rows of 100 to 128 KB and for longer ones
RANGES = [(40, 1000), (12, 50021), (600, 30001), (160, 75001)]


def banned_rows(rows, V, dtype, seed):
    """Rows with a third of the columns banned, other than the targets'."""
    logits, targets, g = rows_of(rows, V, dtype, seed)
    ban = torch.rand(V, generator=g, device="cuda") < 1 / 3
    at = targets.long()[:, None]
    keep = logits.gather(1, at)
    logits.masked_fill_(ban, -math.inf)
    logits.scatter_(1, at, keep)
    return logits, targets, g


@pytest.mark.parametrize("entropy_coef", [0.0, 0.01])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", RANGES, ids=str)
def test_ratios_beyond_fp32(shape, dtype, entropy_coef):
    """Ratios that fp32 does not hold: an advantage of 0 takes no part whatever the ratio, a positive one is clipped,
    and a negative one's slope counts with its weight. The log-probability's error goes into ratio and slope as in
    test_policy_loss."""
    rows, V = shape
    logits, targets, g = banned_rows(rows, V, dtype, 80)
    lp, h = reference(logits, targets, 1.0)
    kind = torch.arange(rows, device="cuda") % 8
    far = torch.tensor([110.0, 800.0, math.inf, 110.0, 91.0, 0.5, -110.0, 91.0], device="cuda", dtype=torch.float64)
    adv = torch.tensor([0.0, 0.0, 0.0, 1.0, -1.0, -2.0, 0.0, 0.5], device="cuda")[kind]
    old = (lp - far[kind]).float()
    steep = kind == 4
    weight = torch.where(steep, 1e-37, 1.0 / rows).float()
    for kl in (0.0, 0.05):
        # the KL term's exponential beyond fp32, in rows of small weight
        ref = (lp + torch.where(steep | (kind == 7), 91.0 if kl else 0.0, 0.3)).float()
        w = torch.where(kind == 7, 1e-37, weight).float() if kl else weight
        kw = dict(ref_logprob=ref, kl_coef=kl, entropy_coef=entropy_coef)
        out = q().policy_loss(logits, targets, old, adv, weight=w, **kw)
        r, u, a = (lp - old.double()).exp(), ref.double() - lp, adv.double()
        ra = torch.where(a == 0, torch.zeros_like(a), r * a)
        fit = r.clamp(0.8, 1.2) * a
        slope = torch.where(ra <= fit, -ra, torch.zeros_like(a)) + kl * (1 - u.exp())
        gh = -entropy_coef * w if entropy_coef else None
        want, bound = reference_grad(logits, targets, 1.0, slope * w.double(), gh)
        size = torch.where(ra <= fit, ra.abs(), torch.zeros_like(a)) + kl * (1 + u.exp())
        _, p, _ = softmax64(logits, 1.0)
        hot = torch.zeros_like(p).scatter_(1, targets.long()[:, None], 1.0)
        close(out.grad, want, bound + (size * w.double() * LP_ATOL * 1.1)[:, None] * (hot + p), "grad")
        row = -torch.minimum(ra, fit) + kl * (u.exp() - u - 1) - entropy_coef * h
        row = torch.where(row > torch.finfo(torch.float32).max, math.inf, row)
        tol = (torch.minimum(ra, fit).abs() + kl * (1 + u.exp())) * LP_ATOL * 1.1 + entropy_coef * H_ATOL
        fits = ~torch.isinf(row)
        close(out.row_loss, torch.where(fits, row, row), torch.where(fits, tol, torch.zeros_like(tol)), "row_loss")
        w = torch.where(fits, w, torch.zeros_like(w))
        out = q().policy_loss(logits, targets, old, adv, weight=w, **kw)
        part = torch.where(fits, row, torch.zeros_like(row)) * w.double()
        lim = torch.where(fits, tol * w.double(), torch.zeros_like(tol)).sum() + part.abs().sum() * EPS
        close(out.loss, part.sum(), lim.item(), "loss")
    bad = old.clone()
    bad[0] = math.nan  # no ratio at all
    out = q().policy_loss(logits, targets, bad, adv, entropy_coef=entropy_coef)
    assert torch.isnan(out.row_loss[0]) and torch.isnan(out.grad[0]).all() and torch.isfinite(out.grad[1].float()).all()


@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", RANGES, ids=str)
def test_infinite_derivatives(shape, dtype, entropy):
    """A derivative that is infinite, or beyond fp32: infinities with their signs where the probability is not 0, zeros
    where it is, and no NaN."""
    rows, V = shape
    logits, targets, g = banned_rows(rows, V, dtype, 81)
    lp, _ = reference(logits, targets, 1.0)
    hot = torch.zeros(rows, V, dtype=torch.bool, device="cuda").scatter_(1, targets.long()[:, None], True)

    def check(grad, sign):
        zero = (logits == -math.inf) & ~hot
        assert (grad[zero] == 0).all()
        assert (grad[hot] == sign * math.inf).all()
        assert (grad[~hot & ~zero] == -sign * math.inf).all()

    coef = 0.01 if entropy else 0.0
    one = torch.ones(rows, device="cuda")
    out = q().policy_loss(logits, targets, (lp - 110).float(), -one, weight=one, entropy_coef=coef)
    check(out.grad, 1)
    fwd = q().token_logprobs(logits, targets, entropy=True)
    kw = dict(entropy=fwd.entropy, grad_entropy=one) if entropy else {}
    check(q().token_logprobs_grad(logits, targets, fwd.stats, math.inf * one, **kw), 1)
    check(q().token_logprobs_grad(logits, targets, fwd.stats, -math.inf * one, **kw), -1)
    logits.masked_fill_(hot, -math.inf)  # a target of probability 0 under a reference that allows it
    out = q().policy_loss(logits, targets, -3 * one, one, ref_logprob=-3 * one, kl_coef=0.1, entropy_coef=coef)
    assert out.loss.item() == math.inf and (out.row_loss == math.inf).all()
    check(out.grad, -1)


def test_sequences_at_the_last_rows_of_31_bits():
    """Sequences whose first row is within a CTA's threads of 2^31: V = 1, so that every log-probability is 0, the loss
    is ln 2 and a row's derivative beta / 2."""
    rows = (1 << 31) - 1
    logits = torch.zeros(rows, 1, dtype=torch.float16, device="cuda")
    targets = torch.zeros(rows, dtype=torch.int32, device="cuda")
    cu = torch.tensor([rows - 180, rows - 120, rows - 20], dtype=torch.int32, device="cuda")
    out = q().preference_loss(logits, targets, cu, grad=False)
    assert (out.seq_logprob == 0).all() and abs(out.loss.item() - math.log(2)) <= EPS
    end = out.row_grad[rows - 200:]
    assert (end[:20] == 0).all() and (end[180:] == 0).all()
    half = torch.tensor(0.1, dtype=torch.float32, device="cuda") / 2  # beta is an fp32 parameter
    assert (end[20:80] == -half).all() and (end[80:180] == half).all()
    assert int(out.row_grad.count_nonzero()) == 160


# rows, V, dtype, with entropy, chunks that the stalled CTA gets: none, in the first row's sums, between its sums and its
# gradient, in a later row; rows of one CTA, of two, and of eight
STALLS = [(600, 30001, torch.float32, False, (0, 1, 5, 9, 16)), (700, 60001, torch.float16, True, (3, 8, 13)),
          (300, 75001, torch.float32, False, (0, 2, 6, 8, 11, 17, 30)), (450, 151936, torch.bfloat16, True, (3, 7, 9, 14, 22)),
          (60 + 148, 1 << 20, torch.float32, False, (5, 19, 21, 30, 60))]


def stalled_calls(case):
    """The call whole, then with one CTA's loads stopped after so many chunks each time, then whole again: yields the
    chunks and (logprob, row_loss, loss, grad), the buffers of all calls."""
    rows, V, dtype, entropy, stops = case
    from quasar_b200.losses import PolicyParams
    logits, targets, g = rows_of(rows, V, dtype, 86)
    old, adv = torch.full((rows,), -9.0, device="cuda"), torch.randn(rows, generator=g, device="cuda")
    prm = PolicyParams(1.0, 0.2, 0.2, 0.0, 0.01 if entropy else 0.0, 64.0)
    h = torch.empty(rows, device="cuda") if entropy else None
    lp, row, loss, grad = (torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty((), device="cuda"),
                           torch.empty_like(logits))
    for chunks in (1 << 30, *stops, 1 << 30):
        for t in (lp, row, loss, grad):
            t.fill_(7.0)
        rc = q().lib().quasar_selftest_stalled_policy_loss(
            20_000_000, chunks, logits.data_ptr(), {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype], V, rows, V,
            targets.data_ptr(), old.data_ptr(), adv.data_ptr(), None, None, ctypes.addressof(prm), lp.data_ptr(),
            None if h is None else h.data_ptr(), row.data_ptr(), loss.data_ptr(), grad.data_ptr(), V,
            torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        yield chunks, (lp, row, loss, grad)


@pytest.mark.parametrize("case", STALLS, ids=lambda c: str(c[:4]))
def test_waits_that_run_out(case):
    """A CTA of the streaming kernel whose loads stop: its waits, and those of the CTAs that sum rows with it, run out
    after 10 ms, and the call ends. Log-probabilities and losses are then as ever or NaN, and the next call is as ever."""
    want = None
    for chunks, out in stalled_calls(case):
        lp, row, loss, grad = out
        if chunks < 1 << 30:
            for x, y in zip((lp, row), want):
                assert bool(((x == y) | torch.isnan(x)).all()), f"{chunks} chunks"
            assert int(torch.isnan(lp).sum()) <= case[0] // 8
            assert torch.equal(torch.isnan(lp), torch.isnan(row)) and torch.isnan(loss) == torch.isnan(row).any()
            assert torch.isnan(grad).any()
        elif want is None:
            want = [t.clone() for t in out]
            assert torch.isfinite(grad.float()).all() and torch.isfinite(loss)
        else:
            assert all(torch.equal(x, y) for x, y in zip(out, want))


@pytest.mark.parametrize("case", STALLS, ids=lambda c: str(c[:4]))
def test_gradients_behind_waits_that_run_out(case):
    """The same call's gradients: every element as ever or NaN, NaN in rows of the stalled clusters alone."""
    want = None
    for chunks, (lp, row, loss, grad) in stalled_calls(case):
        if want is None:
            want = grad.clone()
        elif chunks < 1 << 30:
            lost = torch.isnan(grad).any(1)
            assert 1 <= int(lost.sum()) <= case[0] // 8
            assert not (torch.isnan(lp) & ~lost).any()
            assert bool(((grad == want) | torch.isnan(grad)).all()), f"{chunks} chunks: neither as ever nor NaN"


def test_targets_out_of_range_that_take_no_part():
    """Targets behind the vocabulary in a pair of weight 0, in a pair of offsets out of range and behind the last
    sequence: NaN as log-probability, zeros as gradient. In a pair that takes part: NaN."""
    logits, targets, g = rows_of(14, 50, torch.float32, 82)
    cu = torch.tensor([0, 2, 4, 6, 8, 10, 12], dtype=torch.int32, device="cuda")
    targets[5] = targets[13] = 50
    w = torch.tensor([1.0, 0.0, 1.0], device="cuda")
    out = q().preference_loss(logits, targets, cu, pair_weight=w)
    assert torch.isnan(out.logprob[[5, 13]]).all() and torch.isnan(out.pair_loss[1])
    assert torch.isfinite(out.loss) and torch.isfinite(out.grad).all()
    assert (out.grad[4:8] == 0).all() and (out.grad[12:] == 0).all() and (out.grad[:4] != 0).all()
    out = q().preference_loss(logits, targets, cu, pair_weight=torch.ones(3, device="cuda"))
    assert torch.isnan(out.loss) and torch.isnan(out.grad[4:8]).all() and (out.grad[12:] == 0).all()
    cu[3] = 99  # pair 1 ends behind the rows
    out = q().preference_loss(logits, targets, cu)
    assert torch.isnan(out.loss) and (out.grad[4:8] == 0).all()


def test_autograd_sees_what_is_written():
    """Gradients and outputs written into a caller's tensors count as in-place changes: a graph that saved them refuses
    its backward pass instead of using what was written over."""
    rows, V = 6, 300
    x, targets, g = rows_of(rows, V, torch.float32, 83)
    f = torch.zeros(rows, device="cuda")
    cu = torch.tensor([0, 3, 6], dtype=torch.int32, device="cuda")
    stats = q().token_logprobs(x, targets).stats
    for call in (lambda t: q().token_logprobs_grad(t, targets, stats, f, out=t),
                 lambda t: q().policy_loss(t, targets, f, f, grad=t),
                 lambda t: q().preference_loss(t, targets, cu, grad=t)):
        leaf = x.clone().requires_grad_(True)
        logits = leaf.tanh()  # saves its output
        call(logits.detach())
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            logits.backward(torch.ones_like(logits))
        logits = leaf * 1.0   # saves nothing of it
        call(logits.detach())
        logits.backward(torch.ones_like(logits))
    for make in (lambda **kw: q().token_logprobs(x, targets, entropy=True, **kw),
                 lambda **kw: q().policy_loss(x, targets, f, f, entropy=True, grad=False, **kw),
                 lambda **kw: q().preference_loss(x, targets, cu, grad=False, **kw)):
        out = make()
        before = [None if t is None else t._version for t in out]
        make(out=out)
        assert all(t is None or t._version > b for t, b in zip(out, before))
    with torch.inference_mode():
        buf = torch.empty_like(x)
        assert q().policy_loss(x, targets, f, f, grad=buf).grad is buf


def test_sizes_beyond_32_bits_are_refused():
    """More columns (or rows) than the C entries count: an error, not the first columns alone."""
    wide = torch.empty(1, (1 << 32) + 16, dtype=torch.float16, device="cuda")
    wide[:, :64] = 0
    t, f = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, device="cuda")
    cu = torch.zeros(3, dtype=torch.int32, device="cuda")
    for call in (lambda: q().token_logprobs(wide, t), lambda: q().policy_loss(wide, t, f, f, grad=False),
                 lambda: q().preference_loss(wide, t, cu, grad=False)):
        with pytest.raises(ValueError, match="columns"):
            call()
    rows = (1 << 32) + 2
    tall, t = wide.view(-1, 1)[:rows], torch.empty(rows, dtype=torch.int32, device="cuda")
    t[:64] = 0
    with pytest.raises(ValueError, match="rows"):
        q().token_logprobs(tall, t)


def test_a_failed_launch_is_not_the_next_calls_error():
    """A launch into a stream whose capture is already lost fails; the sampler's next call on another stream does not."""
    cuda = ctypes.CDLL("libcuda.so.1")
    rows, V = 64, 4096
    logits, targets, g = rows_of(rows, V, torch.float32, 84)
    rng = torch.arange(1, rows + 1, dtype=torch.int64, device="cuda")
    out = q().token_logprobs(logits, targets)
    q().pick_batch(logits, rng, params=dict(temperature=0.9))
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    handle, graph = ctypes.c_void_p(stream.cuda_stream), ctypes.c_void_p()
    assert cuda.cuStreamBeginCapture_v2(handle, 2) == 0
    assert cuda.cuStreamSynchronize(handle) != 0  # not allowed while it captures: the capture is lost
    st = q().lib().quasar_token_logprobs(logits.data_ptr(), 0, V, rows, V, targets.data_ptr(), 1.0, out.logprob.data_ptr(),
                                         None, None, handle)
    assert cuda.cuStreamEndCapture(handle, ctypes.byref(graph)) != 0
    assert st == -3, st  # QUASAR_ECUDA
    ids = q().pick_batch(logits, rng, params=dict(temperature=0.9))
    torch.cuda.synchronize()
    assert ((ids >= 0) & (ids < V)).all()


WIDE_ROWS = [(160, torch.float32), (300, torch.float32)]


@pytest.mark.parametrize("rows,dtype", WIDE_ROWS)
def test_sums_of_wide_rows(rows, dtype):
    """Rows masked throughout by a value near -1.5e7, where logits stand a whole number apart, at the largest vocabulary:
    millions of equal terms, whose roundings all have one sign. At most 64 roundings add up (32 terms of a lane, whose
    sums are added with the errors carried on, then 32 lanes): 64 * 2^-24 for the additions, (4 + 3 |t|) 2^-24 for a
    term with |t| < 2, and 4 roundings of parts and of the logarithm."""
    V = 1 << 20
    logits = torch.full((rows, V), -1.5e7 - 1, dtype=dtype, device="cuda")
    logits[:, 12345] = -1.5e7
    targets = torch.full((rows,), 777, dtype=torch.int32, device="cuda")
    s = (V - 1) * math.exp(-1) + 1
    lp, h = -1 - math.log(s), math.log(s) + (V - 1) * math.exp(-1) / s
    bound = (64 + 10 + 4) * EPS
    f = torch.full((rows,), -14.0, device="cuda")
    ref = torch.full((rows,), lp, dtype=torch.float64, device="cuda"), torch.full((rows,), h, dtype=torch.float64, device="cuda")
    for out in (q().token_logprobs(logits, targets, entropy=True),
                q().policy_loss(logits, targets, f, f, entropy=True, grad=logits)):
        close(out.logprob, ref[0], bound, "logprob")
        close(out.entropy, ref[1], 4 * bound, "entropy")  # ln S, and the mean of t (under 2 in size) with S and Q off


# rows, V, dtype, as policy loss with its gradient, additions of a thread's lane (two lanes a thread)
ENTROPIES = [(2000, 1000, torch.float16, False, 16), (2000, 4099, torch.float32, False, 17), (64, 151936, torch.bfloat16, False, 38),
             (600, 30001, torch.float32, True, 59), (600, 50021, torch.float16, True, 98), (400, 75001, torch.float32, True, 59),
             (400, 151936, torch.bfloat16, True, 170)]


@pytest.mark.parametrize("case", ENTROPIES, ids=str)
def test_entropies(case):
    """H = ln S - ln2 Q / S. A lane adds n terms in fp32, each addition off by up to half a step, of random sign: sqrt(n / 3)
    half steps as standard deviation, of sums whose terms' t lie up to 20 over the lane's reference; at the worst one
    lane holds the row's mass, and five such deviations bound 10^4 rows. A common error of the terms cancels in H, the
    rest is at most (4 + 1.4 E|t|) half steps times the spread of ln p. Most rows spread their mass over lanes: their
    errors' median is under a quarter of that. The mean error is ex2.approx's varying part (under 2e-7) and four
    standard errors."""
    rows, V, dtype, policy, n = case
    logits, targets, g = rows_of(rows, V, dtype, 85)
    lnp, p, t = softmax64(logits, 1.0)
    h = -(p * lnp).sum(1)
    et = (p * t.abs()).sum(1)
    spread = (p * (lnp + h[:, None]).abs()).sum(1)
    bound = EPS * (5 * math.sqrt(n / 3) * math.log(2) * (21 + et) + (4 + 1.4 * et) * spread) + h * EPS
    f = torch.full((rows,), -9.0, device="cuda")
    if policy:
        out = q().policy_loss(logits, targets, f, f, entropy=True).entropy
    else:
        out = q().token_logprobs(logits, targets, entropy=True).entropy
    err = out.double() - h
    assert (err.abs() <= bound).all(), f"off by {err.abs().max().item():.3g}, {(err.abs() / bound).max().item():.3g} of the bound"
    assert (err.abs().median() <= bound.median() / 4).all(), f"median {err.abs().median().item():.3g}"
    assert err.mean().abs().item() <= 2e-7 + 4 * err.std().item() / math.sqrt(rows), f"mean {err.mean().item():.3g}"


@pytest.mark.parametrize("shape", [(40, 1000), (600, 30001)], ids=str)
def test_scale_of_zero(shape):
    """A gradient scaled by 0 is zeros, of ratios and KL factors beyond fp32, too."""
    rows, V = shape
    logits, targets, g = rows_of(rows, V, torch.float32, 87)
    lp, _ = reference(logits, targets, 1.0)
    one = torch.ones(rows, device="cuda")
    for far in (1.0, 110.0, 800.0):
        out = q().policy_loss(logits, targets, (lp - far).float(), -one, ref_logprob=(lp + far).float(), kl_coef=0.1, grad_scale=0.0)
        assert (out.grad == 0).all()

"""Token log-probabilities and the losses made of them: the cases that are measured, and their plain forms.

Four operators over rows of logits [rows, V] with int32 targets (a target below 0 marks a row that takes no part):

  logprobs       log-probability of each row's target at a temperature, and the row's entropy
  logprobs_grad  the gradient of the two into the logits
  policy         the clipped policy loss with a KL term and an entropy bonus, and its gradient into the logits
  preference     the paired log-ratio (preference) loss over packed sequences, and its gradient into the logits

A case's plain values: op, rows (preference: pairs and longest), V, pad (columns behind V in the storage of a row), dtype, T (temperature), entropy,
ignored (share of rows whose target is -1), banned (share of columns at -inf, as constrained decoding leaves them) and each loss's own switches.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
CLIP_LOW, CLIP_HIGH = 0.2, 0.28
SCALE = {"f32": 1.0, "f16": 4096.0, "bf16": 1.0}  # loss scaling, without which 16-bit gradients of a mean over many rows vanish
BLOCK = 1 << 26  # values that prepare() and exact() work on at a time


def listed():
    full, shard = 151936, 18992  # the benchmark's vocabulary and its eighth
    return [
        # serving: the log-probability of the one token a decode step has picked
        dict(name="logprobs 1 row", op="logprobs", rows=1, V=full, pad=0, dtype="f32", T=1.0, entropy=False, ignored=0.0, banned=0.0),
        # serving: a batch of 256 sequences, with the entropy of each step's distribution, under constrained decoding
        dict(name="logprobs 256 f32", op="logprobs", rows=256, V=full, pad=0, dtype="f32", T=0.7, entropy=True, ignored=0.0, banned=0.25),
        # scoring of prompts and of rollouts by the old or the reference model
        dict(name="logprobs 8191 bf16", op="logprobs", rows=8191, V=full, pad=0, dtype="bf16", T=1.0, entropy=False, ignored=0.1, banned=0.0),
        # a small step of a loss of the user's own, on a narrow vocabulary
        dict(name="logprobs_grad 64 f32", op="logprobs_grad", rows=64, V=shard, pad=0, dtype="f32", T=1.0, entropy=True, ignored=0.0, banned=0.0),
        # the same for a training batch, some rows of it prompt
        dict(name="logprobs_grad 2047 bf16", op="logprobs_grad", rows=2047, V=full, pad=0, dtype="bf16", T=1.0, entropy=False, ignored=0.2, banned=0.0),
        # policy training: one short rollout
        dict(name="policy 16 f32", op="policy", rows=16, V=full, pad=0, dtype="f32", T=1.0, entropy=False, ignored=0.0, banned=0.0, kl=0.0),
        # a micro-batch of rollouts with a KL term and an entropy bonus
        dict(name="policy 1023 bf16", op="policy", rows=1023, V=full, pad=0, dtype="bf16", T=0.9, entropy=True, ignored=0.3, banned=0.0, kl=0.05),
        # an odd vocabulary, rows packed without padding: no row but the first is aligned
        dict(name="policy 3001 odd f16", op="policy", rows=3001, V=50021, pad=0, dtype="f16", T=1.0, entropy=False, ignored=0.1, banned=0.0, kl=0.05),
        # the benchmark's batch in its type
        dict(name="policy 4096 f32", op="policy", rows=4096, V=full, pad=0, dtype="f32", T=1.0, entropy=False, ignored=0.1, banned=0.0, kl=0.05),
        # preference training: two short pairs
        dict(name="preference 2 pairs bf16", op="preference", pairs=2, longest=24, V=shard, pad=0, dtype="bf16", T=1.0, smoothing=0.0, mean=False, ref=True),
        # a micro-batch of ragged pairs
        dict(name="preference 32 pairs bf16", op="preference", pairs=32, longest=96, V=full, pad=0, dtype="bf16", T=1.0, smoothing=0.0, mean=False, ref=True),
        # length-normalised, without a reference model, on an odd width with padded rows
        dict(name="preference 12 pairs f32", op="preference", pairs=12, longest=150, V=75967, pad=33, dtype="f32", T=1.0, smoothing=0.1, mean=True, ref=False),
    ]


def draw(rng):
    spread = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    op = rng.choice(["logprobs", "logprobs_grad", "policy", "preference"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    V = rng.choice([151936, 18992, spread(260, 151936), spread(260, 151936) | 1])
    pad = rng.choice([0, 0, rng.randrange(1, 64)])
    most = max(1, 4096 * 151936 * 4 // ((V + pad) * SIZE[dtype]) // 3)
    c = dict(op=op, V=V, pad=pad, dtype=dtype, T=rng.choice([1.0, round(rng.uniform(0.4, 1.6), 3)]))
    if op == "preference":
        c["pairs"] = spread(1, max(1, min(256, most // 16)))
        c["longest"] = max(2, spread(2, max(2, min(2048, most // (2 * c["pairs"])))))
        mean = rng.random() < 0.4
        return dict(c, smoothing=rng.choice([0.0, 0.1]), mean=mean, ref=not mean or rng.random() < 0.5)  # sums without a reference would saturate
    c["rows"] = spread(1, min(20000, most))
    c |= dict(entropy=rng.random() < 0.5, ignored=rng.choice([0.0, 0.1, 0.4]), banned=rng.choice([0.0, 0.0, 0.3]))
    return dict(c, kl=rng.choice([0.0, 0.05])) if op == "policy" else c


def lengths(case):
    """The 2 * pairs sequence lengths of a preference case, from one token (now and then none) to the longest."""
    r = random.Random(case["pairs"] * 1000003 + case["longest"])
    n = [r.randint(max(1, case["longest"] // 4), case["longest"]) for _ in range(2 * case["pairs"])]
    if case["pairs"] > 4:
        n[3], n[6] = 1, 0
    return n


def prompt(n):
    """Leading rows of a sequence of n rows that are its prompt."""
    return n * 3 // 10


def rows_of(case):
    """(rows, rows that take part)"""
    if case["op"] == "preference":
        n = lengths(case)
        return sum(n) + 3, sum(x - prompt(x) for x in n)  # three rows of padding behind the last sequence
    return case["rows"], case["rows"] - int(case["rows"] * case["ignored"])


def blocks(rows, V):
    step = max(1, BLOCK // V)
    return [slice(a, min(rows, a + step)) for a in range(0, rows, step)]


def log_probs(logits, targets, T):
    """64-bit log-probabilities of the targets, for making inputs."""
    out = torch.empty(len(targets), dtype=torch.float64, device="cuda")
    for b in blocks(*logits.shape):
        z = logits[b].double() / T
        out[b] = z.gather(1, targets[b].clamp(min=0).long()[:, None])[:, 0] - z.logsumexp(1)
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    normal = lambda *n: torch.randn(*n, generator=g, device="cuda")  # noqa: E731
    (rows, live), V, T = rows_of(case), case["V"], case["T"]
    store = torch.randn(rows, V + case["pad"], generator=g, device="cuda", dtype=DTYPES[case["dtype"]]).mul_(3.0)
    logits = store[:, :V]
    targets = torch.empty(rows, dtype=torch.int32, device="cuda")
    for b in blocks(rows, V):  # tokens drawn from the rows' own distributions, as a rollout's are
        if case.get("banned"):
            logits[b].masked_fill_(torch.rand(V, generator=g, device="cuda") < case["banned"], -math.inf)
        targets[b] = (logits[b].float() / T).sub_(torch.empty(b.stop - b.start, V, device="cuda").exponential_(generator=g).log_()).argmax(1)
    s = dict(case=case, logits=logits, targets=targets)
    if case["op"] == "preference":
        n = lengths(case)
        s["cu"] = torch.tensor([0] + n, device="cuda").cumsum(0).to(torch.int32)
        s["targets"][s["cu"][-1]:] = -1
        at = 0
        for x in n:
            s["targets"][at:at + prompt(x)] = -1
            at += x
        if case["ref"]:  # the reference model is near: sums of the sequences' own log-probabilities, shifted
            lp = log_probs(logits, s["targets"], T).masked_fill(s["targets"] < 0, 0).cumsum(0)
            lp = torch.cat([lp.new_zeros(1), lp])[s["cu"].long()].diff()
            s["ref"] = (lp + normal(len(n)).double() * 4).float()
        return s
    targets[torch.randperm(rows, generator=g, device="cuda")[:rows - live]] = -1
    if case["op"] == "logprobs_grad":
        s["g_logprob"] = normal(rows) / rows
        if case["entropy"]:
            s["g_entropy"] = normal(rows) / rows
        st = {k: torch.empty(rows, dtype=torch.float64, device="cuda") for k in ("max", "sum", "h")}
        for b in blocks(rows, V):  # what the forward pass has left: each row's maximum, its sum of exponentials and its entropy
            l = logits[b].double()
            m = l.amax(1, keepdim=True)
            e = ((l - m) / T).exp()
            st["max"][b], st["sum"][b] = m[:, 0], e.sum(1)
            st["h"][b] = e.sum(1).log() - (e * ((l - m) / T).nan_to_num(neginf=0.0)).sum(1) / e.sum(1)
        s["stats"] = torch.stack([st["max"], st["sum"]], 1).float()
        s["h"] = st["h"].float()
    if case["op"] == "policy":
        lp = log_probs(logits, targets, T)
        d = normal(rows).double() * 0.15  # a policy some steps from the one that made the tokens
        for border in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):
            d = torch.where((d - border).abs() < 1e-4, border + 1e-4, d)  # at a border either side's gradient is right
        s["old"] = (lp - d).float()
        s["advantage"] = normal(rows)
        s["weight"] = (targets >= 0).float() / max(1, live)
        if case["kl"]:
            s["ref"] = (lp + normal(rows).double() * 0.2).float()
    return s


def run(s):
    c = s["case"]
    if own:
        import quasar_b200 as q
        if c["op"] == "logprobs":
            r = q.token_logprobs(s["logits"], s["targets"], temperature=c["T"], entropy=c["entropy"])
            return {"logprob": r.logprob, "entropy": r.entropy}
        if c["op"] == "logprobs_grad":
            return {"grad": q.token_logprobs_grad(s["logits"], s["targets"], s["stats"], s["g_logprob"], entropy=s["h"] if c["entropy"] else None,
                                                  grad_entropy=s.get("g_entropy"), temperature=c["T"])}
        if c["op"] == "policy":
            r = q.policy_loss(s["logits"], s["targets"], s["old"], s["advantage"], ref_logprob=s.get("ref"), weight=s["weight"], temperature=c["T"],
                              clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=c["kl"], entropy_coef=0.01 if c["entropy"] else 0.0,
                              grad_scale=SCALE[c["dtype"]])
            return {"loss": r.loss, "logprob": r.logprob, "entropy": r.entropy, "row_loss": r.row_loss, "grad": r.grad}
        r = q.preference_loss(s["logits"], s["targets"], s["cu"], ref_logprob=s.get("ref"), temperature=c["T"], beta=2.0 if c["mean"] else 0.1,
                              label_smoothing=c["smoothing"], length_normalize=c["mean"], grad_scale=SCALE[c["dtype"]])
        return {"loss": r.loss, "pair_loss": r.pair_loss, "seq_logprob": r.seq_logprob, "logprob": r.logprob, "grad": r.grad}

    l, t = s["logits"].float(), s["targets"].long()
    live = t >= 0
    at = t.clamp(min=0)[:, None]
    if c["op"] == "logprobs_grad":
        p = ((l - s["stats"][:, :1]) / c["T"]).exp_() / s["stats"][:, 1:]
        return {"grad": into_logits(p, at, live, s["g_logprob"], s.get("g_entropy"), s["h"], c["T"], s["logits"].dtype)}
    z = (l - l.amax(1, keepdim=True)) / c["T"]
    e = z.exp()
    total = e.sum(1, dtype=torch.float64)  # a long sum
    lp = torch.where(live, z.gather(1, at)[:, 0].double() - total.log(), 0.0)
    h = None
    if c.get("entropy"):
        h = torch.where(live, total.log() - (e * z.nan_to_num_(neginf=0.0)).sum(1, dtype=torch.float64) / total, 0.0)
    if c["op"] == "logprobs":
        return {"logprob": lp.float(), "entropy": None if h is None else h.float()}
    if c["op"] == "policy":
        w, a = s["weight"].double(), s["advantage"].double()
        ratio = (lp - s["old"].double()).exp()  # 64 bits: it is compared with the borders
        fit = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
        row = -torch.minimum(ratio * a, fit * a)
        g = torch.where(ratio * a <= fit * a, -ratio * a, 0.0)
        if c["kl"]:
            far = s["ref"].double() - lp
            row = row + c["kl"] * (far.exp() - far - 1)
            g = g + c["kl"] * (1 - far.exp())
        if h is not None:
            row = row - 0.01 * h
        row = torch.where(live, row, 0.0)
        loss = (w * row).sum().float()
        w = w * SCALE[c["dtype"]]
        grad = into_logits(e / total.float()[:, None], at, live, (g * w).float(), None if h is None else (-0.01 * w).float(), None if h is None else h.float(),
                           c["T"], s["logits"].dtype)
        return {"loss": loss, "logprob": lp.float(), "entropy": None if h is None else h.float(), "row_loss": row.float(), "grad": grad}
    cu, pairs = s["cu"].long(), c["pairs"]
    n = torch.cat([live.new_zeros(1, dtype=torch.long), live.cumsum(0)])[cu].diff().clamp(min=1)
    seq = torch.cat([lp.new_zeros(1), lp.cumsum(0)])[cu].diff()
    by = n.double() if c["mean"] else torch.ones_like(seq)
    far = seq / by - (s["ref"].double() if c["ref"] else 0.0)
    x = (2.0 if c["mean"] else 0.1) * (far[0::2] - far[1::2])
    tail = (1 + (-x.abs()).exp()).log()
    pair = (1 - c["smoothing"]) * ((-x).clamp(min=0) + tail) + c["smoothing"] * (x.clamp(min=0) + tail)
    g = -(2.0 if c["mean"] else 0.1) * ((1 - c["smoothing"]) / (1 + x.exp()) - c["smoothing"] / (1 + (-x).exp())) / pairs * SCALE[c["dtype"]]
    per_row = torch.stack([g, -g], 1).reshape(-1) / by
    which = torch.searchsorted(cu[1:], torch.arange(len(t), device="cuda"), right=True).clamp(max=2 * pairs - 1)
    grad = into_logits(e / total.float()[:, None], at, live, per_row[which].float(), None, None, c["T"], s["logits"].dtype)
    return {"loss": (pair.sum() / pairs).float(), "pair_loss": pair.float(), "seq_logprob": seq.float(), "logprob": lp.float(), "grad": grad}


def into_logits(p, at, live, g, g_entropy, h, T, dtype):
    """The gradient into the logits of sum(g * logprob + g_entropy * entropy), with the rows' probabilities p."""
    d = p * -g[:, None]
    if g_entropy is not None:
        d -= g_entropy[:, None] * p * (p.log().nan_to_num_(neginf=0.0) + h[:, None])
    d.scatter_add_(1, at, g[:, None])
    return torch.where(live[:, None], d.div_(T), 0.0).to(dtype)


def work(case):
    (rows, live), V, size = rows_of(case), case["V"], SIZE[case["dtype"]]
    read, write = live * V * size, rows * V * size
    if case["op"] == "logprobs":
        return {"bytes": read + rows * (12 if case["entropy"] else 8), "flops": live * V * (6 if case["entropy"] else 4)}
    if case["op"] == "logprobs_grad":
        return {"bytes": read + write + rows * (24 if case["entropy"] else 16), "flops": live * V * (7 if case["entropy"] else 5)}
    if case["op"] == "policy":
        return {"bytes": read + write + rows * (24 + (4 if case["kl"] else 0) + (4 if case["entropy"] else 0)), "flops": live * V * (13 if case["entropy"] else 9)}
    return {"bytes": read + write + rows * 8 + case["pairs"] * 28, "flops": live * V * 9}


def exact(case, seed):
    s = prepare(case, seed)
    rows, V, T = *s["logits"].shape, case["T"]
    t = s["targets"].long()
    on = t >= 0
    lp, h = (torch.zeros(rows, dtype=torch.float64, device="cuda") for _ in range(2))
    for b in blocks(rows, V):
        y = torch.log_softmax(s["logits"][b].double() / T, 1)
        lp[b] = torch.where(on[b], y[torch.arange(len(y)), t[b].clamp(min=0)], 0)
        h[b] = torch.where(on[b], torch.special.entr(y.exp()).sum(1), 0)
    gh = None
    out = {}
    if case["op"] == "logprobs":
        return {"logprob": lp, "entropy": h if case["entropy"] else None}
    if case["op"] == "logprobs_grad":
        g = s["g_logprob"].double()
        gh = s["g_entropy"].double() if case["entropy"] else None
    elif case["op"] == "policy":
        x = lp.clone().requires_grad_(True)
        a, w = s["advantage"].double(), s["weight"].double()
        r = torch.exp(x - s["old"].double())
        row = torch.maximum(-a * r, -a * torch.clamp(r, 1 - CLIP_LOW, 1 + CLIP_HIGH))
        if case["kl"]:
            u = s["ref"].double() - x
            row = row + case["kl"] * (torch.expm1(u) - u)
        if case["entropy"]:
            row = row - 0.01 * h
            gh = -0.01 * w
        row = row * on
        loss = torch.dot(row, w)
        g, = torch.autograd.grad(loss, x)
        out = {"loss": loss.detach(), "logprob": lp, "entropy": h if case["entropy"] else None, "row_loss": row.detach()}
    else:
        x = lp.clone().requires_grad_(True)
        n, beta = lengths(case), 2.0 if case["mean"] else 0.1
        cut = list(torch.split(x[:sum(n)], n))
        seq = torch.stack([v.sum() for v in cut])
        score = torch.stack([v.sum() / max(1, k - prompt(k)) for v, k in zip(cut, n)]) if case["mean"] else seq
        if case["ref"]:
            score = score - s["ref"].double()
        m = beta * (score[0::2] - score[1::2])
        ls = torch.nn.functional.logsigmoid
        pair = -(1 - case["smoothing"]) * ls(m) - case["smoothing"] * ls(-m)
        loss = pair.mean()
        g, = torch.autograd.grad(loss, x)
        out = {"loss": loss.detach(), "pair_loss": pair.detach(), "seq_logprob": seq.detach(), "logprob": lp}
    if case["op"] != "logprobs_grad":
        g = g * SCALE[case["dtype"]]
        gh = None if gh is None else gh * SCALE[case["dtype"]]
    grad = torch.zeros(rows, V, dtype=torch.float64, device="cuda")
    for b in blocks(rows, V):
        y = torch.log_softmax(s["logits"][b].double() / T, 1)
        p = y.exp()
        d = -g[b, None] * p
        d[torch.arange(len(d)), t[b].clamp(min=0)] += g[b]
        if gh is not None:
            d += gh[b, None] * (torch.special.entr(p) - p * h[b, None])
        grad[b] = d / T * on[b, None]
    return out | {"grad": grad}

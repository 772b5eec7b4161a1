"""Log-probabilities of given tokens and the losses made of them, over rows of logits.

The Python side of include/quasar_losses.h: ``token_logprobs`` and its gradient, the clipped
policy loss and the paired preference loss, each over a [rows, V] CUDA tensor of logits
(float32, float16 or bfloat16, unit column stride) and int32 targets, as ``pick_batch`` writes
them. A target below 0 marks a row that takes no part (outputs 0, a gradient of zeros).

Losses return their gradient into the logits with them, so one call is a forward and a backward
pass; a model goes on from there with ``logits.backward(result.grad)``. Nothing is registered
with autograd; tensors of the caller's that are written count as changed in place, so that a graph
which saved them refuses its backward pass. Outputs are allocated on the stream of the call, or given (``out=``, ``grad=``)
and used again. torch is used only for device memory and streams.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

from ._lib import BF16, F16, F32, check, lib

_INT_MAX = 2 ** 31 - 1
_DTYPES = {}  # torch dtype -> the C constant; filled at the first call, torch being imported only then
# the current stream's handle by device index, where torch has a way to it without a Stream object (2 us)
_raw = None


class PolicyParams(ctypes.Structure):
    """ctypes twin of quasar_policy_params."""
    _fields_ = [("temperature", ctypes.c_float), ("clip_low", ctypes.c_float), ("clip_high", ctypes.c_float),
                ("kl_coef", ctypes.c_float), ("entropy_coef", ctypes.c_float), ("grad_scale", ctypes.c_float)]


class PreferenceParams(ctypes.Structure):
    """ctypes twin of quasar_preference_params."""
    _fields_ = [("temperature", ctypes.c_float), ("beta", ctypes.c_float), ("label_smoothing", ctypes.c_float),
                ("grad_scale", ctypes.c_float), ("length_normalize", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor             # [rows] float32
    entropy: Optional[torch.Tensor]   # [rows] float32, or None
    stats: torch.Tensor               # [rows, 2] float32: the row's largest logit, its sum of exp((l - max) / T)


class PolicyLoss(NamedTuple):
    loss: torch.Tensor                # [] float32
    logprob: torch.Tensor             # [rows] float32
    entropy: Optional[torch.Tensor]   # [rows] float32, or None
    row_loss: torch.Tensor            # [rows] float32, without the weights
    grad: Optional[torch.Tensor]      # [rows, V] of the logits' type, or None


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor                # [] float32
    pair_loss: torch.Tensor           # [pairs] float32
    seq_logprob: torch.Tensor         # [2 * pairs] float32: chosen, rejected, chosen, ...
    logprob: torch.Tensor             # [rows] float32
    stats: torch.Tensor               # [rows, 2] float32, as TokenLogprobs.stats
    row_grad: torch.Tensor            # [rows] float32: d loss / d logprob, times grad_scale
    grad: Optional[torch.Tensor]      # [rows, V] of the logits' type, or None


def _torch():
    """torch, imported at the first call; fills the table of types."""
    import torch
    if not _DTYPES:
        global _raw
        _raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        _DTYPES.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16})
    return torch


def _rows(logits, targets):
    """Checks logits and targets; returns (torch, rows, V, the C dtype, the row stride, the device)."""
    torch = _torch()
    dt = _DTYPES.get(logits.dtype)
    if logits.dim() != 2 or dt is None:
        raise ValueError("logits must be a [rows, V] float32, float16 or bfloat16 tensor")
    if not logits.is_cuda:
        raise ValueError("logits must be a CUDA tensor")
    rows, V = logits.shape
    if rows > _INT_MAX or V > _INT_MAX:  # the C entry would take the low 32 bits
        raise ValueError(f"logits have too many {'rows' if rows > _INT_MAX else 'columns'}: {rows} x {V}")
    ld, unit = logits.stride()
    if unit != 1 and V > 1:
        raise ValueError("logits must have unit column stride")
    if rows < 2:
        ld = max(V, 1)  # a tensor of one row or none may have any row stride
    elif ld < V:
        raise ValueError("rows of logits must not overlap")
    device = logits.device
    _vec(targets, "targets", (rows,), torch.int32, device)
    return torch, rows, V, dt, ld, device


def _vec(t, name, shape, dtype, device):
    if t.dtype is not dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {list(shape)} on {device}, got "
                         f"{t.dtype} {list(t.shape)} on {t.device}")


def _ld(t):
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def _like(torch, logits, rows, V, ld):
    """A gradient buffer of the logits' shape whose rows have the 16-byte phase of the logits' rows."""
    phase = logits.data_ptr() & 15
    if ld == V and phase == 0:
        return logits.new_empty((rows, V))
    size = logits.element_size()
    per, first = 16 // size, phase // size
    ld = V + (ld - V) % per  # the shortest stride with the same phases
    return logits.new_empty(first + rows * ld).as_strided((rows, V), (ld, 1), first)


def _check_grad(grad, logits):
    if grad.shape != logits.shape or grad.dtype != logits.dtype or grad.device != logits.device:
        raise ValueError(f"the gradient must be a {logits.dtype} tensor of shape {list(logits.shape)} on {logits.device}")
    if (grad.stride(1) != 1 and grad.shape[1] > 1) or (grad.shape[0] > 1 and grad.stride(0) < grad.shape[1]):
        raise ValueError("the gradient must have unit column stride and rows that do not overlap")


def _grad_arg(torch, grad, logits):
    """Checks the grad argument; returns the buffer that was passed, or None."""
    if grad is True or grad is False:
        return None
    if not isinstance(grad, torch.Tensor):
        raise ValueError("grad must be True (allocate), False (none) or a tensor to write")
    _check_grad(grad, logits)
    return grad


def _p(t):
    return None if t is None else t.data_ptr()


def _wrote(torch, *tensors):
    """Counts the call's writing into a caller's tensors as in-place changes, which autograd refuses to miss."""
    torch.autograd.graph.increment_version([t for t in tensors if t is not None])


def _on(torch, device, stream, tensors, call):
    """call(the C stream) with the logits' device and the stream of the call current, so that what it allocates belongs
    to that stream; keeps the call's tensors from being handed out again before the stream is done."""
    if stream is None and torch.cuda.current_device() == device.index:
        return call(_raw(device.index) if _raw else torch.cuda.current_stream(device).cuda_stream)
    with torch.cuda.device(device):
        current = torch.cuda.current_stream(device)
        if stream is None or stream == current:
            return call(current.cuda_stream)
        if stream.device != device:
            raise ValueError(f"the stream is on {stream.device}, the logits on {device}")
        for t in tensors:
            if t is not None:
                t.record_stream(stream)
        with torch.cuda.stream(stream):
            return call(stream.cuda_stream)


def token_logprobs(logits, targets, *, temperature: float = 1.0, entropy: bool = False,
                   out: Optional[TokenLogprobs] = None, stream=None) -> TokenLogprobs:
    """Log-probability of each row's target under softmax(logits / temperature), and on request the row's entropy.

    targets: [rows] int32; below 0: the row takes no part and its outputs are 0.
    out: a TokenLogprobs of an earlier call whose tensors are written again (its entropy as ``entropy`` asks).
    Launches on ``stream`` (a torch.cuda.Stream; default: the current stream).
    """
    torch, rows, V, dt, ld, device = _rows(logits, targets)
    f32 = torch.float32
    if out is not None:
        _vec(out.logprob, "out.logprob", (rows,), f32, device)
        _vec(out.stats, "out.stats", (rows, 2), f32, device)
        if entropy != (out.entropy is not None):
            raise ValueError("out.entropy must be a tensor if entropy is asked for, and None if not")
        if entropy:
            _vec(out.entropy, "out.entropy", (rows,), f32, device)

    def call(st):
        o = out
        if o is None:
            e = logits.new_empty
            o = TokenLogprobs(e(rows, dtype=f32), e(rows, dtype=f32) if entropy else None, e((rows, 2), dtype=f32))
        check(lib().quasar_token_logprobs(logits.data_ptr(), dt, ld, rows, V, targets.data_ptr(), temperature,
                                          o.logprob.data_ptr(), _p(o.entropy), o.stats.data_ptr(), st),
              "quasar_token_logprobs")
        if out is not None:
            _wrote(torch, *out)
        return o
    return _on(torch, device, stream, (logits, targets, *(out or ())), call)


def token_logprobs_grad(logits, targets, stats, grad_logprob, *, entropy=None, grad_entropy=None,
                        temperature: float = 1.0, out=None, stream=None):
    """Gradient into the logits of sum(grad_logprob * logprob + grad_entropy * entropy).

    stats (and entropy, with grad_entropy): what ``token_logprobs`` gave for the same logits, targets and
    temperature. out: a tensor of the logits' shape and type to write, which may be ``logits`` itself.
    Returns the gradient, of the logits' type.
    """
    torch, rows, V, dt, ld, device = _rows(logits, targets)
    f32 = torch.float32
    _vec(stats, "stats", (rows, 2), f32, device)
    _vec(grad_logprob, "grad_logprob", (rows,), f32, device)
    if (entropy is None) != (grad_entropy is None):
        raise ValueError("pass entropy and grad_entropy together")
    if entropy is not None:
        _vec(entropy, "entropy", (rows,), f32, device)
        _vec(grad_entropy, "grad_entropy", (rows,), f32, device)
    if out is not None:
        _check_grad(out, logits)

    def call(st):
        g = _like(torch, logits, rows, V, ld) if out is None else out
        check(lib().quasar_token_logprobs_grad(logits.data_ptr(), dt, ld, rows, V, targets.data_ptr(), temperature,
                                               stats.data_ptr(), _p(entropy), grad_logprob.data_ptr(), _p(grad_entropy),
                                               g.data_ptr(), _ld(g), st), "quasar_token_logprobs_grad")
        if out is not None:
            _wrote(torch, out)
        return g
    return _on(torch, device, stream, (logits, targets, stats, grad_logprob, entropy, grad_entropy, out), call)


def policy_loss(logits, targets, old_logprob, advantage, *, ref_logprob=None, weight=None, temperature: float = 1.0,
                clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0, entropy_coef: float = 0.0,
                grad_scale: float = 1.0, entropy: bool = False, grad=True, out: Optional[PolicyLoss] = None,
                stream=None) -> PolicyLoss:
    """Clipped policy loss of the rows' tokens, with an optional KL term and entropy bonus, and its gradient.

    ratio = exp(logprob - old_logprob), u = ref_logprob - logprob:
      row_loss = -min(ratio * A, clip(ratio, 1 - clip_low, 1 + clip_high) * A) + kl_coef * (exp(u) - u - 1)
                 - entropy_coef * entropy
      loss     = sum(weight * row_loss)
    old_logprob, advantage, ref_logprob, weight: [rows] float32. weight None: 1/rows each; a weight of 0 leaves the
    row out like a negative target. entropy: return the rows' entropies (they are returned whenever entropy_coef
    is not 0). grad: True to allocate the gradient, a tensor to write (``logits`` itself: in place), False for
    none. grad_scale multiplies the gradient, not the loss. out: a PolicyLoss of an earlier call whose tensors
    other than grad are written again.
    """
    torch, rows, V, dt, ld, device = _rows(logits, targets)
    f32 = torch.float32
    shape = (rows,)
    _vec(old_logprob, "old_logprob", shape, f32, device)
    _vec(advantage, "advantage", shape, f32, device)
    if ref_logprob is not None:
        _vec(ref_logprob, "ref_logprob", shape, f32, device)
    elif kl_coef != 0.0:
        raise ValueError("kl_coef needs ref_logprob")
    if weight is not None:
        _vec(weight, "weight", shape, f32, device)
    want = entropy or entropy_coef != 0.0
    buf = _grad_arg(torch, grad, logits)
    if out is not None:
        _vec(out.loss, "out.loss", (), f32, device)
        _vec(out.logprob, "out.logprob", shape, f32, device)
        _vec(out.row_loss, "out.row_loss", shape, f32, device)
        if want != (out.entropy is not None):
            raise ValueError("out.entropy must be a tensor if the entropy is computed, and None if not")
        if want:
            _vec(out.entropy, "out.entropy", shape, f32, device)
    prm = PolicyParams(temperature, clip_low, clip_high, kl_coef, entropy_coef, grad_scale)

    def call(st):
        g = _like(torch, logits, rows, V, ld) if grad is True else buf
        if out is None:
            e = logits.new_empty
            o = PolicyLoss(e((), dtype=f32), e(rows, dtype=f32), e(rows, dtype=f32) if want else None,
                           e(rows, dtype=f32), g)
        else:
            o = PolicyLoss(out.loss, out.logprob, out.entropy, out.row_loss, g)
        check(lib().quasar_policy_loss(logits.data_ptr(), dt, ld, rows, V, targets.data_ptr(), old_logprob.data_ptr(),
                                       advantage.data_ptr(), _p(ref_logprob), _p(weight), ctypes.addressof(prm),
                                       o.logprob.data_ptr(), _p(o.entropy), o.row_loss.data_ptr(), o.loss.data_ptr(),
                                       _p(g), 0 if g is None else _ld(g), st), "quasar_policy_loss")
        if out is not None:
            _wrote(torch, *o[:4], buf)
        elif buf is not None:
            _wrote(torch, buf)
        return o
    used = (logits, targets, old_logprob, advantage, ref_logprob, weight, buf, *(out or ()))
    return _on(torch, device, stream, used, call)


def preference_loss(logits, targets, cu_seqlens, *, ref_logprob=None, pair_weight=None, temperature: float = 1.0,
                    beta: float = 0.1, label_smoothing: float = 0.0, length_normalize: bool = False,
                    grad_scale: float = 1.0, grad=True, out: Optional[PreferenceLoss] = None,
                    stream=None) -> PreferenceLoss:
    """Preference loss over pairs of packed sequences (chosen, rejected, chosen, ...) and its gradient.

    cu_seqlens: [2 * pairs + 1] int32 row offsets; a row counts if its target is not negative. With a sequence's
    score the sum (length_normalize: the mean) of its log-probabilities less ref_logprob ([2 * pairs] float32):
      x         = beta * (score_chosen - score_rejected)
      pair_loss = -(1 - label_smoothing) * ln sigmoid(x) - label_smoothing * ln sigmoid(-x)
      loss      = sum(pair_weight * pair_loss)                  (pair_weight None: 1/pairs each)
    grad, grad_scale, out: as for ``policy_loss``.
    """
    torch, rows, V, dt, ld, device = _rows(logits, targets)
    f32 = torch.float32
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] % 2 == 0:
        raise ValueError("cu_seqlens must have 2 * pairs + 1 offsets")
    n = cu_seqlens.shape[0] - 1
    if n // 2 > _INT_MAX:
        raise ValueError(f"cu_seqlens has too many offsets: {n + 1}")
    _vec(cu_seqlens, "cu_seqlens", (n + 1,), torch.int32, device)
    if ref_logprob is not None:
        _vec(ref_logprob, "ref_logprob", (n,), f32, device)
    if pair_weight is not None:
        _vec(pair_weight, "pair_weight", (n // 2,), f32, device)
    buf = _grad_arg(torch, grad, logits)
    if out is not None:
        for name, shape in (("loss", ()), ("pair_loss", (n // 2,)), ("seq_logprob", (n,)), ("logprob", (rows,)),
                            ("stats", (rows, 2)), ("row_grad", (rows,))):
            _vec(getattr(out, name), "out." + name, shape, f32, device)
    prm = PreferenceParams(temperature, beta, label_smoothing, grad_scale, 1 if length_normalize else 0, 0)

    def call(st):
        g = _like(torch, logits, rows, V, ld) if grad is True else buf
        if out is None:
            e = logits.new_empty
            o = PreferenceLoss(e((), dtype=f32), e(n // 2, dtype=f32), e(n, dtype=f32), e(rows, dtype=f32),
                               e((rows, 2), dtype=f32), e(rows, dtype=f32), g)
        else:
            o = PreferenceLoss(*out[:6], g)
        check(lib().quasar_preference_loss(logits.data_ptr(), dt, ld, rows, V, targets.data_ptr(),
                                           cu_seqlens.data_ptr(), n // 2, _p(ref_logprob), _p(pair_weight),
                                           ctypes.addressof(prm), o.logprob.data_ptr(), o.seq_logprob.data_ptr(),
                                           o.pair_loss.data_ptr(), o.loss.data_ptr(), o.stats.data_ptr(),
                                           o.row_grad.data_ptr(), _p(g), 0 if g is None else _ld(g), st),
              "quasar_preference_loss")
        if out is not None:
            _wrote(torch, *o[:6], buf)
        elif buf is not None:
            _wrote(torch, buf)
        return o
    used = (logits, targets, cu_seqlens, ref_logprob, pair_weight, buf, *(out or ()))
    return _on(torch, device, stream, used, call)


__all__ = ["TokenLogprobs", "PolicyLoss", "PreferenceLoss", "PolicyParams", "PreferenceParams", "token_logprobs",
           "token_logprobs_grad", "policy_loss", "preference_loss"]

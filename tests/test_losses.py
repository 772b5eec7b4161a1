"""CPU checks of the log-probability and loss entries: the C entries and the
Python wrappers refuse bad arguments before anything reaches a GPU."""
import ctypes
import subprocess
import sys

import pytest

P = ctypes.c_void_p
EINVAL = -1


def _lib():
    import quasar_b200 as q
    return q.lib()


def test_import_needs_no_torch():
    code = "import sys, quasar_b200; assert 'torch' not in sys.modules"
    subprocess.run([sys.executable, "-c", code], check=True)


def logprobs(**kw):
    a = dict(logits=P(4096), dtype=0, ld=16, rows=2, V=16, targets=P(64), T=1.0, logprob=P(128), entropy=None, stats=None)
    a.update(kw)
    return _lib().quasar_token_logprobs(a["logits"], a["dtype"], a["ld"], a["rows"], a["V"], a["targets"], a["T"],
                                        a["logprob"], a["entropy"], a["stats"], None)


def logprobs_grad(**kw):
    a = dict(logits=P(4096), dtype=0, ld=16, rows=2, V=16, targets=P(64), T=1.0, stats=P(64), entropy=None, g=P(64),
             ge=None, grad=P(8192), grad_ld=16)
    a.update(kw)
    return _lib().quasar_token_logprobs_grad(a["logits"], a["dtype"], a["ld"], a["rows"], a["V"], a["targets"], a["T"],
                                             a["stats"], a["entropy"], a["g"], a["ge"], a["grad"], a["grad_ld"], None)


def policy(prm=(1.0, 0.2, 0.2, 0.0, 0.0, 1.0), **kw):
    from quasar_b200.losses import PolicyParams
    a = dict(logits=P(4096), dtype=0, ld=16, rows=2, V=16, targets=P(64), old=P(64), adv=P(64), ref=None, weight=None,
             logprob=P(64), entropy=None, row_loss=P(64), loss=P(64), grad=P(8192), grad_ld=16)
    a.update(kw)
    rec = None if prm is None else PolicyParams(*prm)
    p = None if rec is None else ctypes.addressof(rec)
    return _lib().quasar_policy_loss(a["logits"], a["dtype"], a["ld"], a["rows"], a["V"], a["targets"], a["old"],
                                     a["adv"], a["ref"], a["weight"], p, a["logprob"], a["entropy"], a["row_loss"],
                                     a["loss"], a["grad"], a["grad_ld"], None)


def preference(prm=(1.0, 0.1, 0.0, 1.0, 0, 0), **kw):
    from quasar_b200.losses import PreferenceParams
    a = dict(logits=P(4096), dtype=0, ld=16, rows=2, V=16, targets=P(64), cu=P(64), pairs=1, ref=None, weight=None,
             logprob=P(64), seq=P(64), pair_loss=P(64), loss=P(64), stats=P(64), row_grad=P(64), grad=P(8192),
             grad_ld=16)
    a.update(kw)
    rec = None if prm is None else PreferenceParams(*prm)
    p = None if rec is None else ctypes.addressof(rec)
    return _lib().quasar_preference_loss(a["logits"], a["dtype"], a["ld"], a["rows"], a["V"], a["targets"], a["cu"],
                                         a["pairs"], a["ref"], a["weight"], p, a["logprob"], a["seq"], a["pair_loss"],
                                         a["loss"], a["stats"], a["row_grad"], a["grad"], a["grad_ld"], None)


ROWS = [dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(V=0, ld=0), dict(ld=15), dict(V=(1 << 20) + 1, ld=1 << 21),
        dict(logits=None), dict(targets=None), dict(logits=P(4098)), dict(dtype=1, logits=P(4097)), dict(targets=P(66)),
        dict(ld=1 << 62)]
BAD_T = [0.0, -1.0, float("inf"), float("nan"), 1e-39]


@pytest.mark.parametrize("bad", ROWS, ids=str)
@pytest.mark.parametrize("call", [logprobs, logprobs_grad, policy, preference])
def test_rows_are_checked(call, bad):
    assert call(**bad) == EINVAL


@pytest.mark.parametrize("T", BAD_T)
def test_temperature_is_checked(T):
    assert logprobs(T=T) == EINVAL
    assert logprobs_grad(T=T) == EINVAL
    assert policy(prm=(T, 0.2, 0.2, 0.0, 0.0, 1.0)) == EINVAL
    assert preference(prm=(T, 0.1, 0.0, 1.0, 0, 0)) == EINVAL


# the logits take bytes 4096..4223 (two rows of sixteen floats)
@pytest.mark.parametrize("bad", [dict(grad_ld=15), dict(grad=P(4096 + 64)), dict(grad=P(4096 - 64)), dict(grad=P(4096), grad_ld=17),
                                 dict(grad=P(8194)), dict(grad=P(4220)), dict(grad_ld=1 << 62)], ids=str)
@pytest.mark.parametrize("call", [logprobs_grad, policy, preference])
def test_gradients_are_checked(call, bad):
    assert call(**bad) == EINVAL


def test_buffers_are_checked():
    assert logprobs(logprob=None) == EINVAL
    assert logprobs_grad(stats=None) == EINVAL
    assert logprobs_grad(g=None) == EINVAL
    assert logprobs_grad(grad=None) == EINVAL
    assert logprobs_grad(entropy=P(64)) == EINVAL      # an entropy without its gradient
    assert logprobs_grad(ge=P(64)) == EINVAL
    for name in ("old", "adv", "logprob", "row_loss", "loss"):
        assert policy(**{name: None}) == EINVAL
    assert policy(prm=None) == EINVAL
    for name in ("cu", "logprob", "seq", "pair_loss", "loss", "stats", "row_grad"):
        assert preference(**{name: None}) == EINVAL
    assert preference(prm=None) == EINVAL
    assert preference(pairs=-1) == EINVAL


@pytest.mark.parametrize("prm", [(1.0, -0.1, 0.2, 0.0, 0.0, 1.0), (1.0, 0.2, -0.1, 0.0, 0.0, 1.0),
                                 (1.0, float("nan"), 0.2, 0.0, 0.0, 1.0), (1.0, 0.2, 0.2, 0.1, 0.0, 1.0),
                                 (1.0, 0.2, 0.2, float("nan"), 0.0, 1.0), (1.0, 0.2, 0.2, 0.0, float("inf"), 1.0),
                                 (1.0, 0.2, 0.2, 0.0, 0.0, float("nan"))])
def test_policy_parameters_are_checked(prm):
    assert policy(prm=prm) == EINVAL  # the fourth: a KL term without reference log-probabilities


@pytest.mark.parametrize("prm", [(1.0, float("nan"), 0.0, 1.0, 0, 0), (1.0, 0.1, -0.1, 1.0, 0, 0),
                                 (1.0, 0.1, 1.5, 1.0, 0, 0), (1.0, 0.1, 0.0, float("inf"), 0, 0)])
def test_preference_parameters_are_checked(prm):
    assert preference(prm=prm) == EINVAL


def test_no_rows_is_no_launch():
    assert logprobs(rows=0, logits=None, targets=None, logprob=None) == 0
    assert logprobs_grad(rows=0, logits=None, targets=None, stats=None, g=None, grad=None) == 0


def test_wrappers_refuse_host_tensors():
    import torch
    import quasar_b200 as q
    l, t, f = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32), torch.zeros(2)
    for call in (lambda: q.token_logprobs(l, t), lambda: q.token_logprobs_grad(l, t, torch.zeros(2, 2), f),
                 lambda: q.policy_loss(l, t, f, f), lambda: q.preference_loss(l, t, t)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        q.token_logprobs(l.double(), t)
    with pytest.raises(ValueError, match=r"\[rows, V\]"):
        q.token_logprobs(l[0], t)


def test_parameter_records_match_the_header():
    from quasar_b200.losses import PolicyParams, PreferenceParams
    assert ctypes.sizeof(PolicyParams) == 24
    assert ctypes.sizeof(PreferenceParams) == 24


@pytest.mark.parametrize("wait,chunks", [(-1, 0), ((1 << 32) + 1, 0), (1, -1)])
def test_self_test_arguments_are_checked(wait, chunks):
    from quasar_b200.losses import PolicyParams
    rec = PolicyParams(1.0, 0.2, 0.2, 0.0, 0.0, 1.0)
    assert _lib().quasar_selftest_stalled_policy_loss(wait, chunks, P(4096), 0, 16, 2, 16, P(64), P(64), P(64), None, None,
                                                      ctypes.addressof(rec), P(64), None, P(64), P(64), P(8192), 16,
                                                      None) == EINVAL

"""What the losses on the scores of a vocabulary refuse. Arguments are checked before anything is launched, so no GPU is needed: the
addresses are made up and never followed."""
import ctypes as ct

import pytest

import nnforge_b200.capi as capi

INVALID, UNSUPPORTED = -1, -2
ADDRESS = 1 << 20
F32, BF16, F16, I32, I64 = range(5)


def matrix(rows=4, cols=100, stride=None, type=BF16, data=ADDRESS):
    return capi.Matrix(data, type, rows, cols, cols if stride is None else stride)


def indices(type=I64, data=ADDRESS):
    return capi.Indices(data, type)


def forward(logits=None, tokens=None, logp=ADDRESS, tau=1.0):
    return capi.lib.nnf_token_logp_fwd(None, logp, None, logits, tokens, tau)


def backward(dlogits, logits, tokens=None, dlogp=ADDRESS, saved=ADDRESS, tau=1.0, add=0):
    return capi.lib.nnf_token_logp_bwd(None, dlogits, dlogp, logits, tokens or indices(), saved, tau, add)


def policy(logits=None, dlogits=None, tokens=None, loss=ADDRESS, old=ADDRESS, adv=ADDRESS, low=0.2, high=0.2, add=0, tau=1.0):
    return capi.lib.nnf_policy_loss(None, loss, ADDRESS, None, dlogits, logits or matrix(), tokens or indices(), old, adv, None, None, low, high, 0.0, tau, 1.0, add)


def preference(logits=None, dlogits=None, tokens=None, offsets=None, pairs=2, loss=ADDRESS, saved=ADDRESS, kind=0, beta=0.1, smoothing=0.0, tau=1.0):
    return capi.lib.nnf_preference_loss(None, loss, ADDRESS, ADDRESS, saved, ADDRESS, dlogits, logits or matrix(), tokens or indices(), offsets or indices(), pairs,
                                        ADDRESS, kind, beta, smoothing, 0, tau, 1.0, 0)


def distill(logits=None, dlogits=None, ids=None, top=None, loss=ADDRESS, tau=1.0, add=0):
    return capi.lib.nnf_distill_topk_loss(None, loss, dlogits, logits or matrix(), ids or matrix(cols=8, type=I32), top or matrix(cols=8), None, tau, 1.0, add)


LOGITS = [
    (dict(type=I32), INVALID, "type"), (dict(type=7), INVALID, "type"), (dict(rows=-1), INVALID, "extents"), (dict(cols=0), INVALID, "extents"),
    (dict(stride=99), INVALID, "extents"), (dict(stride=0), INVALID, "extents"), (dict(data=None), INVALID, "null"), (dict(data=ADDRESS + 1), INVALID, "misaligned"),
    (dict(type=F32, data=ADDRESS + 2), INVALID, "misaligned"), (dict(type=F32, cols=(1 << 18) + 1), UNSUPPORTED, "1 MiB"), (dict(cols=(1 << 19) + 1), UNSUPPORTED, "1 MiB"),
]


@pytest.mark.parametrize("bad,status,text", LOGITS)
@pytest.mark.parametrize("call", [lambda x: forward(x, indices()), lambda x: backward(matrix(), x), policy, preference, distill])
def test_logits(call, bad, status, text):
    assert call(matrix(**bad)) == status
    assert text in capi.last_error()


@pytest.mark.parametrize("tau", [0.0, -1.0, float("nan"), float("inf"), 1e-38])
def test_temperatures(tau):
    for status in (forward(matrix(), indices(), tau=tau), backward(matrix(), matrix(), tau=tau), policy(tau=tau), preference(tau=tau), distill(tau=tau)):
        assert status == INVALID and "temperature" in capi.last_error()


@pytest.mark.parametrize("bad", [dict(type=F32), dict(rows=5), dict(cols=101), dict(rows=3)])
def test_gradients_of_another_shape_or_type(bad):
    for status in (backward(matrix(data=1 << 21, **bad), matrix()), policy(dlogits=matrix(data=1 << 21, **bad)), preference(dlogits=matrix(data=1 << 21, **bad)),
                   distill(dlogits=matrix(data=1 << 21, **bad))):
        assert status == INVALID and "another type or shape" in capi.last_error()


def test_gradients_in_the_logits_place():
    for status in (backward(matrix(), matrix(), add=1), policy(dlogits=matrix(), add=1), distill(dlogits=matrix(stride=128)), policy(dlogits=matrix(stride=104))):
        assert status == INVALID and "place" in capi.last_error()
    assert backward(None, matrix()) == INVALID and "dlogits" in capi.last_error()


def test_indices():
    for bad, text in ((indices(type=F32), "type"), (indices(data=None), "null"), (indices(data=ADDRESS + 4), "misaligned"), (indices(type=I32, data=ADDRESS + 2), "misaligned")):
        for status in (forward(matrix(), bad), backward(matrix(data=1 << 21), matrix(), tokens=bad), policy(tokens=bad), preference(tokens=bad), preference(offsets=bad)):
            assert status == INVALID and text in capi.last_error()
    assert forward(matrix(), None) == INVALID and "tokens" in capi.last_error()


def test_null_pointers():
    for status in (forward(matrix(), indices(), logp=None), backward(matrix(data=1 << 21), matrix(), dlogp=None), backward(matrix(data=1 << 21), matrix(), saved=None),
                   policy(loss=None), policy(old=None), policy(adv=None), preference(loss=None), preference(saved=None), distill(loss=None), forward(None, indices())):
        assert status == INVALID and "null" in capi.last_error()


def test_clipping_beta_and_kinds():
    for low, high in ((-0.1, 0.2), (1.5, 0.2), (0.2, -0.1), (float("nan"), 0.2), (0.2, float("nan"))):
        assert policy(low=low, high=high) == INVALID and "ratios" in capi.last_error()
    for bad in (dict(beta=0.0), dict(beta=-1.0), dict(beta=float("nan")), dict(beta=float("inf")), dict(smoothing=-0.1), dict(smoothing=1.1), dict(pairs=-1)):
        assert preference(**bad) == INVALID and "beta" in capi.last_error()
    assert preference(kind=2) == INVALID and "kind" in capi.last_error()
    assert preference(pairs=1 << 30) == UNSUPPORTED


def test_teachers():
    for bad in (dict(ids=matrix(rows=3, cols=8, type=I32)), dict(ids=matrix(cols=9, type=I32)), dict(top=matrix(rows=5, cols=8))):
        assert distill(**bad) == INVALID and "[rows][kept]" in capi.last_error()
    assert distill(ids=matrix(cols=8, type=BF16)) == INVALID and "teacher ids" in capi.last_error()
    assert distill(top=matrix(cols=8, type=I32)) == INVALID and "teacher logits" in capi.last_error()
    assert distill(ids=matrix(cols=1025, type=I64), top=matrix(cols=1025)) == UNSUPPORTED and "1024" in capi.last_error()


def test_nothing_to_do_is_fine():
    assert forward(matrix(rows=0, data=None), None) == 0
    assert backward(matrix(rows=0, data=None), matrix(rows=0, data=None)) == 0
    assert policy(matrix(rows=0, data=None), tokens=indices(data=None)) == 0
    assert preference(pairs=0) == 0
    assert distill(matrix(rows=0), ids=matrix(rows=0, cols=8, type=I32), top=matrix(rows=0, cols=8)) == 0


def test_structures_are_those_of_the_header():
    assert ct.sizeof(capi.Matrix) == 40 and ct.sizeof(capi.Indices) == 16
    assert capi.Matrix.rows.offset == 16 and capi.Indices.type.offset == 8


def test_what_is_no_tensor_of_a_device_is_refused():
    torch = pytest.importorskip("torch")
    x, t, v = torch.zeros(4, 10), torch.zeros(4, dtype=torch.int64), torch.zeros(4)
    calls = [lambda a: capi.token_logp_fwd(v, None, a, t, stream=0), lambda a: capi.token_logp_bwd(x, v, a, t, torch.zeros(2, 4), stream=0),
             lambda a: capi.policy_loss(v, v, a, t, v, v, stream=0), lambda a: capi.preference_loss(v, v, v, v, v, a, t, t, v, stream=0),
             lambda a: capi.distill_topk_loss(v, a, x, x, stream=0)]
    for call in calls:
        with pytest.raises(AssertionError, match="a CUDA tensor"):
            call(x)
        with pytest.raises((TypeError, AssertionError), match="a tensor is expected|a CUDA tensor"):
            call("logits")

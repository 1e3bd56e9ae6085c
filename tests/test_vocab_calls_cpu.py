"""Gradients that overlap the logits, but do not take their place, are refused before anything is launched: the addresses are made up."""
import random

import pytest

import nnforge_b200.capi as capi

INVALID = -1
BASE = 1 << 24
F32, BF16 = 0, 1


def matrix(data, rows, cols, stride, type):
    return capi.Matrix(data, type, rows, cols, stride)


def calls(x, dx):
    tokens = capi.Indices(1 << 20, 4)
    ids, top = matrix(1 << 20, x.rows, 4, 4, 3), matrix(1 << 20, x.rows, 4, 4, F32)
    a = 1 << 20
    yield lambda: capi.lib.nnf_token_logp_bwd(None, dx, a, x, tokens, a, 1.0, 0)
    yield lambda: capi.lib.nnf_policy_loss(None, a, a, None, dx, x, tokens, a, a, None, None, 0.2, 0.2, 0.0, 1.0, 1.0, 0)
    yield lambda: capi.lib.nnf_preference_loss(None, a, a, a, a, a, dx, x, tokens, tokens, 1, a, 0, 0.1, 0.0, 0, 1.0, 1.0, 0)
    yield lambda: capi.lib.nnf_distill_topk_loss(None, a, dx, x, ids, top, None, 1.0, 1.0, 1)


@pytest.mark.parametrize("rows,cols,stride,to_stride,apart", [
    (4, 100, 100, 100, 1), (4, 100, 100, 100, -1), (4, 100, 100, 100, 100), (4, 100, 100, 100, -300), (4, 100, 128, 128, 29), (4, 100, 200, 200, 99),
    (4, 100, 250, 250, 151), (1, 100, 100, 100, 99), (1, 100, 5000, 7000, -99), (4, 100, 200, 100, 0 + 100), (4, 100, 100, 400, -150), (5, 10, 20, 30, 5)])
@pytest.mark.parametrize("type,size", [(F32, 4), (BF16, 2)])
def test_refused(rows, cols, stride, to_stride, apart, type, size):
    for call in calls(matrix(BASE, rows, cols, stride, type), matrix(BASE + apart * size, rows, cols, to_stride, type)):
        assert call() == INVALID
        assert "overlap" in capi.last_error()


def test_refused_where_an_element_is_shared():
    """Random rows and strides: refused where the two sets of elements meet (where they do not, the call would be launched: not made here)."""
    rng = random.Random(7)
    made = 0
    while made < 300:
        rows, cols = rng.randint(1, 6), rng.randint(1, 12)
        stride, to_stride = cols + rng.choice([0, 0, 3, cols, 2 * cols, 17]), cols + rng.choice([0, 0, 3, cols, 2 * cols, 17])
        apart = rng.randint(-90, 90)
        mine = {r * stride + c for r in range(rows) for c in range(cols)}
        its = {apart + r * to_stride + c for r in range(rows) for c in range(cols)}
        if apart == 0 or not mine & its:
            continue
        made += 1
        for call in calls(matrix(BASE, rows, cols, stride, F32), matrix(BASE + 4 * apart, rows, cols, to_stride, F32)):
            assert call() == INVALID and "overlap" in capi.last_error()

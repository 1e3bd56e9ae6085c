"""Calls of the losses on the scores of a vocabulary that the documentation allows and that are not the ordinary ones, against the 64-bit
evaluations of vocab_exact.py (whose tolerances they share) or against another call that has to give the same bits."""
import pytest

import vocab_exact as exact

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def capi():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import nnforge_b200.capi as capi
    return capi


@pytest.fixture(autouse=True)
def errors(capi):
    yield
    assert capi.fused_error_check() == 0
    capi.set_tuning("reset", 0)


def generator(salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(4321 + salt)
    return g


def scores(g, rows, cols, dtype, spread=3.0):
    return (torch.randn(rows, cols, device="cuda", generator=g) * spread).to(dtype)


# ---- the loss alone, with the flag that a gradient would be added --------------------------------------------------


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols,kept", [(4, 100, 5), (40, 1000, 64), (3, 5000, 300), (2, 40000, 17)])
def test_the_loss_alone_is_added_to_nothing(capi, rows, cols, kept, dtype):
    """dlogits None and add_to_destination: there is no gradient to be added to, the loss is that of the call without the flag."""
    g = generator(rows + cols)
    x = scores(g, rows, cols, TYPES[dtype])
    ids = torch.rand(rows, cols, device="cuda", generator=g).topk(kept, dim=1).indices
    top = torch.randn(rows, kept, device="cuda", generator=g)
    loss, flagged = torch.full((rows,), 7.0, device="cuda"), torch.full((rows,), 5.0, device="cuda")
    capi.distill_topk_loss(loss, x, ids, top)
    capi.distill_topk_loss(flagged, x, ids, top, add_to_destination=True)
    exact.check(flagged, *exact.distill(x, ids, top, None, 1.0, 1.0)["loss"], "distillation")
    assert torch.equal(loss, flagged)
    tokens = torch.randint(0, cols, (rows,), device="cuda", generator=g)
    old, adv = torch.full((rows,), -3.0, device="cuda"), torch.randn(rows, device="cuda", generator=g)
    logp, flagged_logp = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    capi.policy_loss(loss, logp, x, tokens, old, adv)
    capi.policy_loss(flagged, flagged_logp, x, tokens, old, adv, add_to_destination=True)
    assert torch.equal(loss, flagged) and torch.equal(logp, flagged_logp)
    if rows == 4:
        offsets = torch.tensor([0, 1, 4], device="cuda")
        given = []
        for add in (False, True):
            given.append([torch.full(size, 7.0, device="cuda") for size in ((1,), (2,), (4,), (2, 4), (4,))])
            capi.preference_loss(*given[-1], x, tokens, offsets, torch.zeros(2, device="cuda"), add_to_destination=add)
        assert all(torch.equal(a, b) for a, b in zip(*given))

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


# ---- outputs in the place of inputs that have an element for each row ----------------------------------------------


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("split", [0, 2, 8])
@pytest.mark.parametrize("rows,cols", [(3, 90), (200, 1500), (6, 5000), (12, 32000), (7, 70001), (300, 40000)])
def test_outputs_in_the_place_of_inputs(capi, rows, cols, split, dtype):
    """A row's numbers are read before another of its CTAs writes its results, so that both calls give the same bits; ratios are far from 1,
    which is what a ratio of logp to itself would be."""
    g = generator(rows * 3 + cols + split)
    x = scores(g, rows, cols, TYPES[dtype])
    tokens = torch.randint(0, cols, (rows,), device="cuda", generator=g)
    tokens[rows // 2] = -100
    old = (exact.token_logp(x, tokens, 1.0)[0] - 0.5 * torch.randn(rows, device="cuda", generator=g)).float()
    adv, ref = torch.randn(rows, device="cuda", generator=g), old + 0.3 * torch.randn(rows, device="cuda", generator=g)
    mask = (torch.rand(rows, device="cuda", generator=g) > 0.2).float() * 0.5
    capi.set_tuning("vocab_split", split)

    def policy(loss, logp, kl, old, adv, ref, mask):
        dx = torch.full_like(x, 7.0)
        capi.policy_loss(loss, logp, x, tokens, old, adv, ref_logp=ref, mask=mask, kl=kl, dlogits=dx, clip_low=0.2, clip_high=0.3, kl_coef=0.1)
        return loss, logp, kl, dx

    def copies():
        return [v.clone() for v in (old, adv, ref, mask)]

    want = policy(*(torch.empty(rows, device="cuda") for _ in range(3)), *copies())
    for loss_at, logp_at, kl_at in ((1, 0, 2), (3, 2, 0), (0, 1, 3)):
        given = copies()
        got = policy(given[loss_at], given[logp_at], given[kl_at], *given)
        for name, a, b in zip(("loss", "logp", "kl", "dlogits"), got, want):
            assert torch.equal(a, b), (name, loss_at, logp_at, kl_at)
    ids = torch.rand(rows, cols, device="cuda", generator=g).topk(20, dim=1).indices
    top = torch.randn(rows, 20, device="cuda", generator=g)
    results = []
    for place in (False, True):
        weights, dx = mask.clone(), torch.full_like(x, 7.0)
        loss = weights if place else torch.empty(rows, device="cuda")
        capi.distill_topk_loss(loss, x, ids, top, mask=weights, dlogits=dx)
        results.append((loss, dx))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("average", [False, True])
def test_rewards_in_the_place_of_the_reference(capi, average):
    """Every thread of a pair's CTA takes the reference before one of them writes the rewards."""
    g = generator(77)
    x = scores(g, 3000, 40, torch.float32)
    tokens = torch.randint(0, 40, (3000,), device="cuda", generator=g)
    offsets = torch.arange(0, 3001, 3, device="cuda")
    ref = torch.randn(1000, device="cuda", generator=g) * 4 - 9
    results = []
    for place in (False, True):
        given = ref.clone()
        rewards = given if place else torch.empty(1000, device="cuda")
        loss, logp, saved, dlogp = torch.empty(500, device="cuda"), torch.empty(3000, device="cuda"), torch.empty(2, 3000, device="cuda"), torch.empty(3000, device="cuda")
        dx = torch.empty_like(x)
        capi.preference_loss(loss, rewards, logp, saved, dlogp, x, tokens, offsets, given, dlogits=dx, beta=0.5, average=average)
        results.append((loss, rewards, logp, saved, dlogp, dx))
    assert all(torch.equal(a, b) for a, b in zip(*results))


# ---- temperatures and sums ------------------------------------------------------------------------------------------


@pytest.fixture(params=["built-in choice", "a CTA a row", "split", "warps"])
def form(request, capi):
    """The forms of the scoring kernels, whatever the sizes for which each is chosen."""
    capi.set_tuning("vocab_form", {"b": 0, "a": 2, "s": 2, "w": 3}[request.param[0]])
    capi.set_tuning("vocab_split", {"a": 1, "s": 4}.get(request.param[0], 0))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("tau", [1e30, 1e33, 1e37])
@pytest.mark.parametrize("rows,cols", [(5, 700), (3, 20001)])
def test_temperatures_as_large_as_the_scores(capi, form, rows, cols, tau, dtype):
    """Scores of three times the temperature, as ordinary scores are at 1: no correction of the exponents may be larger than they are."""
    g = generator(rows + cols)
    x = scores(g, rows, cols, TYPES[dtype], spread=3.0 * tau)
    x[0, cols // 2] = -float("inf")
    tokens = torch.randint(0, cols, (rows,), device="cuda", generator=g)
    tokens[0] = 0
    logp, saved = torch.empty(rows, device="cuda"), torch.empty(2, rows, device="cuda")
    capi.token_logp_fwd(logp, saved, x, tokens, temperature=tau)
    want, want_saved, _, tol, _ = exact.token_logp(x, tokens, float(torch.tensor(tau, dtype=torch.float32)))
    exact.check(logp, want, tol, "logp")
    exact.check(saved[1], want_saved[1], 150 * exact.U * want_saved[1], "sum")


def error_of_sums(x, saved, tau):
    """Relative error of saved[1] in units of 2^-24, a value a row."""
    found = []
    step = max(1, (1 << 27) // x.shape[1])
    for r in range(0, len(x), step):
        want = exact.rows(x[r:r + step], tau)[1]
        found.append((saved[1, r:r + step].double() - want) / want / exact.U)
    return torch.cat(found)


@pytest.mark.parametrize("what,dtype,cols", [("confident", "bf16", 131072), ("confident", "fp32", 131072), ("ascending", "fp32", 131072), ("ascending", "fp32", 262140),
                                             ("ascending", "bf16", 32000), ("flat", "fp32", 131072)])
@pytest.mark.parametrize("rows", ["full turns", 96])
def test_long_sums(capi, form, rows, what, dtype, cols):
    """Rows whose sum has many steps: a score far above a hundred thousand others, scores in ascending order, scores nearly alike. Roundings to
    nearest have no sign, so that over many rows the error's mean shows what is systematic. An approximate power is 0 to 2.3u short
    (u = 2^-24), a term has two of them, and 1.7u are put back: between -3u and 1.7u, and 1u for the sums within a step. 32 rows an SM are
    what the built-in choice gives to warps whatever the rows' length: up to 512 steps."""
    if rows == "full turns":
        rows = 32 * torch.cuda.get_device_properties(0).multi_processor_count
    g = generator(cols)
    if what == "ascending":
        x = (torch.linspace(-1.0, 1.0, cols, device="cuda") + torch.rand(rows, 1, device="cuda", generator=g)).to(TYPES[dtype])
    else:
        x = scores(g, rows, cols, TYPES[dtype], spread=2.5 if what == "confident" else 0.1)
    tokens = torch.randint(0, cols, (rows,), device="cuda", generator=g)
    if what == "confident":
        x.scatter_(1, tokens[:, None], torch.full((rows, 1), 24.0, dtype=x.dtype, device="cuda"))
    logp, saved = torch.empty(rows, device="cuda"), torch.empty(2, rows, device="cuda")
    capi.token_logp_fwd(logp, saved, x, tokens)
    error = error_of_sums(x, saved, 1.0)
    assert float(error.abs().max()) <= 120.0
    assert abs(float(error.mean())) <= 4.0


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("tau", [0.7, 1.0, 1.5, 1.7])
def test_the_mean_error_of_log_probabilities(capi, form, tau, dtype):
    """What a sequence's sum gathers. Roundings to nearest have no sign; what has one is k = log2(e)/tau and 1/tau as floats (2u and 0.5u of
    them at these temperatures, u = 2^-24, times scores that are several tau apart) and the approximate powers, 0.83u short each: two a
    term are put back, a term has one to three. So 0.83u, four standard errors of 8192 rows that are off by 5u each (0.22u), and 0.2u for
    the logarithm."""
    rows, cols = 8192, 16000
    g = generator(16)
    x = torch.randn(rows, cols, device="cuda", generator=g) * 2.5
    tokens = torch.randint(0, cols, (rows,), device="cuda", generator=g)
    x.scatter_add_(1, tokens[:, None], 4.0 + 4.0 * torch.rand(rows, 1, device="cuda", generator=g))
    x = x.to(TYPES[dtype])
    logp = torch.empty(rows, device="cuda")
    capi.token_logp_fwd(logp, None, x, tokens, temperature=tau)
    tau = float(torch.tensor(tau, dtype=torch.float32))
    error = torch.cat([logp[r:r + 1024].double() - exact.token_logp(x[r:r + 1024], tokens[r:r + 1024], tau)[0] for r in range(0, rows, 1024)]) / exact.U
    assert abs(float(error.mean())) <= 1.25


# ---- terms whose coefficient is 0 ------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows,cols", [(6, 100), (5, 5000), (3, 70001)])
def test_a_divergence_that_is_only_watched(capi, rows, cols):
    """kl_coef 0: the reference changes neither loss nor gradient, also where the divergence is infinite (a score of -infinity; logp < -100)."""
    g = generator(cols)
    x = scores(g, rows, cols, torch.float32)
    tokens = torch.randint(0, cols, (rows,), device="cuda", generator=g)
    x[0, tokens[0]] = -float("inf")
    x[1, tokens[1]] = -200.0
    old, adv, ref = torch.full((rows,), -3.0, device="cuda"), torch.randn(rows, device="cuda", generator=g), torch.full((rows,), -2.0, device="cuda")
    results = []
    for r in (None, ref):
        loss, logp, kl, dx = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.full_like(x, 7.0)
        capi.policy_loss(loss, logp, x, tokens, old, adv, ref_logp=r, kl=kl, dlogits=dx)
        results.append((loss, logp, dx))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert bool(torch.isfinite(results[1][0]).all()) and bool(torch.isfinite(results[1][2]).all())
    assert float(kl[1]) == float("inf") and bool(torch.isfinite(kl[2:]).all())


@pytest.mark.parametrize("smoothing", [0.0, 1.0])
def test_a_sequence_that_is_impossible(capi, smoothing):
    """The sequence that is to lose has a token of probability 0: no loss and no gradient without the other term of label smoothing."""
    g = generator(5)
    x = scores(g, 8, 50, torch.float32)
    tokens = torch.randint(0, 50, (8,), device="cuda", generator=g)
    loser = 5 if smoothing == 0.0 else 1   # of the first sequence, rows 0..3, or the second
    x[loser, tokens[loser]] = -float("inf")
    loss, rewards = torch.empty(1, device="cuda"), torch.empty(2, device="cuda")
    logp, dlogp, saved = torch.empty(8, device="cuda"), torch.empty(8, device="cuda"), torch.empty(2, 8, device="cuda")
    dx = torch.full_like(x, 7.0)
    capi.preference_loss(loss, rewards, logp, saved, dlogp, x, tokens, torch.tensor([0, 4, 8], device="cuda"), torch.zeros(2, device="cuda"), dlogits=dx, beta=0.5,
                         label_smoothing=smoothing)
    assert float(loss[0]) == 0.0 and not bool(dlogp.any()) and not bool(dx.any())
    assert float(rewards[1 if smoothing == 0.0 else 0]) == -float("inf")


# ---- where the gradient lies -----------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows,cols", [(1, 40), (6, 100), (5, 5001), (3, 40000)])
@pytest.mark.parametrize("layout", ["side by side", "every second row", "strides of their own", "one behind the other"])
def test_gradients_in_the_logits_buffer(capi, rows, cols, layout):
    """Logits and gradient in one buffer without a shared element, their rows between each other's: not refused, and right."""
    g = generator(rows + cols)
    buffer = torch.full((8 * rows * cols + 64,), 7.0, device="cuda")
    if layout == "side by side":
        x, dx = (torch.as_strided(buffer, (rows, cols), (3 * cols, 1), at) for at in (0, 2 * cols))
    elif layout == "every second row":
        x, dx = (torch.as_strided(buffer, (rows, cols), (2 * cols, 1), at) for at in (cols, 0))
    elif layout == "strides of their own":
        x, dx = torch.as_strided(buffer, (rows, cols), (2 * cols, 1), 0), torch.as_strided(buffer, (rows, cols), (4 * cols, 1), cols)
    else:
        x, dx = torch.as_strided(buffer, (rows, cols), (cols, 1), rows * cols), torch.as_strided(buffer, (rows, cols), (cols, 1), 0)
    x.copy_(scores(g, rows, cols, torch.float32))
    was = x.clone()
    tokens = torch.randint(0, cols, (rows,), device="cuda", generator=g)
    logp, saved, up = torch.empty(rows, device="cuda"), torch.empty(2, rows, device="cuda"), torch.randn(rows, device="cuda", generator=g)
    capi.token_logp_fwd(logp, saved, x, tokens)
    capi.token_logp_bwd(dx, up, x, tokens, saved)
    _, _, on, _, p = exact.token_logp(was, tokens, 1.0)
    want, size = exact.gradient(p, tokens, on, up.double(), up.double().abs(), 1.0)
    exact.check(dx, want, exact.GRAD * size, "dlogits")
    assert torch.equal(x, was) and int((buffer == 7.0).sum()) == buffer.numel() - 2 * rows * cols


# ---- corners ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kept", [341, 700, 1024])
@pytest.mark.parametrize("cols", [30, 1000])
def test_many_kept_logits_of_short_rows(capi, cols, kept, dtype):
    """More shared memory than a launch has without asking for it; more entries than columns, so that most are there several times."""
    g = generator(cols + kept)
    x = scores(g, 50, cols, TYPES[dtype])
    ids = torch.randint(-2, cols + 2, (50, kept), device="cuda", generator=g)
    ids[7] = -1
    top = torch.randn(50, kept, device="cuda", generator=g)
    mask = torch.rand(50, device="cuda", generator=g)
    for add in (False, True):
        loss, dx = torch.empty(50, device="cuda"), torch.zeros_like(x)
        capi.distill_topk_loss(loss, x, ids, top, mask=mask, dlogits=dx, add_to_destination=add)
        want = exact.distill(x, ids, top, mask, 1.0, 1.0)
        exact.check(loss, *want["loss"], "loss")
        exact.check(dx, *want["dlogits"], "dlogits")


def test_pairs_without_rows(capi):
    """Two pairs and no row at all: the reference alone decides."""
    x, none, tokens = torch.empty(0, 100, device="cuda"), torch.empty(0, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda")
    ref = torch.tensor([1.0, 3.0, -2.0, -5.0], device="cuda")
    for squared in (False, True):
        loss, rewards = torch.full((2,), 7.0, device="cuda"), torch.full((4,), 7.0, device="cuda")
        capi.preference_loss(loss, rewards, none, torch.empty(2, 0, device="cuda"), none, x, tokens, torch.zeros(5, dtype=torch.int64, device="cuda"), ref,
                             dlogits=torch.empty_like(x), kind=capi.PREFERENCE_SQUARED if squared else capi.PREFERENCE_LOGISTIC, beta=0.5)
        h = torch.tensor([2.0, -3.0], dtype=torch.float64)   # q = -ref
        want = (h - 1.0) ** 2 if squared else torch.nn.functional.softplus(-0.5 * h)
        # beta*h is exact; the logistic loss has an exponential, a logarithm and a sum of a few roundings each
        exact.check(loss, want, 16 * exact.U * (want + 1.0), "loss")
        assert rewards.tolist() == [-0.5, -1.5, 1.0, 2.5]


@pytest.mark.parametrize("cols", [5000, 131072])
def test_references_on_either_side_of_the_fused_arguments(capi, form, cols):
    """Scores of about 7e5, where x*k passes the 1e6 from which the difference is taken first, in ascending and in descending order, and rows that
    begin with the type's lowest value: parts of both kinds are joined. Scores are multiples of 2^-4, |x - M| < 30."""
    g = generator(cols)
    border = 1.0e6 / 1.4426950408889634
    line = (torch.linspace(-15.0, 15.0, cols, device="cuda", dtype=torch.float64) * 16).round() / 16
    rows = torch.stack([sign * (round(border) + line) for sign in (1.0, -1.0)] + [sign * (round(border) - line) for sign in (1.0, -1.0)]).float()
    low = torch.randn(3, cols, device="cuda", generator=g)
    low[0, :cols // 2] = torch.finfo(torch.float32).min
    low[1, cols // 2:] = torch.finfo(torch.float32).min
    low[2, 1::2] = -1.0e6
    x = torch.cat([rows, low])
    tokens = x.argmax(dim=1)
    tokens[1::2] = (tokens[1::2] + 7) % cols
    logp, saved = torch.empty(7, device="cuda"), torch.empty(2, 7, device="cuda")
    capi.token_logp_fwd(logp, saved, x, tokens)
    want, want_saved, _, tol, _ = exact.token_logp(x, tokens, 1.0)
    exact.check(logp, want, tol, "logp")
    exact.check(saved[0], want_saved[0], torch.zeros_like(tol), "maximum")
    exact.check(saved[1], want_saved[1], 150 * exact.U * want_saved[1], "sum")


def test_a_step_of_training_returns_its_losses(capi):
    """Policy loss and distillation into one gradient: both losses, and the gradient, against their definitions."""
    g = generator(22)
    rows, cols = 96, 1500
    x = scores(g, rows, cols, torch.float32)
    tokens = torch.randint(0, cols, (rows,), device="cuda", generator=g)
    tokens[5] = -100
    logp64 = exact.token_logp(x, tokens, 1.0)[0]
    moved = 0.1 * torch.randn(rows, device="cuda", generator=g).double().clamp(-1.5, 1.5)   # ratios within the borders
    old, adv, ref = (logp64 - moved).float(), torch.randn(rows, device="cuda", generator=g), (logp64 + 0.3).float()
    ids = torch.rand(rows, cols, device="cuda", generator=g).topk(12, dim=1).indices
    top = torch.randn(rows, 12, device="cuda", generator=g)
    loss, logp, dloss, dx = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty_like(x)
    capi.policy_loss(loss, logp, x, tokens, old, adv, ref_logp=ref, kl_coef=0.1, dlogits=dx, scale=1.0 / rows)
    capi.distill_topk_loss(dloss, x, ids, top, dlogits=dx, scale=0.5 / rows, add_to_destination=True)
    policy, teacher = exact.policy(x, tokens, old, adv, ref, None, 0.2, 0.2, 0.1, 1.0, 1.0 / rows), exact.distill(x, ids, top, None, 1.0, 0.5 / rows)
    exact.check(loss, *policy["loss"], "policy loss")
    exact.check(dloss, *teacher["loss"], "distillation")
    a, b = policy["dlogits"], teacher["dlogits"]
    exact.check(dx, a[0] + b[0], a[1] + b[1] + 2 * exact.U * (a[0].abs() + b[0].abs()), "dlogits")


def test_offsets_that_are_wrong_touch_nothing_in_front(capi):
    """Offsets below 0, behind the last row or decreasing: the memory on either side of every output stays as it was."""
    x = scores(generator(12), 12, 100, torch.float32)
    tokens = torch.randint(0, 100, (12,), device="cuda", generator=generator(13))
    for offsets in ([-5, 4, 40], [8, 4, 2], [0, 50, 12], [20, 30, 40], [-9, -7, -3]):
        guard = torch.full((5, 64), 7.0, device="cuda")
        loss, rewards, logp, dlogp, saved = guard[0, 16:17], guard[1, 16:18], guard[2, 16:28], guard[3, 16:28], guard[4, 16:40].view(2, 12)
        capi.preference_loss(loss, rewards, logp, saved, dlogp, x, tokens, torch.tensor(offsets, device="cuda"), torch.zeros(2, device="cuda"))
        for row, count in zip(guard, (1, 2, 12, 12, 24)):
            assert bool((row[:16] == 7.0).all()) and bool((row[16 + count:] == 7.0).all())


def test_kinds_beyond_32_bits(capi):
    def full(*size, dtype=torch.float32):
        return torch.zeros(*size, dtype=dtype, device="cuda")

    for kind in (2, -1, 1 << 32, (1 << 32) + 1, -(1 << 32)):
        with pytest.raises(capi.NnfError, match="kind"):
            capi.preference_loss(full(1), full(2), full(4), full(2, 4), full(4), full(4, 10), full(4, dtype=torch.int64), full(3, dtype=torch.int64), full(2), kind=kind)

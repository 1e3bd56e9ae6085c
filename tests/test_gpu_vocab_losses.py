"""The losses on the scores of a vocabulary against 64-bit evaluations of their definitions: every type, rows that start and end
anywhere, one and many rows, rows split over a cluster, rows that count for nothing, infinities and NaN, accumulation, gradients in the
logits' place, captured calls and other streams."""
import math

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


@pytest.fixture(autouse=True, params=["built-in choice", "shared memory", "shared memory, split", "warps"])
def form(request, capi):
    """Every test runs in each form of the kernels, whatever the sizes for which it is chosen."""
    capi.set_tuning("vocab_form", {"b": 0, "s": 2, "w": 3}[request.param[0]])
    capi.set_tuning("vocab_split", 4 if "split" in request.param else 0)
    yield
    assert capi.fused_error_check() == 0
    capi.set_tuning("reset", 0)


def generator(salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(1234 + salt)
    return g


def scores(g, rows, cols, dtype, stride=None, offset=0, spread=3.0):
    """Rows `stride` elements apart, `offset` elements behind an aligned address; NaN lies between them."""
    stride = stride or cols
    backing = torch.full((rows * stride + offset + 16,), float("nan"), dtype=dtype, device="cuda")
    x = backing[offset:offset + rows * stride].view(rows, stride)[:, :cols]
    x.copy_(torch.randn(rows, cols, device="cuda", generator=g) * spread)
    return x


def somewhere(g, rows, cols, out=True, dtype=torch.int64):
    t = torch.randint(0, cols, (rows,), device="cuda", generator=g)
    if out and rows > 2:
        t[rows // 2] = -100
        if rows > 4:
            t[rows - 1] = cols
            t[1] = cols + 7
    return t.to(dtype)


def room(rows, cols, dtype, stride=None, offset=0, value=7.0):
    stride = stride or cols
    backing = torch.full((rows * stride + offset + 16,), value, dtype=dtype, device="cuda")
    return backing, backing[offset:offset + rows * stride].view(rows, stride)[:, :cols]


def vectors(n, count):
    return [torch.full((n,), 7.0, device="cuda") for _ in range(count)]


SHAPES = [(1, 1), (3, 2), (5, 7), (4, 8), (6, 9), (9, 31), (7, 257), (5, 1000), (6, 1024), (300, 513), (2, 4097), (150, 5000), (3, 8191), (2, 32000), (160, 16390),
          (1, 50021), (150, 40000), (3, 131072), (2, 200003)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_token_logp(capi, rows, cols, dtype):
    g = generator(rows * 7 + cols)
    x = scores(g, rows, cols, TYPES[dtype])
    tokens = somewhere(g, rows, cols, dtype=torch.int32 if rows % 2 else torch.int64)
    tau = [1.0, 0.7, 2.5][(rows + cols) % 3]
    logp, dlogp = vectors(rows, 2)
    saved = torch.full((2, rows), 7.0, device="cuda")
    capi.token_logp_fwd(logp, saved, x, tokens, temperature=tau)
    want, want_saved, on, tol, p = exact.token_logp(x, tokens, tau)
    exact.check(logp, want, tol, "logp")
    exact.check(saved[0], want_saved[0], torch.zeros_like(tol), "maximum")
    exact.check(saved[1], want_saved[1], 150 * exact.U * want_saved[1], "sum")
    other = torch.empty(rows, device="cuda")
    capi.token_logp_fwd(other, None, x, tokens, temperature=tau)
    assert torch.equal(other, logp)
    dlogp.copy_(torch.randn(rows, device="cuda", generator=g))
    if rows > 3:
        dlogp[3] = 0.0
    backing, dx = room(rows, cols, TYPES[dtype])
    capi.token_logp_bwd(dx, dlogp, x, tokens, saved, temperature=tau)
    want_dx, size = exact.gradient(p, tokens, on, dlogp.double(), dlogp.double().abs(), tau)
    exact.check(dx, want_dx, exact.GRAD * size, "dlogits")
    assert bool((backing[rows * cols:] == 7.0).all())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols,stride,offset,to_stride,to_offset", [
    (5, 1000, 1003, 1, 1003, 1), (5, 1000, 1003, 0, 1000, 0), (4, 33, 40, 3, 40, 3), (4, 33, 41, 3, 35, 2), (3, 20001, 20004, 5, 20004, 5), (3, 20001, 20001, 0, 20001, 1),
    (2, 70001, 70003, 2, 70003, 2), (2, 70001, 70008, 0, 70001, 3), (6, 3, 5, 1, 3, 0)])
def test_rows_that_start_anywhere(capi, rows, cols, stride, offset, to_stride, to_offset, dtype):
    """Strides and addresses off the 16-byte boundary, the gradient's other than the logits': the neighbours stay as they were."""
    g = generator(cols + stride)
    x = scores(g, rows, cols, TYPES[dtype], stride, offset)
    tokens = somewhere(g, rows, cols, out=False)
    tokens[0] = cols - 1
    tokens[-1] = 0
    logp, loss, old, adv = vectors(rows, 4)
    saved = torch.empty(2, rows, device="cuda")
    capi.token_logp_fwd(logp, saved, x, tokens)
    want, _, on, tol, p = exact.token_logp(x, tokens, 1.0)
    exact.check(logp, want, tol, "logp")
    up = torch.randn(rows, device="cuda", generator=g)
    want_dx, size = exact.gradient(p, tokens, on, up.double(), up.double().abs(), 1.0)

    def outside(backing, dx):
        mark = torch.zeros_like(backing, dtype=torch.bool)
        mark[to_offset:to_offset + rows * to_stride].view(rows, to_stride)[:, :cols] = True
        assert bool((backing[~mark] == 7.0).all())

    backing, dx = room(rows, cols, TYPES[dtype], to_stride, to_offset)
    capi.token_logp_bwd(dx, up, x, tokens, saved)
    exact.check(dx, want_dx, exact.GRAD * size, "dlogits of logp")
    outside(backing, dx)
    old.copy_(want)
    adv.copy_(up)   # ratio 1: the policy's gradient is that of advantage*logp
    backing, dx = room(rows, cols, TYPES[dtype], to_stride, to_offset)
    capi.policy_loss(loss, logp, x, tokens, old, adv, dlogits=dx, clip_low=1.0, clip_high=10.0)
    exact.check(dx, want_dx, exact.GRAD * size, "dlogits of the policy")
    outside(backing, dx)
    backing, dx = room(rows, cols, TYPES[dtype], to_stride, to_offset)
    ids = torch.stack([tokens, (tokens + 1) % cols], dim=1)
    top = torch.randn(rows, 2, device="cuda", generator=g)
    capi.distill_topk_loss(loss, x, ids, top, dlogits=dx)
    want = exact.distill(x, ids, top, None, 1.0, 1.0)
    exact.check(loss, *want["loss"], "distillation")
    exact.check(dx, *want["dlogits"], "dlogits of the distillation")
    outside(backing, dx)


def policy_inputs(g, x, tokens, tau):
    logp = exact.token_logp(x, tokens, tau)[0]
    rows = len(tokens)
    moved = torch.randn(rows, device="cuda", generator=g).double() * 0.3
    for border in (math.log(0.8), math.log(1.28)):   # a ratio within rounding of a border has two right gradients
        moved = torch.where((moved - border).abs() < 1e-3, moved + 0.01, moved)
    old = (logp - moved).float()
    return old, torch.randn(rows, device="cuda", generator=g), (logp + 0.4 * torch.randn(rows, device="cuda", generator=g)).float()


@pytest.mark.parametrize("reference", [True, False])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(1, 5), (64, 100), (300, 513), (33, 1000), (40, 4100), (20, 32000), (3, 65543), (160, 33000)])
def test_policy_loss(capi, rows, cols, dtype, reference):
    g = generator(rows + 3 * cols)
    x = scores(g, rows, cols, TYPES[dtype])
    tokens = somewhere(g, rows, cols)
    tau = 0.8
    old, adv, ref = policy_inputs(g, x, tokens, tau)
    ref = ref if reference else None
    mask = torch.rand(rows, device="cuda", generator=g).round() * 0.5 if rows > 1 else None
    loss, logp, kl = vectors(rows, 3)
    _, dx = room(rows, cols, TYPES[dtype])
    args = dict(ref_logp=ref, mask=mask, clip_low=0.2, clip_high=0.28, kl_coef=0.1, temperature=tau, scale=0.5)
    capi.policy_loss(loss, logp, x, tokens, old, adv, kl=kl, dlogits=dx, **args)
    want = exact.policy(x, tokens, old, adv, ref, mask, 0.2, 0.28, 0.1, tau, 0.5)
    for name, got in (("loss", loss), ("logp", logp), ("kl", kl), ("dlogits", dx)):
        exact.check(got, *want[name], name)
    alone, alone_logp = vectors(rows, 2)
    capi.policy_loss(alone, alone_logp, x, tokens, old, adv, **args)   # the loss alone
    exact.check(alone, *want["loss"], "the loss alone")
    exact.check(alone_logp, *want["logp"], "its log probabilities")


@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("squared", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cols,offsets,rows", [(37, [0, 1, 2], 2), (500, [0, 0, 3], 3), (1000, [2, 40, 77, 77, 78], 81), (4099, [0, 300, 600, 700, 1100], 1130),
                                               (32000, [0, 5, 20, 21, 60], 60), (70001, [1, 3, 6], 7)])
def test_preference_loss(capi, cols, offsets, rows, dtype, squared, average):
    g = generator(cols + rows)
    x = scores(g, rows, cols, TYPES[dtype])
    tokens = somewhere(g, rows, cols)
    offsets = torch.tensor(offsets, device="cuda", dtype=torch.int32 if average else torch.int64)
    pairs, tau, beta = len(offsets) // 2, 1.3, 0.2
    logp64 = exact.token_logp(x, tokens, tau)[0]
    ends = offsets.tolist()
    ref = torch.stack([logp64[ends[i]:ends[i + 1]].sum() for i in range(2 * pairs)])
    if average:
        ref = ref / offsets.diff().clamp(min=1)
    ref = (ref + torch.randn(2 * pairs, device="cuda", generator=g)).float()
    loss, rewards, logp, dlogp = torch.full((pairs,), 7.0, device="cuda"), *vectors(2 * pairs, 1), *vectors(rows, 2)
    saved = torch.full((2, rows), 7.0, device="cuda")
    _, dx = room(rows, cols, TYPES[dtype])
    args = dict(kind=capi.PREFERENCE_SQUARED if squared else capi.PREFERENCE_LOGISTIC, beta=beta, label_smoothing=0.1, average=average, temperature=tau, scale=0.25)
    capi.preference_loss(loss, rewards, logp, saved, dlogp, x, tokens, offsets, ref, dlogits=dx, **args)
    want = exact.preference(x, tokens, offsets, ref, squared, beta, 0.1, average, tau, 0.25)
    inside = want["inside"]
    exact.check(loss, *want["loss"], "loss")
    exact.check(rewards, *want["rewards"], "rewards")
    for name, got in (("logp", logp), ("dlogp", dlogp), ("dlogits", dx)):
        exact.check(got[inside], *(v[inside] for v in want[name]), name)
        assert bool((got[~inside] == 7.0).all()), name   # left as they were
    assert bool((saved[:, ~inside] == 7.0).all())
    again, again_rewards = torch.empty_like(loss), torch.empty_like(rewards)
    capi.preference_loss(again, again_rewards, logp, saved, dlogp, x, tokens, offsets, ref, **args)   # without dlogits
    assert torch.equal(again, loss) and torch.equal(again_rewards, rewards)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols,kept", [(1, 1, 1), (5, 40, 40), (9, 257, 3), (7, 1000, 100), (4, 5000, 1024), (200, 5003, 64), (3, 32000, 256), (20, 32000, 8),
                                            (2, 65543, 300), (2, 150000, 17)])
def test_distill_topk_loss(capi, rows, cols, kept, dtype):
    g = generator(rows + cols + kept)
    x = scores(g, rows, cols, TYPES[dtype])
    ids = torch.rand(rows, cols, device="cuda", generator=g).topk(kept, dim=1).indices
    teacher_type = [torch.float32, torch.bfloat16, torch.float16][(rows + kept) % 3]
    teacher = (torch.randn(rows, kept, device="cuda", generator=g) * 2).to(teacher_type)
    if kept > 2:
        ids[0, 1] = -1                      # no entry
        teacher[-1, 2] = -math.inf          # an entry without mass
        if rows > 3:
            ids[2] = cols                   # a row without entries
            teacher[3] = -math.inf
    if rows % 2:
        ids = ids.to(torch.int32)
    mask = torch.rand(rows, device="cuda", generator=g) if rows > 1 else None
    if rows > 4:
        mask[4] = 0.0
    tau = 2.0
    loss, = vectors(rows, 1)
    _, dx = room(rows, cols, TYPES[dtype])
    capi.distill_topk_loss(loss, x, ids, teacher, mask=mask, dlogits=dx, temperature=tau, scale=0.5)
    want = exact.distill(x, ids, teacher, mask, tau, 0.5)
    exact.check(loss, *want["loss"], "loss")
    exact.check(dx, *want["dlogits"], "dlogits")
    alone, = vectors(rows, 1)
    capi.distill_topk_loss(alone, x, ids, teacher, mask=mask, temperature=tau, scale=0.5)
    exact.check(alone, *want["loss"], "the loss alone")


@pytest.mark.parametrize("cols", [50, 3000, 33000])
def test_an_index_that_is_there_twice_holds_the_mass_of_both(capi, cols):
    g = generator(cols)
    x = scores(g, 4, cols, torch.float32)
    ids = torch.randint(0, cols, (4, 40), device="cuda", generator=g)
    ids[0, :] = 5
    ids[1, 7] = ids[1, 39] = ids[1, 0]
    ids[2] = torch.arange(40, device="cuda")
    ids[2, 33] = 1
    teacher = torch.randn(4, 40, device="cuda", generator=g)
    for add in (False, True):
        loss, = vectors(4, 1)
        _, dx = room(4, cols, torch.float32, value=0.5)
        capi.distill_topk_loss(loss, x, ids, teacher, dlogits=dx, add_to_destination=add)
        want = exact.distill(x, ids, teacher, None, 1.0, 1.0)
        exact.check(loss, *want["loss"], "loss")
        exact.check(dx, want["dlogits"][0] + (0.5 if add else 0.0), want["dlogits"][1] + exact.U, "dlogits")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cols", [9, 1000, 5001, 40000])
def test_rows_that_count_for_nothing(capi, cols, dtype):
    """NaN and infinities in rows that are masked, whose token is none, or whose gradient is 0 reach nothing; a row of nothing but
    -infinity counts for nothing; one of nothing but the type's lowest value is a uniform distribution."""
    t = TYPES[dtype]
    g = generator(cols + 5)
    x = scores(g, 8, cols, t)
    x[0] = math.nan
    x[1, cols // 2] = math.inf
    x[2] = -math.inf
    x[3] = torch.finfo(t).min
    x[4, 1:] = -math.inf
    x[5, ::2] = torch.finfo(t).min
    x[6, cols - 1] = -math.inf
    tokens = torch.tensor([0, 1, 2, 3, 0, 1, 0, cols - 1], device="cuda") % cols
    out = tokens.clone()
    out[:2] = -100
    logp, dlogp = vectors(8, 2)
    saved = torch.empty(2, 8, device="cuda")
    capi.token_logp_fwd(logp, saved, x, out)
    want, want_saved, on, tol, p = exact.token_logp(x, out, 1.0)
    assert on.tolist() == [False, False, False, True, True, True, True, True]
    exact.check(logp, want, tol, "logp")
    assert saved[:, :3].tolist() == [[0.0] * 3] * 2
    assert abs(float(logp[3]) + math.log(cols)) < 1e-4 and float(logp[4]) == 0.0
    dlogp.fill_(1.0)
    _, dx = room(8, cols, t)
    capi.token_logp_bwd(dx, dlogp, x, out, saved)
    want_dx, size = exact.gradient(torch.nan_to_num(p), out, on, dlogp.double(), dlogp.double(), 1.0)
    exact.check(dx, want_dx, exact.GRAD * size, "dlogits")
    # the same rows out by their mask
    mask = torch.tensor([0.0, 0.0, 1, 1, 1, 1, 1, 1], device="cuda")
    loss, logp, kl = vectors(8, 3)
    old, adv = torch.where(on, want, 0.0).float(), torch.ones(8, device="cuda")
    _, dx = room(8, cols, t)
    capi.policy_loss(loss, logp, x, tokens, old, adv, mask=mask, kl=kl, dlogits=dx, clip_low=1.0, clip_high=10.0)
    exact.check(logp, want, tol, "logp of the policy")
    assert loss[:3].tolist() == [0.0] * 3 and kl[:3].tolist() == [0.0] * 3
    exact.check(dx, want_dx, exact.GRAD * size, "dlogits of the policy")
    ids = torch.stack([tokens, (tokens + 1) % cols], dim=1)
    ids[4:6, 1] = ids[4:6, 0]
    ids[6, 1] = 1
    top = torch.randn(8, 2, device="cuda", generator=g)
    _, dx = room(8, cols, t)
    capi.distill_topk_loss(loss, x, ids, top, mask=mask, dlogits=dx)
    assert loss[:3].tolist() == [0.0] * 3 and not bool(dx[:3].any())
    want = exact.distill(x[3:], ids[3:], top[3:], None, 1.0, 1.0)
    exact.check(loss[3:], *want["loss"], "distillation")
    exact.check(dx[3:], *want["dlogits"], "dlogits of the distillation")
    # an accumulated gradient stays as it was
    backing, dx = room(8, cols, t)
    capi.token_logp_bwd(dx, torch.zeros(8, device="cuda"), x, tokens, saved, add_to_destination=True)
    assert bool((backing == 7.0).all())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cols", [11, 1000, 40000])
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_what_is_no_number_shows(capi, cols, dtype, what):
    x = scores(generator(cols), 2, cols, TYPES[dtype])
    x[1, cols // 3] = what
    tokens = torch.tensor([1, 2], device="cuda")
    logp, loss, old = vectors(2, 3)
    saved = torch.empty(2, 2, device="cuda")
    capi.token_logp_fwd(logp, saved, x, tokens)
    assert math.isfinite(float(logp[0])) and math.isnan(float(logp[1]))
    _, dx = room(2, cols, TYPES[dtype])
    capi.token_logp_bwd(dx, torch.ones(2, device="cuda"), x, tokens, saved)
    assert bool(torch.isfinite(dx[0]).all()) and bool(torch.isnan(dx[1]).any())
    capi.policy_loss(loss, logp, x, tokens, old, torch.ones(2, device="cuda"), dlogits=dx)
    assert math.isfinite(float(loss[0])) and math.isnan(float(loss[1])) and bool(torch.isfinite(dx[0]).all()) and bool(torch.isnan(dx[1]).any())
    capi.distill_topk_loss(loss, x, tokens[:, None], torch.ones(2, 1, device="cuda"), dlogits=dx)
    assert math.isfinite(float(loss[0])) and math.isnan(float(loss[1])) and bool(torch.isfinite(dx[0]).all()) and bool(torch.isnan(dx[1]).any())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(5, 33), (6, 1003), (9, 20000), (3, 70001)])
def test_accumulation_and_gradients_in_the_logits_place(capi, rows, cols, dtype):
    t = TYPES[dtype]
    g = generator(rows + cols)
    x = scores(g, rows, cols, t)
    tokens = somewhere(g, rows, cols)
    before = torch.randn(rows, cols, device="cuda", generator=g).to(t)
    old, adv, ref = policy_inputs(g, x, tokens, 1.0)
    ids = torch.rand(rows, cols, device="cuda", generator=g).topk(8, dim=1).indices
    top = torch.randn(rows, 8, device="cuda", generator=g)
    offsets = torch.tensor([0, rows // 2, rows], device="cuda")
    logp, loss, up = vectors(rows, 3)
    saved = torch.empty(2, rows, device="cuda")
    capi.token_logp_fwd(logp, saved, x, tokens)
    up.copy_(torch.randn(rows, device="cuda", generator=g))
    pair = [torch.empty(1, device="cuda"), torch.empty(2, device="cuda"), torch.empty(rows, device="cuda"), torch.empty(2, rows, device="cuda"),
            torch.empty(rows, device="cuda")]
    ref2 = torch.tensor([-3.0, -4.0], device="cuda")
    calls = {
        "logp": (lambda y, dx, add: capi.token_logp_bwd(dx, up, y, tokens, saved, add_to_destination=add),
                 lambda: exact.gradient(exact.rows(x, 1.0)[2], tokens, exact.token_logp(x, tokens, 1.0)[2], up.double(), up.double().abs(), 1.0), exact.GRAD),
        "policy": (lambda y, dx, add: capi.policy_loss(loss, logp, y, tokens, old, adv, ref_logp=ref, kl_coef=0.1, dlogits=dx, clip_high=0.28, add_to_destination=add),
                   lambda: exact.policy(x, tokens, old, adv, ref, None, 0.2, 0.28, 0.1, 1.0, 1.0)["dlogits"], 1.0),
        "distill": (lambda y, dx, add: capi.distill_topk_loss(loss, y, ids, top, dlogits=dx, add_to_destination=add),
                    lambda: exact.distill(x, ids, top, None, 1.0, 1.0)["dlogits"], 1.0),
        "preference": (lambda y, dx, add: capi.preference_loss(*pair, y, tokens, offsets, ref2, dlogits=dx, add_to_destination=add),
                       lambda: exact.preference(x, tokens, offsets, ref2, False, 0.1, 0.0, False, 1.0, 1.0)["dlogits"], 1.0),
    }
    for name, (call, want, share) in calls.items():
        value, size = want()
        dx = before.clone()
        call(x, dx, True)
        exact.check(dx, before.double() + value, size * share + 2 * exact.U * (before.double().abs() + value.abs()), name + " added")
        y = x.clone()
        call(y, y, False)
        exact.check(y, value, size * share, name + " in place")


def test_gradients_against_differences(capi):
    """Central differences of the loss that the kernel itself returns. A step of 2^-6 leaves a third-order term below step^2/6 times the
    third derivative (below 1 for each of these losses at tau = 1): 4.1e-5; the loss's own error, a few 1e-6, is divided by the step: 3e-4."""
    g = generator(99)
    cols, step = 24, 2.0 ** -6
    x = scores(g, 1, cols, torch.float32, spread=1.0)
    bumped = torch.cat([x + step * torch.eye(cols, device="cuda"), x - step * torch.eye(cols, device="cuda")])
    n = 2 * cols

    def slopes(values):
        return (values[cols:] - values[:cols]).double() / (2 * step)   # the direction in which the loss falls

    def repeat(v):
        return v.expand(n, *v.shape[1:]).contiguous()

    token = torch.tensor([5], device="cuda")
    one = torch.ones(1, device="cuda")
    logp = exact.token_logp(x, token, 1.0)[0]
    for name, kw in (("free", dict(old=logp - 0.05, adv=1.0)), ("held", dict(old=logp - 0.6, adv=0.7)), ("negative", dict(old=logp - 0.6, adv=-0.7))):
        old, adv = kw["old"].float(), one * kw["adv"]
        ref = (logp + 0.3).float()
        loss, lp, dx = torch.empty(1, device="cuda"), torch.empty(1, device="cuda"), torch.empty_like(x)
        capi.policy_loss(loss, lp, x, token, old, adv, ref_logp=ref, kl_coef=0.2, dlogits=dx)
        many, lps = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
        capi.policy_loss(many, lps, bumped, repeat(token), repeat(old), repeat(adv), ref_logp=repeat(ref), kl_coef=0.2)
        assert float((slopes(many) - dx[0].double()).abs().max()) < 1e-3, name
    ids, top = torch.tensor([[3, 9, 20]], device="cuda"), torch.tensor([[1.0, 0.5, -1.0]], device="cuda")
    loss, dx, many = torch.empty(1, device="cuda"), torch.empty_like(x), torch.empty(n, device="cuda")
    capi.distill_topk_loss(loss, x, ids, top, dlogits=dx)
    capi.distill_topk_loss(many, bumped, repeat(ids), repeat(top))
    assert float((slopes(many) - dx[0].double()).abs().max()) < 1e-3, "distill"
    # a pair of two sequences of two rows: the first row's scores are bumped
    rest = scores(g, 3, cols, torch.float32, spread=1.0)
    tokens = torch.tensor([5, 1, 2, 3], device="cuda")
    for kind in (capi.PREFERENCE_LOGISTIC, capi.PREFERENCE_SQUARED):
        def pair(first, dlogits=None):
            count = first.shape[0]
            logits = torch.cat([first[:, None], rest[None].expand(count, 3, cols)], dim=1).reshape(4 * count, cols).contiguous()
            out = [torch.empty(count, device="cuda"), torch.empty(2 * count, device="cuda"), torch.empty(4 * count, device="cuda"),
                   torch.empty(2, 4 * count, device="cuda"), torch.empty(4 * count, device="cuda")]
            capi.preference_loss(*out, logits, tokens.repeat(count), torch.arange(0, 4 * count + 1, 2, device="cuda"),
                                 torch.tensor([-5.0, -6.0], device="cuda").repeat(count), dlogits=dlogits, kind=kind, beta=0.5)
            return out[0]
        dx = torch.empty(4, cols, device="cuda")
        pair(x, dx)
        assert float((slopes(pair(bumped)) - dx[0].double()).abs().max()) < (1e-3 if kind == capi.PREFERENCE_LOGISTIC else 1e-2), kind


def test_offsets_past_32_bits(capi):
    """The last row starts 2^31 elements behind the first one."""
    stride, cols = 1 << 30, 1000
    backing = torch.empty(2 * stride + cols, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(backing, (3, cols), (stride, 1))
    x.copy_(torch.randn(3, cols, device="cuda", generator=generator(3)))
    copy = x.clone()
    tokens = torch.tensor([1, 2, 999], device="cuda")
    logp, up = torch.empty(3, device="cuda"), torch.tensor([1.0, -2.0, 0.5], device="cuda")
    saved = torch.empty(2, 3, device="cuda")
    capi.token_logp_fwd(logp, saved, x, tokens)
    want, _, on, tol, p = exact.token_logp(copy, tokens, 1.0)
    exact.check(logp, want, tol, "logp")
    capi.token_logp_bwd(x, up, x, tokens, saved)
    value, size = exact.gradient(p, tokens, on, up.double(), up.double().abs(), 1.0)
    exact.check(x, value, exact.GRAD * size, "dlogits")
    x.copy_(copy)
    loss = torch.empty(3, device="cuda")
    capi.policy_loss(loss, logp, x, tokens, want.float(), up, dlogits=x, clip_low=1.0, clip_high=10.0)
    exact.check(x, value, exact.GRAD * size, "dlogits of the policy")


def test_many_short_rows(capi):
    g = generator(8)
    x = scores(g, 70001, 17, torch.bfloat16)
    tokens = somewhere(g, 70001, 17)
    logp, loss = vectors(70001, 2)
    dx = torch.empty_like(x)
    old, adv, ref = policy_inputs(g, x, tokens, 1.0)
    capi.policy_loss(loss, logp, x, tokens, old, adv, ref_logp=ref, kl_coef=0.1, dlogits=dx, clip_high=0.28)
    want = exact.policy(x, tokens, old, adv, ref, None, 0.2, 0.28, 0.1, 1.0, 1.0)
    for name, got in (("loss", loss), ("logp", logp), ("dlogits", dx)):
        exact.check(got, *want[name], name)


def test_no_rows_and_no_pairs(capi):
    x, none = torch.empty(0, 100, device="cuda"), torch.empty(0, device="cuda")
    tokens = torch.empty(0, dtype=torch.int64, device="cuda")
    capi.token_logp_fwd(none, torch.empty(2, 0, device="cuda"), x, tokens)
    capi.token_logp_bwd(torch.empty_like(x), none, x, tokens, torch.empty(2, 0, device="cuda"))
    capi.policy_loss(none, none, x, tokens, none, none, dlogits=torch.empty_like(x))
    capi.distill_topk_loss(none, x, torch.empty(0, 4, dtype=torch.int64, device="cuda"), torch.empty(0, 4, device="cuda"))
    capi.preference_loss(none, none, none, torch.empty(2, 0, device="cuda"), none, x, tokens, torch.zeros(1, dtype=torch.int64, device="cuda"), none)
    torch.cuda.synchronize()


def test_offsets_that_are_wrong_stay_within_the_rows(capi):
    """Offsets below 0, behind the last row or decreasing: whatever comes out, nothing outside the rows is touched."""
    g = generator(12)
    x = scores(g, 12, 100, torch.float32)
    tokens = somewhere(g, 12, 100, out=False)
    for offsets in ([-5, 4, 40], [8, 4, 2], [0, 50, 12], [20, 30, 40], [-9, -7, -3]):
        off = torch.tensor(offsets, device="cuda")
        guard = [torch.full((64,), 7.0, device="cuda") for _ in range(3)]
        logp, dlogp, saved = guard[0][16:28], guard[1][16:28], guard[2][16:40].view(2, 12)
        backing = torch.full((14, 100), 7.0, device="cuda")
        capi.preference_loss(torch.empty(1, device="cuda"), torch.empty(2, device="cuda"), logp, saved, dlogp, x, tokens, off,
                             torch.zeros(2, device="cuda"), dlogits=backing[1:13])
        torch.cuda.synchronize()
        assert bool((backing[0] == 7.0).all()) and bool((backing[13] == 7.0).all())
        assert bool((guard[0][:16] == 7.0).all()) and bool((guard[0][28:] == 7.0).all()) and bool((guard[1][28:] == 7.0).all())
        assert bool((guard[2][:16] == 7.0).all()) and bool((guard[2][40:] == 7.0).all())


def step_of(capi, g, rows=64, cols=2000, dtype=torch.bfloat16):
    """The calls of one step over its own buffers: old and reference scores, policy loss, distillation added to its gradient."""
    s = {"x": scores(g, rows, cols, dtype), "r": scores(g, rows, cols, dtype), "tokens": somewhere(g, rows, cols)}
    s["logp"], s["old"], s["ref"], s["loss"], s["dloss"] = vectors(rows, 5)
    s["adv"] = torch.randn(rows, device="cuda", generator=g)
    s["ids"] = torch.rand(rows, cols, device="cuda", generator=g).topk(16, dim=1).indices
    s["top"] = torch.randn(rows, 16, device="cuda", generator=g)
    s["dx"] = torch.zeros(rows, cols, dtype=dtype, device="cuda")

    def step():
        capi.token_logp_fwd(s["old"], None, s["x"], s["tokens"])
        capi.token_logp_fwd(s["ref"], None, s["r"], s["tokens"])
        capi.policy_loss(s["loss"], s["logp"], s["x"], s["tokens"], s["old"], s["adv"], ref_logp=s["ref"], kl_coef=0.1, dlogits=s["dx"])
        capi.distill_topk_loss(s["dloss"], s["x"], s["ids"], s["top"], dlogits=s["dx"], add_to_destination=True)
    return s, step


def test_captured_and_on_another_stream(capi):
    """The same calls give the same bits twice, on another stream, and replayed from two graphs; new inputs are taken up by a replay."""
    s, step = step_of(capi, generator(1))
    names = ("logp", "old", "ref", "loss", "dloss", "dx")
    step()
    torch.cuda.synchronize()
    first = {n: s[n].clone() for n in names}
    other = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        graphs.append(graph)

    def same(what):
        torch.cuda.synchronize()
        for n in names:
            assert torch.equal(s[n], first[n]), (what, n)
            s[n].zero_()
        torch.cuda.synchronize()

    step()
    same("again")
    with torch.cuda.stream(other):
        step()
    same("another stream")
    for k, graph in enumerate(graphs):
        graph.replay()
        same("graph %d" % k)
    s["x"].mul_(0.5)
    graphs[1].replay()
    torch.cuda.synchronize()
    replayed = {n: s[n].clone() for n in names}
    step()
    torch.cuda.synchronize()
    assert all(torch.equal(s[n], replayed[n]) for n in names) and not torch.equal(replayed["loss"], first["loss"])


def test_the_stream_that_is_given(capi):
    x = scores(generator(2), 4, 100, torch.float32)
    tokens = torch.tensor([1, 2, 3, 4], device="cuda")
    want, got = torch.empty(4, device="cuda"), torch.empty(4, device="cuda")
    capi.token_logp_fwd(want, None, x, tokens)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    capi.token_logp_fwd(got, None, x, tokens, stream=stream)
    stream.synchronize()
    assert torch.equal(got, want)


def test_a_step_of_training(capi):
    """Used together: scores from a linear head, policy loss and distillation into one gradient, the head's gradient, the optimiser."""
    g = generator(21)
    rows, width, cols = 96, 64, 1500
    h, w = torch.randn(rows, width, device="cuda", generator=g), torch.randn(cols, width, device="cuda", generator=g) * 0.2
    was = w.clone()
    x = torch.empty(rows, cols, device="cuda")
    torch.mm(h, w.t(), out=x)
    tokens = somewhere(g, rows, cols)
    old, adv, ref = policy_inputs(g, x, tokens, 1.0)
    ids = torch.rand(rows, cols, device="cuda", generator=g).topk(12, dim=1).indices
    top = torch.randn(rows, 12, device="cuda", generator=g)
    loss, logp, dloss = vectors(rows, 3)
    dx = torch.empty_like(x)
    capi.policy_loss(loss, logp, x, tokens, old, adv, ref_logp=ref, kl_coef=0.1, clip_high=0.28, dlogits=dx, scale=1.0 / rows)
    capi.distill_topk_loss(dloss, x, ids, top, dlogits=dx, scale=0.5 / rows, add_to_destination=True)
    want = exact.policy(x, tokens, old, adv, ref, None, 0.2, 0.28, 0.1, 1.0, 1.0 / rows)["dlogits"]
    more = exact.distill(x, ids, top, None, 1.0, 0.5 / rows)["dlogits"]
    total, bound = want[0] + more[0], want[1] + more[1] + 2 * exact.U * (want[0].abs() + more[0].abs())
    exact.check(dx, total, bound, "dlogits")
    gradient = dx.double().t() @ h.double()
    grad32 = gradient.float()
    mean = float(loss.double().sum() + dloss.double().sum())
    capi.apply_gradient([{"data": w, "gradient": grad32.clone(), "learning_rate": 0.5}])
    torch.cuda.synchronize()
    assert float((w.double() - (was.double() + 0.5 * grad32.double())).abs().max()) <= 4 * exact.U * float(was.abs().max() + 1)
    assert math.isfinite(mean)


def test_tensors_that_are_refused(capi):
    def full(*size, dtype=torch.float32):
        return torch.zeros(*size, dtype=dtype, device="cuda")

    x, t, v, saved = full(4, 10), full(4, dtype=torch.int64), full(4), full(2, 4)

    def policy(x=x, t=t, v=v, dx=None):
        capi.policy_loss(v, v, x, t, v, v, dlogits=dx)

    policy(dx=full(4, 10))
    for error, text, kw in ((TypeError, "logits: float32, bfloat16 or float16", dict(x=x.double())), (TypeError, "tokens: int32 or int64", dict(t=v)),
                            (TypeError, "float32 is expected", dict(v=v.half())), (ValueError, r"logits: a tensor \[rows\]\[columns\]", dict(x=v)),
                            (ValueError, "tokens: another number", dict(t=t[:3])), (ValueError, "another number", dict(v=full(5))),
                            (AssertionError, "elements of a row", dict(x=full(10, 4).t())), (AssertionError, "contiguous", dict(v=full(8)[::2])),
                            (AssertionError, "contiguous", dict(t=full(8, dtype=torch.int64)[::2])), (capi.NnfError, "another type or shape", dict(dx=full(4, 11))),
                            (capi.NnfError, "extents", dict(x=full(1, 10).expand(4, 10)))):
        with pytest.raises(error, match=text):
            policy(**kw)
    with pytest.raises(ValueError, match="saved"):
        capi.token_logp_fwd(v, v, x, t)
    with pytest.raises(capi.NnfError, match="null"):
        capi.token_logp_bwd(full(4, 10), v, x, t, None)
    with pytest.raises(TypeError, match="teacher_ids"):
        capi.distill_topk_loss(v, x, full(4, 2), full(4, 2))
    with pytest.raises(ValueError, match="offsets"):
        capi.preference_loss(full(2), full(4), v, saved, v, x, t, full(4, dtype=torch.int64), full(4))
    with pytest.raises(ValueError, match="rewards"):
        capi.preference_loss(full(2), full(3), v, saved, v, x, t, full(5, dtype=torch.int64), full(4))


@pytest.mark.parametrize("dtype,spread,tau", [("fp32", 1e3, 1.0), ("fp32", 1e8, 7.0), ("fp32", 3.0, 1e-4), ("bf16", 300.0, 1.0), ("bf16", 1e7, 1.0), ("fp16", 1e4, 1.0),
                                              ("fp16", 3.0, 0.003)])
@pytest.mark.parametrize("cols", [100, 3001, 33000])
def test_large_scores(capi, cols, dtype, spread, tau):
    """Scores so far apart that a row's maximum has nearly all of the mass, and so large that x*k - M*k would lose it. With |x - M|/tau up to
    T (of those that matter: 104, where exp() leaves fp32) the argument of an exponential is off by 3u*T = 312u, beside the 77u + 4u of the sum:
    GRAD (500u) still holds for p; logp is off by 4u*|x_token - M|/tau + 400u."""
    g = generator(cols)
    rows = 6
    x = scores(g, rows, cols, TYPES[dtype], spread=spread)
    x = torch.where(torch.isfinite(x), x, torch.zeros_like(x))   # (fp16 ends at 65504)
    tokens = x.float().argmax(dim=1)
    tokens[0] = 1
    up = torch.randn(rows, device="cuda", generator=g)
    logp, loss = vectors(rows, 2)
    saved = torch.empty(2, rows, device="cuda")
    capi.token_logp_fwd(logp, saved, x, tokens, temperature=tau)
    want, _, on, tol, p = exact.token_logp(x, tokens, tau)
    exact.check(logp, want, tol + 400 * exact.U, "logp")
    value, size = exact.gradient(p, tokens, on, up.double(), up.double().abs(), tau)
    _, dx = room(rows, cols, TYPES[dtype])
    capi.token_logp_bwd(dx, up, x, tokens, saved, temperature=tau)
    exact.check(dx, value, exact.GRAD * size, "dlogits of logp")
    ids = torch.stack([tokens, (tokens + 1) % cols, (tokens + 2) % cols], dim=1)
    top = torch.tensor([[3.0, 2.0, -4.0]], device="cuda").repeat(rows, 1) * tau
    for add in (False, True):
        _, dx = room(rows, cols, TYPES[dtype], value=0.0)
        capi.policy_loss(loss, logp, x, tokens, want.float().clamp(min=-50), torch.ones(rows, device="cuda"), dlogits=dx, clip_low=1.0, clip_high=10.0, temperature=tau,
                         add_to_destination=add)
        result = exact.policy(x, tokens, want.float().clamp(min=-50), torch.ones(rows, device="cuda"), None, None, 1.0, 10.0, 0.0, tau, 1.0)
        exact.check(dx, result["dlogits"][0], 2 * result["dlogits"][1], "dlogits of the policy")
        _, dx = room(rows, cols, TYPES[dtype], value=0.0)
        capi.distill_topk_loss(loss, x, ids, top, dlogits=dx, temperature=tau, add_to_destination=add)
        result = exact.distill(x, ids, top, None, tau, 1.0)
        exact.check(loss, *result["loss"], "distillation")
        exact.check(dx, *result["dlogits"], "dlogits of the distillation")


@pytest.mark.parametrize("cols", [64, 2000, 33000])
def test_teachers_of_every_kind(capi, cols):
    """The type's lowest value among a teacher's logits, rows of nothing else, NaN and infinity in one row only, a student who excludes what
    the teacher keeps."""
    g = generator(cols + 1)
    low = torch.finfo(torch.float32).min
    x = scores(g, 6, cols, torch.float32)
    ids = torch.rand(6, cols, device="cuda", generator=g).topk(5, dim=1).indices
    top = torch.randn(6, 5, device="cuda", generator=g)
    top[0, 2:] = low
    top[1] = low
    top[2, 1] = math.nan
    top[3, 4] = math.inf
    x[4, ids[4, 0]] = -math.inf
    loss, = vectors(6, 1)
    _, dx = room(6, cols, torch.float32)
    capi.distill_topk_loss(loss, x, ids, top, dlogits=dx)
    keep = torch.tensor([0, 1, 5], device="cuda")
    want = exact.distill(x[keep], ids[keep], top[keep], None, 1.0, 1.0)
    exact.check(loss[keep], *want["loss"], "loss")
    exact.check(dx[keep], *want["dlogits"], "dlogits")
    assert math.isnan(float(loss[2])) and math.isnan(float(loss[3])) and float(loss[4]) == math.inf
    assert bool(torch.isfinite(dx[4]).all())
    want = exact.distill(x[4:5], ids[4:5], top[4:5], None, 1.0, 1.0)
    exact.check(dx[4:5], *want["dlogits"], "dlogits where the student excludes it")


def test_offsets_at_the_ends_of_their_type(capi):
    x = scores(generator(13), 9, 70, torch.float32)
    tokens = somewhere(generator(13), 9, 70, out=False)
    big = 2 ** 63 - 1
    for offsets in ([-big - 1, 4, big], [big, big, big], [big, 3, 0], [-big, -big, -big], [big - 1, big, -1]):
        logp, dlogp = vectors(9, 2)
        backing = torch.full((11, 70), 7.0, device="cuda")
        capi.preference_loss(torch.empty(1, device="cuda"), torch.empty(2, device="cuda"), logp, torch.zeros(2, 9, device="cuda"), dlogp, x, tokens,
                             torch.tensor(offsets, device="cuda"), torch.zeros(2, device="cuda"), dlogits=backing[1:10])
        torch.cuda.synchronize()
        assert bool((backing[0] == 7.0).all()) and bool((backing[10] == 7.0).all())


def test_a_pair_that_is_no_number_stays_alone(capi):
    g = generator(14)
    x = scores(g, 12, 500, torch.bfloat16)
    x[4, 7] = math.nan
    tokens = somewhere(g, 12, 500, out=False)
    offsets = torch.tensor([0, 3, 6, 9, 12], device="cuda")
    loss, rewards, logp, dlogp = torch.empty(2, device="cuda"), *vectors(4, 1), *vectors(12, 2)
    _, dx = room(12, 500, torch.bfloat16)
    capi.preference_loss(loss, rewards, logp, torch.empty(2, 12, device="cuda"), dlogp, x, tokens, offsets, torch.zeros(4, device="cuda"), dlogits=dx)
    assert math.isnan(float(loss[0])) and math.isfinite(float(loss[1]))
    assert bool(torch.isnan(dx[:6]).any()) and bool(torch.isfinite(dx[6:]).all())


def test_two_calls_at_once(capi):
    """Two streams with a step each, many times over, give what they give one after the other."""
    steps = [step_of(capi, generator(30 + k), rows=200, cols=20000) for k in range(2)]
    names = ("logp", "old", "ref", "loss", "dloss", "dx")
    want = []
    for s, step in steps:
        step()
        torch.cuda.synchronize()
        want.append({n: s[n].clone() for n in names})
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(10):
        for (s, step), stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                step()
    torch.cuda.synchronize()
    for (s, _), w in zip(steps, want):
        assert all(torch.equal(s[n], w[n]) for n in names)


def test_the_first_call_of_a_process_may_be_captured(form, capi, request):
    import os
    import subprocess
    import sys
    if "built-in" not in request.node.name:
        pytest.skip("the same in every form")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import torch
from nnforge_b200 import capi
x = torch.randn(8, 20000, device="cuda").bfloat16()
t = torch.arange(8, device="cuda")
v = [torch.zeros(8, device="cuda") for _ in range(4)]
dx = torch.empty_like(x)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    capi.policy_loss(v[0], v[1], x, t, v[2], v[3], dlogits=dx)
graph.replay()
torch.cuda.synchronize()
got = v[1].clone()
capi.policy_loss(v[0], v[1], x, t, v[2], v[3], dlogits=dx)
assert torch.equal(got, v[1]) and float(got.abs().sum()) > 0
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]

"""The losses on the scores of a vocabulary, as cases to be timed and compared.

Kinds (a case names one and gives its sizes; logits are [rows][vocab] of the case's type, one row for each token):

  score       log probabilities of given tokens, forward alone: what the old and the reference policy are asked for
  nll         the same with the backward pass: the gradient of the logits from one gradient for each token
  policy      clipped policy loss with a KL term towards a reference, loss and gradient in one call
  preference  loss of paired sequences (packed, chosen before rejected) over their summed log ratios, loss and gradient in one call
  distill     divergence from a teacher of whom the top K logits are kept, loss and gradient in one call

Where `own` is false, run() computes the operators from elementary torch operations in 32 bits; where it is true, it calls the
framework. Rows that do not count (a prompt's tokens, padding) have a token of -100 or a weight of 0. Gradients are the direction in
which the loss falls, as every backward pass of the framework has them and its optimiser adds them.
"""
import math

import torch

own = False

IGNORED = -100
CLIP_LOW, CLIP_HIGH = 0.2, 0.28
KL_COEF = 0.04
BETA = 0.1
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # the log probabilities of the tokens that a small serving batch has just drawn: latency
        {"name": "score 16 rows", "kind": "score", "rows": 16, "vocab": 32000, "type": "bf16", "temperature": 0.7, "out": 0.0},
        # the old policy is asked about a batch of answers, prompts left out
        {"name": "score 8192 rows", "kind": "score", "rows": 8192, "vocab": 32000, "type": "bf16", "temperature": 1.0, "out": 0.25},
        # fine-tuning in the library's own type on a ragged vocabulary
        {"name": "nll ragged fp32", "kind": "nll", "rows": 1024, "vocab": 50021, "type": "fp32", "temperature": 1.0, "out": 0.1},
        # a policy over a small set of actions, as many rows as a classifier's batch
        {"name": "policy 256x1000 fp32", "kind": "policy", "rows": 256, "vocab": 1000, "type": "fp32", "temperature": 1.0, "out": 0.0, "reference": False},
        # a step of policy optimisation: answers and the prompts in front of them
        {"name": "policy 4096x32000", "kind": "policy", "rows": 4096, "vocab": 32000, "type": "bf16", "temperature": 1.0, "out": 0.4, "reference": True},
        # the same over a large vocabulary
        {"name": "policy 2048x131072", "kind": "policy", "rows": 2048, "vocab": 131072, "type": "bf16", "temperature": 0.9, "out": 0.2, "reference": True},
        # a few short pairs: the micro-batch of a small step
        {"name": "pairs 4 short", "kind": "preference", "rows": 512, "vocab": 32000, "type": "bf16", "temperature": 1.0, "out": 0.3, "pairs": 4,
         "loss": "logistic", "average": False, "tail": 0},
        # an ordinary step of preference optimisation
        {"name": "pairs 16", "kind": "preference", "rows": 8192, "vocab": 32000, "type": "bf16", "temperature": 1.0, "out": 0.3, "pairs": 16,
         "loss": "logistic", "average": False, "tail": 100},
        # a ragged vocabulary, half precision, means over the sequences and the squared loss
        {"name": "pairs ragged fp16", "kind": "preference", "rows": 1500, "vocab": 65537, "type": "fp16", "temperature": 1.0, "out": 0.2, "pairs": 7,
         "loss": "squared", "average": True, "tail": 0},
        # a handful of rows with few kept logits: latency
        {"name": "distill 32 rows", "kind": "distill", "rows": 32, "vocab": 32000, "type": "bf16", "temperature": 1.0, "out": 0.0, "kept": 8},
        # an ordinary step of distillation
        {"name": "distill 4096x32000", "kind": "distill", "rows": 4096, "vocab": 32000, "type": "bf16", "temperature": 2.0, "out": 0.1, "kept": 64},
        # a large vocabulary in the library's own type, many kept logits
        {"name": "distill 1024x131072 fp32", "kind": "distill", "rows": 1024, "vocab": 131072, "type": "fp32", "temperature": 1.5, "out": 0.1, "kept": 256},
    ]


def _scale(case, count):
    """Mean over the rows or pairs; half precision trains with its loss scaled up."""
    return (1024.0 if case["type"] == "fp16" else 1.0) / count


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["score", "nll", "policy", "preference", "distill"])
    kind_type = rng.choice(["bf16", "bf16", "fp32", "fp16"])
    vocab = _log(rng, 256, 131072)
    if rng.random() < 0.6:
        vocab = max(256, vocab // 64 * 64)   # what vocabularies mostly are padded to; the others stay odd
    size = 4 if kind_type == "fp32" else 2
    most = min(8192, (1 << 28) // (vocab * size))
    case = {"kind": kind, "rows": _log(rng, 1, most), "vocab": vocab, "type": kind_type, "temperature": rng.choice([1.0, 1.0, 0.6, 1.7]),
            "out": rng.choice([0.0, 0.1, 0.3, 0.5])}
    if kind == "policy":
        case["reference"] = rng.random() < 0.7
    elif kind == "preference":
        case["rows"] = max(case["rows"], 8)
        case["pairs"] = _log(rng, 1, max(1, case["rows"] // 8))
        case["loss"] = rng.choice(["logistic", "logistic", "squared"])
        case["average"] = case["loss"] == "squared" or rng.random() < 0.2
        case["tail"] = rng.choice([0, 0, 1, case["rows"] // 8])
    elif kind == "distill":
        case["kept"] = _log(rng, 1, 256)
    return case


# ---------------------------------------------------------------------------------------------------------------------
# inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t, v, dtype = case["rows"], case["vocab"], TYPES[case["type"]]

    def normal(*size):
        return torch.randn(*size, device="cuda", generator=g)

    def uniform(*size):
        return torch.rand(*size, device="cuda", generator=g)

    logits = torch.empty(t, v, dtype=dtype, device="cuda")
    tokens = torch.randint(0, v, (t,), device="cuda", generator=g)
    step = max(1, (1 << 26) // v)
    for r in range(0, t, step):
        x = normal(min(step, t - r), v).mul_(2.5)
        # the token that was drawn is one that the model thinks likely
        x.scatter_add_(1, tokens[r:r + step, None], 4.0 + 4.0 * uniform(x.shape[0], 1))
        logits[r:r + step] = x
    # a vocabulary is often padded; the scores of the padding are masked
    pad = v // 500
    if pad:
        tokens = torch.where(tokens >= v - pad, tokens - pad, tokens)
        logits[:, v - pad:] = -math.inf
    out = torch.randperm(t, device="cuda", generator=g) < int(case["out"] * t)
    state = {"case": case, "logits": logits, "tokens": tokens, "logp": torch.zeros(t, device="cuda"), "loss": torch.zeros(t, device="cuda")}
    kind = case["kind"]
    if kind in ("score", "nll", "preference"):
        state["saved"] = torch.zeros(2, t, device="cuda")
    if kind != "score":
        state["dlogits"] = torch.zeros(t, v, dtype=dtype, device="cuda")
    if kind in ("score", "nll"):
        tokens[out] = IGNORED
        state["dlogp"] = uniform(t) * _scale(case, t)
    elif kind == "policy":
        state["mask"] = (~out).float()
        state["advantages"] = normal(t)
        logp = torch.cat([_exact_logp(logits[r:r + step], tokens[r:r + step], case["temperature"])[1] for r in range(0, t, step)])
        # How far the policy has moved since the answers were drawn. A ratio within rounding of a border has two right gradients: none is taken.
        moved = 0.15 * normal(t).double()
        for border in (math.log(1.0 - CLIP_LOW), math.log(1.0 + CLIP_HIGH)):
            near = (moved - border).abs() < 1e-4
            moved = torch.where(near, moved + 3e-4, moved)
        state["old_logp"] = (logp - moved).float()
        state["ref_logp"] = (logp + 0.2 * normal(t)).float() if case["reference"] else None
        state["kl"] = torch.zeros(t, device="cuda")
    elif kind == "preference":
        p, used = case["pairs"], t - case["tail"]
        cuts = torch.sort(torch.randperm(max(1, used - 1), device="cuda", generator=g)[:2 * p - 1] + 1).values
        state["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), cuts, torch.full((1,), used, dtype=torch.int64, device="cuda")])
        # the first part of a sequence is its prompt
        row = torch.arange(t, device="cuda")
        seq = torch.searchsorted(state["offsets"], row, right=True) - 1
        begin = state["offsets"][seq.clamp(max=2 * p - 1)]
        length = state["offsets"].diff()[seq.clamp(max=2 * p - 1)]
        tokens[row - begin < (case["out"] * length).long()] = IGNORED
        sums = torch.zeros(2 * p + 1, dtype=torch.float64, device="cuda")
        logp = torch.cat([_exact_logp(logits[r:r + step], tokens[r:r + step].clamp(min=0), case["temperature"])[1] for r in range(0, t, step)])
        counts = tokens >= 0
        sums.index_add_(0, seq, torch.where(counts, logp, 0.0))
        number = torch.zeros(2 * p + 1, dtype=torch.float64, device="cuda").index_add_(0, seq, counts.double())
        if case["average"]:
            sums = sums / number.clamp(min=1)
        state["ref_logp"] = (sums[:2 * p] + normal(2 * p) * (0.3 if case["average"] else 3.0)).float()
        state["loss"] = torch.zeros(p, device="cuda")
        state["rewards"] = torch.zeros(2 * p, device="cuda")
        state["dlogp"] = torch.zeros(t, device="cuda")
    elif kind == "distill":
        k = min(case["kept"], v)
        state["mask"] = (~out).float()
        ids = torch.randint(0, v - pad, (t, k), device="cuda", generator=g)
        # a teacher's top logits have no index twice: distinct residues
        if k > 1:
            span = (v - pad) // k
            ids = (torch.arange(k, device="cuda")[None, :] * span + ids % max(1, span)).sort(dim=1).values
        ids[:, 0] = torch.where((ids[:, 1:] == tokens[:, None]).any(dim=1) | (tokens >= v - pad), ids[:, 0], tokens)
        state["ids"] = ids.to(torch.int32)
        state["teacher"] = torch.sort(normal(t, k).mul_(2.0).add_(6.0), dim=1, descending=True).values.to(dtype)
    return state


# ---------------------------------------------------------------------------------------------------------------------
# one pass


def run(state):
    case = state["case"]
    return (_framework if own else _plain)(case["kind"], case, state)


def _framework(kind, case, s):
    from nnforge_b200 import capi
    tau = case["temperature"]
    if kind in ("score", "nll"):
        capi.token_logp_fwd(s["logp"], s["saved"], s["logits"], s["tokens"], temperature=tau)
        if kind == "score":
            return {"logp": s["logp"], "saved": s["saved"]}
        capi.token_logp_bwd(s["dlogits"], s["dlogp"], s["logits"], s["tokens"], s["saved"], temperature=tau)
        return {"logp": s["logp"], "saved": s["saved"], "dlogits": s["dlogits"]}
    if kind == "policy":
        capi.policy_loss(s["loss"], s["logp"], s["logits"], s["tokens"], s["old_logp"], s["advantages"], ref_logp=s["ref_logp"], mask=s["mask"], kl=s["kl"],
                         dlogits=s["dlogits"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=KL_COEF, temperature=tau, scale=_scale(case, case["rows"]))
        return {"loss": s["loss"], "logp": s["logp"], "kl": s["kl"], "dlogits": s["dlogits"]}
    if kind == "preference":
        capi.preference_loss(s["loss"], s["rewards"], s["logp"], s["saved"], s["dlogp"], s["logits"], s["tokens"], s["offsets"], s["ref_logp"],
                             dlogits=s["dlogits"], kind=capi.PREFERENCE_SQUARED if case["loss"] == "squared" else capi.PREFERENCE_LOGISTIC, beta=BETA,
                             label_smoothing=0.1, average=case["average"], temperature=tau, scale=_scale(case, case["pairs"]))
        return {"loss": s["loss"], "rewards": s["rewards"], "dlogits": s["dlogits"]}
    capi.distill_topk_loss(s["loss"], s["logits"], s["ids"], s["teacher"], mask=s["mask"], dlogits=s["dlogits"], temperature=tau, scale=_scale(case, case["rows"]))
    return {"loss": s["loss"], "dlogits": s["dlogits"]}


def _rows(logits, tau):
    """Scaled distance from the row's maximum, its exponential's sum, and the probabilities."""
    z = logits.float()
    z = (z - z.amax(dim=1, keepdim=True)) / tau
    e = z.exp()
    total = e.sum(dim=1, keepdim=True)
    return z, total, e / total


def _token_logp(z, total, tokens):
    valid = (tokens >= 0) & (tokens < z.shape[1])
    at = torch.where(valid, tokens, 0)[:, None]
    return valid, at, torch.where(valid, (z.gather(1, at) - total.log())[:, 0], 0.0)


def _token_gradient(p, at, g, tau, dtype):
    """g/tau * (1 at the token - p), rows with g = 0 left empty."""
    d = p * (-g / tau)[:, None]
    d.scatter_add_(1, at, (g / tau)[:, None])
    return torch.where((g != 0)[:, None], d, 0.0).to(dtype)


def _plain(kind, case, s):
    tau, logits, tokens = case["temperature"], s["logits"], s["tokens"]
    z, total, p = _rows(logits, tau)
    if kind == "distill":
        teacher, ids = s["teacher"].float() / tau, s["ids"].long()
        e = (teacher - teacher.amax(dim=1, keepdim=True))
        q = e.exp()
        qt = q.sum(dim=1, keepdim=True)
        q, lnq = q / qt, e - qt.log()
        scale = s["mask"] * _scale(case, case["rows"])
        loss = scale * tau * tau * (q * (lnq - (z.gather(1, ids) - total.log()))).sum(dim=1)
        d = (p * (-scale * tau)[:, None]).scatter_add_(1, ids, q * (scale * tau)[:, None])
        return {"loss": loss, "dlogits": torch.where((scale != 0)[:, None], d, 0.0).to(logits.dtype)}
    valid, at, logp = _token_logp(z, total, tokens)
    if kind in ("score", "nll"):
        # what the backward pass takes up again: the row's maximum and the sum; zeros where the token counts for nothing
        saved = torch.stack([torch.where(valid, logits.amax(dim=1).float(), 0.0), torch.where(valid, total[:, 0], 0.0)])
    if kind == "score":
        return {"logp": logp, "saved": saved}
    if kind == "nll":
        g = torch.where(valid, s["dlogp"], 0.0)
        return {"logp": logp, "saved": saved, "dlogits": _token_gradient(p, at, g, tau, logits.dtype)}
    if kind == "policy":
        on = valid & (s["mask"] != 0)
        logp = torch.where(on, logp, 0.0)
        w = torch.where(on, s["mask"], 0.0) * _scale(case, case["rows"])
        ratio, a = (logp - s["old_logp"]).exp(), s["advantages"]
        free, held = ratio * a, ratio.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * a
        per_token, g = -torch.minimum(free, held), torch.where(free <= held, free, 0.0)
        kl = torch.zeros_like(logp)
        if s["ref_logp"] is not None:
            d = s["ref_logp"] - logp
            kl = torch.where(on, d.expm1() - d, 0.0)
            per_token, g = per_token + KL_COEF * kl, g + KL_COEF * d.expm1()
        g = torch.where(on, w * g, 0.0)
        return {"loss": torch.where(on, w * per_token, 0.0), "logp": logp, "kl": kl, "dlogits": _token_gradient(p, at, g, tau, logits.dtype)}
    # preference
    pairs = case["pairs"]
    row = torch.arange(len(tokens), device=tokens.device)
    seq = torch.searchsorted(s["offsets"], row, right=True) - 1
    valid = valid & (seq < 2 * pairs)
    length = torch.zeros(2 * pairs + 1, dtype=torch.float64, device=tokens.device).index_add_(0, seq, valid.double())
    sums = torch.zeros(2 * pairs + 1, dtype=torch.float64, device=tokens.device).index_add_(0, seq, torch.where(valid, logp, 0.0).double())
    share = 1.0 / length.clamp(min=1) if case["average"] else torch.ones_like(length)
    ratio = ((sums * share)[:2 * pairs] - s["ref_logp"].double()).view(pairs, 2)
    h = ratio[:, 0] - ratio[:, 1]
    scale, smooth = _scale(case, pairs), 0.1
    if case["loss"] == "squared":
        loss, dh = (h - 0.5 / BETA) ** 2, 2.0 * (h - 0.5 / BETA)
    else:
        up, down = 1.0 / (1.0 + (-BETA * h).exp()), 1.0 / (1.0 + (BETA * h).exp())
        loss, dh = -(1.0 - smooth) * up.log() - smooth * down.log(), BETA * (smooth * up - (1.0 - smooth) * down)
    g = torch.cat([torch.stack([-dh, dh], dim=1).view(-1) * share[:2 * pairs] * scale, torch.zeros(1, dtype=torch.float64, device=h.device)])
    g = torch.where(valid, g[seq].float(), 0.0)
    return {"loss": (loss * scale).float(), "rewards": (BETA * ratio).view(-1).float(), "dlogits": _token_gradient(p, at, g, tau, logits.dtype)}


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits


def _exact_logp(logits, tokens, tau):
    x = logits.double() / tau
    lse = torch.logsumexp(x, dim=1)
    return lse, x.gather(1, tokens[:, None])[:, 0] - lse


def exact(case, seed):
    s = prepare(case, seed)
    tau, tokens, t, v = case["temperature"], s["tokens"], case["rows"], case["vocab"]
    valid = (tokens >= 0) & (tokens < v)
    step = max(1, (1 << 26) // v)
    kind = case["kind"]
    if kind == "distill":
        losses, grads = [], []
        for r in range(0, t, step):
            x = s["logits"][r:r + step].double().requires_grad_()
            ids, w = s["ids"][r:r + step].long(), s["mask"][r:r + step].double() * (tau * tau * _scale(case, t))
            lnq = torch.log_softmax(s["teacher"][r:r + step].double() / tau, dim=1)
            lnp = x.gather(1, ids) / tau - torch.logsumexp(x / tau, dim=1, keepdim=True)
            loss = w * (lnq.exp() * (lnq - lnp)).sum(dim=1)
            grads.append(torch.autograd.grad(-loss.sum(), x)[0])
            losses.append(loss.detach())
        return {"loss": torch.cat(losses), "dlogits": torch.cat(grads)}
    logp = torch.cat([_exact_logp(s["logits"][r:r + step], tokens[r:r + step].clamp(min=0), tau)[1] for r in range(0, t, step)])
    logp = torch.where(valid, logp, 0.0)
    lead = logp.clone().requires_grad_()
    found = {}
    if kind in ("score", "nll"):
        top = s["logits"].max(dim=1).values.double()
        lse = torch.cat([torch.logsumexp(s["logits"][r:r + step].double() / tau, dim=1) for r in range(0, t, step)])
        found["logp"] = logp
        found["saved"] = torch.stack([torch.where(valid, top, 0.0), torch.where(valid, torch.exp(lse - top / tau), 0.0)])
        if kind == "score":
            return found
        total = (s["dlogp"].double() * torch.where(valid, lead, 0.0)).sum()
    elif kind == "policy":
        on = s["mask"] > 0
        ratio = torch.exp(lead - s["old_logp"].double())
        gain = torch.stack([ratio * s["advantages"].double(), ratio.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * s["advantages"].double()]).amin(dim=0)
        kl = torch.zeros_like(logp)
        if s["ref_logp"] is not None:
            gap = s["ref_logp"].double() - lead
            kl = gap.exp() - gap - 1.0
        loss = torch.where(on, (KL_COEF * kl - gain) * _scale(case, t), 0.0)
        total = loss.sum()
        found.update(loss=loss.detach(), logp=torch.where(on, logp, 0.0), kl=torch.where(on, kl.detach(), 0.0))
    else:
        ends = s["offsets"].tolist()
        rewards, losses = [], []
        for i in range(2 * case["pairs"]):
            part = lead[ends[i]:ends[i + 1]]
            number = int(valid[ends[i]:ends[i + 1]].sum())
            logsum = torch.where(valid[ends[i]:ends[i + 1]], part, 0.0).sum()
            rewards.append(BETA * ((logsum / max(1, number) if case["average"] else logsum) - s["ref_logp"][i].double()))
        for i in range(case["pairs"]):
            m = rewards[2 * i] - rewards[2 * i + 1]
            if case["loss"] == "squared":
                losses.append((m / BETA - 0.5 / BETA) ** 2 * _scale(case, case["pairs"]))
            else:
                losses.append((0.9 * torch.nn.functional.softplus(-m) + 0.1 * torch.nn.functional.softplus(m)) * _scale(case, case["pairs"]))
        total = torch.stack(losses).sum()
        found.update(loss=torch.stack(losses).detach(), rewards=torch.stack(rewards).detach())
    g = torch.autograd.grad(total if kind == "nll" else -total, lead)[0]
    grads = []
    for r in range(0, t, step):
        x = s["logits"][r:r + step].double().requires_grad_()
        rows = torch.where(valid[r:r + step], _exact_logp(x, tokens[r:r + step].clamp(min=0), tau)[1], 0.0)
        grads.append(torch.autograd.grad((g[r:r + step] * rows).sum(), x)[0])
    found["dlogits"] = torch.cat(grads)
    return found


def work(case):
    t, v = case["rows"], case["vocab"]
    size = 4 if case["type"] == "fp32" else 2
    on = t - int(case["out"] * t)
    read = written = 0
    if case["kind"] == "preference":
        written = (t - case["tail"]) * v * size
        on = (t - case["tail"]) * (1.0 - case["out"])
    elif case["kind"] != "score":
        written = t * v * size
    read = on * v * size
    if case["kind"] == "distill":
        read += on * case["kept"] * (4 + size)
    # a row's scores are read once, each has its distance, exponential and sum, and its gradient one product
    return {"bytes": read + written + 32.0 * t, "flops": on * v * (4.0 if case["kind"] == "score" else 6.0)}

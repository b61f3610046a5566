"""Measured cases of the log-probability objectives (``warpgbm_b200.objectives``).

Four calls: ``label_logprobs`` (with ``label_logprobs_grad``),
``preference_loss``, ``policy_loss`` and ``policy_loss_logits``.  ``run`` makes
them where ``own`` is true and computes the same results with elementary torch
operations in 32 bits where it is false; ``exact`` restates the definitions in
64 bits.

z = logits / temperature; logp = log softmax(z)[label]; a negative label leaves
its row out (zeros in every output).  A sequence is a range of tokens between
two offsets; a false mask entry leaves a token out.
"""
import math

import torch

own = False

DEV = "cuda"
BETA = 0.1
CLIP_LOW, CLIP_HIGH = 0.2, 0.28
KL_COEF, ENTROPY_COEF = 0.05, 0.01
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # one sampled token scored while serving: latency
        dict(name="logprobs_1x131072_bf16", op="logprobs", rows=1, classes=131072, dtype="bfloat16",
             pad=0, grad=False, entropy=False),
        # scoring a batch of sequences under a frozen model, with the entropies
        dict(name="logprobs_4096x131072_bf16", op="logprobs", rows=4096, classes=131072, dtype="bfloat16",
             pad=0, grad=False, entropy=True),
        # a training step's log-probs and gradient; odd class count, logits a slice of a wider buffer
        dict(name="logprobs_train_2047x50001_f16", op="logprobs", rows=2047, classes=50001, dtype="float16",
             pad=15, grad=True, entropy=False),
        # class scores of a boosted multiclass forest: a million rows, few classes
        dict(name="logprobs_train_1000000x7_f32", op="logprobs", rows=1000000, classes=7, dtype="float32",
             pad=0, grad=True, entropy=False),
        # a handful of preference pairs of short answers: latency
        dict(name="preference_8pairs", op="preference", groups=4, per_group=4, pairs=8, mean_length=32,
             loss="sigmoid", average=False, weights=False),
        # a large batch of ragged answers, four to a prompt, answers shared by pairs
        dict(name="preference_4096pairs", op="preference", groups=1024, per_group=4, pairs=4096, mean_length=800,
             loss="sigmoid", average=False, weights=False),
        # a reward model boosted on weighted comparisons of rows: every row is its own sequence
        dict(name="preference_scores_2000000pairs", op="preference", groups=250000, per_group=4, pairs=2000000,
             mean_length=0, loss="sigmoid", average=False, weights=True),
        # one short rollout
        dict(name="policy_tokens_777", op="policy", sequences=3, tokens=777, kl="k3", reduction="token",
             broadcast=False),
        # a large batch of rollouts, one advantage for each answer, mean over answers
        dict(name="policy_tokens_4000000", op="policy", sequences=4001, tokens=4000000, kl="k3",
             reduction="sequence", broadcast=True),
        # the whole policy step on a micro-batch's logits
        dict(name="policy_logits_4096x131072_bf16", op="policy_logits", rows=4096, classes=131072, dtype="bfloat16",
             pad=0, kl="k3", reduction="token", sequences=7),
        # a contextual bandit: ten actions, a million logged decisions
        dict(name="policy_logits_1000000x10_f32", op="policy_logits", rows=1000000, classes=10, dtype="float32",
             pad=0, kl="k2", reduction="token", sequences=1),
        # a small ragged micro-batch in single precision, odd class count
        dict(name="policy_logits_333x32001_f32", op="policy_logits", rows=333, classes=32001, dtype="float32",
             pad=0, kl="k1", reduction="sequence", sequences=9),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "preference", "policy", "policy_logits", "policy_logits"])
    if op in ("logprobs", "policy_logits"):
        dtype = rng.choice(["float32", "bfloat16", "float16"])
        classes = _spread(rng, 2, 200000)
        most = (1 << 28 if dtype == "float32" else 1 << 29) // classes  # logits of the largest listed case
        if op == "logprobs":
            most //= 2
        least = 1 if op == "logprobs" else 4  # a policy step has several tokens
        case = dict(op=op, rows=_spread(rng, least, min(most, 1500000)), classes=classes, dtype=dtype,
                    pad=rng.choice([0, 0, 1, 8, 63]))
        if op == "logprobs":
            case.update(grad=rng.random() < 0.5, entropy=rng.random() < 0.5)
            if case["grad"]:
                case["entropy"] = False
        else:
            case.update(kl=rng.choice(["k1", "k2", "k3"]), reduction=rng.choice(["token", "sequence"]),
                        sequences=_spread(rng, 1, max(1, case["rows"] // 4)))
        return case
    if op == "preference":
        mean_length = 0 if rng.random() < 1 / 3 else _spread(rng, 1, 10000)
        per_group = rng.choice([2, 4, 8])
        groups = _spread(rng, 1, 1000000 // (per_group * max(1, mean_length)))
        return dict(op=op, groups=groups, per_group=per_group,
                    pairs=_spread(rng, 1, max(1, min(2000000, 2 * groups * per_group))), mean_length=mean_length,
                    loss=rng.choice(["sigmoid", "square"]), average=mean_length > 0 and rng.random() < 0.5,
                    weights=rng.random() < 0.5)
    tokens = _spread(rng, 1, 4000000)
    return dict(op=op, sequences=_spread(rng, 1, max(1, tokens // 3)), tokens=tokens,
                kl=rng.choice(["k1", "k2", "k3"]), reduction=rng.choice(["token", "sequence"]),
                broadcast=rng.random() < 0.5)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _uniform(gen, n, lo, hi):
    return torch.rand(n, device=DEV, generator=gen) * (hi - lo) + lo


def _integers(gen, n, hi, dtype=torch.int64):
    return torch.randint(0, hi, (n,), device=DEV, generator=gen, dtype=dtype)


def _log_ratios(gen, n):
    """Log ratios of a policy that has moved a little.  They lie on odd
    multiples of 1/128, away from the logarithms of the clip bounds: on a
    bound the last bit of a log-prob would decide a whole token's gradient."""
    return (torch.floor(torch.randn(n, device=DEV, generator=gen) * 12.0) + 0.5) / 64.0


def _offsets(gen, sequences, tokens):
    """Ragged offsets [sequences + 1] over `tokens` tokens (some sequences may be empty)."""
    cuts = _integers(gen, sequences - 1, tokens + 1).sort().values
    ends = torch.tensor([0, tokens], device=DEV)
    return torch.cat([ends[:1], cuts, ends[1:]])


def _logits(gen, case):
    n, k, dtype = case["rows"], case["classes"], DTYPES[case["dtype"]]
    wide = torch.randn(n, k + case["pad"], device=DEV, generator=gen, dtype=dtype).mul_(2.0)
    logits = wide[:, :k]
    labels = _integers(gen, n, k)
    # the labels were sampled from these logits: likely ones, by and large
    at = torch.arange(n, device=DEV)
    logits[at, labels] += _uniform(gen, n, 0.0, 2.0 + math.log(k)).to(dtype)
    if n >= 16:  # padding at the end of some prompts
        labels = torch.where(torch.rand(n, device=DEV, generator=gen) < 0.05, torch.full_like(labels, -100), labels)
    return logits, labels


def _log_probs(gen, n):
    return 1.5 * _uniform(gen, n, 1e-4, 1.0).log()


def _advantages(gen, shape):
    """Rewards over a baseline that lags behind an improving policy."""
    return torch.randn(shape, device=DEV, generator=gen) + 0.5


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    op = case["op"]
    state = dict(case)
    if op == "logprobs":
        state["logits"], state["labels"] = _logits(gen, case)
        if case["grad"]:
            state["grad_logp"] = torch.randn(case["rows"], device=DEV, generator=gen)
        return state
    if op == "preference":
        per, groups = case["per_group"], case["groups"]
        sequences = per * groups
        tokens = sequences * max(1, case["mean_length"])
        if case["mean_length"]:
            state["offsets"] = _offsets(gen, sequences, tokens)
            state["mask"] = torch.rand(tokens, device=DEV, generator=gen) < 0.8
        state["logp"] = _log_probs(gen, tokens)
        state["ref_logp"] = state["logp"] + 0.1 * torch.randn(tokens, device=DEV, generator=gen)
        first = _integers(gen, case["pairs"], groups) * per
        i = _integers(gen, case["pairs"], per)
        j = (i + 1 + _integers(gen, case["pairs"], per - 1)) % per
        state["chosen"], state["rejected"] = (first + i).int(), (first + j).int()
        if case["weights"]:
            state["weight"] = _uniform(gen, case["pairs"], 0.5, 1.5)
        return state
    if op == "policy":
        tokens, sequences = case["tokens"], case["sequences"]
        state["offsets"] = _offsets(gen, sequences, tokens)
        state["mask"] = torch.rand(tokens, device=DEV, generator=gen) < 0.9
        state["logp"] = _log_probs(gen, tokens)
        state["old_logp"] = state["logp"] - _log_ratios(gen, tokens)
        state["advantages"] = _advantages(gen, (sequences, 1) if case["broadcast"] else (tokens,))
    else:
        state["logits"], state["labels"] = _logits(gen, case)
        n = case["rows"]
        state["offsets"] = _offsets(gen, case["sequences"], n)
        step = max(1, (1 << 28) // case["classes"])
        logp = torch.cat([torch.log_softmax(state["logits"][a:a + step].float(), 1).gather(
            1, state["labels"][a:a + step, None].clamp(min=0))[:, 0] for a in range(0, n, step)])
        state["old_logp"] = logp - _log_ratios(gen, n)
        state["advantages"] = _advantages(gen, (n,))
        tokens = n
    # the policy's own samples are less likely under the reference it has left
    state["ref_logp"] = state["old_logp"] - 0.25 + 0.1 * torch.randn(tokens, device=DEV, generator=gen)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from warpgbm_b200 import objectives as obj
    op = s["op"]
    if op == "logprobs":
        r = obj.label_logprobs(s["logits"], s["labels"], entropy=s["entropy"])
        if s["grad"]:
            return {"logp": r.logp, "lse": r.lse,
                    "grad": obj.label_logprobs_grad(s["logits"], s["labels"], r.lse, s["grad_logp"])}
        return {"logp": r.logp, "lse": r.lse, "entropy": r.entropy}
    if op == "preference":
        r = obj.preference_loss(s["logp"], s["chosen"], s["rejected"], ref_logp=s["ref_logp"],
                                offsets=s.get("offsets"), mask=s.get("mask"), weight=s.get("weight"),
                                beta=BETA, loss=s["loss"], average=s["average"])
        return {"loss": r.loss, "grad": r.grad_logp, "chosen": r.chosen_reward, "rejected": r.rejected_reward}
    if op == "policy":
        r = obj.policy_loss(s["logp"], s["old_logp"], s["advantages"], ref_logp=s["ref_logp"],
                            offsets=s["offsets"], mask=s["mask"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH,
                            kl_coef=KL_COEF, kl=s["kl"], reduction=s["reduction"])
        return {"loss": r.loss, "grad": r.grad_logp, "policy": r.policy, "kl": r.kl, "clipped": r.clip_fraction}
    r = obj.policy_loss_logits(s["logits"], s["labels"], s["old_logp"], s["advantages"], ref_logp=s["ref_logp"],
                               offsets=s["offsets"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=KL_COEF,
                               kl=s["kl"], entropy_coef=ENTROPY_COEF, reduction=s["reduction"],
                               grad_scale=float(s["rows"]))
    return {"loss": r.loss, "grad": r.grad_logits, "logp": r.logp, "policy": r.policy, "kl": r.kl,
            "entropy": r.entropy, "clipped": r.clip_fraction}


def _plain_softmax(logits, labels):
    """(kept rows, label index, z - max, sum of exp, log-prob of the label), in 32 bits."""
    z = logits.float()
    kept = labels >= 0
    y = labels.clamp(min=0)[:, None]
    top = z.max(1, keepdim=True).values
    z = z - top
    e = z.exp()
    total = e.sum(1, keepdim=True)
    logp = z.gather(1, y) - total.log()
    return kept, y, z, e, total, logp[:, 0], (top + total.log())[:, 0]


def _plain_entropy(z, e, total):
    return (total.log() - (e * z).sum(1, keepdim=True) / total)[:, 0]


def _plain_ids(offsets, tokens):
    return torch.bucketize(torch.arange(tokens, device=offsets.device), offsets[1:], right=True)


def _plain_token_weights(kept, offsets, reduction):
    kept = kept.float()
    if reduction == "token":
        return kept / kept.sum().clamp(min=1)
    ids = _plain_ids(offsets, kept.numel())
    count = torch.zeros(offsets.numel() - 1, device=kept.device).index_add_(0, ids, kept)
    return kept / (count.clamp(min=1)[ids] * (count > 0).float().sum().clamp(min=1))


def _plain_policy(logp, old, adv, ref, kl):
    """(policy term, its derivative, kl, its derivative, clipped) of each token."""
    u = logp - old
    clipped = ((adv > 0) & (u > math.log1p(CLIP_HIGH))) | ((adv < 0) & (u < math.log1p(-CLIP_LOW)))
    ratio = u.exp()
    pg = torch.where(clipped, -adv * ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH), -adv * ratio)
    dpg = torch.where(clipped, torch.zeros_like(pg), -adv * ratio)
    d = ref - logp
    if kl == "k1":
        return pg, dpg, -d, torch.ones_like(d), clipped
    if kl == "k2":
        return pg, dpg, 0.5 * d * d, -d, clipped
    return pg, dpg, torch.expm1(d) - d, -torch.expm1(d), clipped


def _plain_total(w, x):
    return torch.where(w > 0, w * x, torch.zeros_like(x)).sum()


def _run_plain(s):
    op = s["op"]
    if op == "logprobs":
        kept, y, z, e, total, logp, lse = _plain_softmax(s["logits"], s["labels"])
        zero = torch.zeros_like(logp)
        out = {"logp": torch.where(kept, logp, zero), "lse": torch.where(kept, lse, zero)}
        if s["grad"]:
            g = torch.where(kept, s["grad_logp"], zero)[:, None]
            grad = (e / total).mul_(-g)
            out["grad"] = grad.scatter_add_(1, y, g).to(s["logits"].dtype)
        else:
            out["entropy"] = torch.where(kept, _plain_entropy(z, e, total), zero) if s["entropy"] else None
        return out
    if op == "preference":
        return _plain_preference(s)
    if op == "policy":
        logp, kept = s["logp"], s["mask"]
        adv = s["advantages"]
        if s["broadcast"]:
            adv = adv[:, 0][_plain_ids(s["offsets"], logp.numel())]
        w = _plain_token_weights(kept, s["offsets"], s["reduction"])
        pg, dpg, kl, dkl, clipped = _plain_policy(logp, s["old_logp"], adv, s["ref_logp"], s["kl"])
        policy, kl_mean = _plain_total(w, pg), _plain_total(w, kl)
        return {"loss": policy + KL_COEF * kl_mean, "grad": w * (dpg + KL_COEF * dkl), "policy": policy, "kl": kl_mean,
                "clipped": _plain_total(w, clipped.float())}
    kept, y, z, e, total, logp, _ = _plain_softmax(s["logits"], s["labels"])
    w = _plain_token_weights(kept, s["offsets"], s["reduction"])
    pg, dpg, kl, dkl, clipped = _plain_policy(logp, s["old_logp"], s["advantages"], s["ref_logp"], s["kl"])
    h = _plain_entropy(z, e, total)
    policy, kl_mean, entropy = _plain_total(w, pg), _plain_total(w, kl), _plain_total(w, h)
    g = (w * (dpg + KL_COEF * dkl) * s["rows"])[:, None]
    ge = (w * (ENTROPY_COEF * s["rows"]))[:, None]
    p = e / total
    grad = p * (ge * (z - total.log() + h[:, None]) - g)
    grad = grad.scatter_add_(1, y, g).to(s["logits"].dtype)
    return {"loss": policy + KL_COEF * kl_mean - ENTROPY_COEF * entropy, "grad": grad,
            "logp": torch.where(kept, logp, torch.zeros_like(logp)), "policy": policy, "kl": kl_mean,
            "entropy": entropy, "clipped": _plain_total(w, clipped.float())}


def _plain_preference(s):
    logp, pairs = s["logp"], s["pairs"]
    d = logp - s["ref_logp"]
    c, r = s["chosen"].long(), s["rejected"].long()
    if "offsets" in s:
        sequences = s["offsets"].numel() - 1
        ids = _plain_ids(s["offsets"], logp.numel())
        kept = s["mask"].float()
        total = torch.zeros(sequences, device=logp.device).index_add_(0, ids, d * kept)
        per_token = kept
        if s["average"]:
            count = torch.zeros_like(total).index_add_(0, ids, kept).clamp(min=1)
            total, per_token = total / count, kept / count[ids]
    else:
        sequences, ids, total, per_token = logp.numel(), None, d, None
    x = total[c] - total[r]
    w = s["weight"] / pairs if "weight" in s else torch.full_like(x, 1.0 / pairs)
    if s["loss"] == "sigmoid":
        h = BETA * x
        each = torch.log1p(torch.exp(-h.abs())) + (-h).clamp(min=0)
        slope = -BETA / (1 + torch.exp(h))
    else:
        each = (x - 0.5 / BETA) ** 2
        slope = 2 * (x - 0.5 / BETA)
    g = torch.zeros(sequences, device=logp.device).index_add_(0, c, w * slope).index_add_(0, r, -w * slope)
    grad = g if ids is None else g[ids] * per_token
    return {"loss": (w * each).sum(), "grad": grad, "chosen": BETA * total[c], "rejected": BETA * total[r]}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op in ("logprobs", "policy_logits"):
        n, size = case["rows"], 4 if case["dtype"] == "float32" else 2
        cells = n * case["classes"]
        if op == "logprobs":
            moved = cells * size * (2 if case["grad"] else 1) + n * (8 + 8 + (4 if case["grad"] or case["entropy"] else 0))
            return {"bytes": moved, "flops": cells * (7 if case["grad"] else 5)}
        return {"bytes": 2 * cells * size + n * (8 + 3 * 4 + 4) + 8 * case["sequences"], "flops": cells * 11}
    if op == "preference":
        sequences = case["groups"] * case["per_group"]
        ragged = case["mean_length"] > 0
        tokens = sequences * max(1, case["mean_length"])
        moved = tokens * (13 if ragged else 12) + case["pairs"] * (20 if case["weights"] else 16)
        return {"bytes": moved + (8 * sequences if ragged else 0), "flops": 3 * tokens + 20 * case["pairs"]}
    adv = case["sequences"] if case["broadcast"] else case["tokens"]
    return {"bytes": case["tokens"] * 17 + 4 * adv + 8 * case["sequences"], "flops": 20 * case["tokens"]}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"logprobs": _exact_logprobs, "preference": _exact_preference, "policy": _exact_policy,
            "policy_logits": _exact_policy_logits}[case["op"]](s)


def _rows(s, fn):
    """fn(logits in 64 bits, labels, row range) over blocks of rows, joined."""
    n, step = s["rows"], max(1, (1 << 27) // s["classes"])
    parts = [fn(s["logits"][a:a + step].double(), s["labels"][a:a + step], slice(a, min(n, a + step)))
             for a in range(0, n, step)]
    return [torch.cat(p) for p in zip(*parts)]


def _exact_logprobs(s):
    def block(z, y, at):
        out = y < 0
        lse = torch.logsumexp(z, 1)
        lp = z - lse[:, None]
        logp = lp[torch.arange(len(y), device=DEV), y.clamp(min=0)]
        zero = torch.zeros_like(lse)
        got = [logp.where(~out, zero), lse.where(~out, zero)]
        if s["grad"]:
            g = s["grad_logp"][at].double().where(~out, zero)
            grad = -lp.exp_() * g[:, None]
            grad[torch.arange(len(y), device=DEV), y.clamp(min=0)] += g
            got.append(grad)
        elif s["entropy"]:
            got.append((-(lp.exp() * lp).sum(1)).where(~out, zero))
        return got
    got = _rows(s, block)
    if s["grad"]:
        return {"logp": got[0], "lse": got[1], "grad": got[2]}
    return {"logp": got[0], "lse": got[1], "entropy": got[2] if s["entropy"] else None}


def _exact_ids(offsets):
    return torch.repeat_interleave(torch.arange(offsets.numel() - 1, device=DEV), offsets.diff())


def _exact_preference(s):
    delta = s["logp"].double() - s["ref_logp"].double()
    if "offsets" in s:
        ids, mask = _exact_ids(s["offsets"]), s["mask"]
        q = s["offsets"].numel() - 1
        score = torch.zeros(q, dtype=torch.float64, device=DEV).index_add_(0, ids[mask], delta[mask])
        scale = torch.ones(q, dtype=torch.float64, device=DEV)
        if s["average"]:
            scale = 1.0 / torch.bincount(ids[mask], minlength=q).clamp(min=1).double()
        score = score * scale
    else:
        score = delta
    score.requires_grad_(True)
    x = score[s["chosen"].long()] - score[s["rejected"].long()]
    each = -torch.nn.functional.logsigmoid(BETA * x) if s["loss"] == "sigmoid" else (x - 1 / (2 * BETA)).square()
    if "weight" in s:
        each = each * s["weight"].double()
    loss = each.mean()
    (g,) = torch.autograd.grad(loss, score)
    grad = g if "offsets" not in s else torch.where(mask, (g * scale)[ids], torch.zeros_like(delta))
    score = score.detach()
    return {"loss": loss.detach(), "grad": grad, "chosen": BETA * score[s["chosen"].long()],
            "rejected": BETA * score[s["rejected"].long()]}


def _exact_terms(s, logp, kept, adv):
    """Each term's mean, the loss without entropy, and the gradient to logp, by differentiation."""
    ids = _exact_ids(s["offsets"])
    if s["reduction"] == "token":
        w = kept.double() / max(1, int(kept.sum()))
    else:
        count = torch.bincount(ids[kept], minlength=s["offsets"].numel() - 1)
        w = kept.double() / (count.clamp(min=1)[ids] * max(1, int((count > 0).sum())))
    logp = logp.clone().requires_grad_(True)
    ratio = (logp - s["old_logp"].double()).exp()
    pg = -torch.minimum(ratio * adv, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv)
    cut = ((adv > 0) & (ratio > 1 + CLIP_HIGH)) | ((adv < 0) & (ratio < 1 - CLIP_LOW))
    d = s["ref_logp"].double() - logp
    kl = {"k1": -d, "k2": d * d / 2, "k3": d.exp() - 1 - d}[s["kl"]]
    policy, kl = (w * pg).sum(), (w * kl).sum()
    loss = policy + KL_COEF * kl
    (g,) = torch.autograd.grad(loss, logp)
    return w, g, loss.detach(), policy.detach(), kl.detach(), (w * cut).sum()


def _exact_policy(s):
    adv = s["advantages"].double()
    if s["broadcast"]:
        adv = adv[_exact_ids(s["offsets"]), 0]
    _, g, loss, policy, kl, cut = _exact_terms(s, s["logp"].double(), s["mask"], adv)
    return {"loss": loss, "grad": g, "policy": policy, "kl": kl, "clipped": cut}


def _exact_policy_logits(s):
    kept = s["labels"] >= 0

    def first(z, y, at):
        lp = torch.log_softmax(z, 1)
        return lp[torch.arange(len(y), device=DEV), y.clamp(min=0)], -(lp.exp() * lp).sum(1)
    logp, h = _rows(s, first)
    w, g, loss, policy, kl, cut = _exact_terms(s, logp, kept, s["advantages"].double())
    entropy = (w * h).sum()
    n = s["rows"]

    def second(z, y, at):
        lp = torch.log_softmax(z, 1)
        p = lp.exp()
        grad = p * (ENTROPY_COEF * w[at, None] * (lp + h[at, None]) - g[at, None])
        grad[torch.arange(len(y), device=DEV), y.clamp(min=0)] += g[at]
        return (grad * n,)
    (grad,) = _rows(s, second)
    return {"loss": loss - ENTROPY_COEF * entropy, "grad": grad, "logp": logp.where(kept, torch.zeros_like(logp)),
            "policy": policy, "kl": kl, "entropy": entropy, "clipped": cut}

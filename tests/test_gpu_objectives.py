"""Log-probability objectives (warpgbm_b200.objectives) against their
definitions in 64 bits, restated here with numpy, and against differences of
the 64-bit losses.

Tolerances come from the kernels' arithmetic.  u = 2^-24 is fp32's rounding.
A row sum adds 2^d with an error of about 2 units (the exponential) plus |d|
units (the rounding of d), weighted by the probabilities, which gives at most
2 + 2 log K units, plus one unit for each addition along a thread's chain and
the tree; the log-sum-exp and the log-prob are then rounded a few times at the
size of the largest |z|.  `row_tol` adds these up.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = {d: torch.finfo(d).eps / 2 for d in (torch.float32, torch.bfloat16, torch.float16)}  # rounding to nearest
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
LOWEST = {d: torch.finfo(d).min for d in DTYPES}


@pytest.fixture(scope="module")
def obj():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from warpgbm_b200 import objectives
    return objectives


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def f64(t):
    return t.detach().double().cpu().numpy()


def make_logits(seed, n, k, dtype, pad=0, shift=0, scale=3.0):
    """[n, k] logits whose rows start `shift` elements into a buffer with `pad` spare columns."""
    buf = torch.randn(n * (k + pad) + shift, device="cuda", generator=gen(seed), dtype=torch.float32) * scale
    buf = buf.to(dtype)
    return buf[shift:].view(n, k + pad)[:, :k]


def make_labels(seed, n, k, dtype=torch.int64):
    return torch.randint(0, k, (n,), device="cuda", generator=gen(seed + 1000), dtype=dtype)


def row_tol(z):
    k = z.shape[1]
    chain = 64 + 2.0 * k / 32  # additions along a thread's share (a warp's row at worst), and the trees
    finite = np.where(np.isfinite(z), np.abs(z), 0.0)
    finite = np.minimum(finite, 1e4).max(1)
    return U * (chain + 2 * math.log(k) + 8 + 4 * finite)


def plain_rows(logits, labels, temperature=1.0):
    """logp, lse, entropy, p (64 bits) of every row; rows left out are zero."""
    z = f64(logits) / temperature
    y = labels.cpu().numpy()
    n, k = z.shape
    logp, lse, ent, p = np.zeros(n), np.zeros(n), np.zeros(n), np.zeros((n, k))
    with np.errstate(all="ignore"):
        for i in range(n):
            if y[i] < 0:
                continue
            if (z[i] == -np.inf).all():
                logp[i] = lse[i] = -np.inf
                continue
            m = z[i].max()
            e = np.exp(z[i] - m)
            lse[i] = m + np.log(e.sum())
            lp = (z[i] - m) - np.log(e.sum())
            p[i] = np.exp(lp)
            logp[i] = lp[y[i]] if y[i] < k else np.nan
            ent[i] = -(p[i] * np.where(p[i] > 0, lp, 0.0)).sum()
    return logp, lse, ent, p


def plain_row_grad(p, logp_all, labels, g, ge, ent):
    """Gradient to z from the gradients to logp and to the entropy."""
    n, k = p.shape
    y = labels.cpu().numpy()
    out = np.zeros((n, k))
    for i in range(n):
        if y[i] < 0 or not p[i].any():
            continue
        out[i] = -g[i] * p[i] - ge[i] * p[i] * (np.where(p[i] > 0, logp_all[i], 0.0) + ent[i])
        out[i, y[i]] += g[i]
    return out


def close(got, want, tol, name=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, name
    assert np.array_equal(np.isnan(got), np.isnan(want)), name
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]) and not np.isinf(got[~inf]).any(), name
    ok = np.isfinite(want)
    err = np.abs(got - want)[ok]
    bound = np.broadcast_to(tol, want.shape)[ok]
    worst = (err - bound).max(initial=-1.0)
    assert worst <= 0, f"{name}: error {err[np.argmax(err - bound)]:.3g} over {bound[np.argmax(err - bound)]:.3g}"


def grad_tol(want, p, logp_all, g, ge, ent, tol, dtype):
    """One rounding to the dtype, and the row's error through p, log p and H."""
    with np.errstate(all="ignore"):
        lp = np.where(p > 0, np.abs(logp_all), 0.0)
    slope = np.abs(g)[:, None] + np.abs(ge)[:, None] * (1 + lp + np.abs(ent)[:, None])
    rel = 4 * tol[:, None] + 8 * U * (1 + lp)
    return p * slope * rel + (np.abs(g)[:, None] * 4 * U) + EPS[dtype] * 1.01 * np.abs(want) + TINY[dtype]


# ---------------------------------------------------------------------------
# label log-probs
# ---------------------------------------------------------------------------

SHAPES = [(1, 1), (5, 2), (33, 3), (1000, 7), (257, 10), (64, 31), (40, 32), (41, 33), (9, 100), (17, 255), (4, 1023),
          (3, 1024), (5, 1025), (2, 4099), (3, 8192), (2, 20001), (1, 50001), (2, 131072), (1, 150001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", SHAPES)
def test_label_logprobs(obj, n, k, dtype):
    x = make_logits(n + k, n, k, dtype, pad=(k % 3) * 5, shift=k % 4)
    y = make_labels(k, n, k, torch.int32 if k % 2 else torch.int64)
    if n > 3:
        y[2] = -100
    for temperature in (1.0, 0.7):
        logp, lse, ent, _ = plain_rows(x, y, temperature)
        tol = row_tol(f64(x) / temperature)
        r = obj.label_logprobs(x, y, temperature=temperature, entropy=True)
        close(f64(r.logp), logp, tol, "logp")
        close(f64(r.lse), lse, tol, "lse")
        close(f64(r.entropy), ent, 4 * tol * (1 + ent), "entropy")
        bare = obj.label_logprobs(x, y, temperature=temperature)
        assert bare.entropy is None
        close(f64(bare.logp), logp, tol, "logp")
        close(f64(bare.lse), lse, tol, "lse")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", SHAPES)
def test_label_logprobs_grad(obj, n, k, dtype):
    x = make_logits(n + k + 1, n, k, dtype, pad=k % 2, shift=k % 3)
    y = make_labels(k, n, k)
    if n > 3:
        y[1] = -1
    g = torch.randn(n, device="cuda", generator=gen(3))
    ge = torch.randn(n, device="cuda", generator=gen(4))
    logp, lse, ent, p = plain_rows(x, y)
    lp = f64(x) - lse[:, None]
    tol = row_tol(f64(x))
    r = obj.label_logprobs(x, y, entropy=True)
    got = obj.label_logprobs_grad(x, y, r.lse, g)
    zero = np.zeros(n)
    want = plain_row_grad(p, lp, y, f64(g), zero, ent)
    assert got.dtype == dtype and got.shape == x.shape
    close(f64(got), want, grad_tol(want, p, lp, f64(g), zero, ent, tol, dtype), "grad")
    got = obj.label_logprobs_grad(x, y, r.lse, g, entropy=r.entropy, grad_entropy=ge)
    want = plain_row_grad(p, lp, y, f64(g), f64(ge), ent)
    close(f64(got), want, grad_tol(want, p, lp, f64(g), f64(ge), ent, 4 * tol * (1 + ent), dtype), "grad with entropy")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [6, 200, 5000, 70001])
def test_masked_places_and_empty_rows(obj, k, dtype):
    x = make_logits(k, 6, k, dtype, pad=3).clone()
    x[0, 1:] = -math.inf                       # one class left, the label
    x[1, :] = -math.inf                        # nothing left
    x[2, ::2] = -math.inf
    x[3, : k - 1] = LOWEST[dtype]              # masked with the type's lowest value
    x[4, :] = LOWEST[dtype]                    # all of them: a uniform row
    y = torch.tensor([0, 2, 2, k - 1, 1, 3], device="cuda")  # row 2's label is masked
    logp, lse, ent, p = plain_rows(x, y)
    tol = row_tol(f64(x))
    r = obj.label_logprobs(x, y, entropy=True)
    assert logp[1] == -np.inf and logp[2] == -np.inf
    close(f64(r.logp), logp, tol, "logp")
    close(f64(r.entropy), ent, 4 * tol * (1 + ent), "entropy")
    close(f64(r.lse), lse, tol + U * np.where(np.isfinite(lse), np.abs(lse), 0), "lse")
    g = torch.ones(6, device="cuda")
    with np.errstate(all="ignore"):
        lp = np.log(p)
    got = obj.label_logprobs_grad(x, y, r.lse, g)
    want = plain_row_grad(p, lp, y, f64(g), np.zeros(6), ent)
    close(f64(got), want, grad_tol(want, p, lp, f64(g), np.zeros(6), ent, tol, dtype), "grad")
    assert not got[1].any()


@pytest.mark.parametrize("k", [9, 3000])
def test_nan_and_infinite_logits_stay_in_their_row(obj, k):
    x = make_logits(k, 5, k, torch.float32).clone()
    y = make_labels(k, 5, k)
    clean = obj.label_logprobs(x, y, entropy=True)
    x[1, 3] = math.nan
    x[3, k - 1] = math.inf
    y[4] = -1
    x[4, :] = math.nan                          # a row that is left out
    r = obj.label_logprobs(x, y, entropy=True)
    for t, c in ((r.logp, clean.logp), (r.lse, clean.lse), (r.entropy, clean.entropy)):
        assert torch.isnan(t[1]) and torch.isnan(t[3])
        assert t[0] == c[0] and t[2] == c[2] and t[4] == 0
    got = obj.label_logprobs_grad(x, y, r.lse, torch.full((5,), 2.0, device="cuda"))
    assert torch.isnan(got[1]).all() and torch.isfinite(got[[0, 2]]).all() and not got[4].any()


def test_label_out_of_range_gives_nan(obj):
    x = make_logits(1, 3, 11, torch.float32)
    y = torch.tensor([0, 11, 10], device="cuda")
    r = obj.label_logprobs(x, y)
    assert torch.isnan(r.logp).tolist() == [False, True, False] and torch.isfinite(r.lse).all()
    g = obj.label_logprobs_grad(x, y, r.lse, torch.ones(3, device="cuda"))
    assert torch.isnan(g).all(1).tolist() == [False, True, False]


def test_no_rows(obj):
    x = torch.empty((0, 5), device="cuda")
    y = torch.empty(0, dtype=torch.int64, device="cuda")
    r = obj.label_logprobs(x, y, entropy=True)
    assert r.logp.shape == r.lse.shape == r.entropy.shape == (0,)
    assert obj.label_logprobs_grad(x, y, r.lse, r.logp).shape == (0, 5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k,pad", [(50, 10, 0), (7, 1500, 5), (3, 40000, 8)])
def test_gradient_in_place_and_into_other_strides(obj, n, k, pad, dtype):
    x = make_logits(7, n, k, dtype, pad=pad)
    y = make_labels(7, n, k)
    g = torch.randn(n, device="cuda", generator=gen(5))
    lse = obj.label_logprobs(x, y).lse
    want = obj.label_logprobs_grad(x, y, lse, g)
    for extra in (1, 3, 8):
        wide = torch.full((n, k + extra), 7.0, dtype=dtype, device="cuda")
        assert obj.label_logprobs_grad(x, y, lse, g, out=wide[:, 1:k + 1] if extra == 8 else wide[:, :k]) is not None
        inner = wide[:, 1:k + 1] if extra == 8 else wide[:, :k]
        assert torch.equal(inner, want)
        outer = wide[:, k + 1:] if extra == 8 else wide[:, k:]
        assert (outer == 7.0).all()
    spare = x.clone() if pad == 0 else x
    got = obj.label_logprobs_grad(spare, y, lse, g, out=spare)
    assert got.data_ptr() == spare.data_ptr() and torch.equal(got, want)


def test_large_row_offsets(obj):
    """Rows whose elements lie beyond 2^31 of the first."""
    n, k = 70000, 40000
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    x = torch.zeros((n, k), dtype=torch.bfloat16, device="cuda")
    y = torch.full((n,), -1, device="cuda")
    y[-1], y[0] = 5, 6
    x[-1, 5], x[0, 6] = 4.0, 2.0
    r = obj.label_logprobs(x, y)
    for i, top in ((-1, 4.0), (0, 2.0)):
        assert abs(float(r.logp[i]) - (top - math.log(math.exp(top) + k - 1))) < 1e-5
    g = torch.ones(n, device="cuda")
    out = obj.label_logprobs_grad(x, y, r.lse, g, out=x)
    assert abs(float(out[-1, 5]) - (1 - math.exp(float(r.logp[-1])))) < 2 ** -8
    assert not out[1:-1].any()


# ---------------------------------------------------------------------------
# preference loss
# ---------------------------------------------------------------------------

def make_offsets(seed, lengths, before=0):
    return torch.tensor([before] + list(before + np.cumsum(lengths)), device="cuda")


def plain_scores(d, offsets, mask, average):
    q = len(offsets) - 1
    score, ids = np.zeros(q), np.full(len(d), -1)
    count = np.zeros(q)
    for s in range(q):
        a, b = offsets[s], offsets[s + 1]
        keep = mask[a:b]
        ids[a:b] = s
        count[s] = keep.sum()
        score[s] = d[a:b][keep].sum()
        if average and count[s]:
            score[s] /= count[s]
    return score, ids, count


def plain_pair(x, kind, beta, smoothing):
    h = beta * x
    sp = lambda v: np.maximum(v, 0) + np.log1p(np.exp(-np.abs(v)))  # noqa: E731
    sig = lambda v: np.where(v >= 0, 1 / (1 + np.exp(-np.abs(v))), np.exp(-np.abs(v)) / (1 + np.exp(-np.abs(v))))  # noqa: E731
    if kind == "sigmoid":
        return (1 - smoothing) * sp(-h) + smoothing * sp(h), beta * (smoothing * sig(h) - (1 - smoothing) * sig(-h))
    if kind == "hinge":
        return np.maximum(0, 1 - h), np.where(h < 1, -beta, 0.0)
    return (x - 0.5 / beta) ** 2, 2 * (x - 0.5 / beta)


def check_preference(obj, lengths, pairs, *, kind="sigmoid", beta=0.3, smoothing=0.0, average=False, ref=True,
                     mask=True, weight=True, index=torch.int32, offset=torch.int64, seed=0, before=0, after=0):
    ragged = lengths is not None
    q = len(lengths) if ragged else 400
    t = before + int(np.sum(lengths)) + after if ragged else q
    g = gen(seed)
    logp = -torch.rand(t, device="cuda", generator=g) * 3
    refp = logp + 0.3 * torch.randn(t, device="cuda", generator=g) if ref else None
    m = (torch.rand(t, device="cuda", generator=g) < 0.7) if ragged and mask else None
    off = make_offsets(seed, lengths, before) if ragged else None
    c = torch.randint(0, q, (pairs,), device="cuda", generator=g).to(index)
    r = torch.randint(0, q, (pairs,), device="cuda", generator=g).to(index)
    w = torch.rand(pairs, device="cuda", generator=g) + 0.5 if weight else None
    got = obj.preference_loss(logp, c, r, ref_logp=refp, offsets=off.to(offset) if ragged else None, mask=m, weight=w,
                              beta=beta, loss=kind, label_smoothing=smoothing, average=average)
    d = f64(logp) - (f64(refp) if ref else 0.0)
    mm = m.cpu().numpy() if m is not None else np.ones(t, bool)
    if ragged:
        score, ids, count = plain_scores(d, off.cpu().numpy(), mm, average)
        size, _, _ = plain_scores(np.abs(d), off.cpu().numpy(), mm, average)
    else:
        score, ids, count, size = d, np.arange(t), np.ones(t), np.abs(d)
    ci, ri = c.long().cpu().numpy(), r.long().cpu().numpy()
    x = score[ci] - score[ri]
    ww = f64(w) if weight else np.ones(pairs)
    each, slope = plain_pair(x, kind, beta, smoothing)
    ex = 2 * U * (size[ci] + size[ri] + np.abs(x))  # rounding of every difference, and of x
    bend = {"sigmoid": beta * beta / 4, "hinge": 0.0, "square": 2.0}[kind]
    loss = (ww * each).sum() / max(pairs, 1)
    close(float(got.loss), loss, ((ww * (np.abs(slope) * ex + 8 * U * (np.abs(each) + 1))).sum() / max(pairs, 1)
                                  + U * abs(loss)), "loss")
    gs, es = np.zeros(q), np.zeros(q)
    np.add.at(gs, ci, ww * slope / max(pairs, 1))
    np.add.at(gs, ri, -ww * slope / max(pairs, 1))
    each_err = ww * (bend * ex + 8 * U * (np.abs(slope) + (beta if kind != "square" else 0))) / max(pairs, 1)
    np.add.at(es, ci, each_err)
    np.add.at(es, ri, each_err)
    keep = mm & (ids >= 0)
    want, tol = np.zeros(t), np.zeros(t)
    per = 1 / np.maximum(count, 1) if average else np.ones(q)
    want[keep] = (gs * per)[ids[keep]]
    tol[keep] = (es * per)[ids[keep]]
    close(f64(got.grad_logp), want, tol + 2 * U * np.abs(want), "grad")
    close(f64(got.chosen_reward), beta * score[ci], beta * 4 * U * (size[ci] + np.abs(score[ci])), "chosen")
    close(f64(got.rejected_reward), beta * score[ri], beta * 4 * U * (size[ri] + np.abs(score[ri])), "rejected")


LENGTHS = {"one": [1, 1], "few": [3, 0, 5, 1, 0, 0, 7], "tile": [1024, 1, 1023, 0, 1025, 2048],
           "long": [40000, 3, 0, 70001], "short": [1, 0, 2, 1] * 700, "mixed": [0, 900, 17, 0, 1, 3000, 33, 31, 32] * 5,
           "nothing": [0, 0, 0]}


@pytest.mark.parametrize("kind,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.1), ("hinge", 0.0), ("square", 0.0)])
@pytest.mark.parametrize("lengths", list(LENGTHS))
def test_preference_ragged(obj, lengths, kind, smoothing):
    n = len(LENGTHS[lengths])
    check_preference(obj, LENGTHS[lengths], 3 * n, kind=kind, smoothing=smoothing, seed=n)
    check_preference(obj, LENGTHS[lengths], n, kind=kind, smoothing=smoothing, seed=n + 1, average=True,
                     weight=False, index=torch.int64, offset=torch.int32)


@pytest.mark.parametrize("ref,mask,before,after", [(False, True, 0, 0), (True, False, 0, 0), (True, True, 5, 1100),
                                                   (False, False, 1500, 3)])
def test_preference_options(obj, ref, mask, before, after):
    check_preference(obj, LENGTHS["mixed"], 100, ref=ref, mask=mask, before=before, after=after)


@pytest.mark.parametrize("pairs", [0, 1, 7, 300, 5000])
@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "square"])
def test_preference_scores(obj, pairs, kind):
    check_preference(obj, None, pairs, kind=kind, beta=1.0, ref=pairs % 2 == 0, seed=pairs)


def test_preference_gradient_against_differences(obj):
    lengths, beta = [4, 3, 5], 0.5
    off = make_offsets(0, lengths)
    t = 12
    logp = -torch.rand(t, device="cuda", generator=gen(1))
    mask = torch.tensor([1, 1, 0, 1, 1, 1, 1, 0, 1, 1, 1, 1], dtype=torch.uint8, device="cuda")
    c, r = torch.tensor([0, 1, 2, 0], device="cuda"), torch.tensor([1, 2, 0, 2], device="cuda")
    for kind in ("sigmoid", "hinge", "square"):
        got = f64(obj.preference_loss(logp, c, r, offsets=off, mask=mask, beta=beta, loss=kind).grad_logp)

        def loss(v):
            s, _, _ = plain_scores(v, off.cpu().numpy(), mask.cpu().numpy().astype(bool), False)
            return plain_pair(s[c.cpu().numpy()] - s[r.cpu().numpy()], kind, beta, 0.0)[0].mean()
        base, h = f64(logp), 1e-5
        for i in range(t):
            up, down = base.copy(), base.copy()
            up[i] += h
            down[i] -= h
            # central differences: h^2 times a third derivative below 1, and 64-bit noise over h
            assert abs(got[i] - (loss(up) - loss(down)) / (2 * h)) < 1e-9 + 16 * U


def test_preference_masked_values_do_not_leak(obj):
    off = make_offsets(0, [3, 3])
    logp = torch.tensor([-1.0, math.nan, -2.0, -0.5, math.inf, -math.inf], device="cuda")
    mask = torch.tensor([1, 0, 1, 1, 0, 0], dtype=torch.bool, device="cuda")
    c, r = torch.tensor([0], device="cuda"), torch.tensor([1], device="cuda")
    got = obj.preference_loss(logp, c, r, offsets=off, mask=mask, beta=1.0)
    x = -3.0 + 0.5
    assert abs(float(got.loss) - math.log1p(math.exp(-x))) < 1e-6
    assert torch.isfinite(got.grad_logp).all() and got.grad_logp[[1, 4, 5]].tolist() == [0, 0, 0]
    mask[:] = False
    got = obj.preference_loss(logp, c, r, offsets=off, mask=mask, beta=1.0)
    assert abs(float(got.loss) - math.log(2)) < 1e-6 and not got.grad_logp.any()


def test_preference_infinite_scores(obj):
    """A sequence that one side gives no probability: limits, not NaN; both sides: NaN."""
    logp = torch.tensor([-math.inf, -1.0, -2.0, -math.inf], device="cuda")
    c = torch.tensor([0], device="cuda")
    lose = obj.preference_loss(logp, c, c + 1, beta=1.0)
    assert float(lose.loss) == math.inf and lose.grad_logp.tolist() == [-1, 1, 0, 0]
    win = obj.preference_loss(logp, c + 1, c, beta=1.0)
    assert float(win.loss) == 0 and not win.grad_logp.any()
    both = obj.preference_loss(logp, c, c + 3, beta=1.0)
    assert math.isnan(float(both.loss)) and torch.isnan(both.grad_logp).tolist() == [True, False, False, True]


def test_preference_index_out_of_range(obj):
    logp = torch.zeros(4, device="cuda")
    for bad in (4, -1):
        got = obj.preference_loss(logp, torch.tensor([0, 1], device="cuda"), torch.tensor([bad, 2], device="cuda"))
        assert math.isnan(float(got.loss)) and math.isnan(float(got.rejected_reward[0]))
        assert torch.isfinite(got.grad_logp[1:]).all()


def test_preference_bounds_of_offsets(obj):
    """Offsets that do not rise, or leave the tokens, touch nothing out of range."""
    logp = -torch.rand(3000, device="cuda", generator=gen(0))
    c, r = torch.tensor([0, 1], device="cuda"), torch.tensor([1, 2], device="cuda")
    for off in ([0, 5000, 9000, 10 ** 10], [-5, 100, 50, 4000], [2000, 1000, 500, 0]):
        got = obj.preference_loss(logp, c, r, offsets=torch.tensor(off, device="cuda"))
        assert got.grad_logp.shape == (3000,) and math.isfinite(float(got.loss))


def test_preference_shared_sequence_sums_do_not_depend_on_order(obj):
    q, p = 50, 20000
    logp = torch.randn(q, device="cuda", generator=gen(2))
    c = torch.randint(0, q, (p,), device="cuda", generator=gen(3))
    r = torch.randint(0, q, (p,), device="cuda", generator=gen(4))
    first = obj.preference_loss(logp, c, r, beta=1.0)
    for seed in range(3):
        perm = torch.randperm(p, device="cuda", generator=gen(seed))
        again = obj.preference_loss(logp, c[perm], r[perm], beta=1.0)
        assert torch.equal(first.grad_logp, again.grad_logp)
    assert torch.equal(first.loss, obj.preference_loss(logp, c, r, beta=1.0).loss)


# ---------------------------------------------------------------------------
# policy loss
# ---------------------------------------------------------------------------

def plain_policy(logp, old, adv, ref, kind, lo, hi):
    with np.errstate(all="ignore"):
        u = logp - old
        ratio = np.exp(u)
        cut = ((adv > 0) & (u > np.log1p(hi))) | ((adv < 0) & (u < np.log1p(-lo)))
        pg = -np.minimum(ratio * adv, np.clip(ratio, 1 - lo, 1 + hi) * adv)
        dpg = np.where(cut, 0.0, -adv * ratio)
        if ref is None:
            return pg, dpg, 0 * u, 0 * u, cut
        d = ref - logp
        kl = {"k1": -d, "k2": d * d / 2, "k3": np.expm1(d) - d}[kind]
        dkl = {"k1": np.ones_like(d), "k2": -d, "k3": -np.expm1(d)}[kind]
    return pg, dpg, kl, dkl, cut


def plain_weights(keep, offsets, reduction):
    t = len(keep)
    if reduction == "token":
        return keep / max(1, keep.sum())
    w, full = np.zeros(t), 0
    for s in range(len(offsets) - 1):
        a, b = offsets[s], offsets[s + 1]
        n = keep[a:b].sum()
        full += n > 0
        w[a:b] = keep[a:b] / max(1, n)
    return w / max(1, full)


def ratios(seed, n):
    """Log ratios away from the logarithms of 0.8 and 1.28, where one rounding decides."""
    return (torch.floor(torch.randn(n, device="cuda", generator=gen(seed)) * 12) + 0.5) / 64


def seq_of(offsets, t):
    ids = np.full(t, -1)
    for s in range(len(offsets) - 1):
        ids[offsets[s]:offsets[s + 1]] = s
    return ids


@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("broadcast", [False, True])
@pytest.mark.parametrize("kl", ["k1", "k2", "k3", None])
@pytest.mark.parametrize("lengths", list(LENGTHS))
def test_policy_tokens(obj, lengths, kl, broadcast, reduction):
    lens = LENGTHS[lengths]
    t = int(np.sum(lens))
    off = make_offsets(0, lens)
    logp = -torch.rand(t, device="cuda", generator=gen(t)) * 4
    old = logp - ratios(t + 1, t)
    ref = old - 0.2 + 0.1 * torch.randn(t, device="cuda", generator=gen(5)) if kl else None
    mask = torch.rand(t, device="cuda", generator=gen(6)) < 0.8 if lengths != "short" else None
    adv = torch.randn((len(lens), 1) if broadcast else (t,), device="cuda", generator=gen(7)) + 0.3
    coef = 0.1 if kl else 0.0
    got = obj.policy_loss(logp, old, adv, ref_logp=ref, offsets=off, mask=mask, clip_low=0.2, clip_high=0.28,
                          kl_coef=coef, kl=kl or "k3", reduction=reduction)
    o = off.cpu().numpy()
    a = f64(adv)[seq_of(o, t), 0] if broadcast else f64(adv)
    keep = mask.cpu().numpy() if mask is not None else np.ones(t, bool)
    w = plain_weights(keep, o, reduction)
    # log ratio, ratio and KL difference are taken from float32 inputs: exact here
    pg, dpg, klt, dkl, cut = plain_policy(f64(logp), f64(old), a, f64(ref) if kl else None, kl, 0.2, 0.28)
    pol, klm = (w * pg).sum(), (w * klt).sum()
    err = 8 * U * (np.abs(a) * 2 + 1) + 8 * U * np.abs(f64(logp))
    tol = (w * err).sum() + 4 * U * (abs(pol) + abs(klm))
    close(float(got.policy), pol, tol, "policy")
    close(float(got.kl), klm, tol, "kl")
    close(float(got.loss), pol + coef * klm, 2 * tol, "loss")
    close(float(got.clip_fraction), (w * cut).sum(), 2 * U, "clipped")
    want = w * (dpg + coef * dkl)
    close(f64(got.grad_logp), want, w * err + 4 * U * np.abs(want), "grad")


def test_policy_without_offsets_or_mask(obj):
    t = 5000
    logp = -torch.rand(t, device="cuda", generator=gen(1))
    old = logp - ratios(2, t)
    adv = torch.randn(t, device="cuda", generator=gen(3))
    got = obj.policy_loss(logp, old, adv)
    pg, dpg, _, _, cut = plain_policy(f64(logp), f64(old), f64(adv), None, "k3", 0.2, 0.2)
    close(float(got.loss), pg.mean(), 16 * U * (np.abs(f64(adv)).mean() + 1), "loss")
    close(f64(got.grad_logp), dpg / t, (16 * U * (np.abs(f64(adv)) + 1)) / t, "grad")
    assert float(got.kl) == 0 and abs(float(got.clip_fraction) - cut.mean()) < 2 * U


def test_policy_masked_values_do_not_leak_and_empty_masks(obj):
    bad = torch.tensor([-1.0, math.nan, math.inf, -math.inf, -2.0], device="cuda")
    good = torch.tensor([-1.0, -1.0, -1.0, -1.0, -2.0], device="cuda")
    mask = torch.tensor([True, False, False, False, True], device="cuda")
    one = torch.ones(5, device="cuda")
    off = torch.tensor([0, 1, 4, 5], device="cuda")
    for reduction in ("token", "sequence"):
        kw = dict(ref_logp=good, kl_coef=0.1, mask=mask, offsets=off, reduction=reduction)
        a = obj.policy_loss(bad, bad, bad.nan_to_num(0, 1, 1) * 0 + one, **kw)
        b = obj.policy_loss(good, good, one, **kw)
        for x, y in zip(a, b):
            assert torch.equal(x, y)
        none = obj.policy_loss(bad, bad, bad, **{**kw, "mask": mask & False})
        assert [float(x) for x in (none.loss, none.policy, none.kl, none.clip_fraction)] == [0, 0, 0, 0]
        assert not none.grad_logp.any()
    empty = torch.empty(0, device="cuda")
    r = obj.policy_loss(empty, empty, empty)
    assert float(r.loss) == 0 and r.grad_logp.shape == (0,)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", [(1, 1), (5, 2), (300, 3), (1000, 10), (70, 33), (40, 500), (9, 1025), (6, 9001),
                                 (3, 50001), (2, 131072), (2, 140001)])
@pytest.mark.parametrize("variant", [0, 1, 2])
def test_policy_logits(obj, n, k, dtype, variant):
    x = make_logits(n + k, n, k, dtype, pad=k % 3, shift=k % 2)
    y = make_labels(n, n, k)
    if n > 4:
        y[3] = -100
    kl = ("k1", "k2", "k3")[variant]
    reduction = "sequence" if variant == 1 else "token"
    temperature = 1.0 if variant else 1.3
    scale = float(n)
    logp, lse, ent, p = plain_rows(x, y, temperature)
    old = torch.from_numpy(logp).float().cuda() - ratios(k, n)
    ref = old - 0.2
    q = min(3, n)
    off = make_offsets(0, [n // q] * (q - 1) + [n - (n // q) * (q - 1)])
    adv = torch.randn((q, 1) if variant == 1 else (n,), device="cuda", generator=gen(9))
    mask = torch.rand(n, device="cuda", generator=gen(10)) < 0.9 if variant == 2 else None
    got = obj.policy_loss_logits(x, y, old, adv, temperature=temperature, ref_logp=ref, offsets=off, mask=mask,
                                 clip_low=0.2, clip_high=0.28, kl_coef=0.1, kl=kl, entropy_coef=0.05,
                                 reduction=reduction, grad_scale=scale)
    keep = (y >= 0).cpu().numpy() & (mask.cpu().numpy() if mask is not None else True)
    o = off.cpu().numpy()
    w = plain_weights(keep, o, reduction)
    a = f64(adv)[seq_of(o, n), 0] if variant == 1 else f64(adv)
    pg, dpg, klt, dkl, cut = plain_policy(logp, f64(old), a, f64(ref), kl, 0.2, 0.28)
    tol = row_tol(f64(x) / temperature) + 4 * U * np.abs(logp)
    close(f64(got.logp), np.where(keep, logp, 0), tol, "logp")
    bend = (np.abs(a) + 1) * 4
    pol, klm, entm = (w * pg).sum(), (w * klt).sum(), (w * ent).sum()
    t = (w * bend * (tol + 8 * U)).sum() + 4 * U * (abs(pol) + abs(klm))
    te = (w * 4 * tol * (1 + ent)).sum() + 4 * U * entm
    close(float(got.policy), pol, t, "policy")
    close(float(got.kl), klm, t, "kl")
    close(float(got.entropy), entm, te, "entropy")
    close(float(got.loss), pol + 0.1 * klm - 0.05 * entm, 2 * t + te, "loss")
    close(float(got.clip_fraction), (w * cut).sum(), 2 * U, "clipped")
    g = w * (dpg + 0.1 * dkl) * scale / temperature
    ge = -0.05 * w * scale / temperature
    lp = f64(x) / temperature - lse[:, None]
    want = plain_row_grad(p, lp, y, g, ge, ent)
    slip = (scale / temperature * w * bend * (tol + 8 * U))[:, None] * (p + np.eye(k)[y.clamp(min=0).cpu().numpy()]
                                                                        if k < 20000 else 1.0)
    close(f64(got.grad_logits), want, grad_tol(want, p, lp, g, ge, ent, 4 * tol * (1 + ent), dtype) + slip, "grad")


@pytest.mark.parametrize("n,k", [(6, 5), (4, 1500)])
def test_policy_logits_gradient_against_differences(obj, n, k):
    x = make_logits(3, n, k, torch.float32, scale=1.0)
    y = make_labels(3, n, k)
    logp = plain_rows(x, y)[0]
    old = torch.from_numpy(logp).float().cuda() - ratios(4, n)
    ref, adv = old - 0.3, torch.randn(n, device="cuda", generator=gen(5))
    got = f64(obj.policy_loss_logits(x, y, old, adv, ref_logp=ref, kl_coef=0.2, entropy_coef=0.1).grad_logits)

    def loss(z):
        lp, _, ent, _ = plain_rows(torch.from_numpy(z), y)
        pg, _, kl, _, _ = plain_policy(lp, f64(old), f64(adv), f64(ref), "k3", 0.2, 0.2)
        return (pg + 0.2 * kl - 0.1 * ent).mean()
    base, h = f64(x), 1e-5
    rng = np.random.RandomState(0)
    for i in range(n):
        for j in {int(y[i]), 0, k - 1, int(rng.randint(k))}:
            up, down = base.copy(), base.copy()
            up[i, j] += h
            down[i, j] -= h
            # h^2 times a third derivative below 10, 64-bit noise over h, and fp32's units at the size of a term
            assert abs(got[i, j] - (loss(up) - loss(down)) / (2 * h)) < 2e-9 + 64 * U / n * (abs(float(adv[i])) + 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [7, 1200, 33000])
def test_policy_logits_in_place_masked_and_empty_rows(obj, k, dtype):
    n = 6
    x = make_logits(k, n, k, dtype).clone()
    y = make_labels(k, n, k)
    x[1, :] = math.nan                                  # left out by the mask
    x[2, :] = math.nan                                  # left out by the label
    y[2] = -1
    x[3, :] = -math.inf                                 # nothing left to choose from
    mask = torch.tensor([1, 0, 1, 1, 1, 1], dtype=torch.bool, device="cuda")
    old = torch.full((n,), -2.0, device="cuda")
    adv = torch.ones(n, device="cuda")
    a = obj.policy_loss_logits(x, y, old, adv, mask=mask, entropy_coef=0.01)
    assert math.isfinite(float(a.loss)) and not a.grad_logits[1:4].any() and a.logp[[1, 2]].tolist() == [0, 0]
    assert float(a.logp[3]) == -math.inf and torch.isfinite(a.grad_logits).all()
    b = obj.policy_loss_logits(x, y, old, adv, mask=mask, entropy_coef=0.01, out=x)
    assert b.grad_logits.data_ptr() == x.data_ptr() and torch.equal(a.grad_logits, x)
    assert torch.equal(a.logp, b.logp) and torch.equal(a.loss, b.loss)


def test_policy_logits_agrees_with_its_parts(obj):
    n, k = 64, 5000
    x, y = make_logits(1, n, k, torch.float32), make_labels(1, n, k)
    r = obj.label_logprobs(x, y, entropy=True)
    old, adv = r.logp - ratios(2, n), torch.randn(n, device="cuda", generator=gen(3))
    parts = obj.policy_loss(r.logp, old, adv, ref_logp=old, kl_coef=0.1)
    whole = obj.policy_loss_logits(x, y, old, adv, ref_logp=old, kl_coef=0.1)
    assert abs(float(parts.loss) - float(whole.loss)) < 1e-6
    g = obj.label_logprobs_grad(x, y, r.lse, parts.grad_logp)
    # both are within a few units of the same gradient, row by row
    assert float((g - whole.grad_logits).abs().max()) < 1e-6 * float(parts.grad_logp.abs().max()) * 8


# ---------------------------------------------------------------------------
# streams, repeatability
# ---------------------------------------------------------------------------

def test_runs_on_the_current_stream_and_repeats_bit_for_bit(obj):
    n, k = 500, 3001
    x, y = make_logits(1, n, k, torch.bfloat16), make_labels(1, n, k)
    logp0 = obj.label_logprobs(x, y).logp
    old, adv = logp0 - ratios(2, n), torch.randn(n, device="cuda", generator=gen(3))
    off = make_offsets(0, [100, 0, 250, 150])
    c, r = torch.tensor([0, 2], device="cuda"), torch.tensor([2, 3], device="cuda")

    def everything():
        a = obj.label_logprobs(x, y, entropy=True)
        b = obj.preference_loss(a.logp, c, r, ref_logp=old, offsets=off)
        d = obj.policy_loss(a.logp, old, adv, offsets=off, reduction="sequence")
        e = obj.policy_loss_logits(x, y, old, adv, offsets=off, reduction="sequence", entropy_coef=0.1)
        return [*a, *b, *d, *e, obj.label_logprobs_grad(x, y, a.lse, b.grad_logp)]
    first = everything()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = everything()
    side.synchronize()
    for u, v in zip(first, second):
        assert torch.equal(u, v)


def test_no_host_wait_and_capturable(obj):
    """The calls queue work only: they can be captured in a CUDA graph."""
    n, k = 40, 2000
    x, y = make_logits(1, n, k, torch.float32), make_labels(1, n, k)
    old, adv = torch.full((n,), -7.0, device="cuda"), torch.randn(n, device="cuda", generator=gen(3))
    want = obj.policy_loss_logits(x, y, old, adv)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = obj.policy_loss_logits(x, y, old, adv)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got.grad_logits, want.grad_logits) and torch.equal(got.loss, want.loss)


# ---------------------------------------------------------------------------
# more rows than blocks: what a block carries from row to row
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("n,k,dtype", [(1500, 9001, torch.bfloat16), (700, 9001, torch.float32), (900, 20480, torch.float16),
                                       (1300, 3001, torch.bfloat16), (400, 70001, torch.bfloat16), (5000, 300, torch.float16),
                                       (3000, 1030, torch.float32), (20000, 90, torch.bfloat16)])
def test_many_rows(obj, n, k, dtype):
    """Every row gives what it gives alone, with rows left out in between."""
    x = make_logits(n, n, k, dtype, pad=k % 2)
    y = make_labels(n, n, k)
    y[::3] = -1
    y[7:40] = -1
    x[11, 5], x[n // 2, 0] = math.nan, math.inf
    g = torch.randn(n, device="cuda", generator=gen(8))
    old = torch.full((n,), -8.0, device="cuda")
    r = obj.label_logprobs(x, y, entropy=True)
    grad = obj.label_logprobs_grad(x, y, r.lse, g)
    pol = obj.policy_loss_logits(x, y, old, g, entropy_coef=0.1, grad_scale=float(n))
    kept = y >= 0
    w = int(kept.sum())
    assert not r.logp[~kept].any() and not r.entropy[~kept].any()
    assert not grad[~kept].any() and not pol.grad_logits[~kept].any() and not pol.logp[~kept].any()
    z = x.float()
    lp = z.log_softmax(1)
    want = lp.gather(1, y.clamp(min=0)[:, None])[:, 0]
    ok = kept & torch.isfinite(want)
    # torch's float32 log-softmax and ours are both within row_tol of the definition
    tol = 2 * torch.from_numpy(row_tol(np.ones((1, k)) * float(z[ok].abs().max()))).max().item()
    assert float((r.logp - want)[ok].abs().max()) < tol
    assert float((pol.logp - want)[ok].abs().max()) < tol
    p = lp.exp()
    wantg = -p * g[:, None]
    wantg[torch.arange(n, device="cuda"), y.clamp(min=0)] += g
    err = (grad.float() - wantg)[ok].abs()
    assert float((err - (EPS[dtype] * 1.01 * wantg[ok].abs() + tol * g[ok].abs()[:, None] * 4 + TINY[dtype])).max()) <= 0
    # the rows alone: the same arithmetic
    for i in ok.nonzero()[:: max(1, w // 5), 0].tolist():
        one = obj.label_logprobs(x[i:i + 1].clone(), y[i:i + 1])
        assert abs(float(one.logp[0]) - float(r.logp[i])) < tol


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", [(600, 70001), (460, 60000), (1500, 8200), (3000, 700), (4000, 70)])
def test_policy_rows_out_of_the_ordinary_among_many(obj, n, k, dtype):
    """Rows left out, masked whole, with the lowest value throughout or with NaN, between plain ones, in place."""
    x = make_logits(k, n, k, dtype, scale=2.0).clone()
    y = make_labels(k, n, k)
    y[5::7] = -1
    empty, lowest, nan = n // 3, n // 3 + 1, n // 2
    y[empty], y[lowest], y[nan] = 1, 2, 3
    x[empty] = -math.inf
    x[lowest] = LOWEST[dtype]
    x[nan, k - 1] = math.nan
    base = obj.label_logprobs(x, y, entropy=True)
    old = torch.where(torch.isfinite(base.logp), base.logp, torch.zeros_like(base.logp)) - ratios(3, n)
    adv = torch.randn(n, device="cuda", generator=gen(4))
    want_logp = -math.log(k)
    assert float(base.logp[empty]) == -math.inf and abs(float(base.logp[lowest]) - want_logp) < 1e-4
    mask = torch.ones(n, dtype=torch.bool, device="cuda")
    mask[[empty, nan]] = False
    a = obj.policy_loss_logits(x, y, old, adv, mask=mask, entropy_coef=0.05, grad_scale=float(n))
    parts = obj.policy_loss(base.logp.nan_to_num(0, 0, 0), old, adv, mask=mask & (y >= 0))
    assert abs(float(a.policy) - float(parts.policy)) < 1e-5 * (1 + abs(float(parts.policy)))
    kept = mask & (y >= 0)
    w = 1.0 / float(kept.sum())
    ent = float((base.entropy[kept].double()).sum() * w)
    assert abs(float(a.entropy) - ent) < 1e-5 * (1 + ent)
    assert torch.equal(a.logp[~kept], torch.zeros_like(a.logp[~kept])) and not a.grad_logits[~kept].any()
    assert torch.isfinite(a.grad_logits).all()
    # the uniform row: p = 1/k in every place, g (1[y] - 1/k), no entropy gradient
    g = float(parts.grad_logp[lowest]) * n
    row = f64(a.grad_logits[lowest])
    want = np.full(k, -g / k)
    want[2] += g
    assert np.abs(row - want).max() < (EPS[dtype] * 1.01 + 1e-4) * abs(g) / 1 + TINY[dtype]
    # rows of the gradient sum to nothing but rounding
    sums = a.grad_logits.double().sum(1)
    size = a.grad_logits.double().abs().sum(1)
    assert float((sums.abs() - (EPS[dtype] * 2 + 1e-4) * size - k * TINY[dtype]).max()) <= 1e-12
    b = obj.policy_loss_logits(x, y, old, adv, mask=mask, entropy_coef=0.05, grad_scale=float(n), out=x)
    assert torch.equal(b.grad_logits, a.grad_logits) and torch.equal(b.loss, a.loss) and torch.equal(b.logp, a.logp)


@pytest.mark.parametrize("n,k,dtype", [(460, 80001, torch.float32), (330, 161003, torch.bfloat16), (170, 160001, torch.float16),
                                       (260, 190001, torch.float32), (160, 380003, torch.bfloat16),
                                       (100, 40001, torch.bfloat16), (140, 17001, torch.float32), (60, 70001, torch.float16)])
def test_policy_rows_shared_by_blocks(obj, n, k, dtype):
    """Long rows: two or four blocks to a row and more rows than clusters, or no more rows than SMs.  Rows left out,
    masked whole, with the lowest value throughout or with NaN lie between plain ones; compared with the plain
    operators, and in place."""
    coef, t = 0.05, 1.25
    x = make_logits(k, n, k, dtype, scale=2.0).clone()
    y = make_labels(k, n, k)
    y[5::7] = -1
    empty, lowest, nan = n // 3, n // 3 + 1, n // 2
    y[empty], y[lowest], y[nan] = 1, 2, 3
    x[empty] = -math.inf
    x[lowest] = LOWEST[dtype]
    x[nan, k - 1] = math.nan
    mask = torch.ones(n, dtype=torch.bool, device="cuda")
    mask[[empty, nan]] = False
    kept = mask & (y >= 0)
    w = 1.0 / float(kept.sum())
    z = x.double() / t
    m = z.max(1, keepdim=True).values
    lp = (z - m) - (z - m).exp().sum(1, keepdim=True).log()
    p = lp.exp()
    want_logp = lp.gather(1, y.clamp(min=0)[:, None])[:, 0]
    old = torch.where(kept, want_logp, torch.zeros_like(want_logp)).float() - ratios(3, n)
    adv = torch.randn(n, device="cuda", generator=gen(4))
    a = obj.policy_loss_logits(x, y, old, adv, mask=mask, entropy_coef=coef, grad_scale=float(n), temperature=t)
    assert not a.logp[~kept].any() and not a.grad_logits[~kept].any() and torch.isfinite(a.grad_logits).all()
    plain = torch.where(kept)[0]
    plain = plain[plain != lowest]
    tol = float(row_tol(np.full((1, k), float(z[plain].abs().max()))).max())
    assert float((a.logp.double() - want_logp)[kept].abs().max()) < tol
    ent = -(p * torch.where(p > 0, lp, torch.zeros_like(lp))).sum(1)
    assert abs(float(a.entropy) - float(ent[kept].sum()) * w) < tol * (1 + math.log(k))
    # the loss's gradient to logp, from the operator on the log-probs that were formed
    parts = obj.policy_loss(a.logp, old, adv, mask=kept)
    g, ge = parts.grad_logp.double() * n, -coef * w * n
    # each of log p, H and g is off by at most `tol` of its size, the scale by a few roundings
    for i in plain.tolist()[:: max(1, n // 24)] + [lowest]:
        want = (-g[i] * p[i] - ge * p[i] * (lp[i] + ent[i])) / t
        want[y[i]] += g[i] / t
        size = (g[i].abs() * p[i] + abs(ge) * p[i] * (lp[i].abs() + ent[i] + 1)) / t
        size[y[i]] += g[i].abs() / t
        err = (a.grad_logits[i].double() - want).abs() - (EPS[dtype] * 1.01 * want.abs() + 4 * tol * size + TINY[dtype])
        assert float(err.max()) <= 0, (i, float(err.max()))
    b = obj.policy_loss_logits(x, y, old, adv, mask=mask, entropy_coef=coef, grad_scale=float(n), temperature=t, out=x)
    assert torch.equal(b.grad_logits, a.grad_logits) and torch.equal(b.loss, a.loss) and torch.equal(b.logp, a.logp)


@pytest.mark.parametrize("n,k,dtype", [(1, 33000, torch.bfloat16), (30, 33000, torch.float16), (70, 66000, torch.bfloat16),
                                       (30, 17000, torch.float32), (20, 12000, torch.float16)])
def test_few_long_rows(obj, n, k, dtype):
    test_label_logprobs(obj, n, k, dtype)
    test_label_logprobs_grad(obj, n, k, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", [(40, 20), (40, 300), (20, 9000)])
def test_gradients_beside_the_logits_and_unlike_aligned(obj, n, k, dtype):
    """Logits and gradient as columns of one buffer, at every alignment to one another."""
    for shift in (0, 1, 3):
        buf = torch.randn(n, 2 * k + 16, device="cuda", generator=gen(k)).to(dtype)
        x, out = buf[:, :k], buf[:, k + 8 + shift:2 * k + 8 + shift]
        y = make_labels(k, n, k)
        old, adv = torch.full((n,), -3.0, device="cuda"), torch.randn(n, device="cuda", generator=gen(4))
        keep = x.clone()
        want = obj.policy_loss_logits(keep, y, old, adv, entropy_coef=0.1)
        got = obj.policy_loss_logits(x, y, old, adv, entropy_coef=0.1, out=out)
        assert torch.equal(x, keep) and got.grad_logits.data_ptr() == out.data_ptr()
        tol = row_tol(f64(keep)).max()
        err = (got.grad_logits.double() - want.grad_logits.double()).abs()
        bound = 2 * EPS[dtype] * 1.01 * want.grad_logits.double().abs() + 8 * tol * float(adv.abs().max()) / n + TINY[dtype]
        assert float((err - bound).max()) <= 0

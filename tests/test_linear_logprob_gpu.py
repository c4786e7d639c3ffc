"""Log probabilities, entropy and top alternatives of a linear head, and their
gradients, against 64 bits.

Tolerances, beside those of the cross entropy (test_linear_ce_gpu.py: E bounds every
logit's error, the log-sum-exp adds its sum's).
  * Entropy: a change of E in every logit changes it by at most 2 E sum p |l + H|.  Its
    two sums have terms of one sign and chains of at most 256 additions, 600 U of
    their quotient and 256 U of the logarithm; the exponents' own rounding, 2 U of
    each |l|, weighs p l^2: 8 U of that sum.
  * G: one rounding to bf16, 8 U of its terms, the errors of p, l and H.
Ranks are compared where they are certain: on inputs whose products and sums are
exact in fp32, where equal logits go by their index.  On others each alternative is
within the logits' error of its place."""
import pytest
import torch

import test_linear_ce_gpu as ce
from aethelstream_amd import loss

pytestmark = pytest.mark.gpu

U = ce.U


def _exact64(x, w, t):
    z = x.double() @ w.double().t()
    lse = torch.logsumexp(z, 1)
    l = z - lse[:, None]
    p = l.exp()
    pl = torch.where(p > 0, p * l, torch.zeros_like(p))
    h = -pl.sum(1)
    kept = t != loss.IGNORE_INDEX
    logp = torch.where(kept, l.gather(1, t.clamp(0, w.shape[0] - 1)[:, None])[:, 0],
                       torch.zeros_like(lse))
    return z, lse, l, p, h, logp


def _entropy_error(e, l, p, h):
    lf = torch.where(p > 0, l, torch.zeros_like(l))
    return 2 * e * (p * (lf + h[:, None]).abs()).sum(1) + U * (
        256 + 600 * h + 8 * (p * lf * lf).sum(1))


def _check_forward(x, w, t, r):
    z, lse, l, p, h, logp = _exact64(x, w, t)
    e = ce._logit_error(x, w)
    bound = e + U * (256 + 4 * lse.abs())
    assert ((r.lse.double() - lse).abs() <= bound).all()
    assert ((r.logp.double() - logp).abs() <= 2 * bound + 4 * U * logp.abs()).all()
    assert (r.logp[t == loss.IGNORE_INDEX] == 0).all()
    off = (r.entropy.double() - h).abs()
    assert (off <= _entropy_error(e, l, p, h)).all(), off.max()
    if r.top_ids is None:
        return
    k = r.top_ids.shape[1]
    assert ((r.top_ids >= 0) & (r.top_ids < w.shape[0])).all()
    assert (r.top_ids.sort(1).values.diff(dim=1) > 0).all()
    at = l.gather(1, r.top_ids)
    assert ((r.top_logp.double() - at).abs() <= (2 * bound + 4 * U * lse.abs())[:, None]
            + 4 * U * at.abs()).all()
    assert (r.top_logp.diff(dim=1) <= 0).all()
    assert ((at - l.topk(k, dim=1).values).abs() <= 2 * e[:, None]).all()


SHAPES = [(1, 1, 8, 1), (1, 40, 64, 32), (2, 32, 16, 32), (1, 1000, 72, 8), (3, 257, 128, 1),
          (17, 3001, 520, 5), (64, 512, 256, 0), (65, 129, 1000, 20), (100, 4099, 192, 32),
          (128, 640, 64, 2), (129, 1023, 320, 0), (257, 513, 136, 7), (300, 2000, 1032, 31),
          (600, 777, 2048, 3), (1000, 17000, 2048, 20), (1500, 9001, 520, 8)]


@pytest.mark.parametrize("m,v,d,k", SHAPES)
def test_forward(m, v, d, k):
    print(m, v, d, k, flush=True)
    x, w, t, _ = ce._inputs(m, v, d, seed=m + v)
    r = loss.linear_log_probs(x, w, t, top_k=k)
    assert (r.top_ids is None) == (k == 0)
    _check_forward(x, w, t, r)
    # The same sums as the cross entropy's, and alternatives change nothing else.
    out, lse = loss.linear_cross_entropy(x, w, t)
    assert (r.logp + out).abs().max() <= 1e-3
    if k > 0:
        s = loss.linear_log_probs(x, w, t)
        for name in ("logp", "lse", "entropy"):
            a, b = getattr(r, name).double(), getattr(s, name).double()
            assert ((a - b).abs() <= 1024 * U * (1 + lse.double().abs())).all()


def _grid(m, v, d, seed, levels=8):
    """Multiples of 1 / 8 and 1 / 64: sums of products are exact in fp32, equal logits
    common."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randint(-levels, levels + 1, (m, d), device="cuda", generator=g) / 8.0
    w = torch.randint(-levels, levels + 1, (v, d), device="cuda", generator=g) / 64.0
    return x.to(torch.bfloat16), w.to(torch.bfloat16)


def _check_ranks(x, w, r, k):
    z = x.double() @ w.double().t()
    want = z.sort(dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(r.top_ids, want)
    assert ((r.top_logp.double() - (z.gather(1, want) - torch.logsumexp(z, 1)[:, None])).abs()
            <= U * (512 + 8 * z.abs().amax(1))[:, None]).all()


@pytest.mark.parametrize("m,v,d,k,levels", [
    (1, 32, 8, 32, 8), (5, 1000, 16, 8, 1), (1, 32000, 64, 20, 2), (33, 5003, 8, 32, 1),
    (130, 12345, 24, 16, 8), (700, 3000, 64, 5, 1), (257, 20000, 8, 32, 1), (16, 50021, 128, 1, 8)])
def test_ranks_and_ties(m, v, d, k, levels):
    x, w = _grid(m, v, d, m + k, levels)
    t = torch.zeros(m, dtype=torch.int64, device="cuda")
    _check_ranks(x, w, loss.linear_log_probs(x, w, t, top_k=k), k)


@pytest.mark.parametrize("m,v", [(3, 600001), (5000, 30000), (16390, 9000)])
@pytest.mark.parametrize("order", ["any", "rising", "falling", "equal"])
def test_pieces_of_the_vocabulary(m, v, order):
    """Several pieces, for few tokens and many, and several chunks of tokens: logits in
    any order, each piece better or worse than those before, and all of them equal."""
    d, k = 8, 9
    x, w = _grid(m, v, d, 3, 1 if order == "any" else 8)
    if order != "any":
        # One element decides: a step each 64 columns.
        x[:] = 0
        x[:, 0] = torch.arange(1, m + 1, device="cuda") % 3 + 1
        step = torch.arange(v, device="cuda") // (v // 250 + 1)
        w[:, 0] = {"rising": step, "falling": 255 - step, "equal": step * 0}[order].to(
            torch.bfloat16)
    t = torch.arange(m, device="cuda") % v
    r = loss.linear_log_probs(x, w, t, top_k=k)
    rows = torch.arange(m, device="cuda")
    if m > 600:
        rows = torch.cat([rows[:200], rows[m // 2:m // 2 + 200], rows[-200:]])
    few = loss.LogProbs(*(None if a is None else a[rows]
                          for a in (r.logp, r.entropy, r.lse, r.top_logp, r.top_ids)))
    _check_ranks(x[rows], w, few, k)
    z, lse, l, p, h, logp = _exact64(x[rows], w, t[rows])
    bound = U * (256 + 4 * lse.abs() + 8 * z.abs().amax(1))
    assert ((few.lse.double() - lse).abs() <= bound).all()
    assert ((few.logp.double() - logp).abs() <= 2 * bound).all()
    assert ((few.entropy.double() - h).abs() <= _entropy_error(0 * lse, l, p, h)).all()


def test_sure_and_undecided_tokens():
    """One logit far above the others, all equal, and logits of thousands."""
    v, d = 3000, 64
    w = torch.zeros(v, d, device="cuda", dtype=torch.bfloat16)
    w[7, 0], w[:, 1] = 1.0, ce._randn((v,), 1)
    x = torch.zeros(4, d, device="cuda", dtype=torch.bfloat16)
    x[0, 0], x[2, 1], x[3, 1] = 40.0, 1000.0, 3.0
    t = torch.tensor([7, 2999, 5, loss.IGNORE_INDEX], device="cuda")
    r = loss.linear_log_probs(x, w, t, top_k=4)
    z, lse, l, p, h, logp = _exact64(x, w, t)
    bound = U * (256 + 4 * lse.abs() + 8 * z.abs().amax(1))
    assert ((r.lse.double() - lse).abs() <= bound).all()
    assert ((r.logp.double() - logp).abs() <= 2 * bound).all()
    assert ((r.entropy.double() - h).abs() <= _entropy_error(U * z.abs().amax(1), l, p, h)).all()
    assert r.top_ids[1].tolist() == [0, 1, 2, 3] and r.top_ids[0].tolist() == [7, 0, 1, 2]
    assert (r.entropy >= 0).all()


def test_what_is_not_finite():
    m, v, d, k = 6, 700, 64, 5
    x, w, t, _ = ce._inputs(m, v, d, seed=3, skip=0.0)
    x[:, 0] = 1.0
    want = loss.linear_log_probs(x, w, t, top_k=k)
    # A token whose row is NaN, targets that are no token, and columns of -inf.
    bad = x.clone()
    bad[2, 5] = float("nan")
    far = t.clone()
    far[3], far[4] = v, -1
    got = loss.linear_log_probs(bad, w, far, top_k=k)
    for a, b in ((want.lse, got.lse), (want.entropy, got.entropy), (want.top_logp, got.top_logp)):
        assert b[2].isnan().all() and torch.equal(torch.cat([a[:2], a[3:]]),
                                                  torch.cat([b[:2], b[3:]]))
    assert got.logp[2:5].isnan().all() and torch.equal(got.logp[:2], want.logp[:2])
    assert ((got.top_ids >= 0) & (got.top_ids < v)).all()
    ids = torch.cat([got.top_ids[:2], got.top_ids[3:]])
    assert torch.equal(ids, torch.cat([want.top_ids[:2], want.top_ids[3:]]))
    low = w.clone()
    low[::2, 0] = float("-inf")
    got = loss.linear_log_probs(x, low, t, top_k=k)
    ref = loss.linear_log_probs(x, w[1::2].contiguous(), t // 2, top_k=k)
    assert ((got.lse - ref.lse).abs() <= 1024 * U * (1 + ref.lse.abs())).all()
    assert ((got.entropy - ref.entropy).abs() <= 2048 * U * (1 + ref.entropy)).all()
    assert torch.equal(got.top_ids, 2 * ref.top_ids + 1)
    assert (got.logp[t % 2 == 0] == float("-inf")).all()
    # Nothing but -inf.
    low[:, 0] = float("-inf")
    got = loss.linear_log_probs(x, low, t, top_k=k)
    assert ((got.top_ids >= 0) & (got.top_ids < v)).all() and got.top_logp.isnan().all()


# -- gradients ----------------------------------------------------------------

def _check_backward(x, w, t, da, dh, r, dx, dw, accumulated=None):
    z, lse, l, p, h, _ = _exact64(x, w, t)
    kept = (t != loss.IGNORE_INDEX).double()
    a = (da.double() * kept)[:, None]
    b = torch.zeros_like(a) if dh is None else dh.double()[:, None]
    hot = torch.zeros_like(p).scatter_(1, t.clamp(min=0)[:, None], 1.0)
    g = hot * a - p * (a + b * (l + h[:, None]))
    e = ce._logit_error(x, w)
    rel = (e + U * (64 + 256 + 8 * lse.abs()))[:, None]
    dist = (a.abs() + b.abs() * (l + h[:, None]).abs())
    off = (2.0 ** -8 + 4 * U) * g.abs() + p * (
        rel * dist + b.abs() * (2 * rel + _entropy_error(e, l, p, h)[:, None])) + 8 * U * (
        p * (a.abs() + b.abs() * (l.abs() + h[:, None])) + hot * a.abs())
    xs, ws = x.double().abs(), w.double().abs()
    sums = 2 * U * x.shape[1]
    want = g @ w.double()
    bound = off @ ws + (2.0 ** -8 + sums) * want.abs() + 64 * U * (g.abs() @ ws) + 1e-30
    assert ((dx.double() - want).abs() <= bound).all()
    want = g.t() @ x.double()
    bound = off.t() @ xs + 64 * U * (g.abs().t() @ xs) + 1e-30
    if accumulated is not None:
        want = want + accumulated.double()
        bound = bound + 2 * U * want.abs()
    elif dw.dtype == torch.bfloat16:
        bound = bound + 2.0 ** -8 * want.abs()
    assert ((dw.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("m,v,d", [s[:3] for s in SHAPES])
@pytest.mark.parametrize("entropy", [True, False])
def test_backward(m, v, d, entropy):
    print(m, v, d, entropy, flush=True)
    x, w, t, da = ce._inputs(m, v, d, seed=m + v)
    dh = ce._randn((m,), 9, 0.5, torch.float32) if entropy else None
    r = loss.linear_log_probs(x, w, t)
    dx, dw = loss.linear_log_probs_bwd(x, w, t, r, da, dh)
    _check_backward(x, w, t, da, dh, r, dx, dw)
    full = torch.empty(v, d, device="cuda")
    dx2, _ = loss.linear_log_probs_bwd(x, w, t, r, da, dh, dw=full)
    assert torch.equal(dx, dx2)
    _check_backward(x, w, t, da, dh, r, dx, full)
    assert torch.equal(full.to(torch.bfloat16), dw)
    base = ce._randn((v, d), 11, 0.1, torch.float32)
    total = base.clone()
    loss.linear_log_probs_bwd(x, w, t, r, da, dh, dw=total, accumulate=True)
    _check_backward(x, w, t, da, dh, r, dx, total, accumulated=base)
    if not entropy:
        zero, _ = loss.linear_log_probs_bwd(x, w, t, r, da, torch.zeros_like(da))
        assert torch.equal(zero, dx)
        # The cross entropy's gradient with the other sign.
        other, _ = loss.linear_cross_entropy_bwd(x, w, t, r.lse, -da)
        assert torch.equal(other, dx)


@pytest.mark.parametrize("m,v,d", [s[:3] for s in SHAPES] + [(3000, 20000, 64), (700, 40007, 256),
                                                             (16384, 3000, 16)])
def test_kept_logits(m, v, d):
    """The gradients from kept logits are those from logits made again, bit for bit, in
    one piece of the vocabulary and in several, and the forward's results the same."""
    print(m, v, d, flush=True)
    x, w, t, da = ce._inputs(m, v, d, seed=m + v)
    dh = ce._randn((m,), 9, 0.5, torch.float32)
    dh[: m // 3] = 0
    da[: m // 4] = 0
    r = loss.linear_log_probs(x, w, t, keep_logits=True)
    s = loss.linear_log_probs(x, w, t, keep_logits=False)
    assert r.logits is not None and s.logits is None
    for name in ("logp", "entropy", "lse"):
        assert torch.equal(getattr(r, name), getattr(s, name))
    kept = loss.linear_log_probs(x, w, t).logits
    assert (kept is not None) == (2 * m <= d)
    assert loss.linear_log_probs(x, w, t, top_k=1).logits is None
    for b in (dh, None):
        got = loss.linear_log_probs_bwd(x, w, t, r, da, b)
        want = loss.linear_log_probs_bwd(x, w, t, s, da, b)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("m,v,d", [(1, 1, 8), (2, 32, 16), (1, 4050, 256), (64, 90, 128),
                                   (40, 8000, 136), (3, 16401, 64), (100, 4097, 64),
                                   (300, 2050, 64)])
def test_workspaces_that_held_something(m, v, d):
    """Workspaces full of NaN before the calls: all that is read of them is written."""
    print(m, v, d, flush=True)
    x, w, t, da = ce._inputs(m, v, d, seed=m + v)
    dh = ce._randn((m,), 9, 0.5, torch.float32)

    def used(backward, k=0):
        n = loss.log_probs_workspace_bytes(m, v, d, k, backward)
        return torch.full((n,), 0xff, dtype=torch.uint8, device="cuda")

    k = min(v, 7)
    r = loss.linear_log_probs(x, w, t, top_k=k, workspace=used(False, k))
    _check_forward(x, w, t, r)
    for keep in (False, True):
        r = loss.linear_log_probs(x, w, t, workspace=used(False), keep_logits=keep)
        _check_forward(x, w, t, r)
        dx, dw = loss.linear_log_probs_bwd(x, w, t, r, da, dh, workspace=used(True))
        _check_backward(x, w, t, da, dh, r, dx, dw)


@pytest.mark.parametrize("m,v", [(1, 100), (33, 700)])
@pytest.mark.parametrize("d", [*range(56, 850, 72), 64, 128, 192, 256, 320, 384, 448, 512, 640])
def test_every_number_of_steps(m, v, d):
    """Reductions of 1 to 14 steps of 64, whole ones and with a rest, through the stages
    of the smallest tiles."""
    x, w, t, da = ce._inputs(m, v, d, seed=d)
    dh = ce._randn((m,), 9, 0.5, torch.float32)
    r = loss.linear_log_probs(x, w, t, top_k=4)
    _check_forward(x, w, t, r)
    for keep in (False, True):
        r = loss.linear_log_probs(x, w, t, keep_logits=keep)
        _check_forward(x, w, t, r)
        dx, dw = loss.linear_log_probs_bwd(x, w, t, r, da, dh)
        _check_backward(x, w, t, da, dh, r, dx, dw)


@pytest.mark.parametrize("m,v,d", [(512, 33500, 264), (300, 66000, 136), (256, 66500, 72)])
def test_columns_behind_whole_rounds(m, v, d):
    """Two launches over the columns, large tiles and the smallest ones."""
    print(m, v, d, flush=True)
    x, w, t, da = ce._inputs(m, v, d, seed=m)
    t[::3] = v - 1 - torch.arange(len(t[::3]), device="cuda") % 700
    dh = ce._randn((m,), 9, 0.5, torch.float32)
    r = loss.linear_log_probs(x, w, t, top_k=9)
    _check_forward(x, w, t, r)
    r = loss.linear_log_probs(x, w, t, keep_logits=True)
    s = loss.linear_log_probs(x, w, t, keep_logits=False)
    _check_forward(x, w, t, r)
    got, want = (loss.linear_log_probs_bwd(x, w, t, o, da, dh) for o in (r, s))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    _check_backward(x, w, t, da, dh, r, *got)


@pytest.mark.parametrize("size", [1e-36, 1e-20, 1e-9])
def test_entropy_far_above_log_probabilities(size):
    """dlogp next to nothing beside dentropy: G stays within its range."""
    m, v, d = 33, 500, 64
    x, w, t, da = ce._inputs(m, v, d, seed=41)
    dh = ce._randn((m,), 9, 1.0, torch.float32)
    r = loss.linear_log_probs(x, w, t)
    dx, dw = loss.linear_log_probs_bwd(x, w, t, r, da * size, dh)
    _check_backward(x, w, t, da * size, dh, r, dx, dw)


def test_nothing_but_minus_infinity():
    x, w, t, _ = ce._inputs(3, 100, 64, seed=5, skip=0.0)
    x[:, 0], w[:, 0] = 1.0, float("-inf")
    r = loss.linear_log_probs(x, w, t)
    assert (r.lse == float("-inf")).all() and r.logp.isnan().all() and r.entropy.isnan().all()


def test_entropy_alone_and_tokens_without_gradients():
    m, v, d = 70, 900, 136
    x, w, t, _ = ce._inputs(m, v, d, seed=21)
    none, dh = torch.zeros(m, device="cuda"), ce._randn((m,), 4, 1.0, torch.float32)
    dh[10:20] = 0
    r = loss.linear_log_probs(x, w, t)
    dx, dw = loss.linear_log_probs_bwd(x, w, t, r, none, dh)
    _check_backward(x, w, t, none, dh, r, dx, dw)
    assert not dx[10:20].any() and dx[:10].any()
    dx, dw = loss.linear_log_probs_bwd(x, w, t, r, none, none)
    assert not dx.any() and not dw.any()
    # No tokens: dw is zero, or what it was.
    e = x[:0].contiguous()
    r = loss.linear_log_probs(e, w, t[:0], top_k=3)
    assert r.top_ids.shape == (0, 3) and r.logp.shape == (0,)
    dx, dw = loss.linear_log_probs_bwd(e, w, t[:0], r, none[:0], none[:0])
    assert dx.shape == (0, d) and not dw.any()


def test_gradients_against_differences():
    """Central differences in 64 bits along random directions.  G is rounded to bf16,
    2^-8 of each entry, and so are the results."""
    m, v, d = 5, 60, 32
    x, w, t, da = ce._inputs(m, v, d, seed=31, skip=0.0)
    dh = ce._randn((m,), 5, 1.0, torch.float32)

    def value(a, b):
        l = torch.log_softmax(a @ b.t(), 1)
        return (l.gather(1, t[:, None])[:, 0] * da.double()).sum() - (
            (l.exp() * l).sum(1) * dh.double()).sum()

    r = loss.linear_log_probs(x, w, t)
    dx, dw = loss.linear_log_probs_bwd(x, w, t, r, da, dh)
    at = [x.double(), w.double()]
    _, _, l, p, h, _ = _exact64(x, w, t)
    a, b = da.double()[:, None], dh.double()[:, None]
    g = torch.zeros_like(p).scatter_(1, t[:, None], a) - p * (a + b * (l + h[:, None]))
    for i, grad in enumerate((dx, dw)):
        step = ce._randn(at[i].shape, 40 + i, 1e-4, torch.float32).double()
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + step, at[i] - step
        want = (value(*up) - value(*down)) / 2
        off = ((2.0 ** -8 + 2.0 ** -12) * g.abs())
        off = off @ at[1].abs() if i == 0 else off.t() @ at[0].abs()
        tol = (step.abs() * (off + 2.0 ** -8 * grad.double().abs())).sum()
        # (and a third derivative of order one times the step cubed)
        assert abs(want - (grad.double() * step).sum()) <= tol + 1e-8


def test_invalid_target_and_nan_rows():
    m, v, d = 8, 300, 64
    x, w, t, da = ce._inputs(m, v, d, seed=41, skip=0.0)
    t[3] = v + 5
    dh = torch.ones(m, device="cuda")
    r = loss.linear_log_probs(x, w, t)
    dx, _ = loss.linear_log_probs_bwd(x, w, t, r, da, dh)
    assert dx[3].isnan().all() and dx[:3].isfinite().all() and dx[4:].isfinite().all()
    t[3] = 0
    x[5, 1] = float("nan")
    r = loss.linear_log_probs(x, w, t)
    for b in (None, dh):
        dx, _ = loss.linear_log_probs_bwd(x, w, t, r, da, b)
        assert dx[5].isnan().all() and dx[:5].isfinite().all() and dx[6:].isfinite().all()


def test_pieces_of_the_gradient():
    m, v, d = 16390, 17000, 64
    print(m, v, d, flush=True)
    x, w, t, da = ce._inputs(m, v, d, seed=5)
    t[:4] = torch.tensor([0, v - 1, 8191, 8192], device="cuda")
    dh = ce._randn((m,), 6, 0.3, torch.float32)
    da[300:-300] = 0
    dh[300:-300] = 0
    rows = torch.cat([torch.arange(300, device="cuda"), torch.arange(m - 300, m, device="cuda")])
    r = loss.linear_log_probs(x, w, t, top_k=2)
    few = loss.LogProbs(r.logp[rows], r.entropy[rows], r.lse[rows], r.top_logp[rows],
                        r.top_ids[rows])
    _check_forward(x[rows], w, t[rows], few)
    dx, dw = loss.linear_log_probs_bwd(x, w, t, r, da, dh)
    assert (dx[300:-300] == 0).all()
    _check_backward(x[rows], w, t[rows], da[rows], dh[rows], few, dx[rows], dw)


def test_past_31_bits():
    """w and dw past 2^31 elements, targets and alternatives at both ends."""
    m, v, d = 40, 65600, 32768
    print(m, v, d, flush=True)
    x, w, t, da = ce._inputs(m, v, d, seed=56)
    t[:4] = torch.tensor([0, v - 1, v - 2, 1], device="cuda")
    w[v - 1] = x[0] * 4
    r = loss.linear_log_probs(x, w, t, top_k=4)
    _check_forward(x, w, t, r)
    assert r.top_ids[0, 0] == v - 1
    dh = torch.full((m,), 0.1, device="cuda")
    dx, dw = loss.linear_log_probs_bwd(x, w, t, r, da, dh)
    _check_backward(x, w, t, da, dh, r, dx, dw)


def test_stream_workspace_and_replays():
    m, v, d, k = 90, 5000, 256, 6
    x, w, t, da = ce._inputs(m, v, d, seed=61)
    dh = ce._randn((m,), 7, 0.2, torch.float32)
    need = loss.log_probs_workspace_bytes(m, v, d, k)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    work_bwd = torch.empty(loss.log_probs_workspace_bytes(m, v, d, backward=True),
                           dtype=torch.uint8, device="cuda")

    def run(a=None, b=None):
        r = loss.linear_log_probs(x, w, t, top_k=k, workspace=a)
        dx, dw = loss.linear_log_probs_bwd(x, w, t, r, da, dh, workspace=b)
        return [r.logp, r.entropy, r.lse, r.top_logp, r.top_ids, dx, dw]

    want = run()
    assert all(torch.equal(a, b) for a, b in zip(run(work, work_bwd), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for replay in range(4):
        x.copy_(ce._randn(x.shape, 70 + replay))
        t.copy_((t * 7 + replay).clamp(min=0) % v)
        da.copy_(ce._randn((m,), 80 + replay, 1.0, torch.float32))
        want = [a.clone() for a in run()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_refusals():
    x, w, t, da = ce._inputs(10, 40, 64, seed=1)
    for kw in (dict(top_k=-1), dict(top_k=33), dict(w=w[:8], top_k=9), dict(x=x.float()),
               dict(w=w.float()), dict(t=t.int()), dict(t=t[:5]), dict(x=x.cpu()),
               dict(x=x[:, ::2]), dict(x=x[:, :32].contiguous()), dict(t=t.cpu()),
               dict(workspace=torch.empty(8, dtype=torch.uint8))):
        a = dict(x=x, w=w, t=t)
        a.update(kw)
        with pytest.raises(ValueError):
            loss.linear_log_probs(a.pop("x"), a.pop("w"), a.pop("t"), **a)
    big = ce._randn((16385, 64), 1)
    for kw in (dict(top_k=1), dict(x=big, t=torch.zeros(16385, dtype=torch.int64, device="cuda"))):
        with pytest.raises(ValueError):
            loss.linear_log_probs(kw.pop("x", x), w, kw.pop("t", t), keep_logits=True, **kw)
    with pytest.raises(RuntimeError):  # d no multiple of 8
        loss.linear_log_probs(x[:, :60].contiguous(), w[:, :60].contiguous(), t)
    r = loss.linear_log_probs(x, w, t)
    for kw in (dict(dlogp=da[:5]), dict(dlogp=da.double()), dict(dentropy=da[:5]),
               dict(dentropy=da.cpu()), dict(accumulate=True), dict(dw=w.half()),
               dict(dw=torch.empty(4, 64, device="cuda")), dict(dw=w.clone(), accumulate=True),
               dict(out=loss.LogProbs(r.logp, r.entropy, r.lse[:5], None, None)),
               dict(out=loss.LogProbs(r.logp, r.entropy[:5], r.lse, None, None)),
               dict(out=loss.LogProbs(r.logp, r.entropy, r.lse, None, None, r.logits[:-4])),
               dict(out=loss.LogProbs(r.logp, r.entropy, r.lse, None, None, r.logits.double()))):
        a = dict(out=r, dlogp=da)
        a.update(kw)
        with pytest.raises(ValueError):
            loss.linear_log_probs_bwd(x, w, t, **a)

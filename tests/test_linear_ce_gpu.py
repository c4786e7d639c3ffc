"""Cross entropy of a linear head and its gradients against 64 bits.

Tolerances.  A logit is an fp32 sum of d products of bf16 values: its error is
taken as U 4 sqrt(d) times the sum of magnitudes (roundings of either sign;
worst-case growth would be d).  The log-sum-exp adds the roundings of its terms
and of a chain of at most 256 additions.  G is rounded to bf16 (8 significant bits: 2^-8 of
each value) and so are dx and dw; p carries the logit's error as a relative one."""
import pytest
import torch

from aethelstream_amd import loss

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _randn(shape, seed, sigma=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * sigma).to(dtype)


def _inputs(m, v, d, seed=0, sx=1.0, sw=None, skip=0.1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = _randn((m, d), seed + 1, sx)
    w = _randn((v, d), seed + 2, 1.5 / d ** 0.5 if sw is None else sw)
    t = torch.randint(0, v, (m,), device="cuda", generator=g)
    t[torch.rand((m,), device="cuda", generator=g) < skip] = loss.IGNORE_INDEX
    dl = _randn((m,), seed + 3, 1.0, torch.float32)
    return x, w, t, dl


def _forward64(x, w, t, ignore=loss.IGNORE_INDEX):
    z = x.double() @ w.double().t()
    lse = torch.logsumexp(z, 1)
    kept = t != ignore
    hit = z.gather(1, t.clamp(0, w.shape[0] - 1)[:, None])[:, 0]
    return z, lse, torch.where(kept, lse - hit, torch.zeros_like(lse))


def _logit_error(x, w):
    """Bound on any logit's error, per token."""
    most = (x.double().abs() @ w.double().abs().t()).amax(1)
    return 4 * U * x.shape[1] ** 0.5 * most


def _check_forward(x, w, t, got):
    _, lse, want = _forward64(x, w, t)
    bound = _logit_error(x, w) + U * (256 + 4 * lse.abs())
    assert ((got[1].double() - lse).abs() <= bound).all()
    assert ((got[0].double() - want).abs() <= 2 * bound + 4 * U * want.abs()).all()
    assert (got[0][t == loss.IGNORE_INDEX] == 0).all()


def _check_backward(x, w, t, dl, lse, dx, dw, accumulated=None):
    z, _, _ = _forward64(x, w, t)
    kept = (t != loss.IGNORE_INDEX).double()
    p = torch.exp(z - lse.double()[:, None])
    scale = (kept * dl.double())[:, None]
    hot = torch.zeros_like(p).scatter_(1, t.clamp(min=0)[:, None], 1.0)
    g = (p - hot) * scale
    rel = (_logit_error(x, w) + U * (64 + 4 * lse.double().abs()))[:, None]
    # Per value of G: one rounding to bf16, three in fp32, the error of p.
    off = (2.0 ** -8 + 4 * U) * g.abs() + (p * rel + U * hot) * scale.abs()
    xs, ws = x.double().abs(), w.double().abs()
    sums = 2 * U * x.shape[1]  # fp32 sums of the products, added in any order
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


SHAPES = [(1, 1, 8), (1, 5, 64), (1, 1000, 72), (3, 257, 128), (17, 3001, 520), (64, 512, 256),
          (65, 129, 1000), (100, 4099, 192), (128, 640, 64), (129, 1023, 320), (257, 513, 136),
          (300, 2000, 1032), (600, 777, 2048), (1000, 17000, 2048), (1500, 9001, 520)]


@pytest.mark.parametrize("m,v,d", SHAPES)
def test_forward_and_backward(m, v, d):
    print(m, v, d, flush=True)
    x, w, t, dl = _inputs(m, v, d, seed=m + v)
    out, lse = loss.linear_cross_entropy(x, w, t)
    _check_forward(x, w, t, (out, lse))
    dx, dw = loss.linear_cross_entropy_bwd(x, w, t, lse, dl)
    _check_backward(x, w, t, dl, lse, dx, dw)
    full = torch.empty(v, d, device="cuda")
    dx2, _ = loss.linear_cross_entropy_bwd(x, w, t, lse, dl, dw=full)
    assert torch.equal(dx, dx2)
    _check_backward(x, w, t, dl, lse, dx, full)
    # The bf16 gradient is the fp32 one, rounded.
    assert torch.equal(full.to(torch.bfloat16), dw)


def test_pieces_of_the_vocabulary():
    """Enough tokens that G comes in several pieces, the last one shorter."""
    m, v, d = 16390, 17000, 64
    print(m, v, d, flush=True)
    x, w, t, dl = _inputs(m, v, d, seed=5)
    t[:4] = torch.tensor([0, v - 1, 8191, 8192], device="cuda")
    need = loss.workspace_bytes(m, v, d, True)
    assert need < m * v * 2
    out, lse = loss.linear_cross_entropy(x, w, t)
    rows = torch.cat([torch.arange(300, device="cuda"), torch.arange(m - 300, m, device="cuda")])
    _check_forward(x[rows], w, t[rows], (out[rows], lse[rows]))
    dl[300:-300] = 0  # so that a few rows make up dw
    dx, dw = loss.linear_cross_entropy_bwd(x, w, t, lse, dl)
    assert (dx[300:-300] == 0).all()
    _check_backward(x[rows], w, t[rows], dl[rows], lse[rows], dx[rows], dw)


def test_accumulate():
    m, v, d = 130, 700, 264
    x, w, t, dl = _inputs(m, v, d, seed=7)
    _, lse = loss.linear_cross_entropy(x, w, t)
    before = _randn((v, d), 8, 0.1, torch.float32)
    dw = before.clone()
    dx, same = loss.linear_cross_entropy_bwd(x, w, t, lse, dl, dw=dw, accumulate=True)
    assert same is dw
    _check_backward(x, w, t, dl, lse, dx, dw, accumulated=before)


@pytest.mark.parametrize("m", [3, 300])
def test_sharp_distributions(m):
    """Logits of several hundred: one column takes everything, exponentials of
    the others vanish, and the loss of its row is the difference of two large
    numbers."""
    v, d = 500, 256
    x, w, t, dl = _inputs(m, v, d, seed=9, sx=8.0, sw=2.0)
    out, lse = loss.linear_cross_entropy(x, w, t)
    assert float(lse.max()) > 300
    _check_forward(x, w, t, (out, lse))
    dx, dw = loss.linear_cross_entropy_bwd(x, w, t, lse, dl)
    _check_backward(x, w, t, dl, lse, dx, dw)


def test_all_targets_ignored_and_another_ignore_index():
    m, v, d = 70, 300, 64
    x, w, t, dl = _inputs(m, v, d, seed=11, skip=2.0)
    out, lse = loss.linear_cross_entropy(x, w, t)
    assert (out == 0).all()
    dx, dw = loss.linear_cross_entropy_bwd(x, w, t, lse, dl)
    assert (dx == 0).all() and (dw == 0).all()
    # An ignored value that is also a column: the column is never a target.
    t = torch.arange(m, device="cuda") % 3
    out, lse = loss.linear_cross_entropy(x, w, t, ignore_index=1)
    assert (out[t == 1] == 0).all() and (out[t != 1] > 0).all()
    dx, _ = loss.linear_cross_entropy_bwd(x, w, t, lse, dl, ignore_index=1)
    assert (dx[t == 1] == 0).all() and (dx[t != 1] != 0).any(1).all()


def test_targets_out_of_range_give_nan():
    m, v, d = 6, 300, 64
    x, w, t, dl = _inputs(m, v, d, seed=12, skip=0.0)
    t[1], t[2], t[3] = v, -1, 2 ** 40
    out, lse = loss.linear_cross_entropy(x, w, t)
    assert torch.isnan(out[1:4]).all() and torch.isfinite(out[[0, 4, 5]]).all()
    assert torch.isfinite(lse).all()
    dx, _ = loss.linear_cross_entropy_bwd(x, w, t, lse, dl)
    assert torch.isnan(dx[1:4]).all() and torch.isfinite(dx[[0, 4, 5]]).all()


@pytest.mark.parametrize("m", [5, 300])
def test_non_finite_rows(m):
    """A NaN in a token's row stays in that row's loss; where the token is ignored
    its loss and its dx are 0.  Columns of logit -inf take no part; a row of
    nothing else has no loss."""
    v, d = 400, 64
    x, w, t, dl = _inputs(m, v, d, seed=13, skip=0.0)
    clean, clean_lse = loss.linear_cross_entropy(x, w, t)
    x2 = x.clone()
    x2[1, 3] = float("nan")
    x2[2, 3] = float("nan")
    t[2] = loss.IGNORE_INDEX
    out, lse = loss.linear_cross_entropy(x2, w, t)
    assert torch.isnan(out[1]) and out[2] == 0 and torch.isnan(lse[2])
    assert torch.equal(out[3:], clean[3:]) and torch.equal(out[0], clean[0])
    dx, _ = loss.linear_cross_entropy_bwd(x2, w, t, lse, dl)
    assert torch.isnan(dx[1]).all() and (dx[2] == 0).all() and torch.isfinite(dx[3:]).all()
    # Column 0 of x at 1, of some of w at -inf: logits -inf there.
    x[:, 0] = 1
    w[:, 0] = 0
    t = torch.full_like(t, 350)
    gone = w.clone()
    gone[:300, 0] = -float("inf")
    out, lse = loss.linear_cross_entropy(x, gone, t)
    _check_forward(x, w[300:].contiguous(), t - 300, (out, lse))
    gone[:, 0] = -float("inf")
    out, lse = loss.linear_cross_entropy(x, gone, t)
    assert (lse == -float("inf")).all() and torch.isnan(out).all()
    # +inf: no finite log-sum-exp either.
    w[7, 0] = float("inf")
    out, lse = loss.linear_cross_entropy(x, w, t)
    assert not torch.isfinite(lse).any() and not torch.isfinite(out).any()


def test_gradients_against_differences():
    m, v, d = 9, 37, 72
    x, w, t, dl = _inputs(m, v, d, seed=14)
    _, lse = loss.linear_cross_entropy(x, w, t)
    dw = torch.empty(v, d, device="cuda")
    dx, _ = loss.linear_cross_entropy_bwd(x, w, t, lse, dl, dw=dw)

    def value(a, b):
        return float((_forward64(a, b, t)[2] * dl.double()).sum())

    step = 1e-5
    a, b = x.double(), w.double()
    for name, grad in (("x", dx), ("w", dw)):
        u = _randn(grad.shape, 15, 1.0, torch.float32).double()
        if name == "x":
            want = (value(a + step * u, b) - value(a - step * u, b)) / (2 * step)
        else:
            want = (value(a, b + step * u) - value(a, b - step * u)) / (2 * step)
        # bf16 roundings of G and of dx, each 2^-8 of what enters the sum.
        z, _, _ = _forward64(x, w, t)
        g = (torch.softmax(z, 1) - torch.zeros_like(z).scatter_(1, t.clamp(min=0)[:, None], 1.0))
        g = (g * (dl.double() * (t != loss.IGNORE_INDEX))[:, None]).abs()
        size = (g @ b.abs() if name == "x" else g.t() @ a.abs()) * u.abs()
        assert abs(float((grad.double() * u).sum()) - want) <= \
            2.0 ** -7 * float(size.sum()) + 1e-6


def test_other_stream_repeats_and_workspace():
    m, v, d = 200, 1500, 256
    x, w, t, dl = _inputs(m, v, d, seed=16)

    def both(**kw):
        out, lse = loss.linear_cross_entropy(x, w, t, **kw)
        return [out, lse, *loss.linear_cross_entropy_bwd(x, w, t, lse, dl, **kw)]

    want = both()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        first = both()
        # A caller's own workspace, full of NaNs.
        work = torch.full((loss.workspace_bytes(m, v, d, True),), 0xff, dtype=torch.uint8,
                          device="cuda")
        second = both(workspace=work)
    side.synchronize()
    for a, b, c in zip(want, first, second):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_no_tokens():
    x, w, t, dl = _inputs(0, 300, 64)
    out, lse = loss.linear_cross_entropy(x, w, t)
    assert out.shape == (0,) and lse.shape == (0,)
    dx, dw = loss.linear_cross_entropy_bwd(x, w, t, lse, dl)
    assert dx.shape == (0, 64) and (dw == 0).all()
    kept = torch.ones(300, 64, device="cuda")
    loss.linear_cross_entropy_bwd(x, w, t, lse, dl, dw=kept, accumulate=True)
    assert (kept == 1).all()


def test_refusals():
    x, w, t, dl = _inputs(4, 30, 64)
    out, lse = loss.linear_cross_entropy(x, w, t)
    for a, b, c in ((x.float(), w, t), (x, w.float(), t), (x, w, t.int()), (x, w, t[:3]),
                    (x, w[:, :32].contiguous(), t), (x.t(), w, t), (x.cpu(), w, t)):
        with pytest.raises(ValueError):
            loss.linear_cross_entropy(a, b, c)
    with pytest.raises(Exception, match="d % 8"):
        loss.linear_cross_entropy(x[:, :12].contiguous(), w[:, :12].contiguous(), t)
    for kw in (dict(accumulate=True),
               dict(dw=torch.zeros(30, 64, device="cuda", dtype=torch.bfloat16), accumulate=True),
               dict(dw=torch.zeros(30, 32, device="cuda")),
               dict(dw=torch.zeros(30, 64, device="cuda", dtype=torch.float16))):
        with pytest.raises(ValueError):
            loss.linear_cross_entropy_bwd(x, w, t, lse, dl, **kw)
    with pytest.raises(ValueError):
        loss.linear_cross_entropy_bwd(x, w, t, lse[:2], dl)

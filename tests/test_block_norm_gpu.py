"""The norms around a block with gate and residual scale, forward and backward,
against the formulas in 64 bits.

Tolerances: U = 2^-24 is the fp32 unit roundoff.  A row's mean is a sum of at most
32 terms a thread, then of 6 and 16 pairs, of products with up to 8 roundings
each: 64 U times the sum of magnitudes covers it, and every value after it has a
few roundings more.  bf16 (8 significant bits) results add 2^-8 of themselves.  Column sums add one
rounding a row."""
import pytest
import torch

from aethelstream_amd import checkpoint, norm

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = 1e-30
ALPHA = 0.7


def _randn(shape, seed, sigma=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * sigma).to(dtype)


def _inputs(m, d, post, gate, seed=0):
    return dict(h=_randn((m, d), seed + 1, 0.5, torch.bfloat16), res=_randn((m, d), seed + 2, 1.5),
                w_pre=1 + _randn((d,), seed + 3, 0.1),
                w_post=1 + _randn((d,), seed + 4, 0.1) if post else None,
                gate=_randn((d,), seed + 5, 0.5) if gate else None)


def _rms(v, eps):
    return (v.square().mean(1, keepdim=True) + eps).sqrt()


def _forward64(s, alpha=ALPHA, eps=norm.EPS):
    """(u, res, y, rms_pre, rms_post) in 64 bits."""
    h = s["h"].double()
    rms_post = None
    if s["w_post"] is not None:
        rms_post = _rms(h, eps)
        h = h / rms_post * s["w_post"].double()
    if s["gate"] is not None:
        h = h * s["gate"].double()
    u = alpha * h
    res = s["res"].double() + u
    rms = _rms(res, eps)
    return u, res, res / rms * s["w_pre"].double(), rms, rms_post


def _within(got, want, bound):
    off = (got.double() - want).abs() - bound
    assert torch.isfinite(got.double()).all()
    assert (off <= 0).all(), f"off by {float((got.double() - want).abs().max())}, " \
                             f"{float(off.max())} past the bound"


SHAPES = [(1, 4), (1, 4096), (3, 68), (5, 1020), (2, 1024), (7, 1028), (4, 2052), (300, 512),
          (33, 5120), (9, 8192), (5, 8196), (3, 12292), (2, 16384), (3, 16388), (2, 32768)]


@pytest.mark.parametrize("post,gate", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("m,d", SHAPES)
def test_forward(m, d, post, gate):
    print(m, d, post, gate, flush=True)
    s = _inputs(m, d, post, gate)
    r = norm.block_norm_fwd(s["h"], s["res"], s["w_pre"], s["w_post"], s["gate"], ALPHA)
    u, res, y, rms, rms_post = _forward64(s)
    _within(r.res, res, U * (res.abs() + 64 * u.abs()) + TINY)
    # The sum that is normed is the rounded one.
    _within(r.rms_pre, rms[:, 0], 64 * U * rms[:, 0])
    if post:
        _within(r.rms_post, rms_post[:, 0], 64 * U * rms_post[:, 0])
    else:
        assert r.rms_post is None
    slack = (64 * U * (res.abs() + u.abs()) / rms * s["w_pre"].double().abs())
    _within(r.y, y, 2.0 ** -8 * y.abs() + 2 * slack + TINY)


def _backward64(s, dy, dres, res, rms_pre, rms_post, alpha=ALPHA):
    """Values and error scales (sums of magnitudes) of every output."""
    dy, dres, res = dy.double(), dres.double(), res.double()
    rms = rms_pre.double()[:, None]
    hat = res / rms
    e = dy * s["w_pre"].double()
    g = dres + (e - hat * (e * hat).mean(1, keepdim=True)) / rms
    gs = dres.abs() + (e.abs() + hat.abs() * (e * hat).abs().mean(1, keepdim=True)) / rms
    out = {"dres": (g, gs), "dw_pre": ((dy * hat).sum(0), (dy * hat).abs().sum(0))}
    if s["h"] is None:
        return out
    hh = s["h"].double()
    if rms_post is not None:
        hh = hh / rms_post.double()[:, None]
    along, alongs = alpha * (g * hh).sum(0), alpha * (gs * hh.abs()).sum(0)
    one = torch.ones_like(along)
    gate = one if s["gate"] is None else s["gate"].double()
    w_post = one if s["w_post"] is None else s["w_post"].double()
    k = alpha * gate * w_post
    kg, kgs = k * g, k.abs() * gs
    if s["w_post"] is not None:
        inv = 1 / rms_post.double()[:, None]
        # The second mean is B - A C / rms: its parts' magnitudes.
        cross = (e * hat).abs().mean(1, keepdim=True) * (k * hh * hat).abs().mean(1, keepdim=True)
        parts = (k * hh).abs() * (dres.abs() + e.abs() / rms)
        kg, kgs = ((kg - hh * (kg * hh).mean(1, keepdim=True)) * inv,
                   (kgs + hh.abs() * (parts.mean(1, keepdim=True) + cross / rms)) * inv)
        out["dw_post"] = (along * gate, alongs * gate.abs())
    if s["gate"] is not None:
        out["dgate"] = (along * w_post, alongs * w_post.abs())
    out["dh"] = (kg, kgs)
    return out


def _check_backward(r, want, m):
    for name, (value, scale) in want.items():
        got = getattr(r, name)
        bound = 128 * U * scale + TINY
        if name == "dh":
            bound = bound + 2.0 ** -8 * value.abs()
        elif name != "dres":
            bound = (128 + m) * U * scale + TINY
        _within(got, value, bound)
    for name in ("dh", "dw_post", "dgate"):
        assert (getattr(r, name) is None) == (name not in want)


@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("post,gate", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("m,d", SHAPES + [(1111, 260), (2050, 1024)])
def test_backward(m, d, post, gate, bits8):
    print(m, d, post, gate, bits8, flush=True)
    s = _inputs(m, d, post, gate, seed=10)
    dy, dres = _randn((m, d), 20, 1e-3, torch.bfloat16), _randn((m, d), 21, 1e-3)
    res = _randn((m, d), 22, 1.5)
    source = checkpoint.encode(res) if bits8 else res
    if bits8:
        res = checkpoint.decode(source)
    rms = _rms(res.double(), norm.EPS)[:, 0].float()
    rms_post = _rms(s["h"].double(), norm.EPS)[:, 0].float() if post else None
    r = norm.block_norm_bwd(dy, dres, source, rms, s["w_pre"], s["h"], rms_post, s["w_post"],
                            s["gate"], ALPHA)
    _check_backward(r, _backward64(s, dy, dres, res, rms, rms_post), m)


@pytest.mark.parametrize("m,d", [(1, 4), (6, 1028), (300, 4096), (3, 16388)])
def test_backward_without_block_or_residual_gradient(m, d):
    """h = None is the RMSNorm backward; dres = None is a zero gradient."""
    s = dict(_inputs(m, d, False, False, seed=30), h=None)
    dy, res = _randn((m, d), 31, 1.0, torch.bfloat16), _randn((m, d), 32)
    rms = _rms(res.double(), norm.EPS)[:, 0].float()
    r = norm.block_norm_bwd(dy, None, res, rms, s["w_pre"])
    _check_backward(r, _backward64(s, dy, torch.zeros_like(res), res, rms, None), m)


@pytest.mark.parametrize("post,gate", [(False, True), (True, True), (True, False)])
def test_backward_against_differences(post, gate):
    """Directional derivatives of the 64-bit forward by central differences."""
    m, d = 6, 132
    s = _inputs(m, d, post, gate, seed=40)
    cy, cr = _randn((m, d), 50, 1.0, torch.bfloat16), _randn((m, d), 51)

    def value(t):
        _, res, y, _, _ = _forward64(t)
        return float((cy.double() * y).sum() + (cr.double() * res).sum())

    f = norm.block_norm_fwd(s["h"], s["res"], s["w_pre"], s["w_post"], s["gate"], ALPHA)
    r = norm.block_norm_bwd(cy, cr, f.res, f.rms_pre, s["w_pre"], s["h"], f.rms_post, s["w_post"],
                            s["gate"], ALPHA)
    grads = {"h": r.dh, "res": r.dres, "w_pre": r.dw_pre, "w_post": r.dw_post, "gate": r.dgate}
    for i, (name, grad) in enumerate(grads.items()):
        if s[name] is None:
            continue
        v = _randn(s[name].shape, 60 + i).double()
        step = 1e-5
        up, down = (value({**{k: (t.double() if t is not None else None) for k, t in s.items()},
                           name: s[name].double() + x * v}) for x in (step, -step))
        want = (up - down) / (2 * step)
        got = float((grad.double() * v).sum())
        # fp32 sums of a few hundred terms, bf16 gradients (dh), step^2 = 1e-10.
        scale = float((grad.double() * v).abs().sum())
        assert abs(got - want) <= (2.0 ** -8 if name == "h" else 1e-5) * scale + 1e-6


def test_backward_where_the_norms_cancel():
    """dy along res gives no gradient through the norm: what is left of the two
    means is rounding of their parts, and dres passes through."""
    m, d = 4, 2048
    s = _inputs(m, d, True, True, seed=70)
    res = _randn((m, d), 71)
    s["w_pre"] = torch.ones(d, device="cuda")
    dy = (res * 3).to(torch.bfloat16)
    res = dy.float() / 3
    dres = _randn((m, d), 72, 1e-3)
    rms = _rms(res.double(), norm.EPS)[:, 0].float()
    rms_post = _rms(s["h"].double(), norm.EPS)[:, 0].float()
    r = norm.block_norm_bwd(dy, dres, res, rms, s["w_pre"], s["h"], rms_post, s["w_post"],
                            s["gate"], ALPHA)
    _check_backward(r, _backward64(s, dy, dres, res, rms, rms_post), m)


def test_zero_rows_and_non_finite_rows_stay_in_their_rows():
    m, d = 5, 1024
    s = _inputs(m, d, True, False, seed=80)
    s["h"][1] = 0
    s["res"][1] = 0
    s["res"][3, 7] = float("inf")
    s["h"][4, 9] = float("nan")
    r = norm.block_norm_fwd(s["h"], s["res"], s["w_pre"], s["w_post"], None, ALPHA)
    assert (r.res[1] == 0).all() and (r.y[1] == 0).all()
    assert abs(float(r.rms_pre[1]) - norm.EPS ** 0.5) < 1e-9
    assert torch.isinf(r.rms_pre[3]) and torch.isnan(r.y[3, 7])
    assert torch.isnan(r.y[4]).all() and torch.isnan(r.res[4]).all()
    clean = norm.block_norm_fwd(s["h"][:3].contiguous(), s["res"][:3].contiguous(), s["w_pre"],
                                s["w_post"], None, ALPHA)
    assert torch.equal(r.y[:3], clean.y) and torch.equal(r.res[:3], clean.res)
    # Backward: the rows' own gradients; the column sums take in every row.
    dy, dres = _randn((m, d), 81, 1.0, torch.bfloat16), _randn((m, d), 82)
    b = norm.block_norm_bwd(dy, dres, r.res, r.rms_pre, s["w_pre"], s["h"], r.rms_post,
                            s["w_post"], None, ALPHA)
    for t in (b.dres, b.dh):
        assert torch.isfinite(t[:3].float()).all() and torch.isnan(t[4].float()).all()


def test_in_place_residuals():
    """The new residual may replace the old, the residual's gradient the one that
    came in: the same values as into new tensors."""
    for d in (1024, 16388):
        s = _inputs(7, d, True, True, seed=90)
        want = norm.block_norm_fwd(s["h"], s["res"], s["w_pre"], s["w_post"], s["gate"], ALPHA)
        res = s["res"].clone()
        got = norm.block_norm_fwd(s["h"], res, s["w_pre"], s["w_post"], s["gate"], ALPHA, out=res)
        assert got.res is res and torch.equal(res, want.res) and torch.equal(got.y, want.y)
        dy, dres = _randn((7, d), 91, 1.0, torch.bfloat16), _randn((7, d), 92)
        args = (want.res, want.rms_pre, s["w_pre"], s["h"], want.rms_post, s["w_post"], s["gate"],
                ALPHA)
        a = norm.block_norm_bwd(dy, dres, *args)
        b = norm.block_norm_bwd(dy, dres, *args, out=dres)
        assert b.dres is dres
        for name in ("dres", "dh", "dw_pre", "dw_post", "dgate"):
            assert torch.equal(getattr(a, name), getattr(b, name))


def test_no_rows():
    s = _inputs(0, 256, True, True)
    r = norm.block_norm_fwd(s["h"], s["res"], s["w_pre"], s["w_post"], s["gate"])
    assert r.y.shape == (0, 256)
    g = norm.block_norm_bwd(r.y, None, r.res, r.rms_pre, s["w_pre"], s["h"], r.rms_post,
                            s["w_post"], s["gate"])
    assert (g.dw_pre == 0).all() and (g.dw_post == 0).all() and (g.dgate == 0).all()


def test_other_stream_and_repeats():
    """On a side stream, twice: bit-identical to the default stream's."""
    m, d = 777, 1024
    s = _inputs(m, d, True, True, seed=100)
    dy, dres = _randn((m, d), 101, 1.0, torch.bfloat16), _randn((m, d), 102)

    def both():
        f = norm.block_norm_fwd(s["h"], s["res"], s["w_pre"], s["w_post"], s["gate"], ALPHA)
        b = norm.block_norm_bwd(dy, dres, f.res, f.rms_pre, s["w_pre"], s["h"], f.rms_post,
                                s["w_post"], s["gate"], ALPHA)
        return [f.res, f.y, b.dres, b.dh, b.dw_pre, b.dw_post, b.dgate]

    want = both()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        first, second = both(), both()
    side.synchronize()
    for a, b, c in zip(want, first, second):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_refusals():
    s = _inputs(4, 64, True, True)
    ok = (s["h"], s["res"], s["w_pre"], s["w_post"], s["gate"])

    def bad(i, t):
        args = list(ok)
        args[i] = t
        with pytest.raises(ValueError):
            norm.block_norm_fwd(*args)

    bad(0, s["h"].float())
    bad(0, s["h"].t())
    bad(0, s["h"].cpu())
    bad(1, s["res"][:3])
    bad(1, s["res"].to(torch.bfloat16))
    bad(2, s["w_pre"][:32])
    bad(4, s["gate"].double())
    r = norm.block_norm_fwd(*ok)
    for kw in (dict(w_post=s["w_post"]), dict(gate=s["gate"]),
               dict(h=s["h"], w_post=s["w_post"])):
        with pytest.raises(ValueError):
            norm.block_norm_bwd(r.y, None, r.res, r.rms_pre, s["w_pre"], **kw)
    with pytest.raises(ValueError):
        norm.block_norm_bwd(r.y, None, None, r.rms_pre, s["w_pre"])

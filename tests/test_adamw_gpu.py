"""AdamW over many tensors against its definition in 64 bits, and the 8-bit moments
bit for bit against the same fp32 operations in numpy.

Tolerances.  U = 2^-24 is half a step of fp32.  m and v are two products and a sum,
the gradient's scaling before them: 8 U of the terms.  The update is a root, two
products, a sum, a quotient and a product behind them, below 32 U of itself; the
decayed parameter 4 U; a bf16 result is rounded once more, 2^-8 of it.
"""
import numpy as np
import pytest
import torch

from aethelstream_amd import optim

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF16 = 2.0 ** -8
LR, BETAS, EPS, WD = 3e-3, (0.9, 0.95), 1e-8, 0.1
OFFSET = np.float32(2.0 ** -15)


def _randn(shape, seed, sigma=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * sigma).to(dtype)


def _tensors(sizes, kinds, seed=0, offset=0):
    """Parameters, gradients and copies; kinds cycles over (param type, grad type,
    copy)."""
    ps, gs, cs = [], [], []
    for i, n in enumerate(sizes):
        pt, gt, copy = kinds[i % len(kinds)]
        ps.append(_randn((n + offset,), seed + 3 * i, 0.02, pt)[offset:])
        gs.append(_randn((n + offset,), seed + 3 * i + 1, 10.0 ** (i % 5 - 4), gt)[offset:])
        cs.append(torch.full((n + offset,), 9.0, device="cuda", dtype=torch.bfloat16)[offset:]
                  if copy else None)
    return ps, gs, cs


F, B = torch.float32, torch.bfloat16
KINDS = [[(F, F, False)], [(B, B, False)], [(F, F, True)], [(F, B, True), (B, F, False)],
         [(F, F, False), (B, F, False), (F, B, False), (B, B, False), (F, F, True), (F, B, True)]]
SIZES = [[1], [128], [127, 129, 7, 4096], [5000, 1, 0, 12345, 65536, 8191],
         [33] * 40 + [2048] * 260, [3_000_001]]


def _step64(p, g, m, v, step, scale, hyper=None):
    c = [float(x) for x in np.float32(optim.coefficients(step, LR, BETAS, EPS, WD))]
    p, g = p.double(), g.double() * scale
    mt = (m * c[0]).abs() + (g * c[1]).abs()
    vt = (v * c[2]).abs() + g * g * c[3]
    m = m * c[0] + g * c[1]
    v = v * c[2] + g * g * c[3]
    upd = m / (v.sqrt() * c[6] + c[7]) * c[5]
    # The numerator's own error counts where its terms cancel.
    updt = mt / (v.sqrt() * c[6] + c[7]) * c[5]
    return p * c[4] - upd, m, v, mt, vt, 4 * U * p.abs() + 32 * U * updt


def _within(got, want, tol):
    bad = ~((got.double() - want).abs() <= tol + 1e-37)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4])


@pytest.mark.parametrize("kinds", range(len(KINDS)))
@pytest.mark.parametrize("sizes", range(len(SIZES)))
@pytest.mark.parametrize("offset", [0, 1])
def test_steps_in_32_bits(kinds, sizes, offset):
    sizes = SIZES[sizes]
    ps, gs, cs = _tensors(sizes, KINDS[kinds], offset=offset)
    state = optim.adamw_state(ps)
    scale = torch.full((1,), 0.25, device="cuda")
    m, v = [p.double() * 0 for p in ps], [p.double() * 0 for p in ps]
    starts = state.starts()
    for step in (1, 2, 7):
        want = [_step64(p, g, a, b, step, 0.25) for p, g, a, b in zip(ps, gs, m, v)]
        optim.adamw_step(ps, gs, state, step, LR, BETAS, EPS, WD, grad_scale=scale, copies=cs)
        for i, (p, a, n) in enumerate(zip(ps, starts, sizes)):
            w = want[i]
            gm, gv = state.m[a:a + n], state.v[a:a + n]
            _within(gm, w[1], 8 * U * w[3])
            _within(gv, w[2], 8 * U * w[4])
            _within(p, w[0], w[5] + (BF16 * w[0].abs() if p.dtype == B else 0))
            if cs[i] is not None:
                assert torch.equal(cs[i], p.to(B))
            m[i], v[i] = gm.double(), gv.double()
    used = torch.zeros_like(state.m, dtype=torch.bool)
    for a, n in zip(starts, sizes):
        used[a:a + n] = True
    assert not state.m[~used].any() and not state.v[~used].any()


# -- 8 bits -----------------------------------------------------------------

def _np_encode(x, mantissa):
    """Magnitude codes and scales of |x| (fp32, whole blocks)."""
    shift = 23 - mantissa
    blocks = np.abs(x).reshape(-1, 128)
    top = blocks.max(1)
    scale = np.where(np.isfinite(top), np.maximum(top, np.float32(2.0 ** -126)),
                     np.float32(np.nan)).astype(np.float32)
    with np.errstate(all="ignore"):
        y = (blocks * (np.float32(1) / scale)[:, None]).astype(np.float32) + OFFSET
    u = y.view(np.uint32) - OFFSET.view(np.uint32)
    u = (u + np.uint32((1 << (shift - 1)) - 1) + ((u >> shift) & 1)) >> shift
    return u.reshape(-1), scale


def _np_value(codes, scale, mantissa):
    u = (codes.astype(np.uint32) << (23 - mantissa)) + OFFSET.view(np.uint32)
    with np.errstate(all="ignore"):
        return ((u.view(np.float32) - OFFSET).reshape(-1, 128) * scale[:, None]).reshape(-1)


def _np_moments(state):
    m, v = state.m.cpu().numpy(), state.v.cpu().numpy()
    ms, vs = state.m_scale.cpu().numpy(), state.v_scale.cpu().numpy()
    mag = _np_value(np.abs(m.astype(np.int32)), ms, 3)
    with np.errstate(all="ignore"):
        r = _np_value(v, vs, 4)
        return np.where(m < 0, -mag, mag), r * r


def _np_step(state, grads, step, scale, hyper=None):
    """Codes and scales after a step, by the same fp32 operations."""
    c = np.float32(optim.coefficients(step, LR, BETAS, EPS, WD))
    m, v = _np_moments(state)
    g = np.zeros_like(m)
    for a, n, t in zip(state.starts(), state.sizes, grads):
        g[a:a + n] = t.float().cpu().numpy()
    with np.errstate(all="ignore"):
        g = g * np.float32(scale)
        m = m * c[0] + g * c[1]
        v = v * c[2] + g * g * c[3]
        r = np.sqrt(v)
    mc, ms = _np_encode(m, 3)
    vc, vs = _np_encode(r, 4)
    vc = np.where((r > 0) & (vc == 0), 1, vc)
    mc = mc.astype(np.int64)
    return np.where(m < 0, -mc, mc).astype(np.int8), vc.astype(np.uint8), ms, vs, m, v


def _check_codes(state, want):
    mc, vc, ms, vs = want[:4]
    gs, hs = state.m_scale.cpu().numpy(), state.v_scale.cpu().numpy()
    assert np.array_equal(gs, ms, equal_nan=True) and np.array_equal(hs, vs, equal_nan=True)
    # Codes of a block that is no number mean nothing.
    for got, w, s in ((state.m, mc, ms), (state.v, vc, vs)):
        fine = np.repeat(np.isfinite(s), 128)
        assert np.array_equal(got.cpu().numpy()[fine], w[fine])


@pytest.mark.parametrize("kinds", [0, 1, 4])
@pytest.mark.parametrize("sizes", range(len(SIZES)))
@pytest.mark.parametrize("offset", [0, 1])
def test_steps_in_8_bits(kinds, sizes, offset):
    sizes = SIZES[sizes]
    ps, gs, cs = _tensors(sizes, KINDS[kinds], offset=offset)
    state = optim.adamw_state(ps, bits=8)
    for step in (1, 2, 9):
        want = _np_step(state, gs, step, 1.0)
        m, v = (torch.from_numpy(t).cuda().double() for t in _np_moments(state))
        p64 = [_step64(p, g, m[a:a + n], v[a:a + n], step, 1.0)
               for p, g, a, n in zip(ps, gs, state.starts(), sizes)]
        optim.adamw_step(ps, gs, state, step, LR, BETAS, EPS, WD, copies=cs)
        _check_codes(state, want)
        for p, w, c in zip(ps, p64, cs):
            _within(p, w[0], w[5] + (BF16 * w[0].abs() if p.dtype == B else 0))
            assert c is None or torch.equal(c, p.to(B))
        a, b = optim.moments(state)
        for got, x in zip((a, b), _np_moments(state)):
            assert np.array_equal(got.cpu().numpy(), x)
        # Within half a step of what was rounded: 2^-4 (m) and 2^-5 (r) of the value,
        # or of the offset, times the scale (and the offset's own sum).
        ms, vs = (np.repeat(s.astype(np.float64), 128) for s in want[2:4])
        err = np.abs(a.cpu().numpy() - want[4].astype(np.float64))
        assert (err <= 2.0 ** -4 * (np.abs(want[4]) + 2.0 ** -15 * ms) + 2.0 ** -23 * ms).all()
        r = np.sqrt(want[5].astype(np.float64))
        err = np.abs(np.sqrt(b.cpu().numpy().astype(np.float64)) - r)
        # (a value that would become zero takes the first code instead)
        assert (err <= np.maximum(2.0 ** -5 * (r + 2.0 ** -15 * vs), 2.0 ** -19 * vs)
                + 2.0 ** -22 * vs).all()
        gs = [_randn(g.shape, 50 + step, 10.0 ** (i % 3 - 3), g.dtype) for i, g in enumerate(gs)]


def test_blocks_of_odd_values():
    """Zeros, one value alone, the smallest and largest numbers, equal values, values
    at and between the codes, and what is no number, which stays in its block."""
    rows = [np.zeros(128), np.eye(1, 128, 77)[0], np.full(128, 1e-45), np.full(128, 1e-40),
            np.full(128, 1e-30), np.full(128, 1e18), np.linspace(-1, 1, 128),
            2.0 ** -np.arange(128), 10.0 ** np.linspace(-18, 18, 128),
            np.r_[np.nan, np.ones(127)], np.r_[np.ones(127), np.inf], np.full(128, 1e30),
            np.ones(128)]
    g = torch.from_numpy(np.stack(rows).astype(np.float32)).reshape(-1).cuda()
    p = torch.zeros_like(g)
    state = optim.adamw_state([p], bits=8)
    for step in (1, 2):
        want = _np_step(state, [g], step, 1.0)
        optim.adamw_step([p], [g], state, step, LR, BETAS, EPS, WD)
        _check_codes(state, want)
        m, v = optim.moments(state)
        wm, wv = _np_moments(state)
        assert np.array_equal(m.cpu().numpy(), wm, equal_nan=True)
        assert np.array_equal(v.cpu().numpy(), wv, equal_nan=True)
        blocks = v.view(-1, 128)
        assert blocks[9].isnan().all() and blocks[10].isnan().all()
        # 1e30 squared is infinite: its v, not its m, is lost.
        assert blocks[11].isnan().all() and not m.view(-1, 128)[11].isnan().any()
        assert not blocks[:9].isnan().any() and not blocks[12].isnan().any()
    assert p.view(-1, 128)[9][1:].isnan().all() and not p.view(-1, 128)[12].isnan().any()


def test_parts_of_one_buffer_and_what_lies_between():
    flat = torch.full((5000,), 3.0, device="cuda")
    copy = torch.full((5000,), 3.0, device="cuda", dtype=B)
    places = [(0, 130), (131, 1000), (1500, 1), (1501, 2000), (3504, 1496)]
    ps, cs = [flat[a:a + n] for a, n in places], [copy[a:a + n] for a, n in places]
    gs = [_randn((n,), i) for i, (_, n) in enumerate(places)]
    for bits in (32, 8):
        state = optim.adamw_state(ps, bits=bits)
        optim.adamw_step(ps, gs, state, 1, LR, BETAS, EPS, WD, copies=cs)
    used = torch.zeros(5000, dtype=torch.bool, device="cuda")
    for a, n in places:
        used[a:a + n] = True
    assert (flat[~used] == 3).all() and (copy[~used] == 3).all() and (flat[used] != 3).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_stream_and_replays(bits):
    """On another stream, and captured with its coefficients on the device: every
    replay is the eager step."""
    ps, gs, _ = _tensors([1000, 77, 4096], KINDS[4], seed=5)
    other = [p.clone() for p in ps]
    state, twin = optim.adamw_state(ps, bits), optim.adamw_state(ps, bits)
    hyper = torch.zeros(8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        optim.adamw_step(ps, gs, state, 1, LR, BETAS, EPS, WD)
    torch.cuda.current_stream().wait_stream(side)
    optim.adamw_step(other, gs, twin, 1, LR, BETAS, EPS, WD)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        optim.adamw_step(ps, gs, state, 0, hyper=hyper)
    for step in range(2, 6):
        for i, g in enumerate(gs):
            g.copy_(_randn(g.shape, 10 * step + i, 1.0, g.dtype))
        hyper.copy_(torch.tensor(optim.coefficients(step, LR, BETAS, EPS, WD)))
        optim.adamw_step(other, gs, twin, step, LR, BETAS, EPS, WD)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip([*ps, state.m, state.v], [*other, twin.m, twin.v]):
            assert torch.equal(a, b)


def test_past_31_bits():
    """A tensor of 2^31 + 4997 elements and one behind it: only the last elements have
    gradients."""
    n = 2 ** 31 + 4997
    p = torch.zeros(n, dtype=B, device="cuda")
    g = torch.zeros(n, dtype=B, device="cuda")
    g[-3000:] = _randn((3000,), 1, 1.0, B)
    q, h = torch.zeros(300, device="cuda"), _randn((300,), 2)
    state = optim.adamw_state([p, q], bits=8)
    print("one step of", n, flush=True)
    optim.adamw_step([p, q], [g, h], state, 1, LR, BETAS, EPS, WD)
    few = [torch.zeros(3077, dtype=B, device="cuda"), torch.zeros(300, device="cuda")]
    small = optim.adamw_state(few, bits=8)
    tail = g[-3077:].clone()  # from the beginning of a block on
    assert (n - 3077) % 128 == 0
    optim.adamw_step(few, [tail, h], small, 1, LR, BETAS, EPS, WD)
    assert torch.equal(p[-3077:], few[0]) and torch.equal(q, few[1])
    k = small.m.numel()
    assert torch.equal(state.m[-k:], small.m) and torch.equal(state.v[-k:], small.v)
    assert not p[:-3077].any() and not state.m[:-k].any() and not state.v[:-k].any()


def test_gradient_in_its_parameters_place():
    p, g = _randn((1000,), 1), _randn((1000,), 1)
    a, b = optim.adamw_state([p]), optim.adamw_state([g])
    q = g.clone()
    optim.adamw_step([p], [g], a, 1, LR, BETAS, EPS, WD)
    optim.adamw_step([q], [q], b, 1, LR, BETAS, EPS, WD)
    assert torch.equal(p, q) and torch.equal(a.m, b.m)


def test_refusals():
    ps, gs, _ = _tensors([256, 100], [(F, F, False)])
    state = optim.adamw_state(ps)

    def bad(params=ps, grads=gs, state=state, step=1, **kw):
        with pytest.raises((ValueError, RuntimeError)):
            optim.adamw_step(params, grads, state, step, LR, **kw)

    bad(params=ps[:1])
    bad(grads=gs[:1])
    bad(copies=[None])
    bad(step=0)
    bad(betas=(1.0, 0.9))
    bad(eps=-1.0)
    bad(weight_decay=-1.0)
    bad(params=[ps[0].half(), ps[1]])
    bad(params=[ps[0][::2], ps[1]], grads=[gs[0][::2], gs[1]])
    bad(params=[ps[0].cpu(), ps[1]])
    bad(grads=[gs[0].cpu(), gs[1]])
    bad(grads=[gs[0].double(), gs[1]])
    bad(grads=[gs[0][:255], gs[1]])
    bad(copies=[ps[0], None])
    bad(copies=[ps[0].bfloat16()[:5], None])
    bad(params=[ps[0].bfloat16(), ps[1]], copies=[ps[0].bfloat16(), None])
    bad(grad_scale=torch.ones(2, device="cuda"))
    bad(grad_scale=torch.ones(1))
    bad(hyper=torch.ones(7, device="cuda"))
    bad(state=optim.AdamWState([256, 100], state.m, state.v[:128]))
    bad(state=optim.AdamWState([256, 100], state.m, state.v, torch.ones(3, device="cuda")))
    bad(state=optim.AdamWState([256, 100], state.m.to(torch.int8), state.v.to(torch.uint8),
                               torch.ones(2, device="cuda"), torch.ones(3, device="cuda")))
    # The same memory twice.
    bad(params=[ps[0], ps[0][100:200]], grads=[gs[0], gs[1]])
    c = torch.zeros(256, dtype=B, device="cuda")
    bad(copies=[c, c[:100]])
    bad(grads=[gs[0], ps[0][:100]])
    bad(params=[state.m[:256], ps[1]])
    with pytest.raises(ValueError):
        optim.adamw_state(ps, bits=16)
    with pytest.raises(ValueError):
        optim.adamw_state([])
    assert torch.equal(state.m, torch.zeros_like(state.m))

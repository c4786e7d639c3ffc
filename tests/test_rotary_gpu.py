"""Norms of queries and keys for each head with the rotation by position, forward
and backward, against the definitions in 64 bits.

Tolerances.  U = 2^-24 is half a step of fp32.  A result is at most half a step of
its type from what the kernel computes, which is off by
  * the angle: 2^-25 of a turn and a sine and cosine of a few steps, below 8 U;
  * the norm: a sum of d squares, at most 16 in a lane and 6 exchanges, a root and
    a division, below 32 U of every value;
  * a handful of products and sums, below 16 U:
64 U of |a| + |b| of the pair covers them.  The backward's row mean adds as much of
its terms' absolute sum; a weight's gradient is summed in lanes, workgroups and
their join, 256 U of the terms' absolute sum for the sizes here.
"""
import math

import numpy as np
import pytest
import torch

from aethelstream_amd import rotary

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-6
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _randn(shape, seed, sigma=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * sigma).to(dtype)


def _angles(positions, turns):
    """cos and sin [M, 1, rot / 2] in 64 bits: position * turns modulo 2^64, exact."""
    with np.errstate(over="ignore"):
        t = positions.cpu().numpy().astype(np.uint64)[:, None] * turns.cpu().numpy().astype(
            np.uint64)
    a = torch.from_numpy(t.astype(np.int64).astype(np.float64) * 2.0 ** -64).cuda() * (2 * math.pi)
    return a.cos()[:, None], a.sin()[:, None]


def _turn64(x, cos, sin, rope):
    half = cos.shape[2]
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if rope.interleaved else (i, i + half)
    y, mag = x.clone(), x.abs()
    y[..., a] = rope.scale * (x[..., a] * cos - x[..., b] * sin)
    y[..., b] = rope.scale * (x[..., b] * cos + x[..., a] * sin)
    both = abs(rope.scale) * (x[..., a].abs() + x[..., b].abs())
    mag[..., a], mag[..., b] = both, both
    return y, mag


def _within(got, want, tol):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4])


def _check_fwd(got, x, w, positions, rope, eps=EPS):
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(2, keepdim=True) + eps).sqrt() * w.double()
    y, mag = _turn64(x, *_angles(positions, rope.turns), rope)
    _within(got, y, HALF_STEP[got.dtype] * y.abs() + 64 * U * mag + 1e-38)


def _check_bwd(got, dw, dy, x, w, positions, rope, eps=EPS):
    cos, sin = _angles(positions, rope.turns)
    dn, mag = _turn64(dy.double(), cos, -sin, rope)
    if w is None:
        _within(got, dn, HALF_STEP[got.dtype] * dn.abs() + 64 * U * mag + 1e-38)
        return
    x, w = x.double(), w.double()
    rms = (x.square().mean(2, keepdim=True) + eps).sqrt()
    hat = x / rms
    e = dn * w
    dx = (e - hat * (e * hat).mean(2, keepdim=True)) / rms
    terms = (mag * w.abs() + hat.abs() * (mag * w.abs() * hat.abs()).mean(2, keepdim=True)) / rms
    _within(got, dx, HALF_STEP[got.dtype] * dx.abs() + 64 * U * terms + 1e-38)
    _within(dw, (dn * hat).sum((0, 1)), 256 * U * (mag * hat.abs()).sum((0, 1)) + 1e-38)


def _rope(rot, interleaved=False, **kw):
    f, scale = rotary.frequencies(rot, **kw)
    return rotary.Rotary.from_frequencies(f, interleaved, scale)


def _inputs(m, hq, hk, d, dtype, norm, seed=0):
    s = dict(q=_randn((m, hq, d), seed, 1.5, dtype), k=_randn((m, hk, d), seed + 1, 1.5, dtype),
             dq=_randn((m, hq, d), seed + 2, 1e-3, dtype),
             dk=_randn((m, hk, d), seed + 3, 1e-3, dtype))
    s["positions"] = torch.arange(m, device="cuda") * 7 % 1000
    s["w_q"] = 1 + _randn((d,), seed + 4, 0.1) if norm else None
    s["w_k"] = 1 + _randn((d,), seed + 5, 0.1) if norm else None
    return s


def _both(s, rope):
    q, k = rotary.apply(s["q"], s["k"], s["positions"], rope, s["w_q"], s["w_k"])
    _check_fwd(q, s["q"], s["w_q"], s["positions"], rope)
    _check_fwd(k, s["k"], s["w_k"], s["positions"], rope)
    g = rotary.apply_bwd(s["dq"], s["dk"], s["positions"], rope, s["q"], s["k"], s["w_q"],
                         s["w_k"])
    _check_bwd(g.dq, g.dw_q, s["dq"], s["q"], s["w_q"], s["positions"], rope)
    _check_bwd(g.dk, g.dw_k, s["dk"], s["k"], s["w_k"], s["positions"], rope)
    return q, k, g


# Heads of 16 to 1024, all lane counts of the vector loads, sizes that only go
# element by element, parts that turn, both orders of the pairs.
SHAPES = [(1, 1, 1, 128, 128), (1, 32, 8, 128, 128), (37, 6, 2, 64, 64), (5, 3, 3, 80, 40),
          (130, 5, 1, 96, 96), (9, 4, 2, 256, 64), (3, 2, 1, 1024, 1024), (7, 3, 2, 512, 256),
          (11, 2, 2, 192, 128), (64, 1, 1, 16, 16), (21, 7, 3, 34, 18), (13, 2, 1, 30, 30),
          (6, 2, 2, 2, 2), (5, 2, 1, 258, 6), (4, 1, 1, 1022, 1020), (300, 9, 4, 128, 32),
          (17, 65, 33, 64, 32), (2, 4096, 1, 8, 8), (700, 1, 1, 32, 16), (50, 2, 2, 112, 56),
          (9, 5, 2, 128, 84), (8, 3, 1, 256, 68), (7, 2, 2, 36, 12), (2, 2, 1, 1000, 500),
          (40, 3, 1, 256, 60), (6, 2, 1, 768, 768)]


@pytest.mark.parametrize("m,hq,hk,d,rot", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("norm", [True, False])
def test_shapes(m, hq, hk, d, rot, dtype, norm):
    for interleaved in (False, True):
        print(m, hq, hk, d, rot, dtype, norm, interleaved, flush=True)
        _both(_inputs(m, hq, hk, d, dtype, norm, seed=d + m), _rope(rot, interleaved))


@pytest.mark.parametrize("m,hq,hk", [(2000, 64, 8), (5000, 1, 1), (9000, 3, 32)])
def test_many_rows(m, hq, hk):
    """Several rows a lane, and several tiles a workgroup in the norms' backward."""
    _both(_inputs(m, hq, hk, 128, torch.bfloat16, True, seed=m), _rope(128))
    _both(_inputs(m, hq, hk, 64, torch.bfloat16, False, seed=m), _rope(32, True))


@pytest.mark.parametrize("factor,trained", [(4.0, None), (16.0, 4096)])
def test_scaled_frequencies(factor, trained):
    rope = _rope(64, factor=factor, trained=trained)
    assert (rope.scale != 1.0) == (trained is not None)
    _both(_inputs(20, 3, 2, 128, torch.float32, True), rope)


@pytest.mark.parametrize("positions", [
    [0, 1, -1, 2 ** 31 - 1, 2 ** 31, 2 ** 33 + 5, -2 ** 40, 2 ** 62 + 12345, -2 ** 63, 2 ** 63 - 1]])
@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions(positions, interleaved):
    m = len(positions)
    s = _inputs(m, 3, 2, 128, torch.float32, False)
    s["positions"] = torch.tensor(positions, device="cuda")
    _both(s, _rope(128, interleaved))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset", [0, 4, 1])
def test_strides_alignment_and_place(dtype, offset):
    """Parts of one wider row, behind an offset that allows 16, 8 (4) or only
    element-wide accesses, token by token or head by head, into new memory, into the
    inputs' place, and into rows of another buffer whose rest stays as it was."""
    m, hq, hk, d = 45, 6, 2, 64
    rope = _rope(32)
    for norm in (True, False):
        s = _inputs(m, hq, hk, d, dtype, norm)
        row = _randn((m, (hq + 2 * hk) * d + 8 + offset), 9, 1.0, dtype)

        def parts(buf):
            return (torch.as_strided(buf, (m, hq, d), (buf.stride(0), d, 1), offset),
                    torch.as_strided(buf, (m, hk, d), (buf.stride(0), d, 1), offset + hq * d))

        q, k = parts(row)
        got = rotary.apply(q, k, s["positions"], rope, s["w_q"], s["w_k"])
        _check_fwd(got[0], q, s["w_q"], s["positions"], rope)
        _check_fwd(got[1], k, s["w_k"], s["positions"], rope)
        other = torch.full_like(row, 7.0)
        oq, ok = parts(other)
        rotary.apply(q, k, s["positions"], rope, s["w_q"], s["w_k"], out_q=oq, out_k=ok)
        assert torch.equal(oq, got[0]) and torch.equal(ok, got[1])
        assert (other[:, :offset] == 7).all() and (other[:, offset + (hq + hk) * d:] == 7).all()
        before = row.clone()
        rotary.apply(q, k, s["positions"], rope, s["w_q"], s["w_k"], out_q=q, out_k=k)
        assert torch.equal(q, got[0]) and torch.equal(k, got[1])
        assert torch.equal(row[:, offset + (hq + hk) * d:], before[:, offset + (hq + hk) * d:])
        # Head by head.
        qh = s["q"].transpose(0, 1).contiguous().transpose(0, 1)
        kh = s["k"].transpose(0, 1).contiguous().transpose(0, 1)
        a = rotary.apply(s["q"], s["k"], s["positions"], rope, s["w_q"], s["w_k"])
        b = rotary.apply(qh, kh, s["positions"], rope, s["w_q"], s["w_k"],
                         out_q=torch.empty_like(qh))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        # The backward in its inputs' place.
        g = rotary.apply_bwd(s["dq"], s["dk"], s["positions"], rope, s["q"], s["k"], s["w_q"],
                             s["w_k"])
        dq, dk = s["dq"].clone(), s["k"].clone()
        h = rotary.apply_bwd(dq, s["dk"], s["positions"], rope, s["q"], dk if norm else None,
                             s["w_q"], s["w_k"], out_q=dq, out_k=dk)
        assert torch.equal(g.dq, dq) and torch.equal(g.dk, dk)
        if norm:
            assert torch.equal(g.dw_q, h.dw_q) and torch.equal(g.dw_k, h.dw_k)


def test_queries_alone_and_broadcast_inputs():
    s = _inputs(33, 4, 4, 128, torch.bfloat16, True)
    rope = _rope(128)
    both = rotary.apply(s["q"], s["k"], s["positions"], rope, s["w_q"], s["w_k"])
    alone = rotary.apply(s["q"], None, s["positions"], rope, s["w_q"])
    assert alone[1] is None and torch.equal(alone[0], both[0])
    g = rotary.apply_bwd(s["dq"], None, s["positions"], rope, s["q"], None, s["w_q"])
    assert g.dk is None and g.dw_k is None
    _check_bwd(g.dq, g.dw_q, s["dq"], s["q"], s["w_q"], s["positions"], rope)
    # One head read for all, one token for all: distances of zero.
    q = s["q"][:, :1].expand(-1, 4, -1)
    k = s["k"][:1].expand(33, -1, -1)
    got = rotary.apply(q, k, s["positions"], rope, s["w_q"], s["w_k"])
    _check_fwd(got[0], q, s["w_q"], s["positions"], rope)
    _check_fwd(got[1], k, s["w_k"], s["positions"], rope)


@pytest.mark.parametrize("norm", [True, False])
def test_no_tokens(norm):
    s = _inputs(0, 4, 2, 64, torch.bfloat16, norm)
    rope = _rope(64)
    q, k = rotary.apply(s["q"], s["k"], s["positions"], rope, s["w_q"], s["w_k"])
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)
    g = rotary.apply_bwd(s["dq"], s["dk"], s["positions"], rope, s["q"], s["k"], s["w_q"],
                         s["w_k"])
    if norm:
        assert not g.dw_q.any() and not g.dw_k.any()


@pytest.mark.parametrize("norm", [True, False])
def test_what_is_not_finite_stays_in_its_head(norm):
    s = _inputs(20, 4, 4, 64, torch.float32, norm)
    rope = _rope(32)
    want = rotary.apply(s["q"], s["k"], s["positions"], rope, s["w_q"], s["w_k"])
    s["q"][3, 1, 40] = float("inf")  # behind what turns
    s["k"][5, 2, 0] = float("nan")
    got = rotary.apply(s["q"], s["k"], s["positions"], rope, s["w_q"], s["w_k"])
    want[0][3, 1], want[1][5, 2] = got[0][3, 1], got[1][5, 2]
    # (The head with an infinity has 0 times it where it is normed: NaN, as in inf / inf.)
    for a, b in zip(want, got):
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())
    if not norm:
        assert got[0][3, 1].isfinite().sum() == 63 and got[0][3, 1, 40] == float("inf")
        assert got[1][5, 2].isnan().sum() == 2  # the pair
    else:
        assert got[1][5, 2].isnan().all()


def test_gradients_against_differences():
    """Central differences in 64 bits of a sum of the results, along random
    directions, against the backward's fp32 gradients."""
    s = _inputs(6, 3, 2, 64, torch.float32, True)
    rope = _rope(48, True)
    cos, sin = _angles(s["positions"], rope.turns)

    def value(q, k, w_q, w_k):
        t = 0.0
        for x, w, dy in ((q, w_q, s["dq"]), (k, w_k, s["dk"])):
            n = x / (x.square().mean(2, keepdim=True) + EPS).sqrt() * w
            t = t + (_turn64(n, cos, sin, rope)[0] * dy.double()).sum()
        return t

    at = [s[n].double() for n in ("q", "k", "w_q", "w_k")]
    g = rotary.apply_bwd(s["dq"], s["dk"], s["positions"], rope, s["q"], s["k"], s["w_q"],
                         s["w_k"])
    for i, grad in enumerate((g.dq, g.dk, g.dw_q, g.dw_k)):
        step = _randn(at[i].shape, 30 + i).double() * 1e-4
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + step, at[i] - step
        want = (value(*up) - value(*down)) / 2
        got = (grad.double() * step).sum()
        # Differences: a third derivative of order one times 1e-8; the gradient: its
        # rounding, 64 U of the terms.
        assert abs(want - got) <= 1e-5 * (grad.double() * step).abs().sum()


def test_stream_and_replays():
    """On a stream of its own, and captured: every replay is the eager result."""
    s = _inputs(70, 4, 2, 128, torch.bfloat16, True)
    rope = _rope(128)
    names = ("q", "k", "dq", "dk")

    def run():
        q, k = rotary.apply(s["q"], s["k"], s["positions"], rope, s["w_q"], s["w_k"])
        g = rotary.apply_bwd(s["dq"], s["dk"], s["positions"], rope, s["q"], s["k"], s["w_q"],
                             s["w_k"])
        return [q, k, g.dq, g.dk, g.dw_q, g.dw_k]

    want = run()
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
        for i, n in enumerate(names):
            s[n].copy_(_randn(s[n].shape, 10 * replay + i, 1.0, s[n].dtype))
        s["positions"].copy_(torch.arange(70, device="cuda") * (replay + 3))
        want = [t.clone() for t in run()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_refusals():
    s = _inputs(10, 4, 2, 64, torch.bfloat16, True)
    q, k, pos, w = s["q"], s["k"], s["positions"], s["w_q"]
    rope = _rope(64)
    bad = [
        dict(q=q.half(), k=k.half()), dict(k=k.float()), dict(q=q.cpu()), dict(k=k[:5]),
        dict(k=k[:, :, :32]), dict(q=q[:, :, ::2], k=None), dict(q=q[0], k=None),
        dict(positions=pos.int()), dict(positions=pos[:5]), dict(positions=pos[::1].cpu()),
        dict(rope=_rope(66)), dict(rope=rotary.Rotary(rope.turns.cpu())),
        dict(rope=rotary.Rotary(rope.turns[:0])), dict(w_q=w), dict(w_k=w),
        dict(w_q=w.bfloat16(), w_k=w.bfloat16()), dict(w_q=w[:32], w_k=w[:32]),
        dict(q=q[:, :, :63], k=None), dict(q=q[:, :0], k=None), dict(k=k[:, :0]),
        dict(out_q=torch.empty_like(q).float()), dict(out_q=q[:, :2]),
        dict(out_q=torch.empty_like(q[:, :1]).expand(-1, 4, -1)),
        dict(out_q=torch.empty_like(q[:1]).expand(10, -1, -1)),
        dict(q=q[:9], k=k[:9], positions=pos[:9], out_q=q[1:]), dict(k=None, out_k=k),
        dict(q=q[:, :2], out_q=k), dict(out_k=q[:, 1:3]),
    ]
    for kw in bad:
        a = dict(q=q, k=k, positions=pos, rope=rope)
        a.update(kw)
        with pytest.raises(ValueError):
            rotary.apply(**a)
    with pytest.raises(ValueError):  # both results in one place
        o = torch.empty_like(k)
        rotary.apply(k.clone(), k, pos, rope, out_q=o, out_k=o)
    dq, dk = s["dq"], s["dk"]
    for kw in (dict(w_q=w, w_k=w), dict(w_q=w, w_k=w, q=q), dict(w_q=w, w_k=w, q=q, k=k[:5]),
               dict(w_q=w, w_k=w, q=q.float(), k=k), dict(out_q=dk), dict(out_k=dq[:, :2]),
               dict(w_q=w, w_k=w, q=q, k=k, workspace=torch.empty(1 << 20, dtype=torch.uint8))):
        with pytest.raises(ValueError):
            rotary.apply_bwd(dq, dk, pos, rope, **kw)


def test_past_31_bits():
    """More than 2^31 elements of q, forward and backward: the first and last tokens as a
    call over them alone, the weights' gradient of a few rows."""
    m, hq, d = 70000, 240, 128
    e = torch.cat([torch.arange(5, device="cuda"), torch.arange(m - 5, m, device="cuda")])
    s = _inputs(5, hq, 2, d, torch.bfloat16, True)
    q = torch.zeros(m, hq, d, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(m, 2, d, dtype=torch.bfloat16, device="cuda")
    q[e], k[e] = _randn((10, hq, d), 1, 1.0, q.dtype), _randn((10, 2, d), 2, 1.0, q.dtype)
    positions = torch.arange(m, device="cuda")
    rope = _rope(128)
    print("forward", m, hq, d, flush=True)
    a, b = rotary.apply(q, k, positions, rope, s["w_q"], s["w_k"])
    c = rotary.apply(q[e], k[e], positions[e], rope, s["w_q"], s["w_k"])
    assert torch.equal(a[e], c[0]) and torch.equal(b[e], c[1])
    assert not a[5:-5].any() and not b[5:-5].any()
    print("backward", flush=True)
    g = rotary.apply_bwd(a, b, positions, rope, q, k, s["w_q"], s["w_k"])
    h = rotary.apply_bwd(a[e], b[e], positions[e], rope, q[e], k[e], s["w_q"], s["w_k"])
    assert torch.equal(g.dq[e], h.dq) and torch.equal(g.dk[e], h.dk)
    assert not g.dq[5:-5].any() and not g.dk[5:-5].any()
    _check_bwd(g.dq[e], g.dw_q, a[e], q[e], s["w_q"], positions[e], rope)


def test_runs_on_the_tensors_device(monkeypatch):
    """With another device current, calls and workspace queries make the tensors' own
    current (here the one device there is, under a wrong report)."""
    s = _inputs(9, 4, 2, 64, torch.bfloat16, True)
    rope = _rope(64)
    want = rotary.apply_bwd(s["dq"], s["dk"], s["positions"], rope, s["q"], s["k"], s["w_q"],
                            s["w_k"])
    seen = []
    real = torch.cuda.device

    def device(index):
        seen.append(index)
        return real(index)

    rotary._bwd_workspace_bytes.cache_clear()
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    got = rotary.apply_bwd(s["dq"], s["dk"], s["positions"], rope, s["q"], s["k"], s["w_q"],
                           s["w_k"])
    monkeypatch.undo()
    assert seen == [0, 0]
    assert torch.equal(got.dq, want.dq) and torch.equal(got.dw_k, want.dw_k)

"""8-bit activation checkpoints: codes and scales bit for bit against the same
fp32 steps in numpy, decode, and the fused decode + RMSNorm against 64 bits."""
import numpy as np
import pytest
import torch

from aethelstream_amd import checkpoint, norm

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _randn(shape, seed, sigma=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=g) * sigma


def _reference(x):
    """(codes, scales) of fp32 x [M, d] in numpy fp32, block by block."""
    x = x.cpu().numpy().astype(np.float32)
    m, d = x.shape
    blocks = -(-d // 128)
    pad = np.zeros((m, blocks * 128), np.float32)
    pad[:, :d] = x
    pad = pad.reshape(m, blocks, 128)
    scale = np.abs(pad).max(2) * (np.float32(1) / np.float32(127))
    # The largest scale: 127 of it are still finite.
    scale = np.clip(scale, np.float32(2.0 ** -126), np.float32(float.fromhex("0x1.020406p+121")))
    inv = np.float32(1) / scale
    q = np.rint(pad * inv[:, :, None]).astype(np.int8)
    return q.reshape(m, -1)[:, :d], scale.astype(np.float32)


SHAPES = [(1, 4), (1, 128), (3, 124), (2, 132), (5, 1024), (7, 1028), (300, 252), (33, 4096),
          (3, 13820), (2, 32768), (4097, 128)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,d", SHAPES)
def test_round_trip(m, d, dtype):
    print(m, d, dtype, flush=True)
    x = _randn((m, d), 1, 2.0)
    x[:, ::97] *= 30
    x = x.to(dtype)
    c = checkpoint.encode(x)
    codes, scales = _reference(x.float())
    assert np.array_equal(c.codes.cpu().numpy(), codes)
    assert np.array_equal(c.scales.cpu().numpy(), scales)
    values = codes.astype(np.float32) * np.repeat(scales, 128, 1)[:, :d]
    assert np.array_equal(checkpoint.decode(c).cpu().numpy(), values)
    back = checkpoint.decode(c, torch.bfloat16)
    assert torch.equal(back, torch.from_numpy(values).cuda().to(torch.bfloat16))
    # Half a step, and the three roundings of s, 1 / s and the product (each 2^-24
    # of at most 127 steps).
    half = torch.from_numpy(np.repeat(scales, 128, 1)[:, :d]).cuda().double() / 2
    assert ((checkpoint.decode(c).double() - x.double()).abs() <= half * (1 + 512 * U)).all()


def test_values_at_the_ends_of_fp32():
    """Zero blocks, subnormal blocks, the largest values, signed zeros."""
    x = torch.zeros(6, 256, device="cuda")
    x[1, :128] = 1e-45
    x[1, 128:] = -2.0 ** -126
    x[2] = _randn((256,), 3) * 2.0 ** -130
    x[3, :3] = torch.tensor([3.4028235e38, -3.4028235e38, 1e30], device="cuda")
    x[4] = -0.0
    x[5, 5] = 2.0 ** -119 * 127
    c = checkpoint.encode(x)
    codes, scales = _reference(x)
    assert np.array_equal(c.codes.cpu().numpy(), codes)
    assert np.array_equal(c.scales.cpu().numpy(), scales)
    back = checkpoint.decode(c)
    assert torch.isfinite(back).all() and (back[0] == 0).all() and (back[4] == 0).all()
    assert float(back[3, 0]) > 3.39e38 and float(back[3, 1]) < -3.39e38


def test_non_finite_blocks_read_back_as_nan():
    for dtype in (torch.float32, torch.bfloat16):
        for bad in (float("inf"), -float("inf"), float("nan")):
            x = _randn((3, 388), 4).to(dtype)
            x[1, 130] = bad
            back = checkpoint.decode(checkpoint.encode(x))
            assert torch.isnan(back[1, 128:256]).all()
            back[1, 128:256] = 0
            assert torch.isfinite(back).all()


@pytest.mark.parametrize("want_x", [True, False])
@pytest.mark.parametrize("m,d", SHAPES)
def test_decode_norm(m, d, want_x):
    print(m, d, want_x, flush=True)
    c = checkpoint.encode(_randn((m, d), 5, 1.5))
    w = 1 + _randn((d,), 6, 0.1)
    x, y, rms = checkpoint.decode_norm(c, w, want_x=want_x)
    plain = checkpoint.decode(c)
    if want_x:
        assert torch.equal(x, plain)
    else:
        assert x is None
    v = plain.double()
    want = (v.square().mean(1) + norm.EPS).sqrt()
    assert ((rms.double() - want).abs() <= 64 * U * want).all()
    want = v / want[:, None] * w.double()
    assert ((y.double() - want).abs() <= (2.0 ** -8 + 128 * U) * want.abs() + 1e-30).all()


def test_large_tensor_offsets():
    """Codes past 2^31: the last rows are coded as the same rows alone."""
    m, d = 70000, 32768  # 2.29e9 elements, bf16: 4.6 GB
    x = torch.zeros(m, d, dtype=torch.bfloat16, device="cuda")
    tail = _randn((3, d), 7).to(torch.bfloat16)
    x[-3:] = tail
    c, alone = checkpoint.encode(x), checkpoint.encode(tail)
    assert torch.equal(c.codes[-3:], alone.codes) and torch.equal(c.scales[-3:], alone.scales)
    del x
    back = checkpoint.decode(c, torch.bfloat16)
    assert torch.equal(back[-3:], checkpoint.decode(alone, torch.bfloat16))
    assert not back[:-3].any()


def test_given_buffers_streams_and_empty():
    x = _randn((65, 516), 8)
    want = checkpoint.encode(x)
    out = checkpoint.Checkpoint8(torch.full_like(want.codes, 99), torch.zeros_like(want.scales))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert checkpoint.encode(x, out) is out
        back = checkpoint.decode(out, out=torch.empty_like(x))
    side.synchronize()
    assert torch.equal(out.codes, want.codes) and torch.equal(out.scales, want.scales)
    assert torch.equal(back, checkpoint.decode(want))
    e = checkpoint.encode(torch.empty(0, 128, device="cuda"))
    assert checkpoint.decode(e).shape == (0, 128)


def test_refusals():
    x = _randn((4, 256), 9)
    c = checkpoint.encode(x)
    for bad in (x.half(), x.t(), x.cpu(), x[0]):
        with pytest.raises(ValueError):
            checkpoint.encode(bad)
    with pytest.raises(Exception, match="d % 4"):
        checkpoint.encode(_randn((4, 6), 1))
    with pytest.raises(ValueError):
        checkpoint.decode(checkpoint.Checkpoint8(c.codes, c.scales[:, :1].contiguous()))
    with pytest.raises(ValueError):
        checkpoint.decode(checkpoint.Checkpoint8(c.codes.view(torch.uint8), c.scales))
    with pytest.raises(ValueError):
        checkpoint.decode(c, torch.float16)
    with pytest.raises(ValueError):
        checkpoint.decode_norm(c, torch.ones(128, device="cuda"))
    with pytest.raises(ValueError):
        checkpoint.encode(x, checkpoint.encode(x[:2]))

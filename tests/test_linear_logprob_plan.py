"""How the log probabilities cut the vocabulary, read from what they ask of memory (CPU
only, for 256 CUs): launches behind whole rounds of large tiles, the smallest tiles for
few tokens, pieces of the gradient.  The shapes are those that the GPU tests of each
(test_linear_logprob_kept_gpu.py, test_linear_logprob_tiles_gpu.py) run, which a changed
rule would leave without what they are for."""
import ctypes

import pytest

from aethelstream_amd import _lib

# Tokens, columns, d; columns of the first launch, in 256-wide tiles, and the width of a
# half tile of the second.  Rests of 16 to 64 columns leave a last half tile of none.
SPLITS = [(1000, 17000, 2048, 16384, 32), (1000, 16400, 2048, 16384, 32),
          (512, 32788, 1024, 32768, 32), (130, 65600, 1024, 65536, 32),
          (4096, 4120, 2048, 4096, 32), (2000, 8212, 1024, 8192, 32),
          (700, 25000, 2048, 21760, 64), (300, 70000, 2048, 65536, 64)]
# Up to 32 tokens whose 64 x 64 tiles take three quarters to all of the places of two a
# CU; and next to that: fewer, more, another token, a shorter reduction.
FEW = [(m, v, d) for m in (1, 32) for v in (24600, 32000, 32768) for d in (2048, 4096)]
NEXT_TO_FEW = [(1, 24500, 2048), (32, 32800, 2048), (33, 32000, 2048), (32, 32000, 2040)]
# Several pieces of the gradient, of one launch over the columns (first launch: None), or
# of two that meet inside a piece.
PIECES = [(16384, 9001, 16, None), (8192, 40007, 64, None), (9000, 33001, 2048, 32768),
          (3000, 100003, 1024, None), (300, 460001, 64, None)]


def _up(a, b):
    return (a + b - 1) // b * b


def _ask(name, *args):
    out = ctypes.c_int64(-1)
    assert getattr(_lib.load(), name)(*args, ctypes.byref(out)) == 0
    return out.value


def columns(m, v, d):
    """Columns of the kept logits: whole tiles of every launch."""
    return _ask("nf4s_linear_logprob_logits_size", m, v, d) // (4 * m)


def forward_bytes(m, slices):
    """Maximum, two sums of each half tile, and the target's logit."""
    return _up(8 * slices * m, 256) + _up(4 * slices * m, 256) + _up(4 * m, 256)


def forward(m, v, d):
    return _ask("nf4s_linear_logprob_workspace_size", m, v, d, 0, 0)


def in_one_launch(m, v, d):
    """Whether some width of tiles, alone, would ask for this."""
    return any(columns(m, v, d) == _up(v, 2 * w)
               and forward(m, v, d) == forward_bytes(m, _up(v, 2 * w) // w) for w in (32, 64, 128))


def in_two_launches(m, v, d, first, width):
    rest = _up(v - first, 2 * width)
    return columns(m, v, d) == first + rest and \
        forward(m, v, d) == forward_bytes(m, first // 128 + rest // width)


@pytest.mark.parametrize("m,v,d,first,width", SPLITS)
def test_two_launches(m, v, d, first, width):
    assert in_two_launches(m, v, d, first, width) and not in_one_launch(m, v, d)


@pytest.mark.parametrize("m,v,d", FEW)
def test_smallest_tiles_of_few_tokens(m, v, d):
    assert columns(m, v, d) == _up(v, 64)
    assert forward(m, v, d) == forward_bytes(m, _up(v, 64) // 32)


@pytest.mark.parametrize("m,v,d", NEXT_TO_FEW)
def test_other_tiles_next_to_them(m, v, d):
    assert forward(m, v, d) != forward_bytes(m, _up(v, 64) // 32)


@pytest.mark.parametrize("m,v,d,first", PIECES)
def test_pieces_of_the_gradient(m, v, d, first):
    # G of all columns would not fit into what the gradients ask for.
    assert _ask("nf4s_linear_logprob_workspace_size", m, v, d, 0, 1) < 2 * m * v
    most = (1 << 28) // (2 * m) // 256 * 256  # columns of 256 MB
    piece = _up(-(-v // -(-v // most)), 256)
    assert piece < v and v % piece != 0
    if first is None:
        assert in_one_launch(m, v, d)
    else:
        assert in_two_launches(m, v, d, first, 64) and first % piece != 0


def test_maxima_that_a_wave_holds():
    """A token's half tiles of a piece of the vocabulary: at most 4096, as LDS holds their
    maxima (4 bytes each, 16 KB).  Of one piece, whose logits the workspace holds."""
    for m in (1, 2, 31, 32, 33, 64, 65, 128, 129, 300, 511, 512, 1000, 4096, 16384):
        for v in (1, 4096, 24600, 32768, 32769, 50021, 65600, 128000, 200000, 262144):
            for d in (8, 2048, 8192):
                piece = min(v, max(min((1 << 28) // (4 * m) // 256 * 256, 1 << 18), 4096))
                assert forward(m, piece, d) <= forward_bytes(m, 4096), (m, v, d, piece)

"""Choices of the launches that the workspace queries show, by the rules' reasons.
CPU only: without a device the queries plan for 256 CUs."""
import ctypes

import pytest
import torch

from aethelstream_amd import _lib

CUS = 256

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="plans for 256 CUs")


def _norm_groups(m, d):
    """Workgroups of the norms' backward: each writes two rows of column sums."""
    out = ctypes.c_int64(0)
    _lib.check(_lib.load().nf4s_block_norm_bwd_workspace_size(m, d, ctypes.byref(out)))
    assert out.value % (8 * d) == 0
    return out.value // (8 * d)


# Columns, and the workgroups that a CU holds at once: of 256 threads and 16 waves
# (1024 columns: four rows side by side are 8 waves), of 12292 to 16384 columns 8
# waves, in workgroups of 7 and 8.
@pytest.mark.parametrize("d,held", [(1024, 2), (4096, 2), (8192, 1), (8196, 1), (12288, 1),
                                    (12292, 1), (13824, 1), (14336, 1), (16384, 1), (16388, 1),
                                    (32768, 1)])
def test_norm_backward_runs_in_one_round(d, held):
    assert _norm_groups(100000, d) == CUS * held
    assert _norm_groups(1, d) == 1


def _forward_bytes(m, v, d):
    out = ctypes.c_int64(0)
    _lib.check(_lib.load().nf4s_linear_ce_workspace_size(m, v, d, 0, ctypes.byref(out)))
    return out.value


# Tokens, columns, length, and the tile width whose forward is the faster one of
# 128 (64 x 128 tiles) and 256 columns (128 or 256 rows), measured in us with w
# from memory.
@pytest.mark.parametrize("m,v,d,narrow,wide", [
    (1, 50021, 4096, 80.2, 90.8), (64, 50021, 4096, 87.0, 92.8), (1, 128000, 1024, 49.4, 55.6),
    (16, 50021, 8192, 151.7, 162.7), (77, 32000, 1024, 21.3, 24.3), (96, 32000, 1024, 22.0, 24.5),
    (77, 32000, 4096, 66.0, 68.8), (128, 32000, 8192, 134.2, 143.6),
    (77, 50021, 4096, 110.9, 92.1), (128, 50021, 4096, 117.5, 93.7),
    (256, 32000, 4096, 114.5, 71.8), (400, 8000, 4096, 50.9, 56.2),
    (512, 32000, 4096, 204.1, 106.5)])
def test_logits_tiles_are_the_faster_ones(m, v, d, narrow, wide):
    width = 128 if narrow < wide else 256
    # Two partial sums of 8 bytes for each tile of a token, up to a multiple of 256
    # bytes, and a logit of 4.
    part = 2 * -(-v // width) * 8 * m
    assert _forward_bytes(m, v, d) == -(-part // 256) * 256 + 4 * m

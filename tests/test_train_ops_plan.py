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

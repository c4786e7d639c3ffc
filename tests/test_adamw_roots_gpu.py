"""The square roots of the AdamW step, which are meant to be correctly rounded (a root in
64 bits, rounded, is: its 53 bits are more than twice 24 and two).  A block of 8-bit
moments whose elements but one are zero has that one's sqrt(v) as its scale, as it is:
v = grad^2 * hyper[3] with hyper[2] = 0."""
import pytest
import torch

from aethelstream_amd import optim

pytestmark = pytest.mark.gpu

BLOCKS = 1 << 24


def _bits(x):
    return x.view(torch.int32)


class _Roots:
    """Steps over BLOCKS blocks of one gradient each."""

    def __init__(self):
        self.p = torch.zeros(BLOCKS * optim.BLOCK, dtype=torch.bfloat16, device="cuda")
        self.grad = torch.zeros(BLOCKS, optim.BLOCK, device="cuda")
        self.state = optim.adamw_state([self.p], bits=8)

    def check(self, d, factor):
        """Whether all roots of d^2 * factor are right; those squares."""
        # One place of the block after the other.
        self.grad.zero_()
        self.grad[torch.arange(BLOCKS, device="cuda"),
                  torch.arange(BLOCKS, device="cuda") % optim.BLOCK] = d
        hyper = torch.tensor([0.0, 1.0, 0.0, factor, 1.0, 0.0, 1.0, 1.0], device="cuda")
        optim.adamw_step([self.p], [self.grad.view(-1)], self.state, 1, hyper=hyper)
        v = d * d * hyper[3]
        want = v.double().sqrt().float()
        assert torch.equal(self.state.v_scale, want)
        return v


def test_every_number_of_two_binades():
    """All 2^24 numbers of [1, 4), by the squares of all of [1, 4) times factors that
    bring other ones about."""
    d = (torch.arange(BLOCKS, dtype=torch.int32, device="cuda") + 0x3f800000).view(torch.float32)
    roots, seen = _Roots(), torch.zeros(BLOCKS, dtype=torch.bool, device="cuda")
    g = torch.Generator().manual_seed(1)
    for i in range(100):
        print("factor", i, flush=True)
        v = roots.check(d, float(0.25 + 0.75 * torch.rand(1, generator=g)))
        seen[_bits(v[(v >= 1) & (v < 4)]).long() - 0x3f800000] = True
        if seen.all():
            break
    assert seen.all(), int((~seen).sum())


@pytest.mark.parametrize("low,high", [(-50, 60), (-63, 63)])
def test_numbers_of_any_size(low, high):
    """Squares of 2^(2 low) to 2^(2 high): those that the quick root takes, and with the
    ones that it leaves in the same waves."""
    g = torch.Generator(device="cuda").manual_seed(2)
    e = torch.randint(low, high, (BLOCKS,), device="cuda", generator=g, dtype=torch.int32)
    frac = torch.randint(0, 1 << 23, (BLOCKS,), device="cuda", generator=g, dtype=torch.int32)
    _Roots().check(((e + 127 << 23) + frac).view(torch.float32), 1.0)

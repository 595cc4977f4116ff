"""Float scales: a value in 8 bits is the e4m3 nearest to the quotient x * 448 / a rounded once to 32 bits, also of 32-bit x, whose product with 448 takes up to 27 digits."""
import pytest
import torch

from .test_fp8 import E4, F32, gen, gpu


def beside_borders(rows, seed):
    """[rows, 5, 128] floats: a block's largest value a first, the others the floats at -2 .. 2 steps from a / 448 times a border between two neighbouring values."""
    values = torch.arange(127, dtype=torch.uint8).view(E4).double()
    borders = (values[1:] + values[:-1]) / 2
    g = gen(seed)
    a = ((1 + torch.rand(rows, generator=g)) * torch.exp2(torch.randint(-60, 60, (rows,), generator=g).float())).float()
    near = (borders * a.double()[:, None] / 448).float()
    x = torch.stack([(near.view(torch.int32) + d).view(torch.float32) for d in range(-2, 3)], 1)
    x = torch.minimum(x, a[:, None, None]) * torch.where(torch.rand(x.shape, generator=g) < 0.5, -1.0, 1.0)
    return torch.cat([a.view(-1, 1, 1).expand(-1, 5, 2), x], 2), a


@gpu
@pytest.mark.parametrize("at", [0, 3])
def test_quotients_beside_borders(at):
    """At the start of a row's block, and three columns into a matrix (other loads)."""
    from jacobiforcing_amd import layer_ops as LO
    x, a = beside_borders(400, 5)
    wide = torch.zeros(2000, 128 + 2 * at)
    wide[:, at:at + 128] = x.reshape(2000, 128)
    r = LO.quantize_fp8(wide.cuda()[:, at:at + 128], F32)
    want = (x.double() * 448 / a.double().view(-1, 1, 1)).float().to(E4).float().view(2000, 128)
    wrong = r.data.float().cpu() != want
    assert not bool(wrong.any()), f"{int(wrong.sum())} of {wrong.numel()} values"


@gpu
def test_units_of_whole_gates_beside_borders():
    """A unit without a linear branch whose gate leaves its value as it is: gelu of numbers so large that it is the identity."""
    from jacobiforcing_amd import layer_ops as LO
    x, a = beside_borders(200, 6)
    up = torch.exp2(30 - torch.floor(torch.log2(a)))    # a power of two: the quotients stay
    x, a = x.abs() * up.view(-1, 1, 1), a * up
    r = LO.gated_act_fp8(x.reshape(1000, 128).cuda(), 0, -1, 128, 3, scale_dtype=F32)
    want = (x.double() * 448 / a.double().view(-1, 1, 1)).float().to(E4).float().view(1000, 128)
    wrong = r.data.float().cpu() != want
    assert not bool(wrong.any()), f"{int(wrong.sum())} of {wrong.numel()} values"

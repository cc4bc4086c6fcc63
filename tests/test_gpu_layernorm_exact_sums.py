"""Gradients of weight and bias where fp32 sums are exact: whole numbers, small enough that no partial sum is rounded.  A row, a group's
or a block's part that is left out or counted twice then shows, however many rows there are."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("types", [(BF, BF), (BF, F32), (F32, F32), (F32, BF)])
@pytest.mark.parametrize("shape", [(1, 768), (2, 5), (64, 768), (9001, 12), (9001, 101), (20000, 40), (4099, 1021), (4099, 257), (2311, 1024), (1500, 4096), (601, 8191),
                                   (333, 9000), (1025, 20001)])
def test_no_row_is_left_out(shape, types):
    """Each row's dy is a number of its own between -64 and 64 in some columns, x between -8 and 8; with mean 0 and rstd 1 given, dw = sum dy x and db = sum dy.
    Sums stay below 20000 * 512 < 2^24."""
    from haste_b200.norm import layer_norm_backward
    rows, D = shape
    xt, gt = types
    gen = torch.Generator(device="cuda").manual_seed(rows + D)
    draw = lambda lo, hi, *s: torch.randint(lo, hi + 1, s, generator=gen, device="cuda").float()
    dy = draw(1, 64, rows, D) * torch.where(torch.rand(rows, D, generator=gen, device="cuda") < 0.5, -1.0, 1.0)       # never 0
    x = draw(1, 8, rows, D) * torch.where(torch.rand(rows, D, generator=gen, device="cuda") < 0.5, -1.0, 1.0)
    mean, rstd = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    _, dw, db = layer_norm_backward(dy.to(gt), x.to(xt), None, mean, rstd, param_dtype=F32)
    assert torch.equal(dw.double(), (dy.double() * x.double()).sum(0)) and torch.equal(db.double(), dy.double().sum(0))
    _, dw1, none = layer_norm_backward(dy.to(gt), x.to(xt), torch.ones(D, device="cuda"), mean, rstd, want_bias=False)
    assert none is None and torch.equal(dw1, dw)

"""What linear layers make of numbers in 8 bits at the ends of their type's range: of fp16 they are as they are from 2^-21 up, multiples of 2^-24 below, infinite from
65520 up, wherever the numbers are widened; of bf16 they are as they are."""
import pytest
import torch

from test_gpu_features import DEV, act64
from test_gpu_layers8 import values

pytestmark = pytest.mark.gpu

POWERS = list(range(-30, 17))


def one_number_a_row(rows, cols, at):
    """Rows of one number each, 1.125 2^k, 1.5 2^k and 1.75 2^k in turn, k from 2^-30 to 2^16."""
    k = torch.tensor(POWERS, device=DEV).repeat(-(-rows // len(POWERS)))[:rows]
    x = torch.zeros((rows, cols), device=DEV)
    x[:, at] = torch.exp2(k.float()) * torch.tensor([1.125, 1.5, 1.75], device=DEV).repeat(-(-rows // 3))[:rows]
    return x


@pytest.mark.parametrize("rows,out", [(94, 3), (94, 700), (3000, 264), (9400, 1030)])     # few rows, and tiles of several shapes
@pytest.mark.parametrize("eight", [False, True], ids=["w16", "w8"])
def test_rows_enter_as_fp16(rows, out, eight):
    from cuke_amd import features
    print("half", rows, out, eight, flush=True)
    r = features.pack8(one_number_a_row(rows, 40, 33))
    held = values(r)
    assert torch.equal(held[:, 33], one_number_a_row(rows, 40, 33)[:, 33].double())
    enters = held[:, 33].half().double()
    same = (held[:, 33] >= 2.0 ** -21) & (held[:, 33] < 65520)
    assert torch.equal(enters[same], held[same, 33]) and bool((enters != held[:, 33]).any()) and bool(enters.isinf().any())
    w = torch.zeros((out, 40), device=DEV)
    w[1, 33], w[2, 33] = 0.25, -4.0
    y = features.linear(r, features.pack8(w) if eight else w.half(), out_dtype=torch.float32, dtype=torch.float16).double()
    fine = enters.isfinite()
    assert torch.equal(y[:, 1], enters * 0.25) and torch.equal(y[:, 2], enters * -4.0) and bool((y[fine, 0] == 0).all()) and bool((y[fine, 3:] == 0).all())


@pytest.mark.parametrize("rows,out", [(94, 700), (3000, 264)])
def test_a_weight_enters_as_fp16(rows, out):
    from cuke_amd import features
    w = features.pack8(one_number_a_row(out, 40, 33))
    enters = values(w)[:, 33].half().double()
    x = torch.zeros((rows, 40), device=DEV)
    x[:, 33] = 0.5
    y = features.linear(features.pack8(x), w, out_dtype=torch.float32, dtype=torch.float16).double()
    assert torch.equal(y, (0.5 * enters).expand(rows, out))


@pytest.mark.parametrize("rows,out", [(94, 3), (3000, 264), (16500, 300)])
def test_the_weights_gradient_of_fp16_rows(rows, out):
    """Each row in a column of its own: a gradient is one product."""
    from cuke_amd import features
    print("half gradient", rows, out, flush=True)
    n = min(rows, 94)
    x = torch.zeros((rows, n), device=DEV)
    at = torch.arange(n, device=DEV)
    x[at * (rows // n), at] = one_number_a_row(n, 1, 0)[:, 0]
    r = features.pack8(x)
    enters = values(r)[at * (rows // n), at].half().double()
    fw = features.linear_forward(r, torch.zeros((out, n), dtype=torch.float16, device=DEV), out_dtype=torch.float32)
    dy = torch.zeros((rows, out), device=DEV)
    dy[:, 2] = 0.5
    g = features.linear_backward(fw, dy).weight.double()
    fine = enters.isfinite()
    assert torch.equal(g[2, fine], (0.5 * enters[fine]).half().double()) and bool(g[2, ~fine].isinf().all()) and bool((g[0, fine] == 0).all())


@pytest.mark.parametrize("rows,out", [(60, 3), (3000, 264)])
@pytest.mark.parametrize("eight", [False, True], ids=["w16", "w8"])
def test_the_smallest_bf16_numbers(rows, out, eight):
    """Numbers down to 2^-133 enter a bf16 layer as they are."""
    from cuke_amd import features
    number = torch.tensor([2.0 ** k for k in range(-133, -113)], dtype=torch.float64, device=DEV).repeat(-(-rows // 20))[:rows]
    x = torch.zeros((rows, 40), device=DEV)
    x[:, 33] = number.float()
    r = features.pack8(x)
    assert torch.equal(values(r)[:, 33], number)
    w = torch.zeros((out, 40), device=DEV)
    w[1, 33] = 2.0 ** 20
    y = features.linear(r, features.pack8(w) if eight else w.bfloat16(), out_dtype=torch.float32, dtype=torch.bfloat16).double()
    assert torch.equal(y[:, 1], number * 2.0 ** 20) and bool((y[:, 0] == 0).all())
    assert torch.equal(features.unpack8(r, torch.bfloat16).double(), values(r))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_what_a_derivative_in_8_bits_is_off_by(act, dtype):
    """A step is 0.005: 0.0025 at most, 0.005 / sqrt(12) = 0.00144 in the mean square (of 65536 values within 1 %), and the gradient's own rounding."""
    from cuke_amd import features
    b = torch.randn(65536, generator=torch.Generator().manual_seed(1)).to(DEV).to(dtype)
    w = torch.zeros((65536, 8), dtype=dtype, device=DEV)
    fw = features.linear_forward(features.pack8(torch.zeros((1, 8), device=DEV)), w, b, act=act)
    got = features.linear_backward(fw, torch.ones_like(fw.y), need_x=False, need_weight=False).bias.double()
    want = act64(b.double(), act)[1]
    half = torch.finfo(dtype).eps / 2
    assert bool(((got - want).abs() <= 0.0025 + half * want.abs() * 1.01 + 1e-6).all())
    kept = (got - want).square().mean().sqrt().item()
    assert 0.0013 <= kept <= (0.00146 ** 2 + (half * want.abs().max().item()) ** 2) ** 0.5

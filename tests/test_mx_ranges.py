"""Block-scaled numbers at the ends of fp32's range: what the containers say that the bytes stand for, the largest
weights, the smallest rows."""
import pytest
import torch

from oracle import mx
from vagus_amd import ops

DEV = 'cuda'
gpu = pytest.mark.gpu


def case(*what):
    print('\n[case]', *what, flush=True)


def test_dequantize_in_64_bits_passes_the_range_of_fp32():
    x = torch.zeros(2, 40)
    x[0, 3], x[1, 35] = torch.finfo(torch.float32).max, -torch.finfo(torch.float32).max      # round up to 256 x 2^120
    q, b = mx.quantize(x, 8)
    rows = ops.MXRows(q.to(torch.float8_e4m3fn), b, 40)
    want = torch.zeros(2, 40, dtype=torch.float64)
    want[0, 3], want[1, 35] = 2.0 ** 128, -2.0 ** 128
    assert torch.equal(rows.dequantize(torch.float64), want)
    assert torch.equal(rows.dequantize(), want.float()) and rows.dequantize(torch.bfloat16).dtype is torch.bfloat16
    values, scales = torch.zeros(1, 1, 4, 16, 16, dtype=torch.uint8), torch.ones(1, 1, 4, 16, 4, dtype=torch.uint8)
    values[0, 0, 0, 5, 1], scales[0, 0, 0, 5, 0] = 0xf6, 254                                # 4 and -6 times 2^127
    got = ops.MXWeight(values, scales, (16, 128)).dequantize(torch.float64)
    assert got[5, 2] == 2.0 ** 129 and got[5, 3] == -6 * 2.0 ** 127 and int((got != 0).sum()) == 2


def test_the_oracles_largest_weights_are_finite_in_bf16():
    w = torch.full((1, 32), torch.finfo(torch.float32).max)
    assert torch.equal(mx.rounded(w, 4), torch.full((1, 32), 1.5 * 2.0 ** 127, dtype=torch.float64))
    for v in (1.75 * 2.0 ** 127, 1.5 * 2.0 ** 127, 2.0 ** 126):           # the first is half a step above the largest
        w[0, 0] = v
        assert float(mx.rounded(w[:, :1], 4)) == min(v, 1.5 * 2.0 ** 127)


@gpu
@pytest.mark.parametrize('dt', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('R', [1, 40])
def test_the_largest_weights(R, dt):
    case('mx_weight of the largest numbers, products with rows of zeros and of small numbers', R, dt)
    top = torch.finfo(dt).max
    w = torch.zeros(32, 256, device=DEV)
    w[0, 0], w[1, 40], w[2, 200], w[3, 5], w[3, 6] = top, -top, 1.75 * 2.0 ** 127, 1.5 * 2.0 ** 127, -2.0 ** 124
    w = w.to(dt)
    got = ops.mx_weight(w)
    assert torch.equal(got.dequantize(torch.float64), mx.rounded(w, 4)) and bool(torch.isfinite(got.dequantize()).all())
    x = torch.zeros(R, 256, device=DEV)
    x[-1, [0, 40, 200, 5]] = 2.0 ** -100
    want = x.double() @ mx.rounded(w, 4).t()                       # powers of two: nothing is rounded
    for rows in (x, x.bfloat16(), ops.mx_quantize(x)):
        assert torch.equal(ops.mx_linear(rows, got, out_dtype=torch.float32).double(), want)


@gpu
@pytest.mark.parametrize('R', [2, 40])
@pytest.mark.parametrize('e', [-100, -115, -122, -126])
def test_small_fp32_rows_are_held_down_to_the_least_of_bf16(R, e):
    """Parts are cut at 2^-133, so an element is off by less than that; 2 (3 K + 64) 2^-24 of sum |x w| for the sums,
    2^-24 of the result for its rounding (as tests/test_mx.py)."""
    case('mx_linear: fp32 rows about 2 to the', e, R)
    K = 200
    g = torch.Generator(DEV).manual_seed(R)
    x = (torch.rand(R, K, generator=g, device=DEV) - 0.5) * 2.0 ** e
    w = ops.mx_weight(torch.randn(40, K, generator=g, device=DEV) * 2.0 ** 110)
    wd = w.dequantize(torch.float64)
    want, A = x.double() @ wd.t(), x.double().abs() @ wd.abs().t()
    tol = 2.0 ** -133 * wd.abs().sum(1) + A * 2 * (3 * K + 64) * 2 ** -24 + want.abs() * 2 ** -24
    assert bool(((ops.mx_linear(x, w).double() - want).abs() <= tol).all())

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

"""Every kernel that the products with 4-bit weights choose among (csrc/gdr_mx_linear.hip, mx_linear_t), by name: the
rule stands here a second time, a test on the CPU holds the shapes to reaching all 44 kernels, and each shape runs
against the 64-bit products of tests/test_mx.py, with its bounds, and again for the same bits.  Rows, columns and
sums end inside a tile wherever the kernel allows it."""
import pytest
import torch

from oracle import mx
from test_mx import BF, DEV, FH, FS, case, gated_bounds, product_error, randn, rows_of, rows_within, within
from vagus_amd import ops

gpu = pytest.mark.gpu
CUS = 256


def kernel_of(kind, gated, out8, R, K, n):
    """(rows as the kernel takes them, gated, (weight tiles, row tiles of 16, waves) or (rows, columns) of a tile)."""
    up = lambda a, b: -(-a // b)  # noqa: E731
    C, N = up(K, 128), n // 2 if gated else n
    tiles = 16 * up(N, 128) if out8 else 2 * up(N, 16) if gated else up(N, 16)
    planes = {'fp32': 3, 'fp16': 2}.get(kind, 1)
    few = lambda mt, nb: up(tiles, mt) * up(R, 16 * nb)  # noqa: E731
    name = lambda x, what: (x, gated, what)  # noqa: E731
    if R <= 32 and (kind in ('fp32', 'fp16') or kind == 'bf16' and K % 128):
        x = 'tail' if kind == 'bf16' else kind
        for mt in () if gated else (1, 2):
            if few(mt, 1) <= CUS:
                return name(x, (mt, 1, 8))
        return name(x, (4, 1, 8))
    x = 'mx8' if kind == 'mx8' else 'bf16'
    total = C * planes
    most = 1 if x == 'mx8' or total <= 6 else 2 if total <= (12 if gated else 16) else 3
    if R <= 32 or few(4, 2) <= most * CUS:
        if not gated:
            for mt, nb in ((1, 1), (2, 1), (2, 2)):
                if few(mt, nb) <= CUS and (nb == 1 or R > 16):
                    return name(x, (mt, nb, 8))
        if R <= 16 or few(4, 1) <= CUS:
            return name(x, (4, 1, 8))
        return name(x, (4, 2, 8 if few(4, 2) <= CUS else 4))
    fills = lambda bm, bn: 4 * up(R, bm) * up(tiles, bn // 16) >= 5 * CUS  # noqa: E731
    for bm, bn in ((128, 256), (64, 256), (64, 128)):
        if fills(bm, bn) and (bm == 64 or x == 'mx8'):
            return name(x, (bm, bn))
    return name(x, (64, 64))


# rows, the sum's length (fp16, fp32, 8 bits: and a few less), columns
PLAIN = [(20, 256, 1000), (37, 256, 2040), (33, 256, 4000), (5, 256, 8300), (35, 256, 5000), (45, 256, 8000), (20, 256, 20000),
         (64, 896, 8200), (130, 256, 4000), (300, 256, 8200), (300, 256, 16400), (600, 256, 16400)]
GATED = [(9, 256, 100), (40, 256, 500), (40, 256, 3900), (20, 256, 8300), (64, 896, 4100), (130, 256, 2000), (300, 256, 4100), (300, 256, 8200),
         (600, 256, 8200)]
FEW = [(20, 250, 1000), (20, 250, 4000), (20, 250, 8300), (3, 250, 8300)]        # of any type, converted on the way

CASES = [(kind, False, R, K - (6 if kind == 'mx8' else 0), N) for kind in ('bf16', 'mx8') for R, K, N in PLAIN] \
    + [(kind, True, R, K - (6 if kind == 'mx8' else 0), 2 * h) for kind in ('bf16', 'mx8') for R, K, h in GATED] \
    + [(kind, False, *s) for kind in ('bf16', 'fp16', 'fp32') for s in FEW] \
    + [(kind, True, 20, 250, 2 * 500) for kind in ('bf16', 'fp16', 'fp32')] \
    + [(kind, False, R, 250, N) for kind in ('fp16', 'fp32') for R, _, N in PLAIN if R > 32] \
    + [(kind, True, R, 250, 2 * h) for kind in ('fp16', 'fp32') for R, _, h in GATED if R > 32] \
    + [('bf16', False, 300, 250, 4100), ('bf16', True, 300, 250, 2 * 2100)]


def test_every_kernel_is_reached():
    every = {(x, g, w) for x in ('fp32', 'fp16', 'tail') for g, ws in ((False, [(1, 1, 8), (2, 1, 8), (4, 1, 8)]), (True, [(4, 1, 8)])) for w in ws}
    every |= {(x, g, w) for x in ('bf16', 'mx8') for g in (False, True)
              for w in ([] if g else [(1, 1, 8), (2, 1, 8), (2, 2, 8)]) + [(4, 1, 8), (4, 2, 8), (4, 2, 4), (64, 256), (64, 128), (64, 64)]
              + ([(128, 256)] if x == 'mx8' else [])}
    assert len(every) == 44
    reached = {kernel_of(kind, gated, False, R, K, n) for kind, gated, R, K, n in CASES}
    assert every == reached, sorted(map(str, every - reached))
    # 8-bit results by every gated kernel too
    gated8 = {kernel_of(kind, True, True, R, K, n) for kind, gated, R, K, n in CASES if gated}
    assert gated8 == {k for k in every if k[1]}
    # rows as bf16 planes, two and three and one of a width that ends inside a tile, by tiles and by few-row kernels
    for kind in ('fp16', 'fp32'):
        planes = {kernel_of(kind, gated, False, R, K, n)[2] for kind_, gated, R, K, n in CASES if kind_ == kind and R > 32}
        assert {len(w) for w in planes} == {2, 3} and len(planes) >= 6


@gpu
@pytest.mark.parametrize('kind, gated, R, K, n', CASES)
def test_a_kernel(kind, gated, R, K, n):
    case(*kernel_of(kind, gated, False, R, K, n), 'of', kind, R, K, n)
    assert torch.cuda.get_device_properties(0).multi_processor_count == CUS
    x, xd = rows_of(kind, R, K, R + K)
    w = ops.mx_weight(randn(n, K, seed=n) * 0.05, gated)
    wd = w.dequantize(torch.float64)
    if gated:
        want, err = gated_bounds(kind, xd, wd)
        f = ops.mx_swiglu
    else:
        want, err = xd @ wd.t(), product_error(kind, xd, wd)
        f = ops.mx_linear
    for dt in ({'bf16': BF, 'fp16': FH, 'fp32': FS, 'mx8': BF}[kind], FS):
        y = f(x, w, out_dtype=dt)
        assert y.shape == want.shape and y.dtype is dt
        within(y, want, err, dt)
        assert torch.equal(f(x, w, out_dtype=dt), y)
    if gated:
        rows = f(x, w, quantize=True)
        rows_within(rows, want, err)
        again = f(x, w, quantize=True)
        assert torch.equal(again.values.view(torch.uint8), rows.values.view(torch.uint8)) and torch.equal(again.scales, rows.scales)


@gpu
@pytest.mark.parametrize('kind', ['bf16', 'fp16', 'fp32'])
@pytest.mark.parametrize('R, K, h', [(3, 256, 384), (70, 640, 1024), (300, 256, 4096), (600, 200, 8192)])
def test_8_bit_results_of_exact_rows_are_the_fp32_result_rounded(R, K, h, kind):
    case('mx_swiglu to 8 bits against mx_quantize of its fp32 result', kind, R, K, h)
    # whole 128s of columns: one kernel for both, one order of the sums
    assert kernel_of(kind, True, True, R, K, 2 * h) == kernel_of(kind, True, False, R, K, 2 * h)
    x, _ = rows_of(kind, R, K, R + K)
    w = ops.mx_weight(randn(2 * h, K, seed=h) * 0.2, gated=True)
    got, want = ops.mx_swiglu(x, w, quantize=True), ops.mx_quantize(ops.mx_swiglu(x, w, out_dtype=FS))
    assert torch.equal(got.scales, want.scales)
    assert torch.equal(got.values.view(torch.uint8), want.values.view(torch.uint8))

"""Block-scaled numbers: rows to 8 bits (ops.mx_quantize, ops.mx_rms_norm), weights to 4 bits (ops.mx_weight), and
the products that take them (ops.mx_linear, ops.mx_swiglu).  The reference has no such operators; the oracle is
oracle/mx.py and fp64 products.

What is rounded to 8 or 4 bits is compared bit by bit: the definition is in exact arithmetic but for the
norm's root, which the kernel forms in 64 bits too (a tie between two of its results within 2^-50 does not occur in
these inputs).  A product's result is off by
  - the rounding of the result, eps / 2 of its type relative to the value;
  - the sum's own error.  Rows of bf16, fp16 and fp32 meet the weights exactly, and of n fp32 additions each
    rounds by 2^-24 of a partial sum, which is at most A = sum |x w|: (K + 64) 2^-24 A, twice that as the matrix
    instructions may cut instead of rounding.  (fp32 rows: three partial products an element, 3 K additions.)
  - with 8-bit rows, the instruction's inner sum of 128 products: it keeps 2^-13 of the largest terms (blocks
    whose scales are far apart lose their low bits to the largest), 2^-12 A in all.
The gated product multiplies errors: silu is 1.1-Lipschitz and at most |a|, so |e| <= 1.1 ea |b| + |a| eb + ea eb, with
the hardware's exponential and reciprocal (|a| 2^-22 + 2^-21 relative) where the result has 16 or 8 bits.
"""
import pytest
import torch

from oracle import mx
from vagus_amd import _lib, ops

DEV = 'cuda'
BF, FH, FS = torch.bfloat16, torch.float16, torch.float32
gpu = pytest.mark.gpu


def case(*what):
    print('\n[case]', *what, flush=True)


def randn(*shape, seed=0, device=DEV):
    return torch.randn(*shape, generator=torch.Generator(device).manual_seed(seed), device=device)


# --- the oracle and the formats, on the CPU ------------------------------------


def test_oracle_rounds_as_torch_does():
    x = randn(64, 96, seed=1, device='cpu') * 60
    assert torch.equal(mx.nearest(x.double().clamp(-448, 448), 8).float(), x.clamp(-448, 448).to(torch.float8_e4m3fn).float())
    every = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(mx.nearest(every, 8), every)
    between = (every[1:] + every[:-1]) / 2                            # ties: the even code
    even = torch.where(torch.arange(126) % 2 == 0, every[:-1], every[1:])
    assert torch.equal(mx.nearest(between, 8), even)
    four = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    assert torch.equal(mx.nearest(four, 4), four)
    assert torch.equal(mx.nearest((four[1:] + four[:-1]) / 2, 4), four[torch.tensor([0, 2, 2, 4, 4, 6, 6])])


def test_oracle_scale_is_the_smallest_that_is_allowed():
    x = torch.cat([randn(50, 32, seed=2, device='cpu') * 10.0 ** torch.arange(-25, 25)[:, None],
                   torch.full((1, 32), 464.0), torch.full((1, 32), 464.1), torch.zeros(1, 32), torch.full((1, 32), 1e-44)])
    q, b = mx.quantize(x, 8)
    s, amax = mx.scales(b[:, 0]), x.double().abs().amax(1)
    assert bool((amax <= 464 * s).all())
    assert bool(((amax > 464 * s / 2) | (b[:, 0] == 1)).all())
    assert b[-4, 0] == 127 and b[-3, 0] == 128 and b[-2, 0] == 1 and bool((b[:, 1:] == 1).all())
    assert bool((q.abs() <= 448).all())


def layout(w, gated):
    """The tiles of vagus_gdr.h, element by element."""
    n, k = w.shape
    half = n // 2 if gated else n
    T, C = (2 if gated else 1) * -(-half // 16), -(-k // 128)
    q, b = mx.quantize(w, 4)
    code = {float(v): i for i, v in enumerate([0, .5, 1, 1.5, 2, 3, 4, 6])}
    values = torch.zeros(T, C, 4, 16, 16, dtype=torch.uint8)
    scales = torch.ones(T, -(-C // 4), 4, 16, 4, dtype=torch.uint8)
    for i in range(n):
        t, r = i // 16, i % 16
        if gated:
            t, r = 2 * (i % half // 16) + i // half, i % half % 16
        for c in range(4 * C):
            scales[t, c // 16, c % 4, r, c // 4 % 4] = b[i, c]
        for j in range(k):
            v = float(q[i, j])
            bits = code[abs(v)] | (8 if v < 0 or (v == 0 and float(w[i, j]) < 0) else 0)
            values[t, j // 128, j % 128 // 32, r, j % 32 // 2] |= bits << 4 * (j % 2)
    return values, scales


@pytest.mark.parametrize('n, k, gated', [(5, 40, False), (33, 130, False), (16, 128, False), (10, 600, True), (64, 128, True)])
def test_weight_tiles_stand_for_the_weights(n, k, gated):
    w = randn(n, k, seed=3, device='cpu')
    values, scales = layout(w, gated)
    got = ops.MXWeight(values, scales, (n, k), gated).dequantize(torch.float64)
    assert torch.equal(got, mx.rounded(w, 4))


def test_rows_stand_for_the_rows():
    x = randn(3, 200, seed=4, device='cpu')
    q, b = mx.quantize(x, 8)
    rows = ops.MXRows(q.to(torch.float8_e4m3fn), b, 200)
    assert rows.shape == (3, 200) and torch.equal(rows.dequantize(torch.float64), mx.rounded(x, 8))


def test_containers_refuse_what_they_cannot_be():
    v, s = torch.zeros(2, 128, dtype=torch.float8_e4m3fn), torch.ones(2, 4, dtype=torch.uint8)
    ops.MXRows(v, s, 100)
    for bad in [(v.float(), s, 100), (v, s.int(), 100), (v, s, 129), (v, s[:, :3], 100), (v, s[:1], 100), (v, s, 0)]:
        with pytest.raises(AssertionError):
            ops.MXRows(*bad)
    v, s = torch.zeros(2, 1, 4, 16, 16, dtype=torch.uint8), torch.ones(2, 1, 4, 16, 4, dtype=torch.uint8)
    ops.MXWeight(v, s, (32, 128))
    ops.MXWeight(v, s, (20, 100), gated=True)
    for bad in [(v, s, (33, 128)), (v, s, (32, 129)), (v.int(), s, (32, 128)), (v, s, (0, 128)), (v, s, (21, 100), True),
                (v.transpose(2, 3).transpose(2, 3)[:, :, :, :, ::2], s, (32, 128))]:
        with pytest.raises(AssertionError):
            ops.MXWeight(*bad)


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 128)
    w = ops.MXWeight(torch.zeros(2, 1, 4, 16, 16, dtype=torch.uint8), torch.ones(2, 1, 4, 16, 4, dtype=torch.uint8), (32, 128))
    rows = ops.MXRows(torch.zeros(2, 128, dtype=torch.float8_e4m3fn), torch.ones(2, 4, dtype=torch.uint8), 128)
    for f in (lambda: ops.mx_quantize(x), lambda: ops.mx_weight(x), lambda: ops.mx_rms_norm(x, x[0]), lambda: ops.mx_linear(x, w),
              lambda: ops.mx_linear(rows, w)):
        with pytest.raises(RuntimeError, match='ROCm GPU'):
            f()


def test_entry_points_check_their_arguments():
    L = _lib.load()
    bad, no = _lib.VGDR_ERR_INVALID, _lib.VGDR_ERR_UNSUPPORTED

    def q(**o):
        a = dict(dt=1, x=4096, ld=128, v=8192, s=12288, rows=2, cols=128) | o
        return L.vgdr_mx_quantize(a['dt'], a['x'], a['ld'], a['v'], a['s'], a['rows'], a['cols'], None)
    assert q(dt=3) == q(dt=-1) == q(x=None) == q(v=None) == q(s=None) == q(v=8200) == q(rows=-1) == q(cols=0) == q(ld=127) == bad
    assert q(v=4096) == q(cols=(1 << 24) + 1, ld=1 << 25) == bad
    assert q(rows=1 << 40) == q(rows=1 << 28) == no                    # more threads than a launch has
    assert q(rows=0, x=None) == _lib.VGDR_OK

    def w(**o):
        a = dict(dt=1, w=4096, ld=128, v=8192, s=12288, rows=2, cols=128, gated=0) | o
        return L.vgdr_mx_weight(a['dt'], a['w'], a['ld'], a['v'], a['s'], a['rows'], a['cols'], a['gated'], None)
    assert w(dt=3) == w(w=None) == w(rows=0) == w(rows=3, gated=1) == w(gated=2) == w(s=12290) == w(rows=(1 << 24) + 1) == bad

    def n(**o):
        a = dict(dt=1, x=4096, r=None, xo=None, g=8192, y=None, v=12288, s=16384, rows=2, dim=128, eps=1e-6) | o
        return L.vgdr_mx_rms_norm(a['dt'], a['x'], a['r'], a['xo'], a['g'], a['y'], a['v'], a['s'], a['rows'], a['dim'], a['eps'], None)
    assert n(dim=4) == n(dim=132) == n(dim=16392) == n(dim=0) == no
    assert n(dt=3) == n(x=4100) == n(v=4096) == n(y=4096) == n(y=12288) == n(eps=-1.0) == n(eps=float('nan')) == n(rows=-1) == bad
    assert n(r=12288) == n(xo=12288) == n(g=None) == bad
    assert n(rows=1 << 24) == no

    def p(**o):
        a = dict(xd=1, x=4096, ld=128, xs=None, v=8192, s=12288, gated=0, od=1, y=16384, ys=None, ws=None, nb=0, rows=2, n=32, k=128) | o
        return L.vgdr_mx_linear(a['xd'], a['x'], a['ld'], a['xs'], a['v'], a['s'], a['gated'], a['od'], a['y'], a['ys'], a['ws'], a['nb'],
                                a['rows'], a['n'], a['k'], None)
    assert p(od=3) == no
    assert p(xd=4) == p(xd=-1) == p(od=4) == p(gated=2) == p(gated=1, n=31) == p(rows=-1) == p(n=0) == p(k=0) == bad
    assert p(k=1 << 25) == p(n=1 << 25) == p(ld=120) == p(ld=132) == p(x=4104) == p(v=None) == p(y=None) == p(y=4096) == bad
    assert p(xd=3) == p(gated=1, od=3) == bad                         # scales of 8-bit rows are missing
    assert p(xd=0, rows=33) == p(xd=2, rows=33) == p(k=100, rows=33) == bad        # the workspace is missing
    assert p(rows=1 << 30) == no
    assert p(xd=0, rows=40, ws=20480, nb=3 * 40 * 256 - 1) == bad and b'workspace' in L.vgdr_last_error()
    size = L.vgdr_mx_linear_workspace_size
    assert size(0, 40, 100) == 3 * 40 * 256 and size(2, 40, 128) == 2 * 40 * 256 and size(1, 33, 130) == 33 * 512
    assert size(1, 40, 128) == size(3, 40, 100) == size(0, 32, 100) == size(0, 0, 100) == 0
    assert p(rows=0, x=None) == _lib.VGDR_OK


# --- rounding, bit by bit --------------------------------------------------------


def same_rows(rows, x, what=''):
    q, b = mx.quantize(x, 8)
    got = rows.values.reshape(q.shape).double()
    assert torch.equal(rows.scales.reshape(b.shape), b), f'{what}: {int((rows.scales.reshape(b.shape) != b).sum())} scales differ'
    nan = torch.isnan(q)
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], q[~nan]), f'{what}: values differ'


@gpu
@pytest.mark.parametrize('dt', [BF, FH, FS])
@pytest.mark.parametrize('R, K', [(1, 1), (3, 31), (5, 32), (2, 128), (7, 200), (33, 1000), (4, 2049), (300, 256)])
def test_rows_to_8_bits(R, K, dt):
    case('mx_quantize', R, K, dt)
    x = (randn(R, K, seed=R + K) * 10 ** (6 * randn(R, 1, seed=K)).clamp(-4, 4)).to(dt)
    same_rows(ops.mx_quantize(x), x)


@gpu
def test_rows_to_8_bits_of_ends_and_odd_layouts():
    case('mx_quantize: zeros, infinities, NaN, the smallest and largest numbers, ties, strides')
    x = randn(12, 128, seed=5)
    x[0] = 0
    x[1, 5], x[1, 40], x[1, 70] = float('inf'), float('-inf'), float('nan')
    x[2] *= 1e-42
    x[3] *= 1e38
    x[3, 3] = torch.finfo(FS).max
    x[4] = 464.0
    x[5] = torch.nextafter(torch.tensor(464.0), torch.tensor(1e9)).item()
    x[6] = torch.arange(128, device=DEV) * 3.5 + 0.25
    x[7] = -0.0
    x[8, :32] = torch.finfo(FS).tiny * 2 ** torch.arange(32, device=DEV)
    x[9, ::2] = 0
    same_rows(ops.mx_quantize(x), x, 'ends')
    same_rows(ops.mx_quantize(x[:, 3:100]), x[:, 3:100], 'misaligned columns')
    same_rows(ops.mx_quantize(x.t()), x.t(), 'transposed')
    same_rows(ops.mx_quantize(x[::2]), x[::2], 'every other row')
    same_rows(ops.mx_quantize(x[:1].expand(5, 128)), x[:1].expand(5, 128), 'one row, broadcast')
    got = ops.mx_quantize(x.view(3, 4, 128))
    assert got.shape == (3, 4, 128)
    same_rows(got, x)
    assert ops.mx_quantize(x[:0]).shape == (0, 128)


@gpu
@pytest.mark.parametrize('dt', [BF, FH, FS])
@pytest.mark.parametrize('n, k, gated', [(1, 1, False), (16, 128, False), (5, 40, False), (33, 700, False), (100, 512, False),
                                         (2, 8, True), (34, 130, True), (96, 1000, True)])
def test_weights_to_4_bits(n, k, gated, dt):
    case('mx_weight', n, k, gated, dt)
    w = (randn(n, k, seed=n + k) * 10 ** randn(n, 1, seed=k)).to(dt)
    w[0, 0] = 0
    got = ops.mx_weight(w, gated)
    values, scales = layout(w.cpu().float(), gated)
    assert torch.equal(got.scales.cpu(), scales)
    assert torch.equal(got.values.cpu(), values)
    assert torch.equal(got.dequantize(torch.float64), mx.rounded(w, 4))
    wide = torch.zeros(n, k + 3, dtype=dt, device=DEV)
    wide[:, 1:k + 1] = w
    assert torch.equal(ops.mx_weight(wide[:, 1:k + 1], gated).values, got.values)


@gpu
def test_a_weight_block_that_is_not_finite_is_nan():
    case('mx_weight: NaN')
    w = randn(20, 200, seed=6)
    w[3, 40], w[7, 199] = float('nan'), float('inf')
    got = ops.mx_weight(w).dequantize()
    bad = torch.zeros(20, 200, dtype=torch.bool, device=DEV)
    bad[3, 32:64] = bad[7, 192:] = True
    assert torch.equal(torch.isnan(got), bad)
    x = randn(3, 200, seed=7)
    for rows in (x, x.bfloat16(), ops.mx_quantize(x), randn(70, 200, seed=8).bfloat16(), ops.mx_quantize(randn(70, 200, seed=8))):
        y = ops.mx_linear(rows, ops.mx_weight(w))
        assert bool(torch.isnan(y[:, [3, 7]]).all()) and int(torch.isnan(y).sum()) == 2 * y.shape[0]


@gpu
@pytest.mark.parametrize('dt', [BF, FH, FS])
@pytest.mark.parametrize('R, D, residual', [(1, 8, True), (3, 128, False), (2, 200, True), (9, 2048, True), (1, 2048, False), (5, 2056, True),
                                            (2, 4104, True), (3, 16384, True)])
def test_norm_to_8_bits(R, D, residual, dt):
    case('mx_rms_norm', R, D, residual, dt)
    x, gamma = randn(R, D, seed=R + D).to(dt), (1 + 0.1 * randn(D, seed=9)).to(dt)
    res = randn(R, D, seed=10).to(dt) if residual else None
    h = x if res is None else (x.double() + res.double()).to(dt)
    got = ops.mx_rms_norm(x, gamma, 1e-6, residual=res, norm_out=True)
    same_rows(got[0], mx.rms_norm(h, gamma, float(torch.tensor(1e-6))))
    if residual:
        assert torch.equal(got[2], h)
    # the norm in x's type: rms_norm's, whose root is fp32: one unit of the type, two with its two roundings
    want = mx.rms_norm(h, gamma, 1e-6)
    tol = 2.02 * torch.finfo(dt).eps
    assert bool(((got[1].double() - want).abs() <= tol * want.abs() + 1e-6 * torch.finfo(dt).tiny).all())


@gpu
def test_norm_to_8_bits_in_place_and_of_odd_rows():
    case('mx_rms_norm: the stream updated in place; zero rows, NaN rows, views')
    x, res, gamma = randn(6, 256, seed=11).bfloat16(), randn(6, 256, seed=12).bfloat16(), randn(256, seed=13).bfloat16()
    x[1], res[1] = 0, 0
    x[2, 7] = float('nan')
    x[3, 200] = float('inf')
    h = (x.float() + res.float()).bfloat16()
    stream = x.clone()
    rows, got = ops.mx_rms_norm(stream, gamma, 1e-6, residual=res, out_residual=stream)
    assert got is stream and torch.equal(stream.view(torch.int16)[[0, 1, 4, 5]], h.view(torch.int16)[[0, 1, 4, 5]])
    live = [0, 1, 4, 5]
    same_rows(ops.MXRows(rows.values[live], rows.scales[live], 256), mx.rms_norm(h[live], gamma, float(torch.tensor(1e-6))))
    assert bool((rows.scales[2] == 255).all())
    # an infinity makes the mean infinite: inf / inf is NaN, everything else is zero
    assert rows.scales[3].tolist() == [1, 1, 1, 1, 1, 1, 255, 1]
    wide = torch.randn(6, 512, device=DEV).bfloat16()
    assert torch.equal(ops.mx_rms_norm(wide[:, 3:259], gamma).values.view(torch.uint8),
                       ops.mx_rms_norm(wide[:, 3:259].contiguous(), gamma).values.view(torch.uint8))
    assert ops.mx_rms_norm(x[:0], gamma).shape == (0, 256)


# --- products ---------------------------------------------------------------------


def rows_of(kind, R, K, seed):
    x = randn(R, K, seed=seed)
    x[:, ::37] *= 8
    if kind == 'mx8':
        rows = ops.mx_quantize(x)
        return rows, rows.dequantize(torch.float64)
    x = x.to({'bf16': BF, 'fp16': FH, 'fp32': FS}[kind])
    return x, x.double()


def product_error(kind, x, w):
    """How far a product's fp32 sums may be from x w^T."""
    A = x.abs() @ w.abs().t()
    K = x.shape[1]
    if kind == 'mx8':
        return A * 2 ** -12
    return A * 2 * ((3 if kind == 'fp32' else 2 if kind == 'fp16' else 1) * K + 64) * 2 ** -24


def within(got, want, err, dt):
    tol = err + torch.finfo(dt).eps / 2 * (want.abs() + err) + torch.finfo(dt).tiny
    off = (got.double() - want).abs() / tol
    assert bool((off <= 1).all()), f'{float(off.max()):.3g} of the tolerance'
    return float(off.max())


SHAPES = [(1, 128, 16), (1, 2048, 512), (1, 1001, 40), (2, 1, 1), (1, 3, 4200), (20, 333, 4100), (32, 700, 8200), (3, 40, 17), (5, 1000, 100), (15, 130, 33), (16, 512, 64), (17, 640, 48),
          (33, 1024, 130), (64, 256, 100), (65, 128, 16), (130, 384, 257), (300, 1000, 70)]


@gpu
@pytest.mark.parametrize('kind', ['bf16', 'fp16', 'fp32', 'mx8'])
@pytest.mark.parametrize('R, K, N', SHAPES)
def test_linear(R, K, N, kind):
    case('mx_linear', R, K, N, kind)
    x, xd = rows_of(kind, R, K, R + K)
    w = ops.mx_weight(randn(N, K, seed=N) * 0.02)
    wd = w.dequantize(torch.float64)
    want = xd @ wd.t()
    for dt in {None, FS}:
        y = ops.mx_linear(x, w, out_dtype=dt)
        assert y.shape == (R, N) and y.dtype == (dt or {'bf16': BF, 'fp16': FH, 'fp32': FS, 'mx8': BF}[kind])
        within(y, want, product_error(kind, xd, wd), y.dtype)


@gpu
@pytest.mark.parametrize('kind', ['bf16', 'fp32', 'mx8'])
def test_linear_of_many_rows(kind):
    case('mx_linear: enough rows and columns for the largest tiles', kind)
    R, K, N = 4099, 256, 4101
    x, xd = rows_of(kind, R, K, 1)
    w = ops.mx_weight(randn(N, K, seed=2) * 0.02)
    wd = w.dequantize(torch.float64)
    y = ops.mx_linear(x, w)
    within(y, xd @ wd.t(), product_error(kind, xd, wd), y.dtype)


def gated_bounds(kind, xd, wd):
    h = wd.shape[0] // 2
    a, b = xd @ wd[:h].t(), xd @ wd[h:].t()
    e = product_error(kind, xd, wd)
    ea, eb = e[:, :h], e[:, h:]
    want = a * torch.sigmoid(a) * b
    return want, 1.1 * ea * b.abs() + a.abs() * eb + 1.1 * ea * eb + want.abs() * (a.abs() * 2 ** -22 + 2 ** -20)


@gpu
@pytest.mark.parametrize('kind', ['bf16', 'fp16', 'fp32', 'mx8'])
@pytest.mark.parametrize('R, K, h', [(1, 128, 16), (1, 2048, 176), (2, 8, 1), (7, 200, 40), (16, 1024, 96), (40, 256, 33), (64, 512, 64),
                                     (70, 128, 130), (257, 640, 100)])
def test_swiglu(R, K, h, kind):
    case('mx_swiglu', R, K, h, kind)
    x, xd = rows_of(kind, R, K, R + K)
    w = ops.mx_weight(randn(2 * h, K, seed=h) * 0.05, gated=True)
    want, err = gated_bounds(kind, xd, w.dequantize(torch.float64))
    y = ops.mx_swiglu(x, w)
    assert y.shape == (R, h)
    within(y, want, err, y.dtype)
    within(ops.mx_swiglu(x, w, out_dtype=FS), want, err, FS)
    rows_within(ops.mx_swiglu(x, w, quantize=True), want, err)


def rows_within(rows, want, err):
    """8-bit rows against the numbers that they round: half a step of the block's scale or of the value; a block's scale
    from its largest element, which may itself be off."""
    assert rows.shape == want.shape
    s = mx.scales(rows.scales).repeat_interleave(32, -1)[:, :want.shape[1]]
    q, b = mx.quantize(want, 8)
    near = (rows.scales.long() - b.long()).abs()
    assert bool((near <= 1).all()) and float((near > 0).double().mean()) < 0.02
    tol = err + (want.abs() + err) * 2 ** -4 + s * 2 ** -10
    assert bool(((rows.dequantize(torch.float64) - want).abs() <= tol).all())
    C = rows.values.shape[-1]
    assert bool((rows.values.float()[:, want.shape[1]:] == 0).all()) and bool((rows.scales[:, -(-want.shape[1] // 32):] == 1).all())


@gpu
@pytest.mark.parametrize('kind', ['bf16', 'mx8'])
def test_swiglu_of_many_rows(kind):
    case('mx_swiglu: enough rows and columns for the largest tiles', kind)
    R, K, h = 4099, 256, 2060
    x, xd = rows_of(kind, R, K, 3)
    w = ops.mx_weight(randn(2 * h, K, seed=4) * 0.05, gated=True)
    want, err = gated_bounds(kind, xd, w.dequantize(torch.float64))
    y = ops.mx_swiglu(x, w)
    within(y, want, err, y.dtype)
    rows_within(ops.mx_swiglu(x, w, quantize=True), want, err)


@gpu
@pytest.mark.parametrize('R', [3, 100])
def test_products_of_odd_layouts(R):
    case('mx_linear: strides, offsets, leading dims, no rows', R)
    K, N = 256, 48
    w = ops.mx_weight(randn(N, K, seed=5))
    for dt in (BF, FS):
        base = randn(R, 2 * K + 8, seed=6).to(dt)
        for x in (base[:, :K], base[:, 8:K + 8], base[:, 3:K + 3], base[:, 1:2 * K:2], base[:1, :K].expand(R, K)):
            assert torch.equal(ops.mx_linear(x, w), ops.mx_linear(x.contiguous(), w))
        x = base[:, :K].reshape(R, 1, K)
        assert ops.mx_linear(x, w).shape == (R, 1, N) and torch.equal(ops.mx_linear(x, w)[:, 0], ops.mx_linear(base[:, :K], w))
        assert torch.equal(ops.mx_linear(base[0, :K], w), ops.mx_linear(base[:1, :K], w)[0])
        assert ops.mx_linear(base[:0, :K], w).shape == (0, N)
    rows = ops.mx_quantize(base[:, :K])
    cut = ops.MXRows(rows.values[1:], rows.scales[1:], K)
    assert torch.equal(ops.mx_linear(cut, w), ops.mx_linear(rows, w)[1:])
    assert ops.mx_linear(ops.MXRows(rows.values[:0], rows.scales[:0], K), w).shape == (0, N)
    odd = ops.MXRows(rows.values.view(R, 256).t().contiguous().t(), rows.scales, K)
    assert torch.equal(ops.mx_linear(odd, w), ops.mx_linear(rows, w))


@gpu
@pytest.mark.parametrize('R', [2, 100])
def test_products_of_infinities_stay_in_their_rows(R):
    case('mx_linear: infinities and NaN', R)
    w = ops.mx_weight(randn(32, 256, seed=7).abs() + 1)
    wd = w.dequantize(torch.float64)
    for dt in (BF, FH, FS):
        x = randn(R, 256, seed=8).to(dt)
        clean = ops.mx_linear(x, w)
        x[1, 5] = float('inf')
        y = ops.mx_linear(x, w)
        hit = wd[:, 5] > 0
        assert bool((y[1][hit] == float('inf')).all())
        assert torch.equal(y[0], clean[0]) and (R < 3 or torch.equal(y[2:], clean[2:]))
        x[1, 5] = float('nan')
        y = ops.mx_linear(x, w)
        assert bool(torch.isnan(y[1]).all()) and torch.equal(y[0], clean[0])
    x = randn(R, 256, seed=8)
    clean = ops.mx_linear(ops.mx_quantize(x), w)
    x[1, 5] = float('inf')
    y = ops.mx_linear(ops.mx_quantize(x), w)
    assert bool(torch.isnan(y[1]).all()) and torch.equal(y[0], clean[0])


@gpu
@pytest.mark.parametrize('R', [2, 100])
def test_a_gated_block_that_is_not_finite(R):
    case('mx_swiglu: an infinity in one row', R)
    w = ops.mx_weight(randn(2 * 96, 256, seed=15), gated=True)
    for rows in (randn(R, 256, seed=16).bfloat16(), randn(R, 256, seed=16)):
        clean = ops.mx_swiglu(rows, w, quantize=True)
        rows[1, 7] = float('inf')
        got = ops.mx_swiglu(rows, w, quantize=True)
        y = ops.mx_swiglu(rows, w)
        assert not bool(torch.isfinite(y[1]).all()) and bool(torch.isfinite(y[0]).all())
        bad = ~torch.isfinite(y.float()).view(R, 3, 32).all(-1)
        assert torch.equal(got.scales[:, :3] == 255, bad) and torch.equal(got.scales[0], clean.scales[0])
        assert torch.equal(torch.isnan(got.dequantize()).view(R, 3, 32).all(-1), bad)
        assert torch.equal(got.values.view(torch.uint8)[0], clean.values.view(torch.uint8)[0])


@gpu
def test_the_largest_numbers():
    case('mx_linear: fp32 rows at the ends of their range, fp16 rows of subnormals')
    w = ops.mx_weight(torch.eye(128, device=DEV))
    x = torch.full((2, 128), torch.finfo(FS).max, device=DEV)
    x[1] = -torch.finfo(FS).max
    assert torch.equal(ops.mx_linear(x, w), x)
    x = (torch.arange(256, device=DEV).reshape(2, 128) * 2.0 ** -24).half()
    assert torch.equal(ops.mx_linear(x, w), x)


@gpu
def test_a_run_of_them_in_a_graph_and_on_a_stream():
    case('norm, gated product, product, recorded and replayed, beside the same on another stream')
    D, h = 256, 320
    w1, w2 = ops.mx_weight(randn(2 * h, D, seed=9) * 0.05, gated=True), ops.mx_weight(randn(D, h, seed=10) * 0.05)
    gamma = randn(D, seed=11).bfloat16()

    def block(x, delta):
        rows, s = ops.mx_rms_norm(x, gamma, residual=delta)
        return s, ops.mx_linear(ops.mx_swiglu(rows, w1, quantize=True), w2), ops.mx_linear(s.float(), w1_plain)
    w1_plain = ops.mx_weight(randn(40, D, seed=12))
    for R in (1, 70):
        x, d = randn(R, D, seed=13).bfloat16(), randn(R, D, seed=14).bfloat16()
        block(x, d)
        side = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = block(x, d)
        for k in range(3):
            x.copy_(randn(R, D, seed=20 + k).bfloat16())
            want = block(x, d)
            graph.replay()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                there = block(x, d)
            torch.cuda.current_stream().wait_stream(side)
            for a, b, c in zip(out, want, there):
                assert torch.equal(a, b) and torch.equal(a, c)


@gpu
def test_calls_that_are_refused():
    w, wg = ops.mx_weight(randn(32, 128)), ops.mx_weight(randn(32, 128), gated=True)
    x = randn(4, 128)
    for f in (lambda: ops.mx_linear(x, wg), lambda: ops.mx_swiglu(x, w), lambda: ops.mx_linear(x[:, :100], w), lambda: ops.mx_linear(x, x),
              lambda: ops.mx_weight(x[0]), lambda: ops.mx_weight(x[:3], gated=True), lambda: ops.mx_weight(x[:0]),
              lambda: ops.mx_rms_norm(x, x[0].half()), lambda: ops.mx_rms_norm(x, x[0], residual=x[:2]),
              lambda: ops.mx_rms_norm(x, x[0], residual=x, out_residual=x.half()), lambda: ops.mx_rms_norm(x, x[0], out_residual=x.clone())):
        with pytest.raises(AssertionError):
            f()
    for f in (lambda: ops.mx_quantize(x.double()), lambda: ops.mx_linear(x.double(), w), lambda: ops.mx_linear(x, w, out_dtype=torch.float64),
              lambda: ops.mx_rms_norm(x[:, :12], x[0, :12]), lambda: ops.mx_linear(x.clone().requires_grad_(), w),
              lambda: ops.mx_quantize(x.clone().requires_grad_()), lambda: ops.mx_rms_norm(x, x[0].clone().requires_grad_())):
        with pytest.raises(NotImplementedError):
            f()
    with pytest.raises(RuntimeError):
        ops.mx_linear(x.cpu(), w)
    with torch.no_grad():
        ops.mx_linear(x.clone().requires_grad_(), w)

"""The operators that serve a model with block-scaled numbers, measured: 4-bit weights, and
rows in 8 bits, each block of 32 elements with a scale that is a power of two.

    quantize  ops.mx_quantize: rows to 8 bits
    norm      ops.mx_rms_norm: the residual's addition, the RMSNorm and its output in 8 bits
    linear    ops.mx_linear: products with 4-bit weights, of 16-bit, fp32 or 8-bit rows
    swiglu    ops.mx_swiglu: the FFN's two input projections, the activation and the
              product, as 16-bit or 8-bit rows

Where ``own`` is false ``run`` computes them in elementary torch operations.  ``exact``
computes the same in 64 bits; its values of 8-bit outputs are those before their rounding.
"""
from __future__ import annotations

import math

import torch

own = False

DT = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
SIZE = {'bf16': 2, 'fp16': 2, 'fp32': 4}


def listed():
    return [
        # one stream of a 1.3B model: the residual's addition and the norm before a block's projections
        dict(name='norm_one', kind='norm', R=1, D=2048, dtype='bf16', residual=True),
        # the same over its 64 packed prompts
        dict(name='norm_prompts', kind='norm', R=65536, D=2048, dtype='bf16', residual=True),
        # the output epilogue's rows of 64 streams, before W_o
        dict(name='quantize_b64', kind='quantize', R=64, K=2048, dtype='bf16'),
        # the same over the prompts
        dict(name='quantize_prompts', kind='quantize', R=65536, K=2048, dtype='bf16'),
        # one stream's q, k, v and output gate projections: latency
        dict(name='linear_one', kind='linear', R=1, K=2048, N=8192, x='bf16'),
        # 64 streams through the FFN's second product
        dict(name='linear_b64', kind='linear', R=64, K=5632, N=2048, x='bf16'),
        # a toy model's odd sizes in fp32
        dict(name='linear_odd_fp32', kind='linear', R=7, K=1000, N=1337, x='fp32'),
        # the projections over the packed prompts, rows in 8 bits
        dict(name='linear_prompts', kind='linear', R=65536, K=2048, N=8192, x='mx8'),
        # W_o over a few prompts, rows in 16 bits
        dict(name='linear_prompts_bf16', kind='linear', R=8192, K=2048, N=2048, x='bf16'),
        # one stream through the FFN's first half
        dict(name='swiglu_one', kind='swiglu', R=1, K=2048, h=5632, x='bf16', out='bf16'),
        # 64 streams
        dict(name='swiglu_b64', kind='swiglu', R=64, K=2048, h=5632, x='bf16', out='bf16'),
        # the prompts, from 8-bit rows to 8-bit rows
        dict(name='swiglu_prompts', kind='swiglu', R=32768, K=2048, h=5632, x='mx8', out='mx8'),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(['norm', 'quantize', 'linear', 'linear', 'linear', 'swiglu', 'swiglu'])
    R = _log(rng, 1, 65536)
    width = lambda lo, hi: _log(rng, lo, hi) if rng.random() < 0.3 else 128 * _log(rng, max(1, lo // 128), hi // 128)  # noqa: E731
    if kind == 'norm':
        D = 8 * _log(rng, 4, 1024)
        return dict(kind=kind, R=max(1, min(R, (1 << 27) // D)), D=D, dtype=rng.choice(['bf16', 'bf16', 'fp16', 'fp32']),
                    residual=rng.random() < 0.7)
    if kind == 'quantize':
        K = width(32, 8192)
        return dict(kind=kind, R=max(1, min(R, (1 << 27) // K)), K=K, dtype=rng.choice(['bf16', 'bf16', 'fp16', 'fp32']))
    K = width(64, 8192)
    x = rng.choice(['bf16', 'bf16', 'mx8', 'mx8', 'fp16', 'fp32'])
    if kind == 'linear':
        N = width(16, 32768)
        return dict(kind=kind, R=max(1, min(R, (1 << 40) // (K * N), (1 << 29) // N)), K=K, N=N, x=x)
    h = width(16, 16384)
    return dict(kind=kind, R=max(1, min(R, (1 << 38) // (K * h), (1 << 28) // h)), K=K, h=h, x=x,
                out=rng.choice(['bf16', 'mx8']) if x == 'mx8' else x)


# --- inputs ------------------------------------------------------------------


def _blocks(v, top):
    """v (R, K) as blocks (R, K / 32, 32) padded with zeros to whole 128s of columns, and the
    blocks' exponents: the smallest s >= -126 with amax <= top 2^s."""
    v = torch.nn.functional.pad(v, (0, -v.shape[1] % 128)).unflatten(1, (-1, 32))
    amax = v.abs().amax(-1)
    m, e = torch.frexp(amax)                                     # amax = m 2^e, m in [1/2, 1)
    tm, te = math.frexp(top)
    s = torch.where(amax > 0, e - te + (m > tm).to(e.dtype), torch.full_like(e, -126)).clamp(min=-126)
    return v, s


def _two(s):
    """2^s as fp32, s in -126 .. 127, by its bits: a power function may be off."""
    return ((s.int() + 127) << 23).view(torch.float32)


def _pack4(w, gated):
    """w (n, K) as 4-bit weights the way ops.MXWeight holds them: codes, two a byte, in tiles of
    16 rows x 128 columns (block of 32, row, 16 bytes), and the blocks' biased exponents in tiles of 16 rows x
    512 columns (block of 32 mod 4, row, tile of 128).  gated: the halves' tiles by turns."""
    if gated:
        h = w.shape[0] // 2
        w = torch.nn.functional.pad(w.unflatten(0, (2, h)), (0, 0, 0, -h % 16)).unflatten(1, (-1, 16)).transpose(0, 1).flatten(0, 2)
    w = torch.nn.functional.pad(w, (0, 0, 0, -w.shape[0] % 16))
    v, s = _blocks(w, 7.0)
    a = v.abs() * _two(-s)[..., None]
    code = ((a > .25).byte() + (a >= .75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte()
            + (a >= 3.5).byte() + (a > 5).byte()) | (v < 0).byte() << 3
    byte = code[..., 0::2] | code[..., 1::2] << 4                # (n, K / 32, 16)
    n, C = byte.shape[0], byte.shape[1] // 4
    values = byte.view(n // 16, 16, C, 4, 16).permute(0, 2, 3, 1, 4).contiguous()
    s = torch.nn.functional.pad((s + 127).byte().view(n, C, 4), (0, 0, 0, -C % 4), value=1)
    scales = s.view(n // 16, 16, -1, 4, 4).permute(0, 2, 4, 1, 3).contiguous()
    return values, scales


def _rows8(v):
    """v as 8-bit rows: e4m3 values, biased exponents."""
    b, s = _blocks(v, 464.0)
    q = (b * _two(-s)[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return q.flatten(1), (s + 127).byte()


def prepare(case, seed):
    """Rows of unit variance, a few of whose columns are ten times as large, as a norm's
    outputs are; weights of standard deviation 0.02, 4-bit once and for all."""
    c = case
    gen = torch.Generator('cuda').manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=gen, device='cuda')

    R, K = c['R'], c.get('D') or c['K']
    x = randn(R, K)
    x *= torch.where(torch.rand(K, generator=gen, device='cuda') < 0.01, 10.0, 1.0)
    s = dict(case=dict(c))
    if c['kind'] in ('norm', 'quantize'):
        dt = DT[c['dtype']]
        s['x'] = x.to(dt)
        if c['kind'] == 'norm':
            s['gamma'] = (1 + 0.1 * randn(K)).to(dt)
            s['residual'] = randn(R, K).to(dt) if c['residual'] else None
        return s
    if c['x'] == 'mx8':
        s['values'], s['scales'] = _rows8(x)
    else:
        s['x'] = x.to(DT[c['x']])
    s['w_values'], s['w_scales'] = _pack4(0.02 * randn(c['N'] if c['kind'] == 'linear' else 2 * c['h'], K), c['kind'] == 'swiglu')
    return s


# --- one pass ----------------------------------------------------------------


def _own(s):
    from vagus_amd import ops
    c = s['case']
    if c['kind'] == 'quantize':
        return _out8(ops.mx_quantize(s['x']))
    if c['kind'] == 'norm':
        r = ops.mx_rms_norm(s['x'], s['gamma'], 1e-6, residual=s['residual'])
        return _out8(r) if s['residual'] is None else dict(_out8(r[0]), h=r[1])
    x = s['x'] if c['x'] != 'mx8' else ops.MXRows(s['values'], s['scales'], c['K'])
    if c['kind'] == 'linear':
        return ops.mx_linear(x, ops.MXWeight(s['w_values'], s['w_scales'], (c['N'], c['K'])))
    y = ops.mx_swiglu(x, ops.MXWeight(s['w_values'], s['w_scales'], (2 * c['h'], c['K']), gated=True), quantize=c['out'] == 'mx8')
    return _out8(y) if c['out'] == 'mx8' else y


def _out8(rows):
    return dict(values=rows.values, scales=rows.scales.view(torch.float8_e8m0fnu))


def _out8_plain(v):
    q, s = _rows8(v)
    return dict(values=q, scales=s.view(torch.float8_e8m0fnu))


def _weights(values, scales, n, K):
    """fp32 (n, K), the rows in the tiles' order."""
    T, C = values.shape[:2]
    size = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], device=values.device)
    code = torch.stack([values & 15, values >> 4], -1).flatten(-2)               # (T, C, 4, 16, 32)
    e = scales.permute(0, 1, 4, 2, 3).reshape(T, -1, 4, 16)[:, :C]               # (T, C, 4, 16)
    w = size[code.int()] * _two(e.int() - 127)[..., None]
    return w.permute(0, 3, 1, 2, 4).reshape(16 * T, 128 * C)[:n, :K]


def _plain(s):
    c = s['case']
    if c['kind'] == 'quantize':
        return _out8_plain(s['x'].float())
    if c['kind'] == 'norm':
        h = s['x'] if s['residual'] is None else (s['x'].float() + s['residual'].float()).to(s['x'].dtype)
        f = h.float()
        y = _out8_plain(f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6) * s['gamma'].float())
        return y if s['residual'] is None else dict(y, h=h)
    K = c['K']
    if c['x'] == 'mx8':
        x = (s['values'].float().unflatten(1, (-1, 32)) * _two(s['scales'].int() - 127)[..., None]).flatten(1)[:, :K]
    else:
        x = s['x'].float()
    dt = DT['bf16' if c['x'] == 'mx8' else c['x']]
    if c['kind'] == 'linear':
        return (x @ _weights(s['w_values'], s['w_scales'], c['N'], K).t()).to(dt)
    h, T = c['h'], s['w_values'].shape[0]
    y = (x @ _weights(s['w_values'], s['w_scales'], 16 * T, K).t()).view(-1, T // 2, 2, 16)
    a, b = y[:, :, 0].flatten(1)[:, :h], y[:, :, 1].flatten(1)[:, :h]
    y = a / (1 + torch.exp(-a)) * b
    return _out8_plain(y) if c['out'] == 'mx8' else y.to(dt)


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    c = case
    R, K = c['R'], c.get('D') or c['K']
    eight = lambda n: R * (n + n / 32)  # noqa: E731
    if c['kind'] in ('norm', 'quantize'):
        e = SIZE[c['dtype']]
        return dict(bytes=R * K * e * (3 if c.get('residual') else 1) + eight(K), flops=6.0 * R * K)
    n, cols = (c['N'], c['N']) if c['kind'] == 'linear' else (2 * c['h'], c['h'])
    x = eight(K) if c['x'] == 'mx8' else R * K * SIZE[c['x']]
    y = eight(cols) if c.get('out') == 'mx8' else R * cols * SIZE.get(c['x'], 2)
    return dict(bytes=n * K * (1 / 2 + 1 / 32) + x + y, flops=2.0 * R * n * K)


# --- the same from the definitions, in 64 bits --------------------------------


def exact(case, seed):
    c, s = case, prepare(case, seed)
    dev = s['x'].device if 'x' in s else s['values'].device

    def power(k):
        return torch.bitwise_left_shift(k.long() + 1023, 52).view(torch.float64)

    def eight(y):
        """Values over their blocks' scales, and the scales, by comparing with the powers themselves."""
        R, K = y.shape
        y = torch.cat([y, y.new_zeros(R, (K + 127) // 128 * 128 - K)], 1).view(R, -1, 32)
        amax = y.abs().max(-1).values
        k = torch.floor(torch.log2(amax / 464.0)).clamp(-126, 127).long()
        k = torch.where(464.0 * power(k) < amax, k + 1, k)
        k = torch.where((464.0 * power(k - 1) >= amax) & (k > -126), k - 1, k)
        scale = power(k)
        return dict(values=(y / scale[..., None]).clamp(-448, 448).flatten(1), scales=scale)

    if c['kind'] == 'quantize':
        return eight(s['x'].double())
    if c['kind'] == 'norm':
        h = s['x'] if s['residual'] is None else (s['x'].double() + s['residual'].double()).to(s['x'].dtype)
        d = h.double()
        out = eight(d / torch.sqrt((d * d).sum(-1, keepdim=True) / c['D'] + 1e-6) * s['gamma'].double())
        return out if s['residual'] is None else dict(out, h=h)
    K, gated = c['K'], c['kind'] == 'swiglu'
    n = 2 * c['h'] if gated else c['N']

    # every weight found by its own place in the tiles
    row, col = torch.arange(n, device=dev)[:, None], torch.arange(K, device=dev)[None]
    tile = row // 16
    r = row % 16
    if gated:
        r = row % c['h'] % 16
        tile = 2 * (row % c['h'] // 16) + row // c['h']
    w = torch.empty(n, K, dtype=torch.float64, device=dev)
    T, C = s['w_values'].shape[:2]
    for a in range(0, n, 4096):                                   # a few rows at a time: the indexes are long
        t, q = tile[a:a + 4096], r[a:a + 4096]
        byte = s['w_values'].flatten()[(((t * C + col // 128) * 4 + col // 32 % 4) * 16 + q) * 16 + col % 32 // 2]
        code = (byte >> (4 * (col % 2)).byte()) & 15
        mag, sign = (code & 7).double(), 1 - 2 * (code >> 3).double()
        v = torch.where(mag < 2, mag / 2, (2 + mag % 2) * power(mag.long() // 2 - 2))
        e = s['w_scales'].flatten()[(((t * ((C + 3) // 4) + col // 512) * 4 + col // 32 % 4) * 16 + q) * 4 + col // 128 % 4]
        w[a:a + 4096] = sign * v * power(e.long() - 127)
    if c['x'] == 'mx8':
        x = s['values'].double()[:, :K] * power(s['scales'].long() - 127).repeat_interleave(32, 1)[:, :K]
    else:
        x = s['x'].double()
    if not gated:
        return x @ w.t()
    a, b = x @ w[:c['h']].t(), x @ w[c['h']:].t()
    y = a * torch.sigmoid(a) * b
    return eight(y) if c['out'] == 'mx8' else y

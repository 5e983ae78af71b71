"""The layer, the model and the generator with 4-bit weights (quantize_weights_), against the same modules
whose nn.Linear weights are the numbers that the 4-bit weights stand for (exact in bf16, fp16 and fp32).

fp32: the same sums in other orders, 1e-5 a product, 1e-4 through the model.  bf16 and fp16: each differs from the exact
value by the roundings of its own chain, the parity bar of 2e-2.

Prompts in 8 bits: the modules' inputs are rounded by the oracle, so both sides round at the same places, but rows
that differ at all (the module rounds a norm to bf16 first, the kernel does not; every later row carries what came
before) may fall to different sides of a tie.  A difference e ahead of a rounding of step s crosses a tie for a share
e / s of the elements, which then move by s: sqrt(e s) behind it, more than e as long as e < s.  So the differences
grow to those of independent roundings, and that is the bound: an element's error is even within half a
step, at most 2^-4 of it, 2^-4 / sqrt(3) = 3.6e-2 rms; two roundings 5.1e-2; a product of many terms keeps its rows'
relative error.  A block rounds four rows one behind the other (the mixer's input, its epilogue, the FFN's input, its
activations, a product of two projections: the third counts twice in amplitude): two blocks, 5.1e-2 sqrt(2 (1 + 1 + 4 + 1))
= 0.19.  What is fed where is therefore checked call by call as well (the operators by themselves: tests/test_mx.py).
"""
import copy

import pytest
import torch
from torch import nn

from oracle import mx
from vagus_amd import ops
from vagus_amd.layer import GatedDeltaNet, MXLinear
from vagus_amd.model import FFN, GDNLM, RaggedGenerator, _ffn

DEV = 'cuda'
gpu = pytest.mark.gpu
BAR = {torch.float32: 1e-4, torch.bfloat16: 2e-2, torch.float16: 2e-2}


def case(*what):
    print('\n[case]', *what, flush=True)


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def model(dtype, gate='scalar', **kw):
    torch.manual_seed(0)
    with torch.device(DEV):
        m = GDNLM(vocab_size=300, dim=256, layer_count=2, head_count=2, key_head_dim=64, value_head_dim=128, gate=gate,
                  la_fused=dtype != torch.float32, **kw)
    return m.to(dtype).eval()


def round_(linear):
    """The weights that 4 bits leave of linear, in place."""
    with torch.no_grad():
        linear.weight.copy_(mx.rounded(linear.weight.double(), 4))


def pair(dtype, head=True, **kw):
    """(the 4-bit model, the same with modules)."""
    m = model(dtype, **kw)
    if head:
        m.head.weight = nn.Parameter(m.head.weight.detach().clone())       # the embedding keeps its own
    want = copy.deepcopy(m)
    for blk in want.blocks:
        for lin in (blk.att.wq, blk.att.wk, blk.att.wv, blk.att.wg, blk.att.wo, blk.ffn.l1, blk.ffn.l2):
            round_(lin)
    if head:
        round_(want.head)
    return m, want


def prompts(n=3, seed=1):
    g = torch.Generator().manual_seed(seed)
    lens = [5, 70, 1, 33, 64][:n]
    ids = torch.cat([torch.randint(0, 300, (k,), generator=g) for k in lens]).to(DEV)
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=DEV)
    return ids, cu, lens


# --- refusals, on the CPU -----------------------------------------------------------


def test_the_gpu_is_where_weights_become_4_bits():
    m = GDNLM(vocab_size=50, dim=64, layer_count=1, head_count=1, key_head_dim=64, value_head_dim=64, gate='scalar')
    with pytest.raises(RuntimeError, match='ROCm GPU'):
        m.quantize_weights_()
    with pytest.raises(AssertionError):
        m.quantize_weights_(prompt_bits=4)
    assert hasattr(m.blocks[0].att, 'wq') and isinstance(m.blocks[0].ffn.l1, nn.Linear) and not m._quantized()


def test_what_4_bit_projections_do_not_stand_for():
    layer = GatedDeltaNet(dim=64, head_count=1, key_head_dim=8, value_head_dim=64, gate='none')
    with pytest.raises(NotImplementedError, match='multiples of 16'):
        layer.quantize_weights_()
    layer = GatedDeltaNet(dim=64, head_count=1, key_head_dim=64, value_head_dim=64, gate='none')
    layer.wk.register_forward_hook(lambda *a: None)
    with pytest.raises(NotImplementedError, match='plain'):
        layer.quantize_weights_()
    ffn = FFN(64, 128)
    ffn.l2 = nn.Linear(128, 64, bias=True)
    with pytest.raises(NotImplementedError, match='plain'):
        ffn.quantize_weights_()
    m = GDNLM(vocab_size=50, dim=64, layer_count=1, head_count=1, key_head_dim=64, value_head_dim=64, gate='scalar')
    m.head = nn.Linear(64, 50, bias=True)
    with pytest.raises(NotImplementedError, match='head'):
        m.quantize_weights_()
    assert isinstance(m.blocks[0].ffn.l1, nn.Linear)
    m.blocks[0].ffn.l1.register_forward_pre_hook(lambda *a: None)         # nothing of the model, not a part of it
    with pytest.raises(NotImplementedError, match='plain'):
        m.quantize_weights_(head=False)
    assert hasattr(m.blocks[0].att, 'wq')


def test_another_module_in_the_place_of_an_ffn_runs():
    h = torch.randn(2, 3, 64)
    with torch.no_grad():
        assert torch.equal(_ffn(nn.Identity(), h), h)
    m = GDNLM(vocab_size=50, dim=64, layer_count=1, head_count=1, key_head_dim=64, value_head_dim=64, gate='scalar')
    m.blocks[0].ffn = nn.Identity()
    assert m._quantized() == []


# --- the layer ------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('gate, kw', [('scalar', {}), ('vector', {}), ('none', {}), ('scalar', dict(delta=False)),
                                      ('scalar', dict(short_conv_size=None)), ('vector', dict(value_head_dim=256)), ('scalar', dict(out_proj=False))])
def test_layer(gate, kw, dtype):
    case('a layer: forward, one-token steps, a longer step, drafts', gate, kw, dtype)
    torch.manual_seed(1)
    args = dict(dim=192, head_count=2, key_head_dim=64, value_head_dim=128, gate=gate, init_std=0.08) | kw
    with torch.device(DEV):
        layer = GatedDeltaNet(**args)
    layer = layer.to(dtype).eval()
    want = copy.deepcopy(layer)
    for n in ('wq', 'wk', 'wv', 'wg') + (('wo',) if layer.out_proj else ()):
        round_(getattr(want, n))
    layer.quantize_weights_()
    layer.quantize_weights_()                                         # again: nothing more to do
    assert not hasattr(layer, 'wq')
    x = torch.randn(3, 37, 192, device=DEV).to(dtype)
    bar = BAR[dtype]
    with torch.no_grad():
        assert rel(layer(x), want(x)) < bar
    for m in (layer, want):
        m.reset_cache(3)
    for a, b in ((0, 1), (1, 2), (2, 20), (20, 21)):
        assert rel(layer.decode_step(x[:, a:b]), want.decode_step(x[:, a:b])) < bar, (a, b)
    assert rel(layer.state, want.state) < bar
    for m in (layer, want):
        m.begin_drafts(4)
    none, some = torch.zeros(3, dtype=torch.int32, device=DEV), torch.tensor([0, 3, 4], dtype=torch.int32, device=DEV)
    assert rel(layer.draft_step(x[:, 21:25], none), want.draft_step(x[:, 21:25], none)) < bar
    assert rel(layer.draft_step(x[:, 25:29], some), want.draft_step(x[:, 25:29], some)) < bar


@gpu
def test_a_layer_whose_gates_are_called_as_modules():
    case('a hooked W_a, a subclass with its own _gates')

    class Mine(GatedDeltaNet):
        def _gates(self, x, **kw):
            g, beta = super()._gates(x, **kw)
            return 0.5 * g, beta
    for cls in (GatedDeltaNet, Mine):
        torch.manual_seed(2)
        with torch.device(DEV):
            layer = cls(dim=128, head_count=1, key_head_dim=64, value_head_dim=64, gate='scalar')
        seen = []
        if cls is GatedDeltaNet:
            layer.wa.register_forward_hook(lambda m, i, o: seen.append(1))
        want = copy.deepcopy(layer)
        for n in ('wq', 'wk', 'wv', 'wg', 'wo'):
            round_(getattr(want, n))
        layer.quantize_weights_()
        x = torch.randn(2, 1, 128, device=DEV)
        for m in (layer, want):
            m.reset_cache(2)
        for _ in range(2):
            assert rel(layer.decode_step(x), want.decode_step(x)) < 1e-4
        assert cls is Mine or len(seen) == 4 or len(seen) == 2


# --- the model ------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('gate', ['scalar', 'vector'])
@pytest.mark.parametrize('head', [True, False])
def test_model_of_16_bit_rows(dtype, gate, head):
    case('logits of prompts and of steps', dtype, gate, head)
    m, want = pair(dtype, head=head, gate=gate)
    assert m.quantize_weights_(prompt_bits=16, head=head) is m
    ids, cu, lens = prompts()
    for k in (m, want):
        k.reset_cache(3)
    assert rel(m.prefill_packed(ids, cu), want.prefill_packed(ids, cu)) < BAR[dtype]
    tok = torch.tensor([[3], [200], [7]], device=DEV)
    for _ in range(3):
        assert rel(m.decode_step(tok), want.decode_step(tok)) < BAR[dtype]
    with torch.no_grad():
        assert rel(m(tok.expand(3, 20)), want(tok.expand(3, 20))) < BAR[dtype]


@gpu
@pytest.mark.parametrize('gate', ['scalar', 'vector'])
def test_model_of_8_bit_prompts(gate):
    case('logits of prompts in 8 bits, and of steps from their states', gate)
    m, want = pair(torch.bfloat16, gate=gate)
    m.quantize_weights_()
    assert m.prompt_bits == 8
    on = [True]

    def hook(_, args):
        x = args[0]
        return (mx.rounded(x.reshape(-1, x.shape[-1]), 8).to(x.dtype).view(x.shape),) if on[0] else None
    for blk in want.blocks:
        for lin in (blk.att.wq, blk.att.wk, blk.att.wv, blk.att.wg, blk.att.wo, blk.ffn.l1, blk.ffn.l2):
            lin.register_forward_pre_hook(hook)
    ids, cu, lens = prompts(5)
    for k in (m, want):
        k.reset_cache(5)
    got = m.prefill_packed(ids, cu)
    # W_a's input and the residual stream are not rounded: only the seven maps' rows are
    assert rel(got, want.prefill_packed(ids, cu)) < 0.19
    for a, b in zip(m.blocks, want.blocks):
        assert rel(a.att.state, b.att.state) < 0.19
    on[0] = False
    tok = torch.full((5, 1), 9, device=DEV)
    assert rel(m.decode_step(tok), want.decode_step(tok)) < 0.19
    # into other rows, in another order, continuing: the same sequences' logits
    m.reset_cache(7)
    assert torch.equal(m.prefill_packed(ids, cu, rows=[6, 2, 0, 1, 5]), got)
    m.reset_cache(5)
    assert torch.equal(m.prefill_packed(ids, cu), got)


@gpu
def test_what_8_bit_prompts_are_fed(monkeypatch):
    case('the calls of a prefill in 8 bits, their inputs and results')
    m, _ = pair(torch.bfloat16)
    m.quantize_weights_()
    calls = []

    def record(name):
        f = getattr(ops, name)

        def g(*a, **kw):
            out = f(*a, **kw)
            calls.append((name, a, kw, out))
            return out
        monkeypatch.setattr(ops, name, g)
    for name in ('mx_rms_norm', 'mx_quantize', 'mx_linear', 'mx_swiglu', 'rms_norm', 'swiglu'):
        record(name)
    ids, cu, _ = prompts()
    m.reset_cache(3)
    x = m.embedding(ids.reshape(1, -1))
    m.prefill_packed(ids, cu, last_logits=False)
    assert [c[0] for c in calls] == 2 * (['mx_rms_norm'] + 4 * ['mx_linear'] + ['mx_quantize', 'mx_linear', 'mx_rms_norm', 'mx_swiglu', 'mx_linear'])
    delta = None
    for k, blk in enumerate(m.blocks):
        norm1, wq, wk, wv, wg, q8, wo, norm2, gated, l2 = calls[10 * k:10 * k + 10]
        assert norm1[2].get('residual') is delta and norm1[1][1] is blk.rmsnorm1.gamma and norm1[2]['norm_out']
        stream = x if delta is None else (x.float() + delta.float()).bfloat16()
        q, b = mx.quantize(mx.rms_norm(stream.reshape(-1, 256), blk.rmsnorm1.gamma.detach(), float(torch.tensor(1e-6))), 8)
        rows = norm1[3][0]
        assert torch.equal(rows.values[0].double(), q) and torch.equal(rows.scales[0], b)
        W, at = blk.att.w_in.weight.dequantize(), 0
        for c, n in zip((wq, wk, wv, wg), (128, 128, 256, 256)):
            assert c[1][0] is rows and torch.equal(c[1][1].dequantize(), W[at:at + n]) and c[3].dtype is torch.bfloat16
            at += n
        assert wo[1][0] is q8[3] and wo[1][1].values is blk.att.wo.values
        assert norm2[2]['residual'] is wo[3] and norm2[1][1] is blk.rmsnorm2.gamma and not norm2[2]['norm_out']
        want = (stream.float() + wo[3].float()).bfloat16()
        q, b = mx.quantize(mx.rms_norm(want.reshape(-1, 256), blk.rmsnorm2.gamma.detach(), float(torch.tensor(1e-6))), 8)
        assert torch.equal(norm2[3][0].values[0].double(), q) and torch.equal(norm2[3][0].scales[0], b)
        assert gated[1][0] is norm2[3][0] and gated[1][1].values is blk.ffn.l1.values and gated[2]['quantize']
        assert l2[1][0] is gated[3] and l2[1][1].values is blk.ffn.l2.values and l2[3].dtype is torch.bfloat16
        x, delta = want, l2[3]


@gpu
def test_no_gradient_passes():
    m, _ = pair(torch.float32)
    m.quantize_weights_()
    tok = torch.randint(0, 300, (2, 8), device=DEV)
    with pytest.raises(NotImplementedError):
        m(tok)
    with torch.no_grad():
        assert m(tok).shape == (2, 8, 300)


# --- the generator ----------------------------------------------------------------------


@gpu
def test_generator():
    case('greedy and drafted generation over 4-bit weights, graph and eager; other weights loaded; a state_dict')
    m, want = pair(torch.float32)
    m.quantize_weights_()
    g = torch.Generator().manual_seed(3)
    texts = [torch.randint(0, 300, (k,), generator=g) for k in (9, 40, 2)]

    def run(mm, **kw):
        gen = RaggedGenerator(mm)
        gen.prefill(texts)
        return gen.generate(12, **kw)
    tokens = run(m)
    assert torch.equal(tokens, run(m, graph=False)) and torch.equal(tokens, run(want, graph=False))
    gen = RaggedGenerator(m)
    gen.prefill(texts)
    assert torch.equal(gen.generate_drafted(12, drafts=3), tokens)
    # the recorded step is made again when the weights change or move
    other = model(torch.float32)
    with torch.no_grad():
        for p in other.parameters():
            p.mul_(1.7)
    other.quantize_weights_()
    gen = RaggedGenerator(m)
    gen.prefill(texts)
    assert torch.equal(gen.generate(12), tokens)
    m.load_state_dict(other.state_dict())
    gen.prefill(texts)
    new = gen.generate(12)
    assert torch.equal(new, run(other, graph=False)) and not torch.equal(new, tokens)
    for blk, src in zip(m.blocks, want.blocks):
        blk.ffn.l1 = MXLinear(ops.mx_weight(src.ffn.l1.weight, gated=True))     # moved
    gen.prefill(texts)
    assert torch.equal(gen.generate(12), run(m, graph=False))


@gpu
def test_weights_quantised_in_inference_mode():
    case('quantize_weights_ within inference_mode, generation outside of it, a state_dict')
    m, want = pair(torch.float32)
    with torch.inference_mode():
        m.quantize_weights_()
    text = [torch.arange(7) % 300]

    def run(mm):
        gen = RaggedGenerator(mm)
        gen.prefill(text)
        return gen.generate(6)
    tokens = run(m)
    assert not any(t.is_inference() for t in m._quantized()) and torch.equal(tokens, run(want))
    m.load_state_dict({n: t.clone() for n, t in m.state_dict().items()})
    assert torch.equal(run(m), tokens)


@gpu
def test_maps():
    case('MXLinear: rows of a weight, buffers, .to')
    w = torch.randn(96, 200, device=DEV)
    lin = MXLinear(ops.mx_weight(w))
    x = torch.randn(4, 200, device=DEV)
    assert torch.equal(ops.mx_linear(x, lin.rows(32, 48)), lin(x)[:, 32:80])
    for bad in ((8, 16), (0, 24), (64, 48), (-16, 16)):
        with pytest.raises(AssertionError):
            lin.rows(*bad)
    lin = lin.to(torch.bfloat16)
    assert lin.values.dtype is torch.uint8 and sorted(lin.state_dict()) == ['scales', 'values']
    with pytest.raises(AssertionError):
        MXLinear(ops.mx_weight(w, gated=True)).rows(0, 16)

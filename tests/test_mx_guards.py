"""What 4-bit modules stand for and what they refuse: layers, FFNs and models of other classes, hooks, modules
put in others' places, and what a generator's recorded step holds.  Where a mistake would let a graph read freed memory
the decision is tested on the CPU, with MXLinear modules whose bytes are never multiplied."""
import copy

import pytest
import torch
from torch import nn

from oracle import mx
from vagus_amd import _lib, ops
from vagus_amd.layer import GatedDeltaNet, MXLinear
from vagus_amd.model import FFN, GDNLM, RaggedGenerator, _ffn

DEV = 'cuda'
gpu = pytest.mark.gpu


def case(*what):
    print('\n[case]', *what, flush=True)


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def round_(linear):
    """The weights that 4 bits leave of linear, in place."""
    with torch.no_grad():
        linear.weight.copy_(mx.rounded(linear.weight.double(), 4))


def blank(n, k, gated=False, device='cpu'):
    """An MXLinear of zeros, on the CPU."""
    T, C = (2 * -(-n // 32) if gated else -(-n // 16)), -(-k // 128)
    return MXLinear(ops.MXWeight(torch.zeros(T, C, 4, 16, 16, dtype=torch.uint8, device=device),
                                 torch.ones(T, -(-C // 4), 4, 16, 4, dtype=torch.uint8, device=device), (n, k), gated))


def small(device='cpu', **kw):
    torch.manual_seed(0)
    with torch.device(device):
        return GDNLM(**(dict(vocab_size=50, dim=64, layer_count=2, head_count=1, key_head_dim=64, value_head_dim=64, gate='scalar') | kw))


class Wrapped(nn.Module):
    """A model of a caller's own over a GDNLM's modules: no _quantized, a map of its own beside the blocks."""

    def __init__(self, m):
        super().__init__()
        self.inner, self.blocks = m, m.blocks
        self.config = m.config

    def __getattr__(self, name):
        if name in ('reset_cache', 'prefill_packed', 'decode_step'):
            return getattr(self._modules['inner'], name)
        return super().__getattr__(name)


# --- what a recorded step holds --------------------------------------------------------


def test_a_recorded_step_knows_every_4_bit_weight():
    m = small()
    for blk in m.blocks:
        blk.ffn.l1, blk.ffn.l2 = blank(2 * blk.ffn.hidden_dim, 64, True), blank(64, blk.ffn.hidden_dim)
    own = Wrapped(m)
    own.extra = nn.ModuleList([blank(32, 64)])
    m.extra = blank(16, 64)
    gens = [RaggedGenerator(own), RaggedGenerator(m)]
    m.reset_cache(2)

    def changes(do, both=True):
        before = [g._fingerprint() for g in gens]
        assert before == [g._fingerprint() for g in gens]
        keep = do()                                           # what it replaced stays alive: its address is not taken again
        after = [g._fingerprint() for g in gens]
        assert before[0] != after[0] and (not both or before[1] != after[1])
        return keep

    def put(mod, name, new):
        old = getattr(mod, name) if isinstance(name, str) else mod[name]
        setattr(mod, name, new) if isinstance(name, str) else mod.__setitem__(name, new)
        return old
    h = m.blocks[1].ffn.hidden_dim
    kept = [changes(lambda: put(m.blocks[1].ffn, 'l1', blank(2 * h, 64, True))),
            changes(lambda: put(m.blocks[0].ffn, 'l2', blank(64, h))),
            changes(lambda: put(m, 'extra', blank(16, 64))),
            changes(lambda: put(own.extra, 0, blank(32, 64)), both=False)]
    kept.append(changes(lambda: m.blocks[0].ffn.l1.values.fill_(3)))            # in place, as load_state_dict
    kept.append(changes(lambda: m.blocks[0].ffn.l1.scales.fill_(3)))
    with torch.no_grad():
        kept.append(changes(lambda: m.blocks[0].att.A_log.add_(1)))
        kept.append(changes(lambda: m.embedding.weight.mul_(2)))


def test_a_recorded_step_of_an_object_that_is_no_module():
    m = small()
    m.blocks[1].ffn.l2 = blank(64, m.blocks[1].ffn.hidden_dim)

    class Plain:
        blocks, parameters = m.blocks, m.parameters
    m.reset_cache(1)
    gen = RaggedGenerator(Plain())
    keys = [gen._fingerprint()]
    for change in (lambda: m.head.weight.mul_(2), lambda: m.blocks[1].ffn.l2.values.fill_(1), lambda: m.blocks[0].ffn.l1.weight.mul_(2)):
        with torch.no_grad():
            change()
        keys.append(gen._fingerprint())
    assert len(set(keys)) == 4 and keys[-1] == gen._fingerprint()


@gpu
def test_a_model_class_of_the_callers_own_is_recorded_again_when_its_4_bit_weights_move():
    case('4-bit layers in another model class: replaced, then loaded into')
    m = small(DEV, key_head_dim=64, value_head_dim=128, dim=128)
    other = copy.deepcopy(m)
    with torch.no_grad():
        for blk in other.blocks:
            blk.ffn.l1.weight.mul_(1.5)
    for k in (m, other):
        for blk in k.blocks:
            blk.att.quantize_weights_()
            blk.ffn.quantize_weights_()
    text = [torch.arange(7), torch.arange(3)]

    def run(gen, **kw):
        gen.prefill(text)
        return gen.generate(10, **kw)
    gen = RaggedGenerator(Wrapped(m))
    first = run(gen)
    assert torch.equal(first, run(RaggedGenerator(m), graph=False))
    for blk, src in zip(m.blocks, other.blocks):
        blk.ffn.l1 = MXLinear(src.ffn.l1.weight)
    torch.cuda.synchronize()
    want = run(RaggedGenerator(other), graph=False)
    assert torch.equal(run(gen), want)


# --- layers of other classes -------------------------------------------------------------


class OwnGates(GatedDeltaNet):
    """_gates as the class documents it to its callers, without the projections that a grouped product hands on."""

    def _gates(self, x, *, raw_gate=False, raw_beta=False):
        g, beta = super()._gates(x, raw_gate=raw_gate, raw_beta=raw_beta)
        return (g if raw_gate else 0.5 * g), beta


class OwnOutput(GatedDeltaNet):
    def _output(self, o, x):
        return self.wo(o.reshape(*x.shape[:2], -1) * torch.sigmoid(self.wg(x)))


def test_a_layer_with_an_output_of_its_own_keeps_its_weights():
    layer = OwnOutput(dim=64, head_count=1, key_head_dim=64, value_head_dim=64, gate='scalar')
    with pytest.raises(NotImplementedError, match='_output'):
        layer.quantize_weights_()
    m = small()
    m.blocks[1].att = layer
    with pytest.raises(NotImplementedError, match='_output'):
        m.quantize_weights_()
    assert isinstance(layer.wq, nn.Linear) and isinstance(m.blocks[0].att.wq, nn.Linear)


@gpu
@pytest.mark.parametrize('gate', ['scalar', 'vector'])
def test_gates_of_a_subclass_take_the_input_alone(gate):
    case('a subclass whose _gates has no proj: every call of a 4-bit layer', gate)
    torch.manual_seed(3)
    with torch.device(DEV):
        layer = OwnGates(dim=128, head_count=2, key_head_dim=64, value_head_dim=64, gate=gate)
    want = copy.deepcopy(layer)
    for n in ('wq', 'wk', 'wv', 'wg', 'wo'):
        round_(getattr(want, n))
    layer.quantize_weights_()
    x = torch.randn(2, 40, 128, device=DEV)
    cu = torch.tensor([0, 9, 40], dtype=torch.int32, device=DEV)
    with torch.no_grad():                                     # fp32 sums in other orders: as tests/test_mx_model.py
        assert rel(layer(x), want(x)) < 1e-4
    for m in (layer, want):
        m.reset_cache(2)
    assert rel(layer.prefill_packed(x[:1], cu), want.prefill_packed(x[:1], cu)) < 1e-4
    for a, b in ((0, 1), (1, 9), (9, 10)):
        assert rel(layer.decode_step(x[:, a:b]), want.decode_step(x[:, a:b])) < 1e-4
    for m in (layer, want):
        m.begin_drafts(4)
    none = torch.zeros(2, dtype=torch.int32, device=DEV)
    assert rel(layer.draft_step(x[:, 10:14], none), want.draft_step(x[:, 10:14], none)) < 1e-4
    assert rel(layer.state, want.state) < 1e-4


# --- FFNs of other classes ------------------------------------------------------------------


class OwnFFN(FFN):
    def forward(self, x):
        return 0.5 * super().forward(x)


def test_an_ffn_with_a_forward_or_an_activation_of_its_own_keeps_its_weights():
    one, gelu, patched, hooked = OwnFFN(64, 128), FFN(64, 128), FFN(64, 128), FFN(64, 128)
    gelu.silu = nn.GELU()
    patched.forward = lambda x: x
    hooked.silu.register_forward_hook(lambda *a: None)
    for ffn in (one, gelu, patched, hooked):
        with pytest.raises(NotImplementedError, match='of its own'):
            ffn.quantize_weights_()
        m = small()
        m.blocks[1].ffn = ffn
        with pytest.raises(NotImplementedError, match='of its own'):
            m.quantize_weights_()
        assert isinstance(ffn.l1, nn.Linear) and isinstance(m.blocks[0].ffn.l1, nn.Linear)


@gpu
@pytest.mark.parametrize('four_bits', [False, True])
@pytest.mark.parametrize('what', ['identity', 'own forward', 'activation', 'hook'])
def test_other_modules_in_the_place_of_an_ffn_run_on_the_gpu(what, four_bits):
    case('another module than the FFN that the fused pass stands for', what, four_bits)
    m = small(DEV, value_head_dim=128, dim=128).to(torch.bfloat16)
    if four_bits:
        m.quantize_weights_()
    with torch.device(DEV):
        ffn = nn.Identity() if what == 'identity' else (OwnFFN if what == 'own forward' else FFN)(128, 256).to(torch.bfloat16)
    if what == 'activation':
        ffn.silu = nn.GELU()
    if what == 'hook':
        ffn.register_forward_hook(lambda mod, args, out: out + 1)
    m.blocks[0].ffn = ffn
    ids, cu = torch.arange(12, device=DEV), torch.tensor([0, 7, 12], dtype=torch.int32, device=DEV)
    m.reset_cache(2)
    assert bool(torch.isfinite(m.prefill_packed(ids, cu)).all()) and bool(torch.isfinite(m.decode_step(ids[:2, None])).all())
    h = torch.randn(1, 5, 128, device=DEV).bfloat16()
    with torch.no_grad():
        assert torch.equal(_ffn(ffn, h), ffn(h))


@pytest.mark.parametrize('where', ['ffn', 'att'])
def test_blocks_of_other_modules_are_refused_as_such(where):
    m = small()
    setattr(m.blocks[1], where, nn.Identity())
    with pytest.raises(NotImplementedError, match='Identity'):
        m.quantize_weights_()
    assert isinstance(m.blocks[0].ffn.l1, nn.Linear)


# --- hooks on 4-bit maps ----------------------------------------------------------------------


def quantised_on_the_cpu(m):
    """m with maps of zeros in the places of its projections, as quantize_weights_ leaves it."""
    for blk in m.blocks:
        a, f = blk.att, blk.ffn
        wide = sum(w.weight.shape[0] for w in (a.wq, a.wk, a.wv, a.wg))
        del a.wq, a.wk, a.wv, a.wg
        a.w_in, a.wo = blank(wide, a.dim), blank(a.dim, a.out_width)
        f.l1, f.l2 = blank(2 * f.hidden_dim, f.dim, True), blank(f.dim, f.hidden_dim)
    return m


@pytest.mark.parametrize('which', ['att.w_in', 'att.wo', 'ffn.l1', 'ffn.l2', 'ffn'])
def test_a_hooked_map_takes_no_8_bit_rows(which):
    m = quantised_on_the_cpu(small())
    assert all(blk._takes8() for blk in m.blocks)
    for register in ('register_forward_hook', 'register_forward_pre_hook'):
        handle = getattr(m.blocks[1].get_submodule(which), register)(lambda *a: None)
        assert m.blocks[0]._takes8() and not m.blocks[1]._takes8()
        handle.remove()
        assert m.blocks[1]._takes8()
    handle = nn.modules.module.register_module_forward_hook(lambda *a: None)
    assert not m.blocks[0]._takes8()
    handle.remove()


def test_a_layer_with_prompts_of_its_own_takes_no_8_bit_rows():
    class Own(GatedDeltaNet):
        def prefill_packed(self, x, cu_seqlens, *, rows=None):
            return 2 * super().prefill_packed(x, cu_seqlens, rows=rows)
    m = small()
    m.blocks[1].att = Own(dim=64, head_count=1, key_head_dim=64, value_head_dim=64, gate='scalar')
    quantised_on_the_cpu(m)
    assert m.blocks[0]._takes8() and not m.blocks[1]._takes8()

    class Around(nn.Module):
        """A layer's calls handed on by name."""

        def __init__(self, layer):
            super().__init__()
            self.layer = layer

        def __getattr__(self, name):
            return super().__getattr__(name) if name == 'layer' else getattr(self._modules['layer'], name)
    m.blocks[0].att = Around(m.blocks[0].att)
    assert not m.blocks[0]._takes8()


@gpu
@pytest.mark.parametrize('dtype, bar', [(torch.float32, 1e-4), (torch.bfloat16, 2e-2)])       # as tests/test_mx_model.py
def test_hooks_on_4_bit_maps_run_on_every_call(dtype, bar):
    case('hooks that scale what each map gives: forward, prompts, steps, drafts', dtype)
    m = small(DEV, dim=256, head_count=2, value_head_dim=128).to(dtype).eval()
    m.head.weight = nn.Parameter(m.head.weight.detach().clone())
    want = copy.deepcopy(m)
    for blk in want.blocks:
        for lin in (blk.att.wq, blk.att.wk, blk.att.wv, blk.att.wg, blk.att.wo, blk.ffn.l1, blk.ffn.l2):
            round_(lin)
        for n in ('wq', 'wk', 'wv', 'wg'):
            getattr(blk.att, n).register_forward_hook(lambda m_, a, o: 2 * o)
        blk.att.wo.register_forward_hook(lambda m_, a, o: -o)
        blk.ffn.l2.register_forward_pre_hook(lambda m_, a: (4 * a[0],))
        blk.ffn.l2.register_forward_hook(lambda m_, a, o: 0.5 * o)
    round_(want.head)
    m.quantize_weights_()
    seen = []

    def hook(name, scale):
        def f(mod, args, out):
            assert torch.is_tensor(args[0]) and args[0].dtype is dtype
            seen.append(name)
            out = scale * out
            return out.transpose(-1, -2).contiguous().transpose(-1, -2) if name == 'w_in' else out      # any view of it
        return f
    for blk in m.blocks:
        for mod, name, scale in ((blk.att.w_in, 'w_in', 2), (blk.att.wo, 'wo', -1), (blk.ffn.l1, 'l1', 4), (blk.ffn.l2, 'l2', 0.5)):
            mod.register_forward_hook(hook(name, scale))

    def both(f):
        seen.clear()
        got = f(m)
        torch.cuda.synchronize()
        assert seen == 2 * ['w_in', 'wo', 'l1', 'l2'], seen
        assert rel(got, f(want)) < bar
    ids = torch.arange(40, device=DEV) % 50
    cu = torch.tensor([0, 30, 40], dtype=torch.int32, device=DEV)
    with torch.no_grad():
        both(lambda k: k(ids.view(2, 20)))
    for k in (m, want):
        k.reset_cache(2)
    both(lambda k: k.prefill_packed(ids, cu))
    both(lambda k: k.decode_step(ids.view(2, 20)[:, :1]))
    both(lambda k: k.decode_step(ids.view(2, 20)[:, :7]))
    for k in (m, want):
        k.begin_drafts(4)
    none = torch.zeros(2, dtype=torch.int32, device=DEV)
    both(lambda k: k.draft_step(ids.view(2, 20)[:, :4], none))


# --- all of a model or nothing ------------------------------------------------------------------


def held(m):
    return {n: t.data_ptr() for n, t in m.state_dict(keep_vars=True).items()}, [type(c) for c in m.modules()]


@pytest.mark.parametrize('good', [0, 1, 2, 3, 5, 7, 8])
def test_a_model_that_cannot_be_quantised_stays_as_it_was(monkeypatch, good):
    m = small()
    before = held(m)
    calls = []

    def mx_weight(w, gated=False):
        calls.append(w.shape)
        if len(calls) > good:
            raise RuntimeError('no room')
        return blank(*w.shape, gated).weight
    monkeypatch.setattr(ops, 'mx_weight', mx_weight)
    with pytest.raises(RuntimeError, match='no room'):
        m.quantize_weights_()
    assert held(m) == before
    good = 100
    calls.clear()
    m.quantize_weights_()                                     # two blocks of four maps, the head
    assert len(calls) == 9 and len(m._quantized()) == 18 and all(blk._takes8() for blk in m.blocks)


@gpu
@pytest.mark.parametrize('what', ['cpu', 'fp64', 'head'])
def test_a_model_with_a_later_part_elsewhere_stays_as_it_was(what):
    case('quantize_weights_ of a model with a part on the CPU or in fp64', what)
    m = small(DEV, value_head_dim=128, dim=128)
    part = m.blocks[1].ffn.l2 if what != 'head' else m.head
    if what == 'head':
        part.weight = nn.Parameter(part.weight.detach().clone())
    part.to('cpu' if what != 'fp64' else torch.float64)
    before = held(m)
    with pytest.raises(NotImplementedError if what == 'fp64' else RuntimeError):
        m.quantize_weights_()
    assert held(m) == before
    part.to(DEV, torch.float32)
    m.quantize_weights_()
    m.reset_cache(2)
    assert bool(torch.isfinite(m.decode_step(torch.ones(2, 1, dtype=torch.int64, device=DEV))).all())


# --- layers that are not 4-bit ---------------------------------------------------------------------


def test_an_ordinary_model_says_how_it_takes_prompts():
    m = small()
    assert m.prompt_bits == 16 and 'prompt_bits' not in m.__dict__


@gpu
def test_a_layer_that_is_not_4_bit_searches_for_no_4_bit_map():
    case('attributes that the calls of an ordinary layer look for in vain')
    missed = []

    class Watched(GatedDeltaNet):
        def __getattr__(self, name):
            try:
                return super().__getattr__(name)
            except AttributeError:
                missed.append(name)
                raise
    with torch.device(DEV):
        layer = Watched(dim=128, head_count=1, key_head_dim=64, value_head_dim=64, gate='scalar')
    x = torch.randn(2, 8, 128, device=DEV)
    layer(x).sum().backward()
    layer.reset_cache(2)
    with torch.no_grad():
        layer(x)
    layer.prefill_packed(x[:1], torch.tensor([0, 3, 8], dtype=torch.int32, device=DEV))
    layer.decode_step(x[:, :1])
    layer.decode_step(x)
    layer.begin_drafts(4)
    layer.draft_step(x[:, :4], torch.zeros(2, dtype=torch.int32, device=DEV))
    assert 'w_in' not in missed, missed


# --- results that lie in what is read ----------------------------------------------------------------


def test_a_norm_refuses_results_that_overlap():
    """Every call here is refused before a launch: the addresses are none."""
    L = _lib.load()

    def n(**o):
        a = dict(dt=1, x=1 << 20, r=2 << 20, xo=None, g=3 << 20, y=4 << 20, v=5 << 20, s=6 << 20, rows=4, dim=128) | o
        return L.vgdr_mx_rms_norm(a['dt'], a['x'], a['r'], a['xo'], a['g'], a['y'], a['v'], a['s'], a['rows'], a['dim'], 1e-6, None)
    row, total = 256, 1024                                    # bf16: bytes of a row, of x
    for base in (1 << 20, 2 << 20):                           # x, the residual: shifted by rows either way
        for at in (base - total + 16, base - row, base + 16, base + row, base + total - 16):
            assert n(xo=at) == n(y=at) == _lib.VGDR_ERR_INVALID, at
            assert b'alias' in L.vgdr_last_error()
        for at in (base, base + 16, base + total - 16):                   # the bytes are fewer: 512 and 16
            assert n(v=at) == n(s=at) == n(v=at - 496) == _lib.VGDR_ERR_INVALID, at
    for at in (3 << 20, (3 << 20) + 16, (3 << 20) + row - 16):            # gamma
        assert n(xo=at) == n(y=at) == n(v=at) == n(s=at) == _lib.VGDR_ERR_INVALID, at
    assert n(y=1 << 20) == n(v=2 << 20) == n(xo=4 << 20) == n(s=(5 << 20) + 16) == n(xo=(5 << 20) + 496) == _lib.VGDR_ERR_INVALID
    assert n(dt=0, xo=(1 << 20) + 2 * total - 16) == n(xo=1 << 20, y=1 << 20) == _lib.VGDR_ERR_INVALID


@gpu
def test_a_norm_in_place_and_beside_what_it_reads():
    case('mx_rms_norm into x, into the residual, beside x in one buffer, shifted by a row')
    D = 256
    buf = torch.randn(12, D, device=DEV).bfloat16()
    gamma, res = torch.randn(D, device=DEV).bfloat16(), torch.randn(5, D, device=DEV).bfloat16()
    x = buf[:5]
    want, h = ops.mx_rms_norm(x, gamma, residual=res)
    for out in (buf[5:10], buf[7:12]):
        rows, got = ops.mx_rms_norm(x, gamma, residual=res, out_residual=out)
        assert got is out and torch.equal(got, h) and torch.equal(rows.values.view(torch.uint8), want.values.view(torch.uint8))
    for out in (buf[1:6], buf[4:9]):
        with pytest.raises(AssertionError, match='alias'):
            ops.mx_rms_norm(x, gamma, residual=res, out_residual=out)
    r = res.clone()
    rows, got = ops.mx_rms_norm(x, gamma, residual=r, out_residual=r)
    assert got is r and torch.equal(r, h) and torch.equal(rows.scales, want.scales)
    rows, got = ops.mx_rms_norm(x, gamma, residual=res, out_residual=x)
    assert got is x and torch.equal(x, h) and torch.equal(rows.scales, want.scales)

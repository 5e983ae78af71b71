"""What 4-bit modules stand for and what they refuse: layers, FFNs and models of other classes, hooks, modules
put in others' places, and what a generator's recorded step holds.  Where a mistake would let a graph read freed memory
the decision is tested on the CPU, with MXLinear modules whose bytes are never multiplied."""
import copy

import pytest
import torch
from torch import nn

from vagus_amd import ops
from vagus_amd.layer import MXLinear
from vagus_amd.model import GDNLM, RaggedGenerator

DEV = 'cuda'
gpu = pytest.mark.gpu


def case(*what):
    print('\n[case]', *what, flush=True)


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

"""Speculative decoding as it is used: a layer's drafted blocks against its one-token steps, and
the generator's drafted decoding (lookup, block, verification together) against its
greedy decoding.

Bars. A layer in fp32: both sides compute the same sums of at most dim = 128 products in fp32
in another order, through four matrix products and the recurrence: 1e-5 of the output's norm is
some 170 half steps of 2^-24. In bf16 the one-token step rounds the conv's, SiLU's, norm's and
recurrence's results (2^-8 each, five in a row) where the block does not, the state carrying them:
2e-2, the other tests' bar against the oracle. Tokens: fp32 logits of 211 random ids
are not within 1e-5 of each other at their top, so greedy tokens are equal.
"""
import contextlib
import gc

import pytest
import torch

from test_model import prompts, tiny
from vagus_amd.layer import GatedDeltaNet
from vagus_amd.model import GDNLM, RaggedGenerator


def layer(gate, dtype, **kw):
    torch.manual_seed(3)
    kw = {'dim': 128, 'head_count': 2, 'key_head_dim': 64, 'value_head_dim': 64, 'gate_rank': 16, **kw}
    m = GatedDeltaNet(gate=gate, **kw)
    with torch.no_grad():
        m.o_norm.gamma.uniform_(0.5, 1.5)
        if m.short_conv_size is not None:
            for n in ('conv_q', 'conv_k', 'conv_v'):
                getattr(m, n).conv.weight.normal_(0, 0.5)
    return m.to(device='cuda', dtype=dtype).eval()


def varied(dtype, gate='scalar', seed=0):
    """A model whose next token depends on its text: a head of its own, logits of 2.3 a standard
    deviation (tied to its embedding the tiny model repeats each stream's last token for ever)."""
    torch.manual_seed(seed)
    m = GDNLM(vocab_size=211, dim=128, layer_count=2, head_count=2, key_head_dim=64, value_head_dim=64, gate=gate,
              gate_rank=16, tie_embedding=False)
    with torch.no_grad():
        for blk in m.blocks:
            blk.att.o_norm.gamma.uniform_(0.5, 1.5)
            for n in ('conv_q', 'conv_k', 'conv_v'):
                getattr(blk.att, n).conv.weight.normal_(0, 0.5)
            blk.att.wo.weight.normal_(0, 0.2)
            blk.ffn.l1.weight.normal_(0, 0.1)
            blk.ffn.l2.weight.normal_(0, 0.1)
        m.embedding.weight.normal_(0, 0.3)
        m.head.weight.normal_(0, 0.2)
    return m.to(device='cuda', dtype=dtype).eval()


def rel(x, ref):
    return ((x.double() - ref.double()).norm() / ref.double().norm().clamp_min(1e-30)).item()


@pytest.mark.gpu
@pytest.mark.parametrize('gate,dtype,kw', [
    ('scalar', torch.float32, {}), ('vector', torch.float32, {}), ('none', torch.float32, {}),
    ('scalar', torch.float32, dict(delta=False)), ('vector', torch.float32, dict(gate_lower_bound=-3.0)),
    ('scalar', torch.float32, dict(short_conv_size=3)), ('vector', torch.float32, dict(short_conv_size=None)),
    ('scalar', torch.float32, dict(key_head_dim=32, value_head_dim=128)),
    ('scalar', torch.float32, dict(out_proj=False, value_head_dim=128)),
    ('scalar', torch.bfloat16, {}), ('vector', torch.bfloat16, dict(value_head_dim=256))])
def test_layer_blocks_are_its_one_token_steps(gate, dtype, kw):
    """Blocks of 4 with 0 to 4 tokens that stand: every output, the state and the conv caches are those of
    one-token steps over the tokens that stood before it."""
    m = layer(gate, dtype, **kw)
    N, L, bar = 3, 4, 1e-5 if dtype == torch.float32 else 2e-2
    r = torch.Generator().manual_seed(7)
    counts = [[0, 0, 0], [4, 1, 0], [2, 4, 3], [0, 1, 4]]
    xs = [torch.randn(N, L, 128, generator=r).to('cuda', dtype) for _ in counts]
    m.reset_cache(N)
    m.begin_drafts(L)
    outs = [m.draft_step(x, torch.tensor(a, device='cuda')) for x, a in zip(xs, counts)]
    m.commit_drafts(torch.tensor([1, 0, 2], device='cuda'))
    got = m.export_cache()
    stood = counts[1:] + [[1, 0, 2]]
    ref = layer(gate, dtype, **kw)
    for b in range(N):
        ref.reset_cache(1)
        for x, o, a in zip(xs, outs, stood):
            keep = ref.export_cache()
            for t in range(L):
                want = ref.decode_step(x[b:b + 1, t:t + 1])
                assert rel(o[b:b + 1, t:t + 1], want) <= bar
            ref.load_cache(keep)
            for t in range(a[b]):
                ref.decode_step(x[b:b + 1, t:t + 1])
        end = ref.export_cache()
        assert rel(got['state'][b], end['state'][0]) <= bar
        if m.short_conv_size is not None:
            for n in ('qp_cache', 'kp_cache', 'vp_cache'):
                # the projections' order of sums differs between one row and twelve
                assert rel(got[n][b], end[n][0]) <= (1e-5 if dtype == torch.float32 else 2 ** -8)


@pytest.mark.gpu
@pytest.mark.parametrize('gate', ['scalar', 'vector', 'none'])
def test_many_rows(gate):
    """70 streams of 4 tokens: more rows than one projection launch takes (256), as the blocks of 10
    streams each, which it does."""
    m = layer(gate, torch.float32)
    x = torch.randn(70, 4, 128, generator=torch.Generator().manual_seed(8)).cuda()
    zero, two = (torch.full((70,), n, dtype=torch.int32, device='cuda') for n in (0, 2))
    m.reset_cache(70)
    m.begin_drafts(4)
    m.draft_step(x, zero)
    got, state = m.draft_step(x.flip(1), two), m.state.clone()
    for b in range(0, 70, 10):
        m.reset_cache(10)
        m.begin_drafts(4)
        m.draft_step(x[b:b + 10], zero[:10])
        want = m.draft_step(x[b:b + 10].flip(1), two[:10])
        assert rel(got[b:b + 10], want) <= 1e-5 and rel(state[b:b + 10], m.state) <= 1e-5


@pytest.mark.gpu
def test_layer_refusals():
    m = layer('scalar', torch.float32)
    x, a = torch.zeros(2, 3, 128, device='cuda'), torch.zeros(2, dtype=torch.int32, device='cuda')
    with pytest.raises(AssertionError, match='No state'):
        m.begin_drafts(3)
    m.reset_cache(2)
    with pytest.raises(AssertionError, match='begin_drafts'):
        m.draft_step(x, a)
    m.begin_drafts(2)
    with pytest.raises(AssertionError, match='1 to 2 tokens'):
        m.draft_step(x, a)
    m.begin_drafts(3)
    with pytest.raises(AssertionError, match='Batch size'):
        m.draft_step(x[:1], a[:1])
    with pytest.raises(NotImplementedError, match='1 to 16'):
        m.begin_drafts(17)

    class Write(GatedDeltaNet):
        def _write(self, x, k, g, beta):
            return beta, k

    w = Write(128, 2, 64, 64, gate='vector').cuda()
    w.reset_cache(2)
    with pytest.raises(NotImplementedError, match='write of its own'):
        w.begin_drafts(3)


def repeating(lens, seed=1, vocab=211):
    """Prompts whose phrases come again."""
    out = []
    for i, p in enumerate(prompts(lens, seed, vocab)):
        n = max(1, p.numel() // 3)
        out.append(p[torch.arange(p.numel()) % n])
    return out


@pytest.mark.gpu
@pytest.mark.parametrize('gate', ['scalar', 'vector'])
def test_drafted_tokens_are_the_greedy_ones(gate):
    m = varied(torch.float32, gate)
    ps = repeating([5, 70, 19, 1, 2])
    gen = RaggedGenerator(m)
    gen.prefill(ps)
    want = gen.generate(41)
    states = [blk.att.export_cache() for blk in m.blocks]
    for drafts, graph in ((4, True), (1, True), (15, True), (7, False)):
        gen.prefill(ps)
        got = gen.generate_drafted(41, drafts=drafts, graph=graph)
        assert torch.equal(got, want), drafts
        # the caches stand where 41 one-token steps leave them
        for blk, s in zip(m.blocks, states):
            assert rel(blk.att.state, s['state']) <= 41e-5         # a step's bar, 41 steps
            assert rel(blk.att.kp_cache, s['kp_cache']) <= 41e-5
        assert gen.fed_len == [n - 1 + 41 for n in (5, 70, 19, 1, 2)]
    assert len(set(want[1].tolist())) > 5              # a text, not one token


def test_drafted_steps_are_the_last_calls():
    """drafted_steps is there before the first call, and 0 behind a call that takes none."""
    gen = RaggedGenerator(Chain())
    assert gen.drafted_steps == 0
    gen.prefill(prompts([5], 6, 97))
    gen.drafted_steps = 9                              # as an earlier call leaves it
    assert gen.generate_drafted(0).shape == (1, 0) and gen.drafted_steps == 0


@pytest.mark.gpu
def test_drafted_and_one_token_calls_in_turn():
    """generate, generate_drafted and generate again go on where the last call ended; a
    second prefill replays the recorded step."""
    m = varied(torch.float32)
    ps = repeating([12, 33, 8], seed=4)
    gen = RaggedGenerator(m)
    gen.prefill(ps)
    want = gen.generate(40)
    for _ in range(2):
        gen.prefill(ps)
        got = torch.cat([gen.generate(7), gen.generate_drafted(13), gen.generate_drafted(0), gen.generate_drafted(1),
                         gen.generate(9), gen.generate_drafted(10)], 1)
        assert torch.equal(got, want)
    with torch.no_grad():                              # a parameter changed in place, and one that moved: recorded again
        m.blocks[0].ffn.l1.weight.mul_(1.5)
        m.blocks[1].att.wq.weight = torch.nn.Parameter(m.blocks[1].att.wq.weight * 0.5)
    gen.prefill(ps)
    want = gen.generate(20)
    gen.prefill(ps)
    assert torch.equal(gen.generate_drafted(20), want)


@pytest.mark.gpu
def test_a_recorded_step_knows_every_tensor_of_its_blocks():
    """A block's log-decays that lie elsewhere: the step is recorded again."""
    m = varied(torch.float32)
    ps = repeating([12, 33, 8], seed=4)
    gen = RaggedGenerator(m)
    gen.prefill(ps)
    want = gen.generate_drafted(30)
    att = m.blocks[1].att
    for name in ('k', 'u', 'g'):
        key, old = gen._drafted_fingerprint(), getattr(att._drafted, name)
        setattr(att._drafted, name, torch.zeros_like(old))
        assert gen._drafted_fingerprint() != key
    gen.prefill(ps)
    assert torch.equal(gen.generate_drafted(30), want)


@pytest.mark.gpu
def test_sampled_decoding():
    """The same uniform numbers give the same tokens, eagerly and replayed; at a temperature near 0
    they are the greedy ones; every token is in the vocabulary."""
    m = varied(torch.float32)
    ps = repeating([12, 33, 8, 20], seed=5)
    gen = RaggedGenerator(m)

    def run(T, graph, seed=1):
        gen.prefill(ps)
        return gen.generate_drafted(25, drafts=3, temperature=T, graph=graph,
                                    generator=torch.Generator('cuda').manual_seed(seed))

    a, b = run(0.8, False), run(0.8, True)
    assert torch.equal(a, b) and int(a.min()) >= 0 and int(a.max()) < 211
    assert not torch.equal(run(0.8, True, seed=2), a)
    assert torch.equal(run(1e-4, True), run(0.0, True))


@pytest.mark.gpu
def test_bf16_model_runs():
    """bf16: steps over 64 streams of blocks of 5 (320 rows: the stacked projections) and of 2."""
    m = varied(torch.bfloat16, 'vector')
    ps = repeating([3 + i % 40 for i in range(64)], seed=6)
    gen = RaggedGenerator(m)
    for drafts in (4, 1):
        gen.prefill(ps)
        out = gen.generate_drafted(12, drafts=drafts)
        assert out.shape == (64, 12) and int(out.min()) >= 0 and int(out.max()) < 211
        for blk in m.blocks:
            assert torch.isfinite(blk.att.state).all()


@pytest.mark.gpu
@pytest.mark.parametrize('drafts,graph', [(4, True), (1, True), (15, False)])
def test_drafts_stand(drafts, graph):
    """A model that repeats each stream's last token for ever: behind one step, whose drafts may fall, the
    text ends in that token twice and every draft is it, so that each step makes drafts + 1 tokens."""
    m = tiny(torch.float32)
    lens, steps = [5, 70, 19, 1, 2], 41
    ps = [p.clone() for p in prompts(lens)]
    gen = RaggedGenerator(m)
    gen.prefill(ps)
    want = gen.generate(steps)
    assert torch.equal(want.cpu(), torch.stack([p[-1].expand(steps) for p in ps]))        # the premise
    states = [blk.att.export_cache()['state'] for blk in m.blocks]
    gen.prefill(ps)
    assert torch.equal(gen.generate_drafted(steps, drafts=drafts, graph=graph), want)
    assert -(-steps // (drafts + 1)) <= gen.drafted_steps <= 1 + -(-(steps - 1) // (drafts + 1))
    for blk, s in zip(m.blocks, states):
        assert rel(blk.att.state, s) <= 41e-5          # a step's bar, 41 steps


@pytest.mark.gpu
def test_sampled_drafts_stand():
    """At a temperature too: one that leaves the repeated token nearly all of the mass."""
    m = tiny(torch.float32)
    ps = prompts([5, 70, 19])
    gen = RaggedGenerator(m)
    gen.prefill(ps)
    got = gen.generate_drafted(41, drafts=4, temperature=1e-3, generator=torch.Generator('cuda').manual_seed(3))
    assert torch.equal(got.cpu(), torch.stack([p[-1].expand(41) for p in ps]))
    assert 9 <= gen.drafted_steps <= 1 + 8


@pytest.mark.gpu
@pytest.mark.parametrize('gate', ['scalar', 'vector'])
def test_bf16_logits_of_a_block(gate):
    """Blocks of 5 through 64 bf16 streams (320 rows: the stacked projections), all of the first one's tokens
    standing: each token's logits against the one-token steps'. Either is within 2e-2 of the oracle's by the
    model's own bar, so they are within twice that of each other."""
    m = tiny(torch.bfloat16, gate)
    toks = torch.stack(prompts([10] * 64, seed=10)).cuda()
    m.reset_cache(64)
    want = torch.cat([m.decode_step(toks[:, t:t + 1]) for t in range(10)], 1)
    m.reset_cache(64)
    m.begin_drafts(5)
    counts = torch.zeros(64, dtype=torch.int32, device='cuda')
    got = torch.cat([m.draft_step(toks[:, :5], counts), m.draft_step(toks[:, 5:], counts + 5)], 1)
    for t in range(10):
        assert rel(got[:, t], want[:, t]) <= 4e-2, t


@pytest.mark.gpu
def test_generator_refusals():
    m = varied(torch.float32)
    gen = RaggedGenerator(m)
    with pytest.raises(AssertionError, match='prefill first'):
        gen.generate_drafted(4)
    gen.prefill(repeating([5]))
    with pytest.raises(AssertionError, match='drafts a step'):
        gen.generate_drafted(4, drafts=16)
    with pytest.raises(AssertionError, match='temperature'):
        gen.generate_drafted(4, temperature=-1)


@pytest.mark.gpu
def test_model_logits_of_a_block():
    """GDNLM.draft_step's logits are decode_step's, token by token."""
    m = varied(torch.float32, 'vector')
    toks = prompts([6, 6], seed=9)
    block = torch.stack(toks).cuda()
    m.reset_cache(2)
    want = torch.cat([m.decode_step(block[:, t:t + 1]) for t in range(6)], 1)
    m.reset_cache(2)
    m.begin_drafts(6)
    got = m.draft_step(block, torch.zeros(2, dtype=torch.int32, device='cuda'))
    assert rel(got, want) <= 1e-4


class Chain(torch.nn.Module):
    """Stands for a model on the CPU: the token behind t is 5 t + 3 modulo 97."""
    blocks = ()

    def __init__(self):
        super().__init__()
        self.scale = torch.nn.Parameter(torch.ones(1))

    def reset_cache(self, batch_size):
        pass

    def prefill_packed(self, tokens, cu_seqlens, *, rows=None, last_logits=True):
        pass

    def decode_step(self, tokens, *, return_logits=True):
        return torch.nn.functional.one_hot((5 * tokens + 3) % 97, 97).float()


def test_texts_of_the_streams():
    """The streams' texts: their prompts and what every call made since, of any length; a prefill starts anew."""
    gen = RaggedGenerator(Chain())
    for lens, calls in (([5, 1, 9], (3, 0, 1, 600, 2, 1300)), ([5, 1, 9], ()), ([2], (1, 255, 1)), ([4, 300], (7,))):
        ps = prompts(lens, 6, 97)
        gen.prefill((torch.cat(ps), torch.tensor([0] + lens).cumsum(0)))
        outs = []
        for n in calls:
            out = gen.generate(n, graph=False)
            outs.append(out.clone())
            out.fill_(-7)                              # the caller's to write
        text, length = gen._texts(11)
        assert text.shape[1] >= int(length.max()) + 11 and length.dtype == torch.int32
        for b, p in enumerate(ps):
            want = torch.cat([p] + [o[b] for o in outs])
            assert length[b] == want.numel() and torch.equal(text[b, :want.numel()], want)
            assert not text[b, want.numel():].any()


def test_one_token_calls_hold_no_tensors_of_their_own():
    """A server of one-token calls that never drafts: as many tensors behind 300 of them as behind two."""
    gen = RaggedGenerator(Chain())
    gen.prefill(prompts([5, 9], 6, 97))

    def held():
        gc.collect()
        return sum(type(t) is torch.Tensor for t in gc.get_objects())

    for _ in range(2):
        gen.generate(1, graph=False)
    before = held()
    for _ in range(300):
        gen.generate(1, graph=False)
    assert held() <= before


def test_steps_are_recorded_on_the_models_gpu(monkeypatch):
    """The capture stream is one of the generator's device, whichever is current: seen with torch's calls replaced."""
    gen = RaggedGenerator(Chain())
    gen.prefill(prompts([5, 9], 6, 97))
    seen = []

    class Graph:
        def replay(self):
            gen._step()

    @contextlib.contextmanager
    def entered(*args, **kw):
        seen.append((args, kw))
        yield

    monkeypatch.setattr(torch.cuda, 'CUDAGraph', Graph)
    monkeypatch.setattr(torch.cuda, 'graph', entered)
    monkeypatch.setattr(torch.cuda, 'device', entered)
    monkeypatch.setattr(torch.cuda, 'Stream', lambda device=None, **kw: ('stream', device))
    gen.generate(3)
    assert seen[0] == ((gen.device,), {})
    assert seen[1][1] == dict(stream=('stream', gen.device))


def test_calls_within_and_outside_inference_mode():
    """The text that one call leaves in inference mode is the next one's to write on outside of it."""
    gen = RaggedGenerator(Chain())
    gen.prefill(prompts([5, 9], 6, 97))
    with torch.inference_mode():
        a = gen.generate(3, graph=False)
    b = gen.generate(2, graph=False)
    text, length = gen._texts(1)
    assert torch.equal(text[0, 5:10], torch.cat([a, b], 1)[0]) and length.tolist() == [10, 14]


@pytest.mark.gpu
@pytest.mark.parametrize('graph', [True, False])
def test_drafted_calls_within_and_outside_inference_mode(graph):
    m = varied(torch.float32)
    ps = repeating([12, 33, 8], seed=4)
    gen = RaggedGenerator(m)
    gen.prefill(ps)
    want = gen.generate(30)
    gen.prefill(ps)
    with torch.inference_mode():
        a = gen.generate_drafted(10, graph=graph)
    b = gen.generate_drafted(10, graph=graph)
    with torch.inference_mode():
        c = gen.generate_drafted(10, graph=graph)
    assert torch.equal(torch.cat([a, b, c], 1), want)

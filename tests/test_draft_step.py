"""A drafted block through a layer's recurrence (ops.hip_draft_step,
ops.commit_drafts): the accepted tokens of the last block committed, the new block's
outputs and what it leaves pending, against the recurrence walked token by token in 64
bits on the same inputs.

Bars, by arithmetic. Inside everything is fp32 (half a step: 2^-24). A value is a sum of at
most dk + 2 L + K products behind some 30 further roundings (activation, norm, gate, decay,
epilogue), so its error is under (dk + 2 L + K + 30) 2^-24 of the terms' size, and the
2-norm of a whole tensor's errors, whose signs differ, under that part of the tensor's
norm. o is then rounded once to its type: half a step more, 2^-8 (bf16) or 2^-11 (fp16) of
each value. Caches and raw inputs are copies: equal bits.
"""
import ctypes

import pytest
import torch
import torch.nn.functional as F

from vagus_amd import _lib, ops

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make(N, L, H, dk, dv, *, P=None, dtype=torch.float32, gate='scalar', delta=True, K=4, epilogue=True, act=True,
         l2norm=True, seed=0, wide=False, logits=True):
    """Inputs on the CPU: a state, a pending block of P tokens, and L new tokens."""
    P = P or L
    r = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=r)  # noqa: E731
    gs = {'none': None, 'scalar': (H,), 'vector': (H, dk)}[gate]
    c = dict(N=N, L=L, H=H, dk=dk, dv=dv, P=P, gate=gate, delta=delta, K=K, act=act and gate == 'vector', l2norm=l2norm,
             logits=logits and delta, dtype=dtype)
    c['state'] = 0.2 * randn(N, H, dk, dv)
    c['k'] = F.normalize(randn(N, P, H, dk), dim=-1)
    c['u'] = randn(N, P, H, dv)
    c['g'] = None if gs is None else F.logsigmoid(randn(N, P, *gs) + 3)
    y = randn(N, L, 2 * H * (dk + dv)).to(dtype)
    c['q_in'], c['k_in'], c['v_in'], c['out_gate'] = y.split([H * dk, H * dk, H * dv, H * dv], -1)
    c['y'] = y
    c['wide'] = wide
    c['beta'] = (randn(N, L, H) if logits else torch.rand(N, L, H, generator=r)) if delta else None
    c['g_in'] = F.logsigmoid(randn(N, L, H) + 3) if gate == 'scalar' else None
    if gate == 'vector':
        c['g_in'] = randn(N, L, H, dk).to(dtype) if c['act'] else F.logsigmoid(randn(N, L, H, dk) + 3)
    c['A_log'], c['dt_bias'] = torch.rand(H, generator=r), randn(H * dk) - 2
    if gate == 'scalar' and act == 'scalar':
        c['act'], c['g_in'], c['dt_bias'] = True, randn(N, L, H).to(dtype), c['dt_bias'][:H]
    c['lower'] = None
    c['gamma'] = 1 + 0.2 * randn(dv) if epilogue else None
    D = (H * dk, H * dk, H * dv)
    c['w'] = [randn(d, K).to(dtype) for d in D] if K else None
    c['cache'] = [randn(N, K, d).to(dtype) for d in D] if K else None
    c['x'] = [randn(N, P, d).to(dtype) for d in D] if K else None
    return c


def reference(c, accepted):
    """Token by token in 64 bits, stream by stream; the committed state, the caches, o and the
    new pending block."""
    N, L, H, dk, dv, K = c['N'], c['L'], c['H'], c['dk'], c['dv'], c['K']
    S = c['state'].double().clone()
    cache = [t.clone() for t in c['cache']] if K else None
    o, pk, pu, pg = [], [], [], []

    def decay(M, g):
        return M if g is None else (g.double().exp()[..., None] if g.dim() == 2 else g.double().exp()[:, None, None]) * M

    for n in range(N):
        a = max(0, min(c['P'], int(accepted[n])))
        for t in range(a):
            S[n] = decay(S[n], None if c['g'] is None else c['g'][n, t])
            S[n] += c['k'][n, t].double()[..., None] * c['u'][n, t].double()[:, None]
        rows = []
        for i, name in enumerate(('q_in', 'k_in', 'v_in')):
            raw = c[name][n]
            if not K:
                rows.append(raw.double())
                continue
            line = torch.cat([c['cache'][i][n], c['x'][i][n, :a]])[a:]
            cache[i][n] = line
            line = torch.cat([line, raw]).double()
            y = torch.stack([(line[t + 1:t + 1 + K] * c['w'][i].double().T).sum(0) for t in range(L)])
            rows.append(y * torch.sigmoid(y))
        q, k, v = (t.reshape(L, H, -1) for t in rows)
        if c['l2norm']:
            q, k = (t / torch.sqrt((t * t).sum(-1, keepdim=True) + 1e-6) for t in (q, k))
        M = S[n].clone()
        for t in range(L):
            g = None if c['g_in'] is None else c['g_in'][n, t].double()
            if c['act']:
                z = g + c['dt_bias'].double().view(g.shape)
                A = c['A_log'].double().exp().view((H,) + (1,) * (g.dim() - 1))
                g = -A * F.softplus(z) if c['lower'] is None else c['lower'] * torch.sigmoid(A * z)
            M = decay(M, g)
            u = v[t]
            if c['delta']:
                b = c['beta'][n, t].double()
                u = (torch.sigmoid(b) if c['logits'] else b)[:, None] * (v[t] - (M * k[t][..., None]).sum(1))
            M = M + k[t][..., None] * u[:, None]
            y = (M * q[t][..., None]).sum(1) * dk ** -0.5
            if c['gamma'] is not None:
                z = c['out_gate'][n, t].double().view(H, dv)
                y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * c['gamma'].double() * z * torch.sigmoid(z)
            o.append(y)
            pk.append(k[t])
            pu.append(u)
            pg.append(g)
    sh = lambda ts: torch.stack(ts).reshape(N, L, *ts[0].shape)  # noqa: E731
    return dict(state=S, cache=cache, o=sh(o), k=sh(pk), u=sh(pu), g=None if c['g_in'] is None else sh(pg))


def device(c, dev='cuda'):
    """The case's tensors on the GPU and the arguments of the call."""
    mv = lambda t: None if t is None else t.to(dev)  # noqa: E731
    y = mv(c['y'])
    H, dk, dv = c['H'], c['dk'], c['dv']
    parts = y.split([H * dk, H * dk, H * dv, H * dv], -1)
    if not c['wide']:
        parts = [t.contiguous() for t in parts]
    cache = [mv(t) for t in c['cache']] if c['K'] else None
    pending = ops.DraftBlock(mv(c['k']), mv(c['u']), mv(c['g']), [mv(t) for t in c['x']] if c['K'] else None)
    kw = dict(scale=dk ** -0.5, delta=c['delta'], conv_weights=[mv(t) for t in c['w']] if c['K'] else None,
              conv_cache=cache, l2norm=c['l2norm'], beta_logits=c['logits'])
    if c['act']:
        kw.update(gate_in_kernel=True, A_log=mv(c['A_log']), dt_bias=mv(c['dt_bias']), lower_bound=c['lower'])
    if c['gamma'] is not None:
        kw.update(out_gate=parts[3], out_norm_weight=mv(c['gamma']))
    return list(parts[:3]), mv(c['g_in']), mv(c['beta']), mv(c['state']), pending, cache, kw


def check(c, o, state, pending, cache, ref):
    L, K = c['L'], c['K']
    bar = (c['dk'] + 2 * L + K + 30) * 2.0 ** -24

    def near(name, x, want, half=0.0):
        x, want = x.double().cpu(), want.double()
        assert torch.isfinite(x).all(), name
        rel = ((x - want).norm() / want.norm().clamp_min(1e-30)).item()
        assert rel <= bar + half, f'{name}: rel_l2 {rel:.3g} over {bar + half:.3g}'

    near('state', state, ref['state'])
    near('o', o, ref['o'], HALF[c['dtype']])
    near('pending k', pending.k[:, :L], ref['k'])
    near('pending u', pending.u[:, :L], ref['u'])
    if ref['g'] is not None:
        near('pending g', pending.g[:, :L], ref['g'])
    if K:
        for i, name in enumerate(('q_in', 'k_in', 'v_in')):
            assert torch.equal(cache[i].cpu(), ref['cache'][i])
            assert torch.equal(pending.x[i][:, :L].cpu(), c[name])
    # rows behind the block stay as they were
    for new, old in ((pending.k, c['k']), (pending.u, c['u'])) + (((pending.g, c['g']),) if c['g'] is not None else ()):
        assert torch.equal(new[:, L:].cpu(), old[:, L:])


def run(c, accepted, dev='cuda'):
    (q, k, v), g, beta, state, pending, cache, kw = device(c, dev)
    o = ops.hip_draft_step(q, k, v, g, beta, state, pending, torch.tensor(accepted, dtype=torch.int32, device=dev), **kw)
    return o, state, pending, cache


CASES = [
    # sizes, gates, types: one token to the longest block, none to all of the last one accepted
    dict(N=1, L=1, H=1, dk=64, dv=64),
    dict(N=2, L=5, H=3, dk=128, dv=128, dtype=torch.bfloat16, wide=True),
    dict(N=3, L=16, H=2, dk=128, dv=128, dtype=torch.bfloat16),
    dict(N=2, L=8, H=2, dk=128, dv=256, dtype=torch.bfloat16, gate='vector'),
    dict(N=2, L=16, H=1, dk=64, dv=256, gate='vector'),
    dict(N=3, L=9, H=2, dk=64, dv=128, gate='vector', act=False, dtype=torch.float16),
    dict(N=2, L=7, H=2, dk=128, dv=64, gate='none', K=0, epilogue=False),
    dict(N=5, L=3, H=5, dk=48, dv=96, gate='vector', K=3, wide=True),
    dict(N=2, L=4, H=2, dk=8, dv=8, gate='scalar', K=1),
    dict(N=2, L=6, H=2, dk=72, dv=200, gate='scalar', K=8, dtype=torch.bfloat16, wide=True),
    dict(N=2, L=6, H=2, dk=120, dv=136, gate='none', K=2, l2norm=False, logits=False),
    dict(N=3, L=5, H=2, dk=64, dv=64, delta=False, gate='scalar'),
    dict(N=2, L=16, H=2, dk=128, dv=128, delta=False, gate='vector', dtype=torch.float16),
    # a short block behind a longer one
    dict(N=4, L=2, P=7, H=2, dk=64, dv=64),
    dict(N=4, L=1, P=16, H=2, dk=128, dv=128, dtype=torch.bfloat16, gate='vector'),
    dict(N=1, L=5, P=6, H=2, dk=128, dv=64, wide=True),
    # the scalar gate's activation in the kernel
    dict(N=3, L=5, H=3, dk=64, dv=64, act='scalar'),
    dict(N=2, L=11, H=2, dk=128, dv=128, act='scalar', dtype=torch.bfloat16),
    dict(N=2, L=4, H=5, dk=64, dv=128, act='scalar', dtype=torch.float16, delta=False),
]


@pytest.mark.gpu
@pytest.mark.parametrize('i', range(len(CASES)))
def test_step_matches_the_recurrence_in_64_bits(i):
    c = make(**CASES[i], seed=i)
    P = c['P']
    accepted = [(0, P, 1, P // 2, P - 1)[(n + i) % 5] for n in range(c['N'])]
    print(f'\n[case] {CASES[i]} accepted {accepted}', flush=True)
    check(c, *run(c, accepted), reference(c, accepted))


@pytest.mark.gpu
def test_bounded_gate_and_counts_outside_the_room():
    c = make(3, 4, 2, 64, 64, gate='vector', seed=50)
    c['lower'] = -3.0
    check(c, *run(c, [-5, 100, 2]), reference(c, [-5, 100, 2]))


@pytest.mark.gpu
def test_rejected_tokens_leave_no_trace():
    """What is pending behind the accepted count, whatever it holds, reaches nothing."""
    for gate in ('none', 'scalar', 'vector'):
        c = make(2, 6, 2, 64, 64, gate=gate, seed=60)
        a = [2, 0]
        o, state, pending, cache = run(c, a)
        for n in range(2):
            for t in ([c['k'], c['u']] + ([c['g']] if c['g'] is not None else []) + c['x']):
                t[n, a[n]:] = float('nan')
        o2, state2, pending2, cache2 = run(c, a)
        assert torch.equal(o, o2) and torch.equal(state, state2)
        assert all(torch.equal(x, y) for x, y in zip(cache, cache2))
        assert torch.equal(pending.u, pending2.u) and torch.equal(pending.k, pending2.k)


@pytest.mark.gpu
@pytest.mark.parametrize('L,gate', [(6, 'scalar'), (14, 'scalar'), (6, 'vector'), (14, 'vector'), (6, 'none')])
def test_no_token_depends_on_a_later_one(L, gate):
    """A padded batch: streams of fewer drafts hold anything in the rows behind them."""
    at = L // 2
    c = make(2, L, 2, 64, 128, gate=gate, seed=61)
    o, state, pending, cache = run(c, [1, L])
    for t in (c['y'], c['beta']) + ((c['g_in'],) if c['g_in'] is not None else ()):
        t[:, at:] = float('nan')
    o2, state2, pending2, cache2 = run(c, [1, L])
    assert torch.equal(o[:, :at], o2[:, :at]) and torch.equal(state, state2)
    assert torch.equal(pending.u[:, :at], pending2.u[:, :at]) and torch.equal(pending.k[:, :at], pending2.k[:, :at])
    # an infinite value of one column stays in that column up to the norm over the row
    c = make(2, L, 2, 64, 128, gate=gate, epilogue=False, K=0, seed=62)
    o, _, pending, _ = run(c, [1, L])
    c['v_in'][:, at, 3] = float('inf')
    o2, _, pending2, _ = run(c, [1, L])
    assert torch.equal(o[:, :at], o2[:, :at]) and torch.equal(pending.u[:, :at], pending2.u[:, :at])


@pytest.mark.gpu
@pytest.mark.parametrize('gate', ['scalar', 'vector'])
def test_strong_decays(gate):
    """Log-decays of -inf, -1e30 and -200 between weak ones, in the pending block and the new one: what
    lies behind them is the recurrence's, not a difference of large sums."""
    for L in (7, 12):
        c = make(2, L, 2, 64, 64, gate=gate, act=False, K=0, epilogue=False, seed=70 + L)
        for t in (c['g'], c['g_in']):
            t[:, 1] = float('-inf')
            t[:, 3] = -1e30
            t[:, 5] = -200.0
        ref = reference(c, [L, 5])
        o, state, pending, cache = run(c, [L, 5])
        bar = (c['dk'] + 2 * L + 30) * 2.0 ** -24
        for x, want in ((o, ref['o']), (state, ref['state']), (pending.u[:, :L], ref['u'])):
            assert torch.isfinite(x).all()
            assert ((x.double().cpu() - want).norm() / want.norm()).item() <= bar


@pytest.mark.gpu
def test_commit_alone_and_steps_in_a_row():
    """Four steps with random counts and a last commit, against one walk over the tokens that stood."""
    N, L, H, dk, dv = 3, 5, 2, 64, 128
    for gate, dtype in (('scalar', torch.bfloat16), ('vector', torch.float32)):
        cs = [make(N, L, H, dk, dv, gate=gate, dtype=dtype, seed=80 + s) for s in range(4)]
        for c in cs[1:]:
            for name in ('w', 'gamma', 'A_log', 'dt_bias'):
                c[name] = cs[0][name]
        r = torch.Generator().manual_seed(5)
        counts = [[0] * N] + [torch.randint(0, L + 1, (N,), generator=r).tolist() for _ in range(4)]
        (_, _, _, state, pending, cache, _) = device(cs[0])
        ref = dict(state=cs[0]['state'], cache=cs[0]['cache'])
        prev = None
        for c, a in zip(cs, counts):
            c['state'], c['cache'] = ref['state'], ref['cache']
            if prev is not None:
                c['k'], c['u'], c['g'] = prev['k'], prev['u'], prev['g']
                c['x'] = [cp[n] for n in ('q_in', 'k_in', 'v_in')]
            (q, k, v), g, beta, _, _, _, kw = device(c)
            kw['conv_cache'] = cache
            o = ops.hip_draft_step(q, k, v, g, beta, state, pending, torch.tensor(a, device='cuda'), **kw)
            ref = reference(c, a)
            bar = 5 * (dk + 2 * L + 34) * 2.0 ** -24                   # the errors of up to five steps
            for x, want, half in ((o, ref['o'], HALF[dtype]), (state, ref['state'], 0.0)):
                assert ((x.double().cpu() - want).norm() / want.norm()).item() <= bar + half
            prev, cp = ref, c
        a = counts[4]
        before = [t.clone() for t in (pending.k, pending.u, *pending.x)]
        ops.commit_drafts(state, pending, torch.tensor(a, device='cuda'), conv_weights=kw['conv_weights'], conv_cache=cache)
        c = dict(cs[3], state=ref['state'], cache=ref['cache'], k=prev['k'], u=prev['u'], g=prev['g'],
                 x=[cp[n] for n in ('q_in', 'k_in', 'v_in')])
        want = reference(c, a)
        assert ((state.double().cpu() - want['state']).norm() / want['state'].norm()).item() <= bar
        assert all(torch.equal(x.cpu(), y) for x, y in zip(cache, want['cache']))
        assert all(torch.equal(x, y) for x, y in zip(before, (pending.k, pending.u, *pending.x)))


@pytest.mark.gpu
def test_streams_and_graphs():
    """The same bits on a side stream, and from a graph replayed between eager calls."""
    c = make(4, 5, 4, 128, 128, dtype=torch.bfloat16, seed=90)
    accepted = torch.tensor([0, 5, 2, 3], dtype=torch.int32, device='cuda')
    (q, k, v), g, beta, state, pending, cache, kw = device(c)
    held = (state, pending.k, pending.u, pending.g, *pending.x, *cache)
    start = [t.clone() for t in held]

    def reset():
        for t, s in zip(held, start):
            t.copy_(s)

    want = ops.hip_draft_step(q, k, v, g, beta, state, pending, accepted, **kw)
    after = [t.clone() for t in held]
    reset()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.hip_draft_step(q, k, v, g, beta, state, pending, accepted, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and all(torch.equal(t, s) for t, s in zip(held, after))
    reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.hip_draft_step(q, k, v, g, beta, state, pending, accepted, **kw)
    for _ in range(4):
        reset()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(torch.equal(t, s) for t, s in zip(held, after))
        reset()
        assert torch.equal(ops.hip_draft_step(q, k, v, g, beta, state, pending, accepted, **kw), want)


@pytest.mark.gpu
@pytest.mark.parametrize('L', [1, 4])
def test_layouts_of_the_inputs(L):
    """(N, L, H, d) operands, rows of one buffer at any place, transposed streams: the same bits."""
    c = make(3, L, 2, 64, 128, gate='vector', dtype=torch.bfloat16, seed=97)
    accepted = [0, L, 1]
    want, want_state = run(c, accepted)[:2]
    acc = torch.tensor(accepted, device='cuda')

    def again(f):
        (q, k, v), g, beta, state, pending, cache, kw = device(c)
        kw['out_gate'] = f(kw['out_gate'])
        g, beta = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (g, beta))
        return ops.hip_draft_step(f(q), f(k), f(v), g, beta, state, pending, acc, **kw), state

    shift = lambda t: torch.cat([t[..., :3], t], -1)[..., 3:]  # noqa: E731 -- rows 6 bytes off their alignment
    for f in (lambda t: t.view(3, L, 2, -1), shift, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
              lambda t: torch.cat([t, t], 1)[:, :L], lambda t: t.view(3, L, 2, -1).transpose(1, 2).contiguous().transpose(1, 2)):
        o, s = again(f)
        assert torch.equal(o, want) and torch.equal(s, want_state)


@pytest.mark.gpu
def test_no_streams():
    c = make(1, 3, 2, 64, 64, seed=95)
    (q, k, v), g, beta, state, pending, cache, kw = device(c)
    cut = lambda t: t[:0]  # noqa: E731
    p = ops.DraftBlock(cut(pending.k), cut(pending.u), cut(pending.g), [cut(t) for t in pending.x])
    kw.update(conv_cache=[cut(t) for t in cache], out_gate=cut(kw['out_gate']))
    o = ops.hip_draft_step(cut(q), cut(k), cut(v), cut(g), cut(beta), cut(state), p,
                           torch.zeros(0, dtype=torch.int32, device='cuda'), **kw)
    assert o.shape == (0, 3, 2, 64)


@pytest.mark.gpu
def test_refusals():
    c = make(2, 3, 2, 64, 64, seed=96)
    (q, k, v), g, beta, state, pending, cache, kw = device(c)
    acc = torch.zeros(2, dtype=torch.int32, device='cuda')
    call = lambda q=q, k=k, v=v, g=g, beta=beta, state=state, pending=pending, acc=acc, **over: ops.hip_draft_step(  # noqa: E731
        q, k, v, g, beta, state, pending, acc, **{**kw, **over})
    with pytest.raises(AssertionError, match='1 to 3 tokens'):
        call(*(torch.cat([t, t], 1) for t in (q, k, v)))
    with pytest.raises(AssertionError, match='1 to 3 tokens'):
        call(*(t[:, :0] for t in (q, k, v)))
    with pytest.raises(AssertionError, match='accepted'):
        call(acc=acc[:1])
    with pytest.raises(AssertionError, match='accepted'):
        call(acc=acc.float())
    with pytest.raises(AssertionError, match='accepted'):
        call(acc=acc.cpu().cuda().bool())
    with pytest.raises(AssertionError, match='state'):
        call(state=state.bfloat16())
    with pytest.raises(AssertionError, match='state'):
        call(state=state.transpose(2, 3))
    with pytest.raises(AssertionError, match='another gate'):
        call(g=None)
    with pytest.raises(AssertionError, match='conv'):
        call(conv_weights=None)
    with pytest.raises(AssertionError, match='conv cache'):
        call(conv_cache=[t[:, :3].contiguous() for t in cache])
    with pytest.raises(AssertionError, match='beta'):
        call(beta=None)
    with pytest.raises(AssertionError, match='no beta to activate'):
        call(delta=False)
    with pytest.raises(AssertionError, match='needs A_log'):
        call(gate_in_kernel=True)
    with pytest.raises(AssertionError, match='A_log has 2 and dt_bias 2'):
        call(gate_in_kernel=True, A_log=torch.zeros(2, device='cuda'), dt_bias=torch.zeros(128, device='cuda'))
    with pytest.raises(AssertionError, match='bounded'):
        call(gate_in_kernel=True, A_log=torch.zeros(2, device='cuda'), dt_bias=torch.zeros(2, device='cuda'), lower_bound=-2.0)
    with pytest.raises(NotImplementedError, match='share one'):
        call(k=k.half())
    with pytest.raises(NotImplementedError, match='backward'):
        call(q=q.clone().requires_grad_())
    with pytest.raises(RuntimeError, match='ROCm GPU'):
        call(q=q.cpu())
    with pytest.raises(NotImplementedError, match='1 to 16'):
        ops.DraftBlock.empty(state, 17, gate='scalar')
    s = torch.zeros(1, 1, 60, 64, device='cuda')
    z = torch.zeros(1, 1, 64, device='cuda')
    with pytest.raises(NotImplementedError, match='multiples of 8'):
        ops.hip_draft_step(z[..., :60], z[..., :60], z, None, torch.zeros(1, 1, 1, device='cuda'), s,
                           ops.DraftBlock.empty(s, 1, gate='none'), acc[:1], scale=1.0)


@pytest.mark.gpu
def test_without_a_gate_log_decays_are_not_looked_at():
    """The C entry without a gate: log-decays, or room for them in the block, change no bit and stay as they are."""
    c = make(3, 4, 2, 64, 64, gate='none', K=0, epilogue=False, l2norm=False, logits=False, seed=98)
    accepted = torch.tensor([0, 4, 2], dtype=torch.int32, device='cuda')
    lib = _lib.load()

    def call(g, room):
        (q, k, v), _, beta, state, pending, _, _ = device(c)
        pg = torch.full((3, 4, 2), -1.5, device='cuda') if room else None
        gs = torch.full((3, 4, 2), -0.5, device='cuda') if g else None
        blk = _lib.DraftBlock(pending.k.data_ptr(), pending.u.data_ptr(), pg.data_ptr() if room else None, None, None, None, 4)
        outs = []
        for L in (4, 0):                                   # a block behind the last one's, and its commit alone
            o = torch.zeros(3, 4, 2, 64, device='cuda')
            _lib.check(lib.vgdr_draft_step(
                _lib.VGDR_F32, _lib.VGDR_GATE_NONE, 1, q.data_ptr(), k.data_ptr(), v.data_ptr(), gs.data_ptr() if g else None,
                beta.data_ptr(), o.data_ptr(), state.data_ptr(), ctypes.byref(blk), accepted.data_ptr(), 3, L, 2, 64, 64, 128, 128,
                0.125, None, None, None, torch.cuda.current_stream().cuda_stream))
            outs += [o, state.clone()]
        assert not room or bool((pg == -1.5).all())
        return [*outs, pending.k, pending.u]

    want = call(False, False)
    for g, room in ((True, True), (False, True), (True, False)):
        assert all(torch.equal(x, y) for x, y in zip(call(g, room), want)), (g, room)


@pytest.mark.parametrize('dtype', [torch.int64, torch.uint32, torch.int32, torch.int16, torch.uint8])
def test_counts_of_wider_types_do_not_wrap(dtype):
    """Counts are clamped by the kernels: one that int32 does not hold must not come in as another."""
    counts = [n for n in (0, 5, 127, 2 ** 31 - 1, 2 ** 31, 2 ** 32 - 1, 2 ** 32 + 3, 2 ** 62, -1, -2 ** 32 + 3)
              if torch.iinfo(dtype).min <= n <= torch.iinfo(dtype).max]
    t = torch.tensor(counts, dtype=torch.int64).to(dtype)
    got = ops._stream_counts('counts', t, len(counts), -1)
    assert got.dtype == torch.int32
    room = 2 ** 31 - 1                                         # as the kernels clamp, for the largest room there is
    assert [min(max(n, 0), room) for n in got.tolist()] == [min(max(n, 0), room) for n in counts]


@pytest.mark.gpu
def test_counts_that_int32_does_not_hold():
    """2^32 + 1 accepted tokens are as many as there is room for, -2^32 + 1 are none."""
    c = make(2, 4, 2, 64, 64, seed=51)
    args, g, beta, state, pending, cache, kw = device(c)
    o = ops.hip_draft_step(*args, g, beta, state, pending, torch.tensor([2 ** 32 + 1, -2 ** 32 + 1], device='cuda'), **kw)
    check(c, o, state, pending, cache, reference(c, [4, 0]))


def _call(**over):
    blk = _lib.DraftBlock(16, 32, 48, 64, 80, 96, over.pop('P', 4))
    a = dict(dtype=1, gate=1, delta=1, q=16, k=32, v=48, g=64, beta=80, o=96, state=112, pending=blk, acc=128, B=2, L=3,
             H=2, dk=64, dv=64, ld_qk=128, ld_v=128, scale=1.0, fz=None, conv=None, ep=None)
    a.update(over)
    import ctypes
    ref = lambda s: None if s is None else ctypes.byref(s)  # noqa: E731
    return _lib.load().vgdr_draft_step(a['dtype'], a['gate'], a['delta'], a['q'], a['k'], a['v'], a['g'], a['beta'], a['o'],
                                       a['state'], ref(a['pending']), a['acc'], a['B'], a['L'], a['H'], a['dk'], a['dv'],
                                       a['ld_qk'], a['ld_v'], a['scale'], ref(a['fz']), ref(a['conv']), ref(a['ep']), None)


def test_entry_point_refuses_before_it_launches():
    """Every call here ends in its argument checks: there is no device."""
    bad, no = _lib.VGDR_ERR_INVALID, _lib.VGDR_ERR_UNSUPPORTED
    assert _call(dtype=7) == bad and _call(gate=3) == bad and _call(B=-1) == bad and _call(L=-1) == bad
    assert _call(L=5) == bad and b'room' in _lib.load().vgdr_last_error()
    assert _call(P=17) == no and _call(P=0) == no and _call(pending=None) == bad
    assert _call(dk=60) == no and _call(dk=136) == no and _call(dv=264) == no and _call(dv=0) == no
    assert _call(state=None) == bad and _call(acc=None) == bad and _call(q=None) == bad and _call(g=None) == bad
    assert _call(beta=None) == bad and _call(state=113) == bad and _call(q=18) == bad
    assert _call(ld_qk=120) == bad and _call(ld_v=132) == bad
    assert _call(pending=_lib.DraftBlock(16, 32, None, None, None, None, 4)) == bad
    conv = _lib.ShortConv(16, 32, 48, 64, 80, 96, 4, 1)
    assert _call(conv=conv, pending=_lib.DraftBlock(16, 32, 48, None, None, None, 4)) == bad
    assert _call(conv=_lib.ShortConv(16, 32, 48, 64, 80, 96, 9, 1)) == no
    assert _call(fz=_lib.Fusion(1, 1, 0, 0, None, None, 0, 0.0), delta=0) == bad
    assert _call(gate=0, fz=_lib.Fusion(1, 0, 1, 0, 16, 32, 0, 0.0)) == bad           # no gate to activate
    assert _call(fz=_lib.Fusion(1, 0, 1, 0, 16, 32, 1, -2.0)) == bad                  # the scalar gate has no bounded form
    assert _call(fz=_lib.Fusion(1, 0, 1, 0, None, 32, 0, 0.0)) == bad
    assert _call(ep=_lib.Epilogue(None, 16, 0, 1e-6)) == bad
    assert _call(H=1 << 19, ld_qk=1 << 25, ld_v=1 << 25) == no and _call(B=1 << 31) == no
    assert _call(B=0) == _lib.VGDR_OK


def test_more_heads_than_a_launch_holds_are_refused():
    """A workgroup of 128 (dk, dv up to 64), 256 (up to 128) or 512 threads a (stream, head): under 2^32 threads a launch."""
    no = _lib.VGDR_ERR_UNSUPPORTED
    for d, threads in (((64, 64), 128), ((128, 128), 256), ((128, 256), 512)):
        ld = [max(2 * n, 128) for n in d]
        assert _call(B=(1 << 31) // threads, H=2, dk=d[0], dv=d[1], ld_qk=ld[0], ld_v=ld[1]) == no
        assert b'too many' in _lib.load().vgdr_last_error()

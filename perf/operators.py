"""The operators of speculative decoding, measured: drafts looked up in a stream's
own text, a drafted block through a gated delta-rule layer whose state takes only
the tokens that stand, and the drafts' verification against the target's
probabilities.

    draft    ops.hip_draft_step: the last block's accepted tokens committed to the
             state and the conv caches, the next block's outputs formed, its own
             writes left pending; from the projections to the input of W_o
    verify   ops.verify_drafts: which drafts stand and the token after them, from
             given uniform numbers
    lookup   ops.lookup_drafts: what followed the latest earlier occurrence of a
             stream's last tokens

Where ``own`` is false ``run`` computes them in elementary torch operations.
``exact`` computes the same in 64 bits, token by token or by other formulas.
"""
from __future__ import annotations

import math

import torch

own = False

DT = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
SIZE = {'bf16': 2, 'fp16': 2, 'fp32': 4}
NEG = float('-inf')


def listed():
    return [
        # one stream of a 1.3B model's layer, four drafts behind the last token: latency
        dict(name='draft_one_stream', kind='draft', N=1, L=5, H=16, dk=128, dv=128, dtype='bf16', gate='scalar',
             delta=True, conv=4, epilogue=True),
        # 64 streams of that layer, the serving batch of the 1.3B generation workload
        dict(name='draft_b64', kind='draft', N=64, L=5, H=16, dk=128, dv=128, dtype='bf16', gate='scalar',
             delta=True, conv=4, epilogue=True),
        # a KDA layer of wide value heads, the gate's activation in the kernel
        dict(name='draft_kda_wide', kind='draft', N=64, L=8, H=4, dk=128, dv=256, dtype='bf16', gate='vector',
             delta=True, conv=4, epilogue=True),
        # the longest block on a large batch
        dict(name='draft_longest', kind='draft', N=128, L=16, H=16, dk=128, dv=128, dtype='bf16', gate='scalar',
             delta=True, conv=4, epilogue=True),
        # a toy model's heads of an odd number and size, fp32, without the conv and the epilogue
        dict(name='draft_odd_fp32', kind='draft', N=7, L=3, H=5, dk=48, dv=96, dtype='fp32', gate='vector',
             delta=True, conv=0, epilogue=False),
        # one greedy stream: latency
        dict(name='verify_greedy_one', kind='verify', N=1, K=4, V=32000, dtype='bf16', probs=False, temps='greedy'),
        # the 1.3B generation workload's batch and vocabulary, sampled
        dict(name='verify_b64', kind='verify', N=64, K=4, V=32000, dtype='bf16', probs=False, temps='one'),
        # drafts of a draft model with its probabilities, streams of their own temperatures, greedy ones among them
        dict(name='verify_probs', kind='verify', N=64, K=7, V=32000, dtype='bf16', probs=True, temps='mixed'),
        # an odd vocabulary, fp32 logits, few streams
        dict(name='verify_odd_fp32', kind='verify', N=5, K=3, V=50257, dtype='fp32', probs=True, temps='mixed'),
        # a large vocabulary and batch
        dict(name='verify_large', kind='verify', N=128, K=7, V=131072, dtype='bf16', probs=False, temps='one'),
        # the prompts and the text so far of the 1.3B generation workload's streams
        dict(name='lookup_b64', kind='lookup', N=64, cap=2304, K=4, longest=3, shortest=1, dtype='int64'),
        # long documents
        dict(name='lookup_long', kind='lookup', N=64, cap=131072, K=8, longest=4, shortest=2, dtype='int64'),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(['draft', 'draft', 'draft', 'verify', 'verify', 'lookup'])
    if kind == 'draft':
        N, L, H = _log(rng, 1, 128), rng.randint(1, 16), rng.choice([1, 2, 3, 4, 5, 8, 16])
        gate = rng.choice(['scalar', 'scalar', 'vector', 'none'])
        dk, dv = rng.choice([(64, 64), (128, 128), (128, 128), (128, 256), (64, 128), (128, 64), (48, 96), (96, 192)])
        N = max(1, min(N, 128 * 16 * 128 * 128 // (H * dk * dv), (1 << 28) // (H * L * L * dk) if gate == 'vector' else N))
        return dict(kind=kind, N=N, L=L, H=H, dk=dk, dv=dv, dtype=rng.choice(['bf16', 'bf16', 'fp16', 'fp32']), gate=gate,
                    delta=rng.random() < 0.85, conv=rng.choice([4, 4, 4, 3, 0]), epilogue=rng.random() < 0.8)
    if kind == 'verify':
        K, V = rng.randint(0, 8), _log(rng, 1000, 131072)
        probs = K > 0 and rng.random() < 0.5
        N = max(1, min(_log(rng, 1, 128), (1 << (24 if probs else 27)) // ((K + 1) * V)))
        return dict(kind=kind, N=N, K=K, V=V, dtype=rng.choice(['bf16', 'bf16', 'fp16', 'fp32']) if N * K * V < 1 << 26 else 'bf16',
                    probs=probs, temps=rng.choice(['one', 'mixed', 'mixed', 'greedy']))
    cap = _log(rng, 64, 131072)
    longest = rng.randint(1, 5)
    return dict(kind=kind, N=max(1, min(_log(rng, 1, 256), (1 << 23) // cap)), cap=cap, K=rng.randint(1, 15), longest=longest,
                shortest=rng.randint(1, longest), dtype=rng.choice(['int64', 'int32']))


# --- inputs ------------------------------------------------------------------


def _unit(x):
    return x / x.square().sum(-1, keepdim=True).sqrt()


def _prepare_draft(c, gen):
    """Streams some way into their text: the state, the conv caches and the last
    block's writes (its keys unit vectors, its decays logsigmoid(N + 4)); of that
    block 0 to all tokens stand. The new block's projections are column blocks of
    one product's output, the beta logits and a scalar log-decay the gate kernel's."""
    N, L, H, dk, dv, K = c['N'], c['L'], c['H'], c['dk'], c['dv'], c['conv']
    dt = DT[c['dtype']]

    def randn(*s):
        return torch.randn(*s, generator=gen, device='cuda')

    def decay(*s):
        return -torch.log1p(torch.exp(-(randn(*s) + 4)))

    gs = {'none': None, 'scalar': (H,), 'vector': (H, dk)}[c['gate']]
    s = dict(state=0.1 * randn(N, H, dk, dv), accepted=torch.randint(0, L + 1, (N,), generator=gen, device='cuda',
                                                                   dtype=torch.int32))
    s['pending'] = dict(k=_unit(randn(N, L, H, dk)), u=0.5 * randn(N, L, H, dv), g=None if gs is None else decay(N, L, *gs))
    y = randn(N, L, H * (2 * dk + 2 * dv)).to(dt)
    s['q'], s['k'], s['v'], s['out_gate'] = y.split([H * dk, H * dk, H * dv, H * dv], -1)
    s['beta'] = randn(N, L, H) if c['delta'] else None
    s['g'] = decay(N, L, H) if c['gate'] == 'scalar' else None
    if c['gate'] == 'vector':
        s['g'] = randn(N, L, H, dk).to(dt)                     # the activation's input
        r = torch.rand(H + H * dk, generator=gen, device='cuda')
        step = torch.exp(r[H:] * math.log(100.0) + math.log(1e-3))
        s['A_log'], s['dt_bias'] = (1 + 15 * r[:H]).log(), step + torch.log(-torch.expm1(-step))
    s['gamma'] = 1 + 0.1 * randn(dv) if c['epilogue'] else None
    if K:
        D = (H * dk, H * dk, H * dv)
        s['conv_weights'] = [(randn(d, K) / K ** 0.5).to(dt) for d in D]
        s['conv_cache'] = [randn(N, K, d).to(dt) for d in D]
        s['pending']['x'] = [randn(N, L, d).to(dt) for d in D]
    return s


def _prepare_verify(c, gen):
    """Logits of a peaked and a broad part: a draft has between a tenth and nine
    tenths of its row's mass, so some are refused; with probabilities, those of a
    draft model that is near the target; one stream in four has fewer drafts."""
    N, K, V = c['N'], c['K'], c['V']
    x = 2 * torch.randn(N, K + 1, V, generator=gen, device='cuda')
    drafts = torch.randint(0, V, (N, K), generator=gen, device='cuda')
    T = torch.ones(N, device='cuda')
    if c['temps'] == 'mixed':
        T = 0.3 + torch.rand(N, generator=gen, device='cuda')
        T = torch.where(torch.rand(N, generator=gen, device='cuda') < 0.2, torch.zeros_like(T), T)
    elif c['temps'] == 'greedy':
        T = torch.zeros_like(T)
    if K:
        peak = torch.rand(N, K, 1, generator=gen, device='cuda') * 4 - 1 + math.log(V) + 2
        x[:, :K].scatter_(2, drafts[..., None], peak)
    s = dict(logits=x.to(DT[c['dtype']]), drafts=drafts, temperature=T, draft_probs=None,
             uniforms=torch.rand(N, K + 1, generator=gen, device='cuda'))
    fewer = torch.rand(N, generator=gen, device='cuda') < 0.25
    some = torch.randint(0, K + 1, (N,), generator=gen, device='cuda', dtype=torch.int32)
    s['n_drafts'] = torch.where(fewer, some, torch.full_like(some, K))
    if c['probs']:
        near = x[:, :K] + 0.5 * torch.randn(N, K, V, generator=gen, device='cuda')
        s['draft_probs'] = torch.softmax(near, -1)
    return s


def _prepare_lookup(c, gen):
    """Text over 32,000 token ids in which phrases come again: every stream is
    copied, from a random place on, out of its own earlier part, and one in four
    ends in tokens that it has not had."""
    N, cap = c['N'], c['cap']
    dt = {'int64': torch.int64, 'int32': torch.int32}[c['dtype']]
    text = torch.randint(0, 32000, (N, cap), generator=gen, device='cuda', dtype=dt)
    n = torch.randint(max(1, cap // 2), cap + 1, (N, 1), generator=gen, device='cuda')
    at = torch.arange(cap, device='cuda')[None]
    back = 1 + (torch.rand(N, 1, generator=gen, device='cuda') * (n - 1)).long()   # how far back the copy comes from
    copied = 1 + (torch.rand(N, 1, generator=gen, device='cuda') * torch.clamp(n - back - 1, min=0)).long()
    fresh = torch.rand(N, 1, generator=gen, device='cuda') < 0.25
    source = torch.where((at >= n - torch.minimum(copied, back)) & (at >= back) & ~fresh, at - back, at)
    return dict(history=text.gather(1, source), lengths=n[:, 0].to(torch.int32))


def prepare(case, seed):
    gen = torch.Generator('cuda').manual_seed(seed)
    make = {'draft': _prepare_draft, 'verify': _prepare_verify, 'lookup': _prepare_lookup}[case['kind']]
    return dict(make(case, gen), case=dict(case))


# --- one pass ----------------------------------------------------------------


def _draft_own(s):
    from vagus_amd import ops
    c = s['case']
    p = s['pending']
    pending = ops.DraftBlock(k=p['k'], u=p['u'], g=p['g'], x=p.get('x'))
    more = dict(out_gate=s['out_gate'], out_norm_weight=s['gamma']) if c['epilogue'] else {}
    if c['gate'] == 'vector':
        more.update(gate_in_kernel=True, A_log=s['A_log'], dt_bias=s['dt_bias'])
    return ops.hip_draft_step(s['q'], s['k'], s['v'], s['g'], s['beta'], s['state'], pending, s['accepted'],
                              scale=c['dk'] ** -0.5, delta=c['delta'], beta_logits=c['delta'],
                              conv_weights=s.get('conv_weights'), conv_cache=s.get('conv_cache'), **more)


def _silu(x):
    return x / (1 + torch.exp(-x))


def _conv_plain(raw, weight, cache, pending, a):
    """SiLU of the causal conv of raw (N, L, D) behind the a accepted inputs of the
    last block, and the cache of the last K inputs up to there."""
    K, L = weight.shape[1], raw.shape[1]
    at = a.long()[:, None] + torch.arange(K, device=raw.device)
    kept = torch.cat([cache, pending], 1).gather(1, at[..., None].expand(-1, -1, cache.shape[2]))
    taps = torch.cat([kept[:, 1:], raw], 1).float().unfold(1, K, 1)               # (N, L, D, K)
    pending[:, :L].copy_(raw)
    cache.copy_(kept)
    return _silu((taps * weight.float()).sum(-1))


def _inverse_of_unit_lower(A):
    """(I + A)^-1 for strictly lower A of up to 16 rows: (I - A)(I + A^2)(I + A^4)(I + A^8)."""
    eye = torch.eye(A.shape[-1], device=A.device)
    A2 = A @ A
    A4 = A2 @ A2
    return (eye - A) @ (eye + A2) @ (eye + A4) @ (eye + A4 @ A4)


def _draft_plain(s):
    c, S, p = s['case'], s['state'], s['pending']
    N, L, H, dk, dv = c['N'], c['L'], c['H'], c['dk'], c['dv']
    a = s['accepted']
    stands = torch.arange(L, device=S.device) < a[:, None]                        # (N, P)
    # the accepted tokens' writes join the state, decayed by the tokens after them
    kw = torch.where(stands[..., None, None], p['k'], 0.0)
    uw = torch.where(stands[..., None, None], p['u'], 0.0)
    new = S
    if p['g'] is not None:
        gw = p['g'] if c['gate'] == 'vector' else p['g'][..., None]
        gw = torch.where(stands[..., None, None], gw, 0.0).double()
        kw = kw * torch.exp(gw.sum(1, keepdim=True) - gw.cumsum(1)).float()
        new = torch.exp(gw.sum(1)).float()[..., None] * S
    new = new + kw.permute(0, 2, 3, 1) @ uw.transpose(1, 2)                        # (N, H, dk, P) (N, H, P, dv)
    S.copy_(new)
    # the new block's q, k, v
    if c['conv']:
        q, k, v = (_conv_plain(r, w, cc, x, a) for r, w, cc, x in
                   zip((s['q'], s['k'], s['v']), s['conv_weights'], s['conv_cache'], p['x']))
    else:
        q, k, v = (s[n].float() for n in 'qkv')
    q, k, v = (t.reshape(N, L, H, -1).transpose(1, 2) for t in (q, k, v))         # (N, H, L, d)
    q, k = (t * torch.rsqrt(t.square().sum(-1, keepdim=True) + 1e-6) for t in (q, k))
    if c['gate'] == 'none':
        qg, kg, between = q, k, torch.ones(1, device=S.device)
        A, B = k @ k.transpose(2, 3), q @ k.transpose(2, 3)
    else:
        g = s['g']
        if c['gate'] == 'vector':
            z = g.float() + s['dt_bias'].view(H, dk)
            g = -torch.exp(s['A_log'])[:, None] * torch.where(z > 20, z, torch.log1p(torch.exp(z.clamp(max=20))))
        p['g'].copy_(g)
        G = (g if c['gate'] == 'vector' else g[..., None]).transpose(1, 2).double().cumsum(2)   # (N, H, L, dk or 1)
        qg, kg = (t * torch.exp(G).float() for t in (q, k))
        later = torch.ones(L, L, device=S.device).tril()[..., None] > 0
        between = torch.exp(torch.where(later, G[:, :, :, None] - G[:, :, None], NEG)).float()   # (N, H, t, j, dk or 1)
        A, B = (((t[:, :, :, None] * between) * k[:, :, None]).sum(-1) for t in (k, q))
    x = v
    if c['delta']:
        beta = (1 / (1 + torch.exp(-s['beta']))).transpose(1, 2)[..., None]
        x = _inverse_of_unit_lower((beta * A).tril(-1)) @ (beta * (v - kg @ new))
    o = c['dk'] ** -0.5 * (qg @ new + B.tril() @ x).transpose(1, 2)               # (N, L, H, dv)
    p['k'].copy_(k.transpose(1, 2))
    p['u'].copy_(x.transpose(1, 2))
    if c['epilogue']:
        gate = s['out_gate'].reshape(N, L, H, dv).float()
        o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + 1e-6) * s['gamma'] * _silu(gate)
    return o.to(s['q'].dtype)


def _verify_plain(s):
    x = s['logits'].double()
    N, L, V = x.shape
    K = L - 1
    drafts, u, T = s['drafts'], s['uniforms'].double(), s['temperature'].double()[:, None, None]
    top = x.amax(-1, keepdim=True)
    ids = torch.arange(V, device=x.device)
    lowest = torch.where(x == top, ids, V).amin(-1, keepdim=True)
    w = torch.where(T > 0, torch.exp((x - top) / torch.where(T > 0, T, 1.0)), (ids == lowest).double())
    p = w / w.sum(-1, keepdim=True)
    rows = torch.arange(N, device=x.device)
    n_drafts = s['n_drafts'].long()
    pd = p[:, :K].gather(2, drafts[..., None])[..., 0]
    qd = 1.0 if s['draft_probs'] is None else s['draft_probs'].gather(2, drafts[..., None])[..., 0].double()
    stands = (u[:, :K] * qd < pd) & (torch.arange(K, device=x.device) < n_drafts[:, None])
    accepted = stands.long().cumprod(1).sum(1)
    r = p[rows, accepted]
    if K:
        at = accepted.clamp(max=K - 1)
        taken = (ids == drafts[rows, at][:, None]).double() if s['draft_probs'] is None else s['draft_probs'][rows, at].double()
        left = torch.clamp(r - taken, min=0)
        refused = (accepted < n_drafts) & (left.sum(1) > 0)
        r = torch.where(refused[:, None], left, r)
    C = r.cumsum(1)
    token = (C <= u[:, K:] * C[:, -1:]).sum(1)
    at = torch.arange(L, device=x.device)
    tokens = torch.where(at < accepted[:, None], torch.cat([drafts, token[:, None]], 1), -1)
    return torch.where(at == accepted[:, None], token[:, None], tokens), accepted.to(torch.int32)


def _lookup_plain(s):
    c, h, n = s['case'], s['history'], s['lengths'].long()[:, None]
    cap, K = c['cap'], c['K']
    back = torch.arange(c['longest'], device=h.device)[:, None]
    ends = torch.arange(cap, device=h.device) - back                             # (longest, cap)
    last = h.gather(1, (n - 1 - back[:, 0]).clamp(min=0))                        # (N, longest): the last token first
    same = (h[:, ends.clamp(min=0)] == last[..., None]) & (ends >= 0)
    length = same.long().cumprod(1).sum(1)                                       # the suffix's length that ends there
    end = torch.arange(cap, device=h.device)
    key = torch.where((length >= c['shortest']) & (end < n - 1), length * cap + end, -1).amax(1, keepdim=True)
    start = key % cap + 1
    take = (start + torch.arange(K, device=h.device) % (n - start).clamp(min=1)).clamp(max=cap - 1)
    found = key >= 0
    return torch.where(found, h.gather(1, take).long(), 0), torch.where(found[:, 0], K, 0).to(torch.int32)


def run(state):
    s = state
    kind = s['case']['kind']
    if kind == 'draft':
        o = _draft_own(s) if own else _draft_plain(s)
        return dict(o=o, state=s['state'], cache=s.get('conv_cache'), pending=s['pending'])
    if own:
        from vagus_amd import ops
        if kind == 'verify':
            return ops.verify_drafts(s['logits'], s['drafts'], s['uniforms'], temperature=s['temperature'],
                                     draft_probs=s['draft_probs'], n_drafts=s['n_drafts'])
        c = s['case']
        return ops.lookup_drafts(s['history'], s['lengths'], c['K'], max_ngram=c['longest'], min_ngram=c['shortest'])
    return _verify_plain(s) if kind == 'verify' else _lookup_plain(s)


def work(case):
    c = case
    if c['kind'] == 'draft':
        e, N, L, H, dk, dv = SIZE[c['dtype']], c['N'], c['L'], c['H'], c['dk'], c['dv']
        g = {'none': 0, 'scalar': 4, 'vector': 4 * dk}[c['gate']]
        token = e * (2 * dk + (3 if c['epilogue'] else 2) * dv) + 4 + {'none': 0, 'scalar': 4, 'vector': e * dk}[c['gate']]
        half = 4 * (dk + dv) + g                                # a pending token: written; half of the last block's read
        raw = e * (2 * dk + dv) if c['conv'] else 0
        per = 8 * dk * dv + L * (token + 1.5 * half + 1.5 * raw) + 2 * c['conv'] * raw
        flops = 2 * dk * dv * (L / 2 + (2 if c['delta'] else 1) * L) + 2 * L * L * (dk + dv)
        return dict(bytes=N * H * per, flops=N * H * flops)
    if c['kind'] == 'verify':
        row = c['V'] * SIZE[c['dtype']]
        return dict(bytes=c['N'] * ((c['K'] + 1) * row + (4 * c['V'] if c['probs'] else 0)), flops=4.0 * c['N'] * (c['K'] + 1) * c['V'])
    return dict(bytes=0.75 * c['N'] * c['cap'] * (8 if c['dtype'] == 'int64' else 4), flops=0.75 * c['N'] * c['cap'])


# --- the same from the definitions, in 64 bits --------------------------------


def exact(case, seed):
    def draft(s):
        """Every token in turn: the accepted writes one by one, then the block walked on
        a copy of the state."""
        c, p = s['case'], s['pending']
        N, L, H, dk, dv, K = c['N'], c['L'], c['H'], c['dk'], c['dv'], c['conv']
        S, a, out = s['state'].double(), s['accepted'].long(), {}
        per_key = (lambda g: g.double().exp()[..., None] if c['gate'] == 'vector' else g.double().exp()[..., None, None])
        for t in range(L):
            step = S if p['g'] is None else per_key(p['g'][:, t]) * S
            step = step + p['k'][:, t].double()[..., None] * p['u'][:, t].double()[..., None, :]
            S = torch.where((t < a)[:, None, None, None], step, S)
        out['state'] = S
        x = {n: s[n].double() for n in 'qkv'}
        out['cache'] = None
        if K:
            out['cache'], pending_x = [], []
            for i, n in enumerate('qkv'):
                every = torch.cat([s['conv_cache'][i], p['x'][i]], 1)
                kept = torch.stack([every[b, a[b]:a[b] + K] for b in range(N)])
                out['cache'].append(kept)
                pending_x.append(s[n])
                line, w = torch.cat([kept, s[n]], 1).double(), s['conv_weights'][i].double()
                y = torch.stack([sum(w[:, j] * line[:, 1 + t + j] for j in range(K)) for t in range(L)], 1)
                x[n] = y * torch.sigmoid(y)
        q, k, v = (x[n].reshape(N, L, H, -1) for n in 'qkv')
        q, k = (t / torch.sqrt((t * t).sum(-1, keepdim=True) + 1e-6) for t in (q, k))
        g = s['g']
        if c['gate'] == 'vector':
            g = -s['A_log'].double().exp()[:, None] * torch.nn.functional.softplus(g.double() + s['dt_bias'].double().view(H, dk))
        M, o, u = S, [], []
        for t in range(L):
            M = M if g is None else per_key(g[:, t]) * M
            u.append(v[:, t] if not c['delta'] else
                     torch.sigmoid(s['beta'][:, t].double())[..., None] * (v[:, t] - (M * k[:, t][..., None]).sum(2)))
            M = M + k[:, t][..., None] * u[-1][..., None, :]
            o.append((M * q[:, t][..., None]).sum(2) / math.sqrt(dk))
        o = torch.stack(o, 1)
        if c['epilogue']:
            gate = s['out_gate'].double().reshape(N, L, H, dv)
            o = o / torch.sqrt((o * o).mean(-1, keepdim=True) + 1e-6) * s['gamma'].double() * gate * torch.sigmoid(gate)
        out['o'] = o
        out['pending'] = dict(k=k, u=torch.stack(u, 1), g=g)
        if K:
            out['pending']['x'] = pending_x
        return out

    def verify(s):
        """Stream by stream."""
        N, L, V = s['logits'].shape
        tokens, counts = torch.full((N, L), -1, dtype=torch.int64), torch.zeros(N, dtype=torch.int32)
        for b in range(N):
            x, T, n = s['logits'][b].double(), float(s['temperature'][b]), int(s['n_drafts'][b])
            if T > 0:
                p = torch.softmax(x / T, -1)
            else:
                p = torch.zeros_like(x)
                for i in range(L):
                    p[i, int((x[i] == x[i].max()).nonzero()[0])] = 1
            i = 0
            while i < n:
                d = int(s['drafts'][b, i])
                q = 1.0 if s['draft_probs'] is None else float(s['draft_probs'][b, i, d])
                if not float(s['uniforms'][b, i]) * q < float(p[i, d]):
                    break
                tokens[b, i] = d
                i += 1
            r = p[i].clone()
            if i < n:
                if s['draft_probs'] is None:
                    r[int(s['drafts'][b, i])] = 0
                else:
                    r = (r - s['draft_probs'][b, i].double()).clamp(min=0)
                r = r if float(r.sum()) > 0 else p[i]
            C = r.cumsum(0)
            tokens[b, i] = int(torch.searchsorted(C, float(s['uniforms'][b, L - 1]) * C[-1], right=True))
            counts[b] = i
        return tokens.cuda(), counts.cuda()

    def lookup(s):
        """Stream by stream, the longest suffix first."""
        c = s['case']
        N, K = c['N'], c['K']
        out, counts = torch.zeros(N, K, dtype=torch.int64), torch.zeros(N, dtype=torch.int32)
        for b in range(N):
            h = s['history'][b, :int(s['lengths'][b])]
            n = h.numel()
            for m in range(min(c['longest'], n - 1), c['shortest'] - 1, -1):
                at = (h[:-1].unfold(0, m, 1) == h[n - m:]).all(1).nonzero()
                if at.numel():
                    text, start = h.tolist(), int(at[-1]) + m
                    for i in range(K):
                        text.append(text[start + i])
                    out[b], counts[b] = torch.tensor(text[n:]), K
                    break
        return out.cuda(), counts.cuda()

    return {'draft': draft, 'verify': verify, 'lookup': lookup}[case['kind']](prepare(case, seed))

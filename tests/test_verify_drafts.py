"""Drafted tokens against the target's probabilities (ops.verify_drafts) and drafts looked up
in a stream's own text (ops.lookup_drafts), against plain code in 64 bits. The results are
whole numbers and have to be equal: weights and sums are 64-bit on both sides, so a border
falls on different sides only where a uniform number lies within some 2^-40 of it, and the
uniforms are multiples of 2^-24 drawn without regard to the borders.
"""
import pytest
import torch

from vagus_amd import _lib, ops


def reference(logits, drafts, uniforms, temperature, probs=None, n_drafts=None):
    """Stream by stream on the CPU."""
    N, L, V = logits.shape
    x = logits.double()
    x = torch.where(x.isnan(), float('-inf'), x)
    tokens, counts = torch.full((N, L), -1), torch.zeros(N, dtype=torch.int32)
    for b in range(N):
        T = float(temperature[b])
        p = torch.zeros(L, V, dtype=torch.float64)
        for i in range(L):
            top = x[b, i].max()
            if T > 0:
                w = torch.where(x[b, i] == top, 1.0, torch.exp((x[b, i] - top) / T))
                p[i] = w / w.sum()
            else:
                p[i, int((x[b, i] == top).nonzero()[0])] = 1
        n = L - 1 if n_drafts is None else max(0, min(L - 1, int(n_drafts[b])))
        i = 0
        while i < n:
            d = int(drafts[b, i])
            if not 0 <= d < V:
                break
            q = 1.0 if probs is None else float(probs[b, i, d])
            if not float(uniforms[b, i]) * q < float(p[i, d]):
                break
            tokens[b, i] = d
            i += 1
        r = p[i].clone()
        if i < n:
            d = int(drafts[b, i])
            if probs is not None:
                r = (r - probs[b, i].double()).clamp(min=0)
            elif 0 <= d < V:
                r[d] = 0
            r = r if float(r.sum()) > 0 else p[i]
        C = r.cumsum(0)
        tokens[b, i] = int((C > float(uniforms[b, L - 1]) * C[-1]).nonzero()[0])
        counts[b] = i
    return tokens, counts


def make(N, K, V, dtype=torch.bfloat16, probs=False, seed=0):
    r = torch.Generator().manual_seed(seed)
    x = 2 * torch.randn(N, K + 1, V, generator=r)
    drafts = torch.randint(0, V, (N, K), generator=r)
    if K:
        peak = torch.log(torch.tensor(float(V))) + 2 + 4 * torch.rand(N, K, 1, generator=r) - 1
        x[:, :K].scatter_(2, drafts[..., None], peak)
    q = torch.softmax(x[:, :K] + 0.5 * torch.randn(N, K, V, generator=r), -1) if probs else None
    return x.to(dtype), drafts, torch.rand(N, K + 1, generator=r), q


def check(x, drafts, u, T, q=None, n=None):
    mv = lambda t: t.cuda() if isinstance(t, torch.Tensor) else t  # noqa: E731
    tokens, counts = ops.verify_drafts(mv(x), mv(drafts), mv(u), temperature=mv(T), draft_probs=mv(q), n_drafts=mv(n))
    want = reference(x, drafts, u, T if isinstance(T, torch.Tensor) else [T] * x.shape[0], q, n)
    assert tokens.dtype == torch.int64 and counts.dtype == torch.int32
    assert torch.equal(counts.cpu(), want[1]), (counts.cpu(), want[1])
    assert torch.equal(tokens.cpu(), want[0])
    return tokens, counts


@pytest.mark.gpu
@pytest.mark.parametrize('N,K,V,dtype,probs', [
    (1, 4, 32000, torch.bfloat16, False), (3, 7, 32000, torch.bfloat16, True), (5, 3, 50257, torch.float32, True),
    (4, 1, 1, torch.float32, False), (6, 2, 2, torch.float16, True), (3, 0, 1001, torch.bfloat16, False),
    (2, 64, 300, torch.float16, True), (7, 5, 2047, torch.bfloat16, False), (7, 5, 2048, torch.float32, False),
    (7, 5, 2049, torch.float16, True), (2, 3, 131071, torch.bfloat16, True), (33, 8, 777, torch.bfloat16, True)])
def test_matches_plain_code(N, K, V, dtype, probs):
    for seed in range(3):
        x, d, u, q = make(N, K, V, dtype, probs, seed)
        print(f'\n[case] N {N} K {K} V {V} {dtype} probs {probs} seed {seed}', flush=True)
        r = torch.Generator().manual_seed(seed + 100)
        T = 0.2 + torch.rand(N, generator=r)
        T[torch.rand(N, generator=r) < 0.25] = 0
        n = torch.randint(0, K + 1, (N,), generator=r)
        for args in ((1.0, q, None), (T, q, n.int()), (0.0, q, n), (T, None, None), (0.05, None, n)):
            check(x, d, u, *args)
        if q is not None:
            check(x, d, u, T, q.to(torch.bfloat16), n)


@pytest.mark.gpu
def test_borders_of_the_uniform_numbers():
    """u = 0 takes a draft of any mass and the lowest id that has any; the largest u below 1 the last."""
    x, d, u, q = make(4, 3, 500, torch.float32, True, seed=4)
    for value in (0.0, 1 - 2.0 ** -24):
        check(x, d, torch.full_like(u, value), 1.0, q)
        check(x, d, torch.full_like(u, value), 0.0, q)
        check(x, d, torch.full_like(u, value), 0.7)


@pytest.mark.gpu
@pytest.mark.parametrize('V,dtype,probs', [(32000, torch.bfloat16, False), (1003, torch.float32, True), (131071, torch.float16, True)])
def test_uniforms_at_the_acceptance_border(V, dtype, probs):
    """Uniform numbers that are the fp32 neighbours of p(d) / q(d), half a step (2^-24) from it or less:
    what an fp32 sum cannot tell, and 64 bits can."""
    N = 24
    x, d, u, q = make(N, 2, V, dtype, probs, seed=12)
    if probs:
        q = q.to(torch.float16)
    p = torch.softmax(x.double(), -1)
    pd = p[:, :2].gather(2, d[..., None])[..., 0]
    if probs:
        pd = pd / q.double().gather(2, d[..., None])[..., 0]
    at = pd.float().clamp(max=1 - 2.0 ** -24)
    for way in (0.0, 2.0, None):
        u[:, :2] = at if way is None else torch.nextafter(at, torch.full_like(at, way)).clamp(0, 1 - 2.0 ** -24)
        _, counts = check(x, d, u, 1.0, q)
        if way is not None and not probs:
            assert int((counts > 0).sum()) == (N if way == 0.0 else 0)


@pytest.mark.gpu
def test_masks_infinities_and_nan():
    V = 600
    x, d, u, q = make(6, 2, V, torch.float32, True, seed=5)
    low = torch.finfo(torch.float32).min
    x[0, :, 1:] = float('-inf')                      # one token allowed
    x[1, :] = float('-inf')                          # none: every token alike
    x[2, :] = low                                    # none, by the type's lowest value
    x[3, :, ::2] = float('nan')                      # NaN has no mass
    x[4, :, 7] = float('inf')                        # +inf has all of it,
    x[4, :, 300] = float('inf')                      # shared
    x[5, :, :599] = low
    x[5, 0, 10] = float('nan')
    for T in (1.0, 0.3, 0.0):
        for probs in (None, q):
            for seed in range(4):
                u = torch.rand(6, 3, generator=torch.Generator().manual_seed(seed))
                tokens, _ = check(x, d, u, T, probs)
                assert int(tokens[:, 0].min()) >= 0 and int(tokens.max()) < V
    x[:] = float('nan')
    check(x, d, u, 1.0, q)


@pytest.mark.gpu
def test_drafts_outside_the_vocabulary_and_counts_outside_the_block():
    x, d, u, q = make(4, 3, 100, torch.float32, True, seed=6)
    d[0, 0], d[1, 1], d[2, 2] = -1, 100, 2 ** 40
    for T in (1.0, 0.0):
        for probs in (None, q):
            want = reference(x, d.clamp(-1, 100), u, [T] * 4, None if probs is None else probs)
            got = ops.verify_drafts(x.cuda(), d.cuda(), u.cuda(), temperature=T,
                                    draft_probs=None if probs is None else probs.cuda(),
                                    n_drafts=torch.tensor([3, 99, 3, 3], device='cuda'))
            assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    got = ops.verify_drafts(x.cuda(), d.cuda(), u.cuda(), n_drafts=torch.tensor([-4, 0, 0, 0], device='cuda'))
    assert torch.equal(got[1].cpu(), torch.zeros(4, dtype=torch.int32)) and bool((got[0][:, 1:] == -1).all())


@pytest.mark.gpu
def test_probabilities_that_cover_the_targets():
    """A refused draft whose q is p everywhere (or above): nothing is left over, the token comes from p."""
    x, d, u, _ = make(3, 2, 64, torch.float32, seed=7)
    q = torch.full((3, 2, 64), 2.0)
    u[:, :2] = 0.999
    check(x, d, u, 1.0, q)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_strided_rows(dtype):
    """Logits as a slice of a padded vocabulary, every second position, streams expanded."""
    x, d, u, q = make(3, 4, 1003, dtype, True, seed=8)
    want = ops.verify_drafts(x.cuda(), d.cuda(), u.cuda(), draft_probs=q.cuda())
    for pad in (1, 5, 21):
        wide = torch.full((3, 10, 1003 + pad), 9.0, dtype=dtype, device='cuda')
        wide[:, ::2, pad:] = x.cuda()
        qw = torch.full((3, 4, 1003 + pad), 9.0, device='cuda')
        qw[:, :, pad:] = q.cuda()
        got = ops.verify_drafts(wide[:, ::2, pad:], d.cuda(), u.cuda(), draft_probs=qw[:, :, pad:])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = ops.verify_drafts(x.cuda().transpose(0, 1).contiguous().transpose(0, 1), d.cuda(), u.cuda(), draft_probs=q.cuda())
    assert torch.equal(got[0], want[0])
    got = ops.verify_drafts(x.cuda().transpose(1, 2).contiguous().transpose(1, 2), d.cuda(), u.cuda(), draft_probs=q.cuda())
    assert torch.equal(got[0], want[0])
    one = x[:1].cuda().expand(3, -1, -1)
    got = ops.verify_drafts(one, d.cuda(), u.cuda())
    want = ops.verify_drafts(one.contiguous(), d.cuda(), u.cuda())
    assert torch.equal(got[0], want[0])


@pytest.mark.gpu
def test_tokens_follow_the_targets_distribution():
    """Drafts drawn from q, verified: the first token's frequencies are p's. 40,000 streams over 8 ids: a
    frequency is off by more than 6 standard deviations, sqrt(p (1 - p) / n), with probability 1e-8."""
    n, V = 40000, 8
    r = torch.Generator().manual_seed(9)
    x, q = torch.randn(V, generator=r) * 1.5, torch.softmax(torch.randn(V, generator=r) * 1.5, -1)
    d = torch.multinomial(q.expand(n, V), 1, generator=r)
    u = torch.rand(n, 2, generator=r)
    p = torch.softmax(x.double(), -1)
    logits = x.expand(n, 2, V).cuda()
    for probs in (q.expand(n, 1, V).cuda(), None):
        dd = d if probs is not None else torch.full((n, 1), 3)
        tokens, _ = ops.verify_drafts(logits, dd.cuda(), u.cuda(), draft_probs=probs)
        freq = torch.bincount(tokens[:, 0].cpu(), minlength=V).double() / n
        assert bool(((freq - p).abs() <= 6 * torch.sqrt(p * (1 - p) / n)).all()), (freq, p)


@pytest.mark.gpu
def test_streams_and_graphs():
    x, d, u, q = (t.cuda() for t in make(8, 4, 5000, torch.bfloat16, True, seed=10))
    want = ops.verify_drafts(x, d, u, draft_probs=q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.verify_drafts(x, d, u, draft_probs=q)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.verify_drafts(x, d, u, draft_probs=q)
        hist = torch.zeros(2, 40, dtype=torch.int64, device='cuda')
        looked = ops.lookup_drafts(hist, torch.full((2,), 40, device='cuda', dtype=torch.int32), 3)
    for step in range(4):
        u.copy_(torch.rand(8, 5, generator=torch.Generator().manual_seed(step)))
        graph.replay()
        torch.cuda.synchronize()
        want = ops.verify_drafts(x, d, u, draft_probs=q)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        assert looked[1].tolist() == [3, 3]


@pytest.mark.gpu
def test_two_graphs_replayed_in_turn():
    """Each recorded call has its own workspace; other work runs between the replays."""
    sides = []
    for seed in (1, 2):
        x, d, u, q = (t.cuda() for t in make(6, 3, 9001, torch.bfloat16, True, seed))
        h = torch.randint(0, 3, (3, 30000), device='cuda', generator=torch.Generator('cuda').manual_seed(seed))
        n = torch.tensor([30000, 7, 12345], device='cuda', dtype=torch.int32)
        ops.verify_drafts(x, d, u, draft_probs=q), ops.lookup_drafts(h, n, 5, max_ngram=16)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.verify_drafts(x, d, u, draft_probs=q) + ops.lookup_drafts(h, n, 5, max_ngram=16)
        sides.append((graph, out, (x, d, u, q, h, n)))
    for step in range(3):
        for graph, out, (x, d, u, q, h, n) in sides:
            u.copy_(torch.rand(6, 4, generator=torch.Generator().manual_seed(step)))
            h[1, :7] = torch.tensor([1, 2, step, 9, 1, 2, step], device='cuda')
        for graph, out, _ in sides + sides[::-1]:
            graph.replay()
        torch.cuda.synchronize()
        for graph, out, (x, d, u, q, h, n) in sides:
            want = ops.verify_drafts(x, d, u, draft_probs=q) + ops.lookup_drafts(h, n, 5, max_ngram=16)
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_more_streams_than_a_grid_dimension():
    n = 40000
    h = torch.arange(12, device='cuda').remainder(5).expand(n, 12).contiguous()
    h[:, -1] = torch.arange(n, device='cuda') % 5
    drafts, counts = ops.lookup_drafts(h, torch.full((n,), 12, device='cuda'), 2, max_ngram=2)
    want = [looked_up(h[b].tolist(), 12, 2, 2, 1) for b in range(5)]
    for b in range(5):
        assert bool((drafts[b::5] == torch.tensor(want[b][0], device='cuda')).all())
    assert bool((counts == 2).all())
    empty = ops.lookup_drafts(h[:3, :0], torch.tensor([0, 5, -1], device='cuda'), 2)
    assert empty[0].tolist() == [[0, 0]] * 3 and empty[1].tolist() == [0, 0, 0]


@pytest.mark.gpu
@pytest.mark.parametrize('K', [0, 1])
def test_eight_million_streams(K):
    """2^23 streams, sampled and greedy: the choosing workgroups' threads pass 2^32."""
    n, V = 1 << 23, 3
    r = torch.Generator('cuda').manual_seed(12)
    x = torch.randn(n, K + 1, V, generator=r, device='cuda')
    T = (torch.arange(n, device='cuda') % 4 > 0).float()
    drafts = torch.randint(0, V, (n, K), generator=r, device='cuda')
    u = torch.rand(n, K + 1, generator=r, device='cuda')
    tokens, accepted = ops.verify_drafts(x, drafts, u, temperature=T)
    p = torch.where(T[:, None, None] > 0, x.double().softmax(-1),
                    torch.nn.functional.one_hot(x.argmax(-1), V).double())
    stood = u[:, 0].double() < p[:, 0].gather(1, drafts)[:, 0] if K else torch.zeros(n, dtype=torch.bool, device='cuda')
    # the row behind what stands, without a refused draft
    rest = p[torch.arange(n, device='cuda'), stood.long()]
    if K:
        refused = (~stood[:, None] & (T[:, None] > 0)) & (torch.arange(V, device='cuda')[None] == drafts)
        rest = torch.where(refused, 0.0, rest)
    one, two = rest[:, 0], rest[:, 0] + rest[:, 1]
    goal = u[:, K].double() * (two + rest[:, 2])
    last = torch.where(one > goal, 0, torch.where(two > goal, 1, 2))
    want = torch.full((n, K + 1), -1, device='cuda')
    if K:
        want[:, 0] = torch.where(stood, drafts[:, 0], last)
        want[:, 1] = torch.where(stood, last, -1)
    else:
        want[:, 0] = last
    assert torch.equal(accepted, stood.int()) and torch.equal(tokens, want)


@pytest.mark.gpu
def test_refusals():
    x, d, u, q = (t.cuda() for t in make(2, 3, 50, torch.float32, True, seed=11))
    with pytest.raises(AssertionError, match='drafts'):
        ops.verify_drafts(x, d[:, :2], u)
    with pytest.raises(AssertionError, match='drafts'):
        ops.verify_drafts(x, d.float(), u)
    with pytest.raises(AssertionError, match='uniforms'):
        ops.verify_drafts(x, d, u[:, :3])
    with pytest.raises(AssertionError, match='uniforms'):
        ops.verify_drafts(x, d, u.double())
    with pytest.raises(AssertionError, match='temperature'):
        ops.verify_drafts(x, d, u, temperature=-1.0)
    with pytest.raises(AssertionError, match='temperature'):
        ops.verify_drafts(x, d, u, temperature=torch.ones(3, device='cuda'))
    with pytest.raises(AssertionError, match='draft_probs'):
        ops.verify_drafts(x, d, u, draft_probs=q[:, :2])
    with pytest.raises(AssertionError, match='n_drafts'):
        ops.verify_drafts(x, d, u, n_drafts=torch.ones(2, device='cuda'))
    with pytest.raises(NotImplementedError, match='logits'):
        ops.verify_drafts(x.double(), d, u)
    with pytest.raises(NotImplementedError, match='at most 64'):
        ops.verify_drafts(torch.zeros(1, 66, 4, device='cuda'), torch.zeros(1, 65, dtype=torch.int64, device='cuda'),
                          torch.zeros(1, 66, device='cuda'))
    with pytest.raises(NotImplementedError, match='backward'):
        ops.verify_drafts(x.clone().requires_grad_(), d, u)
    with pytest.raises(RuntimeError, match='ROCm GPU'):
        ops.verify_drafts(x.cpu(), d, u)
    h = torch.zeros(2, 9, dtype=torch.int64, device='cuda')
    n = torch.full((2,), 9, device='cuda')
    with pytest.raises(AssertionError, match='64 drafts'):
        ops.lookup_drafts(h, n, 0)
    with pytest.raises(AssertionError, match='ngram'):
        ops.lookup_drafts(h, n, 3, max_ngram=1, min_ngram=2)
    with pytest.raises(NotImplementedError, match='int32 or int64'):
        ops.lookup_drafts(h.float(), n, 3)
    with pytest.raises(AssertionError, match='lengths'):
        ops.lookup_drafts(h, n[:1], 3)
    tokens, counts = ops.verify_drafts(x[:0], d[:0], u[:0])
    assert tokens.shape == (0, 4) and counts.shape == (0,)
    assert ops.lookup_drafts(h[:0], n[:0], 3)[0].shape == (0, 3)


def looked_up(row, n, K, longest, shortest):
    text = row[:max(0, min(n, len(row)))]
    n = len(text)
    for m in range(min(longest, n - 1), shortest - 1, -1):
        for s in range(n - 1 - m, -1, -1):
            if text[s:s + m] == text[n - m:]:
                out = list(text)
                for i in range(K):
                    out.append(out[s + m + i])
                return out[n:], K
    return [0] * K, 0


@pytest.mark.gpu
@pytest.mark.parametrize('N,cap,K,longest,shortest,ids,dtype', [
    (3, 1, 2, 3, 1, 3, torch.int64), (4, 2, 3, 3, 1, 2, torch.int64), (9, 40, 5, 3, 1, 4, torch.int64),
    (9, 300, 7, 4, 2, 6, torch.int32), (5, 1000, 15, 16, 1, 2, torch.int64), (6, 513, 4, 2, 2, 30, torch.int32),
    (3, 5000, 64, 3, 3, 12, torch.int64), (2, 40000, 8, 5, 2, 50, torch.int32)])
def test_lookup_matches_plain_code(N, cap, K, longest, shortest, ids, dtype):
    for seed in range(3):
        r = torch.Generator().manual_seed(seed)
        wide = torch.randint(0, ids, (N, cap + 3), generator=r).to(dtype)
        n = torch.randint(0, cap + 1, (N,), generator=r)
        n[0], n[-1] = cap, min(cap, 2)
        for h in (wide[:, :cap].contiguous(), wide[:, :cap], wide[:, 3:]):
            wide_dev = wide.cuda()
            hd = h.cuda() if h.is_contiguous() else wide_dev[:, :cap] if h.data_ptr() == wide.data_ptr() else wide_dev[:, 3:]
            drafts, counts = ops.lookup_drafts(hd, n.cuda(), K, max_ngram=longest, min_ngram=shortest)
            for b in range(N):
                want = looked_up(h[b].tolist(), int(n[b]), K, longest, shortest)
                assert (drafts[b].tolist(), int(counts[b])) == (want[0], want[1]), (seed, b)


@pytest.mark.gpu
def test_lookup_takes_the_longest_then_the_latest():
    rows = [[1, 2, 3, 9, 9, 7, 3, 8, 8, 1, 2, 3],            # the trigram at 0 before the 3 at 6
            [5, 1, 5, 2, 5, 0, 0, 0, 0, 0, 0, 5],            # the latest 5
            [4, 4, 4, 4, 4, 4, 4, 4, 4, 4, 4, 4],            # a period of one
            [1, 2, 1, 2, 1, 2, 1, 2, 1, 2, 1, 2],            # of two
            [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12]]         # nothing
    h = torch.tensor(rows, device='cuda')
    drafts, counts = ops.lookup_drafts(h, torch.full((5,), 12, device='cuda'), 4)
    assert counts.tolist() == [4, 4, 4, 4, 0]
    assert drafts.tolist() == [[9, 9, 7, 3], [0, 0, 0, 0], [4] * 4, [1, 2, 1, 2], [0] * 4]
    _, counts = ops.lookup_drafts(h, torch.tensor([-3, 0, 1, 2, 99], device='cuda'), 4)
    assert counts.tolist() == [0, 0, 0, 0, 0]


def test_entry_points_refuse_before_they_launch():
    L, bad = _lib.load(), _lib.VGDR_ERR_INVALID

    def verify(**over):
        a = dict(dt=1, x=16, ls=400, lr=100, d=32, u=48, T=64, q=None, qdt=0, qs=0, qr=0, n=None, tok=80, acc=96, ws=112,
                 nb=1 << 20, B=2, K=3, V=100)
        a.update(over)
        return L.vgdr_verify_drafts(*a.values(), None)
    assert verify(dt=5) == bad and verify(B=-1) == bad and verify(V=0) == bad and verify(x=None) == bad
    assert verify(K=65) == _lib.VGDR_ERR_UNSUPPORTED and verify(lr=99) == bad and verify(q=16, qr=99) == bad
    assert verify(q=16, qdt=9, qr=100) == bad and verify(ws=None) == bad and verify(nb=1) == bad and verify(u=None) == bad
    assert verify(B=0) == _lib.VGDR_OK
    assert L.vgdr_verify_drafts_workspace_size(2, 3, 0) == 0

    def lookup(**over):
        a = dict(h=16, tb=8, ld=100, cap=100, n=32, d=48, c=64, ws=80, nb=1 << 20, B=2, K=3, hi=3, lo=1)
        a.update(over)
        return L.vgdr_lookup_drafts(*a.values(), None)
    assert lookup(tb=2) == bad and lookup(ld=99) == bad and lookup(K=0) == bad and lookup(K=65) == bad
    assert lookup(hi=17) == bad and lookup(lo=0) == bad and lookup(hi=1, lo=2) == bad and lookup(h=None) == bad
    assert lookup(cap=-1) == bad and lookup(B=0) == _lib.VGDR_OK


def test_row_counts_past_64_bits_are_refused():
    """B (K + 1) rows are counted without an overflow."""
    L = _lib.load()
    for B, K in ((1 << 62, 3), ((1 << 63) - 1, 1), (1 << 24, 1)):
        assert L.vgdr_verify_drafts_workspace_size(B, K, 100) == 0 and b'too many rows' in L.vgdr_last_error()
        rc = L.vgdr_verify_drafts(0, 16, 400, 100, 32, 48, 64, None, 0, 0, 0, None, 80, 96, 112, 1 << 62, B, K, 100, None)
        assert rc == _lib.VGDR_ERR_INVALID and b'too many rows' in L.vgdr_last_error()

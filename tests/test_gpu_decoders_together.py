"""Windowed attention, linear attention and the choice of a token together on the GPU: a model that trains with them and answers
with them, the calls that a model makes beside the plain ones, and sizes whose offsets pass 32 bits."""
import numpy as np
import pytest
import torch

import _decoders as D
import _sequence as R
from tensorgrad_amd import nn
from tensorgrad_amd import ops as O
from tensorgrad_amd.compile import compile_forward
from tensorgrad_amd.compile import compile as tg_compile
from tensorgrad_amd.module import Module
from test_gpu_decoders import check_linear, check_sample, check_window, decays, f32, forward, linear_inputs, rng

pytestmark = pytest.mark.gpu

VOCAB, DIM, HEADS, KV, WINDOW, SINKS = 29, 32, 4, 2, 6, 2
SLOPES = [0.5, 0.25, 0.125, 0.0625]
DECAY = [0.5, 0.9, 0.97, 1.0]


class Model(Module):
    """A layer that looks at a window and the first positions, and one that carries a state."""

    def __init__(self):
        self.emb = nn.Embedding(VOCAB, DIM)
        for a in ('w', 'l'):
            for n, d in (('q', DIM), ('k', DIM * KV // HEADS), ('v', DIM * KV // HEADS), ('o', DIM)):
                setattr(self, a + n, nn.Linear(DIM, d, bias=False))
        self.head = nn.Linear(DIM, VOCAB)


def heads_of(p, a, x):
    return (O.split_heads(getattr(p, a + n).fwd(x), h) for n, h in (('q', HEADS), ('k', KV), ('v', KV)))


def after(p, x, y, i, lengths=None):
    """What follows the first attention's result y: (logits, the last state)."""
    x = O.add(x, p.wo.fwd(O.merge_heads(y)))
    q, k, v = heads_of(p, 'l', x)
    y, state = O.linear_attention(q, k, v, DECAY, state=i['state'], documents=i.get('documents'), lengths=lengths)
    return p.head.fwd(O.add(x, p.lo.fwd(O.merge_heads(y)))), state


def logits_of(p, i):
    x = p.emb.fwd(i['tokens'])
    q, k, v = heads_of(p, 'w', x)
    return after(p, x, O.attention(q, k, v, slopes=SLOPES, window=WINDOW, documents=i['documents']), i)[0]


def plain_logits(w, tokens, documents, state, sinks):
    """The same in f64 torch, for autograd: one pair of positions at a time through masks, no states but the given one."""
    B, T = tokens.shape
    at = torch.arange(T)
    far = (at[:, None] - at[None, :]).double()
    x = w['emb.W'][tokens.long()]

    def heads(a, x):
        h = lambda n, h: (x @ w[f'{a}{n}.W']).reshape(B, T, h, -1).transpose(1, 2)  # noqa: E731
        return h('q', HEADS), h('k', KV).repeat_interleave(HEADS // KV, 1), h('v', KV).repeat_interleave(HEADS // KV, 1)
    back = lambda y, o: y.transpose(1, 2).reshape(B, T, DIM) @ w[o + '.W']  # noqa: E731
    d = documents
    there = (d >= 0)[:, None, :] & (d >= 0)[:, :, None] & (far >= 0)
    same = torch.ones(B, T, T, dtype=torch.bool)             # no other document between
    for b in range(B):
        for t in range(T):
            for s in range(t):
                same[b, t, s] = bool((d[b, s:t + 1] == d[b, t]).all())
    q, k, v = heads('w', x)
    ok = (there & (d[:, :, None] == d[:, None, :]) & ((far < WINDOW) | (at < sinks)))[:, None]
    sc = q @ k.transpose(-1, -2) / 8 ** 0.5 - torch.tensor(SLOPES).double()[:, None, None] * far.abs()
    P = torch.softmax(sc.masked_fill(~ok, -1e300), -1).masked_fill(~ok, 0)
    x = x + back(P @ v, 'wo')
    q, k, v = heads('l', x)
    lam = torch.tensor(DECAY).double()[:, None, None]
    W = torch.where((there & same)[:, None], lam ** far.clamp(min=0), 0.0)
    opens = (there & same)[:, None, :, 0]                    # the given state reaches what goes on from position 0
    c = torch.where(opens, lam[:, :, 0] ** (at + 1).double(), 0.0)
    y = ((W * (q @ k.transpose(-1, -2))) @ v + c[..., None] * (q @ state.double())) / 8 ** 0.5
    return (x + back(y, 'lo')) @ w['head.W'] + w['head.b']


def batch_of(B, T, seed):
    r = rng(B, T, seed)
    doc = np.sort(r.integers(0, 3, (B, T), dtype=np.int32), 1)
    doc[:, T - 2:] = -1
    return {'tokens': r.integers(0, VOCAB, (B, T), dtype=np.int32), 'targets': r.integers(0, VOCAB, (B, T), dtype=np.int32),
            'documents': doc, 'state': f32(r.standard_normal((B, HEADS, 8, 8)))}


def decl_of(arrays):
    return {n: {'shape': list(a.shape), 'dtype': 'i32' if a.dtype == np.int32 else 'f32'} for n, a in arrays.items()}


def trainer(batch, optimizer, seed):
    return tg_compile(Model(), lambda p, i: nn.cross_entropy(logits_of(p, i), i['targets']), decl_of(batch), optimizer, seed=seed)


@pytest.mark.parametrize('B,T', [(2, 12), (2, 150)])
def test_a_model_of_them_trains_as_in_64_bits(B, T):
    """One SGD step at rate 1 from known weights: what the weights moved by is the gradient. Chains of some ten f32 operations and
    sums over B T positions: 2e-5 of each gradient's norm is about 300 roundings."""
    batch = batch_of(B, T, 1)
    t = trainer(batch, {'kind': 'sgd', 'lr': 1.0}, 3)
    before = t.download_params()
    shapes = t.ir.param_shapes()
    r = t.step(batch)
    assert r.kind == 'completed', r.error
    moved = t.download_params()
    w = {n: torch.from_numpy(a.reshape(shapes[n])).double().requires_grad_(True) for n, a in before.items()}
    i = {n: torch.from_numpy(a) for n, a in batch.items()}
    logits = plain_logits(w, i['tokens'], i['documents'], i['state'], 0)
    loss = torch.nn.functional.cross_entropy(logits.reshape(-1, VOCAB), i['targets'].long().reshape(-1))
    assert abs(r.loss - float(loss.detach())) <= 1e-5 * abs(float(loss.detach()))
    for n, g in zip(w, torch.autograd.grad(loss, list(w.values()))):
        got = (before[n].astype(np.float64) - moved[n]).reshape(shapes[n])
        # the difference of two f32 weights carries their own rounding
        assert np.linalg.norm(got - g.numpy()) <= 2e-5 * np.linalg.norm(g) + 2 * R.U * np.linalg.norm(before[n]), n
    kinds = [n['kind'] for n in t._rt.describe()['nodes']]
    assert [kinds.count(k) for k in ('attend', 'attend_grad', 'linear', 'linear_grad')] == [1, 1, 1, 1]
    t.destroy()


def test_a_model_of_them_steps_alike_captured_and_launched(monkeypatch):
    """Captured steps, replayed with eager work and waits between, against steps launched one by one: the same bits."""
    batches = [batch_of(2, 300, n) for n in range(5)]

    def train(graph):
        monkeypatch.setenv('TG_GRAPH', graph)
        t = trainer(batches[0], {'kind': 'adam', 'lr': 0.01}, 4)
        losses = []
        for b in batches:
            r = t.step(b)
            assert r.kind == 'completed', r.error
            losses.append(r.loss)
            torch.randn(1 << 20, device='cuda').sum()
            torch.cuda.synchronize()
        w = t.download_params()
        t.destroy()
        return losses, w
    (l0, w0), (l1, w1) = train('0'), train('1')
    assert l0 == l1 and all(np.array_equal(w0[n], w1[n]) for n in w0)


def test_a_model_of_them_answers():
    """Prompts of uneven length read at once, then a token at a time from the cache and the state, on a stream of its own without
    a wait on the host: each step's logits as of the whole sequence in 64 bits, each token as chosen from them."""
    B, T, MORE = 3, 12, 20
    cap = T + MORE
    r = rng(41)
    n = np.array([7, 12, 1], np.int32)
    batch = batch_of(B, T, 5)
    t = trainer(batch, {'kind': 'sgd', 'lr': 0.1}, 6)
    shapes = t.ir.param_shapes()
    w = {m: torch.from_numpy(a.reshape(shapes[m])).double() for m, a in t.download_params().items()}

    def prompt(p, i):
        x = p.emb.fwd(i['tokens'])
        q, k, v = heads_of(p, 'w', x)
        y = O.attention(q, k, v, slopes=SLOPES, window=WINDOW, sinks=SINKS)
        logits, state = after(p, x, y, i, i['lengths'])
        return [logits, O.mul(k, 1.0), O.mul(v, 1.0), state]

    def keys(p, i):                                          # of one new position
        x = p.emb.fwd(i['tokens'])
        return [O.mul(z, 1.0) for z in (x, *heads_of(p, 'w', x))]

    def answer(p, i):
        y = O.attention(i['q'], i['k'], i['v'], slopes=SLOPES, window=WINDOW, sinks=SINKS, lengths=i['lengths'])
        logits, state = after(p, i['x'], y, i)
        logits = O.reshape(logits, [B, VOCAB])
        return [logits, state, O.sample(logits, i['u'], temperature=0.8, top_k=9, top_p=0.95)]
    tokens = batch['tokens']
    state = np.zeros((B, HEADS, 8, 8), np.float32)
    one = {'q': [B, HEADS, 1, 8], 'k': [B, KV, cap, 8], 'v': [B, KV, cap, 8], 'x': [B, 1, DIM], 'state': list(state.shape), 'u': [B],
           'lengths': {'shape': [B], 'dtype': 'i32'}}
    f = t.attach(prompt, decl_of({'tokens': tokens, 'lengths': n, 'state': state}))
    g = t.attach(keys, {'tokens': {'shape': [B, 1], 'dtype': 'i32'}})
    h = t.attach(answer, one)
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    new = lambda *s: torch.empty(s, device='cuda')  # noqa: E731
    u = f32(r.random((MORE, B)))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    logits, chosen, keep = [], [], []
    with torch.cuda.stream(stream):
        def call(ex, ins, outs):
            res = ex.run_device(ins, outs, stream.cuda_stream)
            assert res.error is None, res.error
            keep.append((ins, outs))
            return outs
        first, k0, v0, s = call(f, {'tokens': dev(tokens), 'lengths': dev(n), 'state': dev(state)},
                                [new(B, T, VOCAB), new(B, KV, T, 8), new(B, KV, T, 8), new(B, HEADS, 8, 8)])
        kc, vc = (torch.full((B, KV, cap, 8), float('nan'), device='cuda') for _ in range(2))
        for b in range(B):
            kc[b, :, :n[b]], vc[b, :, :n[b]] = k0[b, :, :n[b]], v0[b, :, :n[b]]
        rows = torch.arange(B, device='cuda')
        at = dev(n).long()
        now = torch.stack([first[b, n[b] - 1] for b in range(B)])
        token = now.argmax(1).int()
        start = token.clone()
        for step in range(MORE):
            x, q, k1, v1 = call(g, {'tokens': token[:, None].contiguous()}, [new(B, 1, DIM), new(B, HEADS, 1, 8), new(B, KV, 1, 8), new(B, KV, 1, 8)])
            kc[rows, :, at], vc[rows, :, at] = k1[:, :, 0], v1[:, :, 0]
            at = at + 1
            lg, s, token = call(h, {'q': q, 'k': kc.clone(), 'v': vc.clone(), 'x': x, 'state': s, 'u': dev(u[step]), 'lengths': at.int()},
                                [new(B, VOCAB), new(B, HEADS, 8, 8), torch.empty(B, dtype=torch.int32, device='cuda')])
            logits.append(lg)
            chosen.append(token)
    torch.cuda.synchronize()
    first = first.cpu().numpy()
    for b in range(B):
        said = [int(start[b])] + [int(c[b]) for c in chosen]
        seq = np.concatenate([tokens[b, :n[b]], np.array(said[:MORE], np.int32)])
        want = plain_logits(w, torch.from_numpy(seq)[None], torch.zeros(1, len(seq), dtype=torch.int32), torch.from_numpy(state[:1]), SINKS)[0].numpy()
        # chains of some ten f32 operations on sums of some hundred terms, as above
        assert np.linalg.norm(first[b, :n[b]] - want[:n[b]]) <= 1e-5 * np.linalg.norm(want[:n[b]])
        got = np.stack([x[b].cpu().numpy() for x in logits])
        assert np.linalg.norm(got - want[n[b]:]) <= 1e-5 * np.linalg.norm(want[n[b]:])
        for step in range(MORE):
            assert said[step + 1] == D.sample(got[step], float(u[step, b]), 0.8, 9, 0.95), (b, step)
    t.destroy()


# ---- other calls ------------------------------------------------------------------------------------

def test_calls_follow_the_stream():
    """Producer, call and consumer on one stream, then on several, without the host waiting between: workspaces are one call's at a
    time."""
    a = linear_inputs(1, 4, 2, 700, 64, 64, 51, True)
    a['logits'], a['u'] = f32(3 * rng(52).standard_normal((3, 40000))), f32(rng(53).random(3))

    def fn(m, i):
        y, s = O.linear_attention(i['q'], i['k'], i['v'], decays(4), state=i['state'])
        z = O.attention(i['q'], i['k'], i['v'], window=90, sinks=3)
        grads = [*O.linear_attention_grad(i['q'], i['k'], i['v'], i['dy'], decays(4), state=i['state'], dstate=i['dstate']),
                 *O.attention_grad(i['q'], i['k'], i['v'], z, i['dy'], window=90, sinks=3)]
        return [y, s, z, *grads, O.sample(i['logits'], i['u'], temperature=0.9, top_p=0.9)]
    ex = compile_forward(Module(), fn, decl_of(a), seed=0)
    g = ex.graph_for(a).graph
    new = lambda: [torch.empty(g.tensors[t].shape, device='cuda', dtype=torch.int32 if g.tensors[t].dtype == 'i32' else torch.float32)  # noqa: E731
                   for t in g.outputs]
    first, second = ({n: torch.from_numpy(x if k == 0 or n == 'u' else x[..., ::-1].copy()).cuda() for n, x in a.items()} for k in (0, 1))
    torch.cuda.synchronize()
    wants = []
    for ins in (first, second):
        o = new()
        assert ex.run_device(ins, o).error is None
        torch.cuda.synchronize()
        wants.append([x.cpu() for x in o])
    streams, keep = [torch.cuda.Stream() for _ in range(3)], []
    for turn in range(9):
        with torch.cuda.stream(streams[turn % 3]):
            ins = {n: x.clone() for n, x in (first, second)[turn % 2].items()}
            o = new()
            assert ex.run_device(ins, o, streams[turn % 3].cuda_stream).error is None
            keep.append((ins, [x.clone() for x in o], o))
    torch.cuda.synchronize()
    for turn, (_, got, _) in enumerate(keep):
        for x, want in zip(got, wants[turn % 2]):
            assert torch.equal(x.cpu(), want), turn
    ex.destroy()


@pytest.mark.parametrize('T', [1, 300])
def test_linear_gradients_of_the_state_alone_with_wide_values(T):
    """No gradient of y, and values of many more features than the queries have."""
    a = linear_inputs(1, 1, 1, T, 4, 128, 61, True)
    del a['dy']
    check_linear(a, [0.9])


@pytest.mark.parametrize('T', [40, 300])
def test_linear_queries_get_no_gradient_from_an_infinite_state_alone(T):
    """Without a gradient of y nothing reaches the queries, whatever the state holds."""
    a = linear_inputs(1, 2, 1, T, 32, 32, 68, True)
    a['state'][0, 0, 3, 4], a['state'][0, 1, 5, 6] = np.inf, np.nan
    a['v'][0, 0, T // 2, 7] = np.inf
    def fn(i):
        return list(O.linear_attention_grad(i['q'], i['k'], i['v'], None, decays(2), state=i['state'], dstate=i['dstate']))
    dq, _, dv, _ = forward(fn, {n: x for n, x in a.items() if n != 'dy'})
    assert not dq.any() and np.isfinite(dv).all()


@pytest.mark.parametrize('shape', [(16, 4, 2, 512, 16, 16), (9, 6, 2, 900, 32, 20), (2, 4, 2, 140, 16, 19)])
def test_linear_shared_heads_in_turn_and_apart(shape):
    """Enough blocks that one takes all query heads of a key head, and so few that each is taken alone."""
    check_linear(linear_inputs(*shape, 62, True), decays(shape[1]), what=str(shape))


@pytest.mark.parametrize('T', [128, 129, 400])
@pytest.mark.parametrize('size', [16, 15], ids=['aligned', 'odd'])
def test_linear_gradients_without_the_forward_of_heads_in_place(T, size):
    """Gradients alone, of heads that are strided views of one product, written to heads of one."""
    C = 4 * size
    r = rng(T, size, 63)
    a = {n: f32(r.standard_normal((2, T, C))) for n in ('q', 'k', 'v', 'dy')}

    def fn(i):
        q, k, v, dy = (O.split_heads(O.mul(i[n], 1.0), 4) for n in ('q', 'k', 'v', 'dy'))
        return [O.merge_heads(x) for x in O.linear_attention_grad(q, k, v, dy, decays(4))]
    got = forward(fn, a)
    heads = {n: x.reshape(2, T, 4, size).transpose(0, 2, 1, 3) for n, x in a.items()}
    want, tol = D.linear(heads['q'], heads['k'], heads['v'], decays(4), dy=heads['dy'])
    for n, x in zip(('dq', 'dk', 'dv'), got):
        R.check(x, *(z[n].transpose(0, 2, 1, 3).reshape(2, T, C) for z in (want, tol)), n)


def test_one_tensor_as_every_operand():
    """Queries, keys and values that are one tensor."""
    r = rng(64)
    x, dy = f32(r.standard_normal((2, 3, 200, 32))), f32(r.standard_normal((2, 3, 200, 32)))
    got = forward(lambda i: [*O.linear_attention(i['x'], i['x'], i['x'], decays(3)), *O.linear_attention_grad(i['x'], i['x'], i['x'], i['dy'], decays(3))],
                  dict(x=x, dy=dy))
    want, tol = D.linear(x, x, x, decays(3), dy=dy)
    for n, z in zip(('y', 'state', 'dq', 'dk', 'dv'), got):
        R.check(z, want[n], tol[n], n)
    got = forward(lambda i: [O.attention(i['x'], i['x'], i['x'], window=33, sinks=1)], dict(x=x))[0]
    want, tol = D.attention(x, x, x, window=33, sinks=1)
    R.check(got, want['y'], tol['y'], 'y')


def test_windows_of_keys_shared_by_many_queries():
    check_window(*(f32(rng(65, n).standard_normal(s)) for n, s in enumerate([(1, 28, 260, 48), (1, 4, 260, 48), (1, 4, 260, 48), (1, 28, 260, 48)])),
                 dict(window=100, sinks=70), {})


@pytest.mark.parametrize('how', [dict(top_k=1024, top_p=0.97), dict(top_k=1025, top_p=0.97), dict(top_k=1025), dict(top_p=1e-30), dict(top_p=1 - 2.0 ** -40),
                                 dict(top_k=2, top_p=0.999999, min_p=1.0), dict(min_p=1e-12), dict(temperature=2.0 ** -149)],
                         ids=lambda h: '+'.join(f'{n}={x}' for n, x in h.items()))
@pytest.mark.parametrize('rows,V', [(2, 2048), (3, 2049), (5, 8193), (130, 8193), (2, 24576), (2, 24577), (129, 24577), (2, 30011)])
def test_sample_limits_where_the_way_changes(rows, V, how):
    r = rng(rows, V, 66)
    check_sample(f32(2 * r.standard_normal((rows, V))), f32(r.random(rows)), **how)


@pytest.mark.parametrize('rows,V', [(12, 20000), (140, 9000)])
def test_sample_rows_of_every_kind_in_one_call(rows, V):
    """Rows without a limit, with each limit, all equal, greedy, empty, side by side, in both forms of the work."""
    r = rng(rows, V, 67)
    logits, u = f32(2 * r.standard_normal((rows, V))), f32(r.random(rows))
    logits[3::12] = 1.5
    logits[4::12] = -np.inf
    logits[5::12, ::3] = -np.inf
    heat, k, p, m = (np.full(rows, x, t) for x, t in ((1, np.float32), (0, np.int32), (1, np.float32), (0, np.float32)))
    heat[1::12], k[2::12], p[3::12], k[5::12], p[6::12], k[6::12], m[7::12] = 0, 40, 0.7, 5000, 0.9, 3000, 0.2
    heat[8::12] = np.finfo(np.float32).max
    k[9::12], p[10::12], m[11::12] = 2 ** 31 - 1, 0.99, 3.0
    got = check_sample(logits, u, temperature=heat, top_k=k, top_p=p, min_p=m)
    heat[8::12] = np.inf                                     # weighs all alike, as the largest number does
    arrays = dict(logits=logits, u=u, temperature=heat, top_k=k, top_p=p, min_p=m)
    again = forward(lambda i: [O.sample(i['logits'], i['u'], i['temperature'], i['top_k'], i['top_p'], i['min_p'])], arrays)[0]
    assert np.array_equal(got, again)


# ---- offsets beyond 32 bits ---------------------------------------------------------------------------

def on_device(fn, ins, shapes, dtypes):
    decl = {n: {'shape': list(x.shape), 'dtype': 'i32' if x.dtype == torch.int32 else 'f32'} for n, x in ins.items()}
    ex = compile_forward(Module(), lambda m, i: fn(i), decl, output='i32' if dtypes[0] == torch.int32 else 'f32', seed=0)
    outs = [torch.empty(s, device='cuda', dtype=d) for s, d in zip(shapes, dtypes)]
    torch.cuda.synchronize()
    r = ex.run_device(ins, outs)
    assert r.error is None, r.error
    torch.cuda.synchronize()
    ex.destroy()
    return outs


def test_linear_of_more_than_2_31_elements():
    """The last positions of a sequence whose queries alone fill 8 GiB; the decay forgets what is 200 positions back."""
    T = (1 << 25) + 77
    gen = torch.Generator(device='cuda').manual_seed(71)
    ins = {n: torch.randn((1, 1, T, 64), generator=gen, device='cuda') for n in 'qkv'}
    y, state = on_device(lambda i: list(O.linear_attention(i['q'], i['k'], i['v'], [0.5])), ins, [(1, 1, T, 64), (1, 1, 64, 64)], [torch.float32] * 2)
    tail = {n: np.ascontiguousarray(x[:, :, -400:].cpu().numpy()) for n, x in ins.items()}
    want, tol = D.linear(**tail, decay=[0.5])
    R.check(y[:, :, -200:].cpu().numpy(), want['y'][:, :, 200:], tol['y'][:, :, 200:], 'y')
    R.check(state.cpu().numpy(), want['state'], tol['state'], 'state')


def test_window_in_a_cache_of_more_than_2_31_elements():
    T = (1 << 25) + 77
    gen = torch.Generator(device='cuda').manual_seed(72)
    ins = {'k': torch.randn((1, 1, T, 64), generator=gen, device='cuda'), 'v': torch.randn((1, 1, T, 64), generator=gen, device='cuda')}
    for Tq in (1, 40):
        ins['q'] = torch.randn((1, 2, Tq, 64), generator=gen, device='cuda')
        y, = on_device(lambda i: [O.attention(i['q'], i['k'], i['v'], window=300, sinks=5)], ins, [(1, 2, Tq, 64)], [torch.float32])
        part = {n: torch.cat([ins[n][:, :, :5], ins[n][:, :, -600:]], 2).cpu().numpy() for n in 'kv'}
        want, tol = D.attention(ins['q'].cpu().numpy(), part['k'], part['v'], window=300, sinks=5)
        R.check(y.cpu().numpy(), want['y'], tol['y'], str(Tq))


def test_sample_of_more_than_2_31_logits():
    rows, V = 130, 1 << 24
    gen = torch.Generator(device='cuda').manual_seed(73)
    ins = {'logits': torch.randn((rows, V), generator=gen, device='cuda'), 'u': torch.rand(rows, generator=gen, device='cuda')}
    got, = on_device(lambda i: [O.sample(i['logits'], i['u'], temperature=0.2, top_k=500)], ins, [(rows,)], [torch.int32])
    for r in (0, rows - 1):
        assert int(got[r]) == D.sample(ins['logits'][r].cpu().numpy(), float(ins['u'][r]), 0.2, 500), r
    one = {n: x[-1:].clone() for n, x in ins.items()}
    again, = on_device(lambda i: [O.sample(i['logits'], i['u'], temperature=0.2, top_k=500)], one, [(1,)], [torch.int32])
    assert int(again[0]) == int(got[-1])

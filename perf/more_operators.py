"""Operators of decoders whose memory does not grow with what they have read, as cases that can be timed and checked:
attention over a sliding window with first positions that stay, linear attention with a decay for each head (with its
state), both with their gradients, and the choice of the next token.

`own = False` computes them from elementary torch operations; `own = True` calls this package on the same tensors, which
stay on the device from the call's inputs to its outputs.
"""
import math

import torch

own = False

DEV = 'cuda'


# ---- cases ------------------------------------------------------------------------------------

def listed():
    window = dict(op='window', cap=0.0, slopes=False, documents=0, prefix=False, sinks=0, lengths=False, grad=True)
    linear = dict(op='linear', state=False, documents=0, lengths=False, grad=True)
    sample = dict(op='sample', temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, each=False, ties=False)
    return [
        # the longest training sequence through a layer that looks back 512 positions and at the first four
        dict(window, name='window_long', b=1, h=16, hk=4, tq=4096, tk=4096, d=128, window=512, sinks=4),
        # a packed batch of ragged length with capped scores; a window that is no multiple of anything
        dict(window, name='window_documents', b=4, h=8, hk=2, tq=1000, tk=1000, d=64, cap=30.0, documents=4, window=100),
        # one new token a sequence against a long cache of which the window and the first positions count
        dict(window, name='window_token', b=8, h=16, hk=4, tq=1, tk=16000, d=128, window=1024, sinks=4, lengths=True, grad=False),
        # a training step's layer of a sample-sized transformer: launches are all there is
        dict(linear, name='linear_small', b=64, h=4, hk=4, t=16, d=16, dv=16),
        # a packed batch of ragged length, shared key heads, values of another size than keys
        dict(linear, name='linear_documents', b=3, h=8, hk=2, t=1777, d=96, dv=80, documents=5),
        # a training step of long sequences: the most operations
        dict(linear, name='linear_long', b=4, h=16, hk=16, t=4096, d=128, dv=128),
        # prompts of uneven length read at once, for the states that answering starts from
        dict(linear, name='linear_prompt', b=8, h=16, hk=16, t=2048, d=64, dv=64, lengths=True, grad=False),
        # one new token for each sequence of a large batch
        dict(linear, name='linear_token', b=64, h=16, hk=16, t=1, d=128, dv=128, state=True, grad=False),
        # characters, as a sample-sized transformer writes them
        dict(sample, name='sample_characters', rows=64, vocab=65, temperature=0.8, top_k=20),
        # a few sequences answered at once: few rows, long ones
        dict(sample, name='sample_few', rows=4, vocab=128000, temperature=0.7, top_k=50, top_p=0.9),
        # a hot nucleus of many thousand tokens
        dict(sample, name='sample_nucleus', rows=32, vocab=200000, temperature=1.6, top_p=0.95),
        # a serving batch where every request has its own settings
        dict(sample, name='sample_batch', rows=256, vocab=50001, each=True),
    ]


MOST_FLOPS = 5.2e10        # of the largest listed case in operations (linear_long)
MOST_BYTES = 1.2e9         # and in bytes
MOST_SCORES = 1 << 28      # scores that the plain form holds at once, as in window_long
MOST_LOGITS = 1.3e7        # logits that are sorted at once, as in sample_batch


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['window', 'linear', 'linear', 'sample', 'sample'])
    if op == 'sample':
        c = dict(op=op, vocab=_log(rng, 27, 200000), temperature=round(rng.uniform(0.4, 2.0), 2), top_k=0, top_p=1.0, min_p=0.0,
                 each=rng.random() < 0.3, ties=rng.random() < 0.15)
        if rng.random() < 0.5:
            c['top_k'] = min(_log(rng, 1, 2000), c['vocab'])
        if rng.random() < 0.5:
            c['top_p'] = round(rng.uniform(0.3, 0.999), 3)
        if rng.random() < 0.3:
            c['min_p'] = round(10 ** rng.uniform(-3, -0.5), 4)
        c['rows'] = max(1, min(_log(rng, 1, 512), int(MOST_LOGITS) // c['vocab']))
        return c
    hk = rng.choice([1, 2, 3, 4, 8])
    if op == 'window':
        c = dict(op=op, h=hk * rng.choice([1, 1, 2, 4, 7]), hk=hk, d=rng.choice([16, 32, 40, 64, 80, 96, 128, rng.randint(1, 128)]),
                 cap=rng.choice([0.0, 0.0, 0.0, 30.0]), slopes=rng.random() < 0.2, prefix=False, documents=0, sinks=0, lengths=False)
        kind = rng.choice(['train', 'train', 'chunk', 'token'])
        c['tk'] = _log(rng, 8, 4096)
        c['tq'] = c['tk'] if kind == 'train' else 1 if kind == 'token' else rng.randint(2, max(2, c['tk'] // 8))
        c['window'] = _log(rng, 1, c['tk'])
        c['grad'] = kind == 'train'
        more = rng.choice(['sinks', 'sinks', 'documents', 'prefix', 'none'])
        if more == 'sinks':
            c['sinks'] = rng.randint(1, 40)
        elif more == 'prefix':
            c['prefix'] = True
        elif more == 'documents' and kind == 'train':
            c['documents'] = rng.choice([3, 9])
        if kind != 'train':
            c['lengths'] = rng.random() < 0.7
            c['tk'] = max(c['tq'], c['tk'])
        c['b'] = _log(rng, 1, 64)
        heavy = lambda: c['b'] * c['h'] * c['tq'] * c['tk'] > MOST_SCORES  # noqa: E731
        while c['b'] > 1 and (heavy() or work(c)['flops'] > MOST_FLOPS or work(c)['bytes'] > MOST_BYTES):
            c['b'] //= 2
        while heavy():
            c['hk'], c['h'] = 1, c['h'] // c['hk']
            c['tk'] = c['tk'] * 3 // 4
            c['tq'] = min(c['tq'], c['tk'])
        return c
    c = dict(op=op, h=hk * rng.choice([1, 1, 1, 2, 4]), hk=hk, d=rng.choice([16, 32, 48, 64, 96, 128, rng.randint(1, 128)]),
             documents=0, lengths=False, state=rng.random() < 0.4)
    c['dv'] = c['d'] if rng.random() < 0.6 else rng.choice([16, 32, 64, 80, 128, rng.randint(1, 128)])
    kind = rng.choice(['train', 'train', 'prompt', 'token'])
    c['t'] = _log(rng, 1, 4 if kind == 'token' else 4096)
    c['grad'] = kind == 'train'
    if kind == 'train':
        c['documents'] = rng.choice([0, 0, 3, 9])
    elif kind == 'prompt':
        c['lengths'] = rng.random() < 0.7
    else:
        c['state'] = True
    c['b'] = _log(rng, 1, 64)
    while c['b'] > 1 and (work(c)['flops'] > MOST_FLOPS or work(c)['bytes'] > MOST_BYTES):
        c['b'] //= 2
    return c


# ---- inputs -----------------------------------------------------------------------------------

class State:
    """A case's tensors and, where the package runs it, its compiled graph (freed with the state)."""

    def __init__(self, case, tensors):
        self.case, self.t, self.handle = case, tensors, None

    def __del__(self):
        if self.handle is not None:
            self.handle.destroy()


def _slopes(c):
    """The usual distance slopes: a geometric sequence over the heads from 2^(-8/H) to 2^-8."""
    return [2.0 ** (-8.0 * (i + 1) / c['h']) for i in range(c['h'])] if c['slopes'] else None


def _decay(c):
    """The usual decays: from heads that forget within some thirty positions to heads that keep for thousands."""
    return [1.0 - 2.0 ** (-5.0 - 7.0 * i / max(1, c['h'] - 1)) for i in range(c['h'])]


def _tensors(c, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed) * 7919 + 29)
    normal = lambda *s: torch.randn(s, generator=gen, device=DEV)  # noqa: E731
    uniform = lambda *s: torch.rand(s, generator=gen, device=DEV)  # noqa: E731
    ints = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=gen, device=DEV, dtype=torch.int32)  # noqa: E731

    def packed(b, t):                                        # documents laid end to end, the last places unused (-1)
        ids = torch.cumsum((uniform(b, t) < c['documents'] / t).int(), 1, dtype=torch.int32)
        return torch.where(torch.arange(t, device=DEV) < t - t // 50, ids, -1).int()
    t = {}
    if c['op'] == 'window':
        b, tq, tk, d = c['b'], c['tq'], c['tk'], c['d']
        t['q'] = 1.5 * normal(b, c['h'], tq, d)              # scores of the size that trained heads have
        t['k'] = normal(b, c['hk'], tk, d) + 0.5 * normal(1, c['hk'], 1, d)
        t['v'] = normal(b, c['hk'], tk, d)
        if c['documents']:
            t['documents'] = packed(b, tk)
        if c['prefix']:
            t['prefix'] = ints(0, tk // 4 + 1, b)
        if c['lengths']:                                     # a cache filled to somewhere in its second half
            t['lengths'] = ints(max(tq, tk // 2), tk + 1, b)
        if c['grad']:
            t['dy'] = normal(b, c['h'], tq, d)
    elif c['op'] == 'linear':
        b, n, d, dv = c['b'], c['t'], c['d'], c['dv']
        t['q'], t['k'], t['v'] = normal(b, c['h'], n, d), normal(b, c['hk'], n, d), normal(b, c['hk'], n, dv)
        if c['state']:                                       # what some dozen positions leave
            t['state'] = 5 * normal(b, c['h'], d, dv)
        if c['documents']:
            t['documents'] = packed(b, n)
        if c['lengths']:
            t['lengths'] = ints(n // 2, n + 1, b)
        if c['grad']:
            t['dy'] = normal(b, c['h'], n, dv)
            if c['state']:
                t['dstate'] = normal(b, c['h'], d, dv)
    else:
        r, v = c['rows'], c['vocab']
        t['logits'] = 2.5 * normal(r, v) + 4 * (uniform(r, v) < 10.0 / v)      # some tokens stand out, as after a prompt
        if c['ties']:                                        # logits that were rounded to few bits
            t['logits'] = torch.round(t['logits'] * 4) / 4
        t['u'] = uniform(r)
        if c['each']:                                        # greedy and free requests among the others
            t['temperature'] = 0.3 + 1.2 * uniform(r)
            t['temperature'][::7] = 0
            t['top_k'] = ints(1, 200, r)
            t['top_k'][::3] = 0
            t['top_p'] = 0.5 + 0.6 * uniform(r)              # from 1 on: everything
            t['min_p'] = 0.1 * uniform(r)
            t['min_p'][::2] = 0
    return t


def prepare(case, seed):
    s = State(case, _tensors(case, seed))
    if own:
        s.handle = _compiled(case, s.t)
    return s


# ---- the package's calls ----------------------------------------------------------------------

def _compiled(c, t):
    """The case as a compiled forward graph whose outputs are the operator's result and its gradients."""
    import tensorgrad_amd.ops as O
    from tensorgrad_amd.compile import compile_forward
    from tensorgrad_amd.module import Module

    def window(m, i):
        how = dict(window=c['window'], sinks=c['sinks'], softcap=c['cap'] or None, slopes=_slopes(c), documents=i.get('documents'),
                   prefix=i.get('prefix'), lengths=i.get('lengths'))
        y = O.attention(i['q'], i['k'], i['v'], **how)
        return [y, *O.attention_grad(i['q'], i['k'], i['v'], y, i['dy'], **how)] if c['grad'] else [y]

    def linear(m, i):
        how = dict(state=i.get('state'), documents=i.get('documents'), lengths=i.get('lengths'))
        y, state = O.linear_attention(i['q'], i['k'], i['v'], _decay(c), **how)
        if not c['grad']:
            return [y, state]
        return [y, *O.linear_attention_grad(i['q'], i['k'], i['v'], i['dy'], _decay(c), dstate=i.get('dstate'), **how)]

    def sample(m, i):
        how = ({n: i[n] for n in ('temperature', 'top_k', 'top_p', 'min_p')} if c['each'] else
               dict(temperature=c['temperature'], top_k=c['top_k'] or None, top_p=None if c['top_p'] >= 1 else c['top_p'],
                    min_p=c['min_p'] or None))
        return [O.sample(i['logits'], i['u'], **how)]

    decl = {n: {'shape': list(x.shape), 'dtype': 'i32' if x.dtype == torch.int32 else 'f32'} for n, x in t.items()}
    return compile_forward(Module(), {'window': window, 'linear': linear, 'sample': sample}[c['op']], decl,
                           output='i32' if c['op'] == 'sample' else 'f32', seed=0)


def _outputs(c):
    """Names and shapes that a pass writes."""
    if c['op'] == 'window':
        q, k = (c['b'], c['h'], c['tq'], c['d']), (c['b'], c['hk'], c['tk'], c['d'])
        return {'y': q, 'dq': q, 'dk': k, 'dv': k} if c['grad'] else {'y': q}
    if c['op'] == 'linear':
        b, h, hk, n, d, dv = (c[x] for x in ('b', 'h', 'hk', 't', 'd', 'dv'))
        if not c['grad']:
            return {'y': (b, h, n, dv), 'state': (b, h, d, dv)}
        out = {'y': (b, h, n, dv), 'dq': (b, h, n, d), 'dk': (b, hk, n, d), 'dv': (b, hk, n, dv)}
        return dict(out, dstate=(b, h, d, dv)) if c['state'] else out
    return {'tokens': (c['rows'],)}


def run(state):
    c, t = state.case, state.t
    if own:
        kind = torch.int32 if c['op'] == 'sample' else torch.float32
        out = {n: torch.empty(s, dtype=kind, device=DEV) for n, s in _outputs(c).items()}
        r = state.handle.run_device(t, list(out.values()), stream=torch.cuda.current_stream().cuda_stream)
        if r.error is not None:
            raise r.error
        return out
    return {'window': _window, 'linear': _linear, 'sample': _sample}[c['op']](c, t)


# ---- plain forms, in 32 bits ------------------------------------------------------------------

def _seen(c, t):
    """[B, 1, Tq, Tk] which key a query sees, and [B, 1, Tq, Tk] their distance."""
    b, tq, tk = c['b'], c['tq'], c['tk']
    n = t['lengths'].long() if c['lengths'] else torch.full((b,), tk, device=DEV)
    p = (n[:, None] - tq + torch.arange(tq, device=DEV))[:, :, None]
    j = torch.arange(tk, device=DEV)[None, None, :]
    seen = (j <= p) & ((j > p - c['window']) | (j < c['sinks']))
    if c['prefix']:
        seen = seen | (j < t['prefix'].long()[:, None, None])
    seen = seen & (p >= 0) & (j < n[:, None, None])
    if c['documents']:
        doc = t['documents']
        mine = torch.gather(doc, 1, p[:, :, 0].clamp(min=0))
        seen = seen & (mine[:, :, None] == doc[:, None, :]) & (doc[:, None, :] >= 0)
    return seen[:, None], (p - j).abs()[:, None].float()


def _window(c, t):
    b, h, hk, tq, tk, d = (c[n] for n in ('b', 'h', 'hk', 'tq', 'tk', 'd'))
    g, scale, cap = h // hk, 1 / math.sqrt(d), c['cap']
    q = t['q'].reshape(b * hk, g * tq, d)
    k, v = t['k'].reshape(b * hk, tk, d), t['v'].reshape(b * hk, tk, d)
    seen, far = _seen(c, t)
    s = (q @ k.transpose(1, 2).contiguous()).reshape(b, h, tq, tk) * scale
    if cap:
        th = torch.tanh(s / cap)
        s = cap * th
    if c['slopes']:
        s = s - torch.tensor(_slopes(c), device=DEV)[:, None, None] * far
    s = torch.where(seen, s, -math.inf)
    top = s.max(-1, keepdim=True).values
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    rows = lambda x: x.reshape(b * hk, g * tq, -1)  # noqa: E731
    y = (rows(p) @ v).reshape(b, h, tq, d)
    if not c['grad']:
        return {'y': y}
    dy = t['dy']
    dp = (rows(dy) @ v.transpose(1, 2).contiguous()).reshape(b, h, tq, tk)
    ds = p * (dp - (dy * y).sum(-1, keepdim=True)) * scale
    if cap:
        ds = ds * (1 - th * th)
    return {'y': y, 'dq': (rows(ds) @ k).reshape(b, h, tq, d),
            'dk': (rows(ds).transpose(1, 2).contiguous() @ q).reshape(b, hk, tk, d),
            'dv': (rows(p).transpose(1, 2).contiguous() @ rows(dy)).reshape(b, hk, tk, d)}


CHUNK = 128


def _linear(c, t):
    """In chunks: products of pairs within a chunk, states between chunks."""
    b, h, hk, n, d, dv = (c[x] for x in ('b', 'h', 'hk', 't', 'd', 'dv'))
    g, scale, C = h // hk, 1 / math.sqrt(d), min(CHUNK, n)
    m = -(-n // C)
    pad = m * C - n
    lam = torch.tensor(_decay(c), dtype=torch.float64, device=DEV)
    there = torch.ones(b, n, dtype=torch.bool, device=DEV)
    if c['lengths']:
        there = torch.arange(n, device=DEV)[None] < t['lengths'][:, None]
    run_id = torch.zeros(b, n, dtype=torch.int64, device=DEV)                # rows of one document
    if c['documents']:
        doc = t['documents']
        there = there & (doc >= 0)
        run_id = torch.cumsum(torch.cat([torch.zeros_like(doc[:, :1]), (doc[:, 1:] != doc[:, :-1]).int()], 1), 1)
    last = t['lengths'].long() - 1 if c['lengths'] else torch.full((b,), n - 1, device=DEV)

    def rows(x, shared):                                                     # [b, h, m, C, width], nothing in hidden rows
        x = torch.where(there[:, None, :, None], x, 0.0)
        if shared and g > 1:
            x = x.repeat_interleave(g, 1)
        return torch.nn.functional.pad(x, (0, 0, 0, pad)).reshape(b, h, m, C, -1)
    q, k, v = rows(t['q'], False), rows(t['k'], True), rows(t['v'], True)
    ids = torch.nn.functional.pad(run_id, (0, pad), value=-1).reshape(b, 1, m, C)
    at = torch.arange(C, device=DEV)
    near = (at[:, None] - at[None, :]).clamp(min=0)
    weight = torch.where(at[:, None] >= at[None, :], lam[:, None, None] ** near, 0.0).float()[None, :, None] \
        * (ids[..., :, None] == ids[..., None, :])                           # [b, h, m, C, C]
    before = torch.cat([torch.zeros_like(ids[:, :, :1, 0]), ids[:, :, :-1, -1]], 2)      # the row before the chunk
    comes = (lam[:, None] ** (at + 1)).float()[None, :, None] * (ids == before[..., None])    # what came in, at each row
    final = ids[..., -1:].clone()
    stop = torch.full((b, 1, m, 1), C - 1, device=DEV)                       # the chunk's last row that counts
    lm, lc = last.clamp(min=0) // C, last.clamp(min=0) % C
    here = torch.arange(m, device=DEV)[None, None, :, None] == lm[:, None, None, None]
    final = torch.where(here, ids.gather(3, lc[:, None, None, None].expand(b, 1, m, 1)), final)
    stop = torch.where(here, lc[:, None, None, None], stop)
    power = lambda e: torch.exp(e.double() * torch.log(lam)[None, :, None, None]).float()  # noqa: E731
    goes = power((stop - at).clamp(min=0))
    goes = goes * ((ids == final) & (at <= stop))                            # what a row leaves at the chunk's end
    stays = power(stop + 1) * (final == before[..., None])                   # of what came in
    after = torch.arange(m, device=DEV)[None, None, :, None] > lm[:, None, None, None]   # chunks behind the last row
    none = (last < 0)[:, None, None, None]
    stays = torch.where(after | none, 1.0, stays)[..., None]
    goes = torch.where(after | none, 0.0, goes)

    flat = lambda x: x.reshape(b * h * m, x.shape[-2], x.shape[-1])  # noqa: E731
    un = lambda x: x.reshape(b, h, m, x.shape[-2], x.shape[-1])  # noqa: E731
    cross = lambda x, y: un(flat(x).transpose(1, 2).contiguous() @ flat(y))  # noqa: E731
    T = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731

    def carried(first, add):                                                 # states before each chunk, and the last
        states = []
        for i in range(m):
            states.append(first)
            first = first * stays[:, :, i] + add[:, :, i]
        return torch.stack(states, 2), first
    zero = torch.zeros(b, h, d, dv, device=DEV)
    S, end = carried(t['state'] if c['state'] else zero, cross(k * goes[..., None], v))
    pairs = un(flat(q) @ flat(T(k))) * weight * scale
    y = un(flat(pairs) @ flat(v)) + un(flat(q * comes[..., None]) @ flat(S)) * scale
    back = lambda x: torch.where(there[:, None, :, None], x.reshape(b, h, m * C, -1)[:, :, :n], 0.0)  # noqa: E731
    if not c['grad']:
        return {'y': back(y), 'state': end}
    dy = rows(t['dy'], False)
    add = cross(q * comes[..., None], dy) * scale
    states, first = [], t['dstate'] if c['state'] else zero                  # gradients of the states behind each chunk
    for i in reversed(range(m)):
        states.append(first)
        first = first * stays[:, :, i] + add[:, :, i]
    G = torch.stack(states[::-1], 2)
    ds = un(flat(dy) @ flat(T(v))) * weight * scale
    dq = un(flat(ds) @ flat(k)) + un(flat(dy * comes[..., None]) @ flat(T(S))) * scale
    dk = cross(ds, q) + un(flat(v * goes[..., None]) @ flat(T(G)))
    dv_ = cross(pairs, dy) + un(flat(k * goes[..., None]) @ flat(G))
    shared = lambda x: back(x).reshape(b, hk, g, n, -1).sum(2)  # noqa: E731
    out = {'y': back(y), 'dq': back(dq), 'dk': shared(dk), 'dv': shared(dv_)}
    return dict(out, dstate=first) if c['state'] else out


def _settings(c, t):
    """temperature, top_k, top_p, min_p as [rows, 1] in 64 bits."""
    names = ('temperature', 'top_k', 'top_p', 'min_p')
    if c['each']:
        return [t[n].double()[:, None] for n in names]
    return [torch.full((c['rows'], 1), float(c[n]), dtype=torch.float64, device=DEV) for n in names]


def _sample(c, t):
    """Sorted, since every limit keeps a first part of the order; weights and sums in 64 bits, as borders are close."""
    heat, top_k, top_p, min_p = _settings(c, t)
    x = t['logits']
    v = x.shape[1]
    ordered, index = torch.sort(x, dim=1, descending=True, stable=True)
    z = (ordered.double() - ordered[:, :1].double()) / torch.where(heat > 0, heat, 1.0)
    w = torch.exp(z)
    rank = torch.arange(v, device=DEV)
    keep = (rank < torch.where(top_k > 0, top_k, v)) & (rank < torch.where(heat > 0, v, 1))
    w = torch.where(keep, w, 0.0)
    sums = torch.cumsum(w, 1)
    keep = keep & ((sums - w < top_p * sums[:, -1:]) | (top_p >= 1)) & (w >= min_p)
    w = torch.zeros_like(w).scatter_(1, index, torch.where(keep, w, 0.0))      # back in the vocabulary's order
    sums = torch.cumsum(w, 1)
    passed = (sums > t['u'].double()[:, None] * sums[:, -1:]) & (w > 0)
    return {'tokens': passed.int().argmax(1).int()}


# ---- work -------------------------------------------------------------------------------------

def work(case):
    c = case
    if c['op'] == 'window':
        q, k = c['b'] * c['h'] * c['tq'] * c['d'], c['b'] * c['hk'] * c['tk'] * c['d']
        n = c['tk'] * 3 // 4 if c['lengths'] else c['tk']    # lengths lie between half and all of the cache
        if c['documents']:
            n = max(1, n // c['documents'])                  # about so many documents a row
        first = max(0, n - c['tq'])
        stay = c['sinks'] + (c['tk'] // 8 if c['prefix'] else 0)
        w = min(c['window'] + stay, n)                       # keys a query sees, fewer near the start
        full = max(0, n - max(first, w))                     # queries that see all of them
        some = min(c['tq'], n) - full
        pairs = full * w + some * (first + 1 + min(first + some, w)) // 2
        if c['documents']:
            pairs *= c['documents']
        if c['tq'] < c['tk']:                                # keys that any query sees
            k = k * min(c['tk'], c['window'] + stay + c['tq'] - 1) // c['tk']
        products = 2 * c['b'] * c['h'] * max(1, pairs) * c['d']
        return {'bytes': 4 * (4 * q + 4 * k), 'flops': 7 * products} if c['grad'] else {'bytes': 4 * (2 * q + 2 * k), 'flops': 2 * products}
    if c['op'] == 'linear':
        b, h, hk, n, d, dv = (c[x] for x in ('b', 'h', 'hk', 't', 'd', 'dv'))
        n = n * 3 // 4 if c['lengths'] else n
        rows = b * n * (h * (d + dv) + hk * (d + dv))        # q and y, k and v
        state = b * h * d * dv
        step = 2 * b * h * n * d * dv                        # a state's update, or a row's product with it
        if not c['grad']:
            return {'bytes': 4 * (rows + (2 if c['state'] else 1) * state), 'flops': 2 * step}
        # q, k, v, dy read, y, dq, dk, dv written
        return {'bytes': 4 * (2 * rows + (3 * state if c['state'] else 0)), 'flops': 6 * step}
    return {'bytes': 4 * c['rows'] * c['vocab'] + 8 * c['rows'], 'flops': 3 * c['rows'] * c['vocab']}


# ---- the same in 64 bits ----------------------------------------------------------------------

def _exact_window(c, t):
    out = {n: torch.zeros(s, dtype=torch.float64, device=DEV) for n, s in _outputs(c).items()}
    tq, tk, g = c['tq'], c['tk'], c['h'] // c['hk']
    slopes = _slopes(c)
    for b in range(c['b']):
        n = int(t['lengths'][b]) if c['lengths'] else tk
        stay = max(c['sinks'], 0)
        pos = torch.arange(n - tq, n, device=DEV)[:, None]
        key = torch.arange(tk, device=DEV)[None, :]
        back = pos - key
        hidden = (back < 0) | ((back >= c['window']) & (key >= stay))
        if c['prefix']:
            hidden = hidden & (key >= int(t['prefix'][b]))
        hidden = hidden | (key >= n) | (pos < 0)
        if c['documents']:
            doc = t['documents'][b]
            hidden = hidden | (doc[pos.clamp(min=0)] != doc[key]) | (doc[key] < 0)
        none = hidden.all(1, keepdim=True)
        for h in range(c['h']):
            q, k, v = (t[m][b, i].double().requires_grad_(c['grad']) for m, i in (('q', h), ('k', h // g), ('v', h // g)))
            s = torch.mm(q, k.t()) / math.sqrt(c['d'])
            if c['cap']:
                s = torch.tanh(s / c['cap']) * c['cap']
            if slopes:
                s = s - slopes[h] * back.abs()
            w = torch.softmax(s.masked_fill(hidden, -1e300), 1).masked_fill(hidden | none, 0.0)
            y = torch.mm(w, v)
            out['y'][b, h] = y.detach()
            if c['grad']:
                gq, gk, gv = torch.autograd.grad(y, (q, k, v), t['dy'][b, h].double())
                out['dq'][b, h] = gq
                out['dk'][b, h // g] += gk
                out['dv'][b, h // g] += gv
    return out


def _exact_linear(c, t):
    """All pairs of one head at a time: y = (decay mask * scale q k^T) v, and what the first state adds."""
    out = {n: torch.zeros(s, dtype=torch.float64, device=DEV) for n, s in _outputs(c).items()}
    n, g, grad = c['t'], c['h'] // c['hk'], c['grad']
    at = torch.arange(n, device=DEV)
    for b in range(c['b']):
        end = min(max(int(t['lengths'][b]), 0), n) if c['lengths'] else n
        live = at < end
        since = torch.zeros_like(at)                         # the first row of a row's document
        if c['documents']:
            doc = t['documents'][b]
            live = live & (doc >= 0)
            starts = torch.zeros_like(at)
            starts[1:] = torch.where(doc[1:] != doc[:-1], at[1:], 0)
            since = torch.cummax(starts, 0).values
        far = (at[:, None] - at[None, :]).double()
        pairs = (far >= 0) & (at[None, :] >= since[:, None]) & live[:, None] & live[None, :]
        opens = live & (since == 0)                          # rows that the first state reaches
        for h in range(c['h']):
            lam = _decay(c)[h]
            q, k, v = (t[m][b, i].double().requires_grad_(grad) for m, i in (('q', h), ('k', h // g), ('v', h // g)))
            s0 = t['state'][b, h].double().requires_grad_(grad) if c['state'] else torch.zeros(c['d'], c['dv'], dtype=torch.float64, device=DEV)
            w = torch.where(pairs, torch.pow(lam, far.clamp(min=0)), 0.0)
            y = torch.mm(w * torch.mm(q, k.t()), v)
            y = (y + torch.where(opens, lam ** (at + 1).double(), 0.0)[:, None] * torch.mm(q, s0)) / math.sqrt(c['d'])
            if end == 0:
                last = s0
            else:
                e = end - 1
                tail = torch.where(live & (at >= since[e]) & live[e], lam ** (e - at).clamp(min=0).double(), 0.0)
                last = torch.mm((k * tail[:, None]).t(), v) + (lam ** end if bool(opens[e]) else 0.0) * s0
            out['y'][b, h] = y.detach()
            if not grad:
                out['state'][b, h] = last
                continue
            total = (y * t['dy'][b, h].double()).sum()
            if c['state']:
                total = total + (last * t['dstate'][b, h].double()).sum()
            grads = torch.autograd.grad(total, (q, k, v, s0) if c['state'] else (q, k, v))
            out['dq'][b, h] = grads[0]
            out['dk'][b, h // g] += grads[1]
            out['dv'][b, h // g] += grads[2]
            if c['state']:
                out['dstate'][b, h] = grads[3]
    return out


def _exact_sample(c, t):
    """Row by row: how many tokens each limit keeps, then the first token where the kept weights' sum passes u of them all."""
    heat, top_k, top_p, min_p = (x[:, 0].tolist() for x in _settings(c, t))
    u = t['u'].double().tolist()
    out = []
    for r in range(c['rows']):
        x = t['logits'][r].double()
        order = torch.argsort(x, descending=True, stable=True)
        if heat[r] <= 0:
            out.append(order[0])
            continue
        p = torch.exp((x[order] - x[order[0]]) / heat[r])
        n = int(top_k[r]) if 0 < top_k[r] < len(p) else len(p)
        p = p[:n]
        mass = torch.cumsum(p, 0)
        if top_p[r] < 1:
            n = min(n, 1 + int((mass[:-1] < top_p[r] * mass[-1]).sum()))
        n = min(n, max(1, int((p >= min_p[r]).sum())))
        kept, _ = torch.sort(order[:n])
        mass = torch.cumsum(torch.exp((x[kept] - x[order[0]]) / heat[r]), 0)
        at = int((mass <= u[r] * mass[-1]).sum())
        out.append(kept[min(at, n - 1)])
    return {'tokens': torch.stack(out).int()}


def exact(case, seed):
    t = _tensors(case, seed)
    return {'window': _exact_window, 'linear': _exact_linear, 'sample': _exact_sample}[case['op']](case, t)

"""The sequence operators as cases that can be timed and checked: attention with capped scores, distance bias, document,
prefix and length masks; rotary positions of several axes; the gated linear recurrence. Each with its gradients.

`own = False` computes them from elementary torch operations; `own = True` calls this package on the same tensors, which
stay on the device from the call's inputs to its outputs.
"""
import math

import torch

own = False

DEV = 'cuda'


# ---- cases ------------------------------------------------------------------------------------

def listed():
    attention = dict(op='attention', causal=True, cap=0.0, slopes=False, documents=0, prefix=False, lengths=False, grad=True)
    rope = dict(op='rope', per_axis=False, grad=True)
    scan = dict(op='scan', start=False, grad=True)
    return [
        # a training step's attention of a sample-sized transformer, with a distance bias: launches are all there is
        dict(attention, name='attention_small', b=64, h=4, hk=4, tq=16, tk=16, d=16, slopes=True),
        # a packed batch: ragged length, short documents, capped scores, shared key heads
        dict(attention, name='attention_documents', b=8, h=8, hk=2, tq=1000, tk=1000, d=64, cap=30.0, documents=6),
        # a prefix that every position of it sees (an image or a question), an odd length and a head size of 96
        dict(attention, name='attention_prefix', b=4, h=8, hk=8, tq=777, tk=777, d=96, prefix=True, slopes=True),
        # the longest training sequence: capped scores, shared key heads; the most operations
        dict(attention, name='attention_long', b=1, h=16, hk=4, tq=4096, tk=4096, d=128, cap=50.0),
        # one new token a sequence against a long, unevenly filled cache
        dict(attention, name='attention_token', b=8, h=16, hk=4, tq=1, tk=16000, d=128, lengths=True, grad=False),
        # a chunk of new tokens against a cache, as a prompt is read in pieces
        dict(attention, name='attention_chunk', b=2, h=8, hk=4, tq=64, tk=5000, d=64, lengths=True, slopes=True, grad=False),
        # positions of a sample-sized transformer over small images
        dict(rope, name='rope_small', b=64, h=4, hk=4, t=16, d=16, sections='4,4', per_axis=True),
        # video: time, height and width of long sequences, with the gradient
        dict(rope, name='rope_video', b=4, h=16, hk=4, t=4096, d=128, sections='16,24,24'),
        # one token at a far position, part of each head turned
        dict(rope, name='rope_token', b=32, h=16, hk=4, t=1, d=96, sections='8,12,12', grad=False),
        # recurrent layer of a sample-sized model
        dict(scan, name='scan_small', b=64, t=16, c=64),
        # an odd length and width, a state carried in from the sequence before
        dict(scan, name='scan_odd', b=3, t=1777, c=333, start=True),
        # a recurrent layer over a long sequence: the most bytes
        dict(scan, name='scan_long', b=4, t=8192, c=1024, start=True),
    ]


MOST_FLOPS = 2.4e11        # of the largest listed case in operations (attention_long)
MOST_BYTES = 9.3e8         # and in bytes (scan_long)
MOST_SCORES = 1 << 28      # scores that the plain form holds at once, as in attention_long


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['attention', 'attention', 'rope', 'scan'])
    if op == 'attention':
        hk = rng.choice([1, 2, 3, 4, 8])
        c = dict(op=op, h=hk * rng.choice([1, 1, 2, 4, 7]), hk=hk, d=rng.choice([16, 24, 32, 40, 64, 80, 96, 128, rng.randint(1, 128)]),
                 cap=rng.choice([0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.3, prefix=False, documents=0, lengths=False)
        kind = rng.choice(['train', 'train', 'forward', 'chunk', 'token'])
        c['tk'] = _log(rng, 8, 4096)
        c['tq'] = c['tk'] if kind in ('train', 'forward') else 1 if kind == 'token' else rng.randint(2, max(2, c['tk'] // 8))
        c['grad'] = kind == 'train'
        c['causal'] = kind != 'forward' or rng.random() < 0.5
        if kind in ('train', 'forward'):
            c['prefix'] = c['causal'] and rng.random() < 0.25
            c['documents'] = rng.choice([0, 0, 3, 9])
        else:
            c['lengths'] = rng.random() < 0.7
            c['tk'] = max(c['tq'], c['tk'])
        c['b'] = _log(rng, 1, 64)
        while c['b'] > 1 and (c['b'] * c['h'] * c['tq'] * c['tk'] > MOST_SCORES or work(c)['flops'] > MOST_FLOPS
                              or work(c)['bytes'] > MOST_BYTES):
            c['b'] //= 2
        while c['b'] * c['h'] * c['tq'] * c['tk'] > MOST_SCORES:
            c['hk'], c['h'] = 1, c['h'] // c['hk']
            c['tk'] = c['tk'] * 3 // 4
            c['tq'] = min(c['tq'], c['tk'])
        return c
    if op == 'rope':
        hk = rng.choice([1, 2, 4, 8])
        d = rng.choice([16, 32, 64, 80, 96, 128, 2 * rng.randint(3, 64)])
        pairs = rng.randint(3, d // 2) if rng.random() < 0.5 else d // 2
        axes = rng.choice([1, 2, 3])
        cuts = sorted(rng.sample(range(1, pairs), axes - 1)) if axes > 1 else []
        sizes = [e - s for s, e in zip([0] + cuts, cuts + [pairs])]
        c = dict(op=op, h=hk * rng.choice([1, 2, 4]), hk=hk, d=d, sections=','.join(map(str, sizes)), t=_log(rng, 1, 4096),
                 per_axis=rng.random() < 0.5, grad=rng.random() < 0.6)
        c['b'] = _log(rng, 1, 64)
    else:
        c = dict(op=op, t=_log(rng, 1, 8192), c=_log(rng, 8, 2048), start=rng.random() < 0.5, grad=rng.random() < 0.7)
        c['b'] = _log(rng, 1, 64)
    while c['b'] > 1 and work(c)['bytes'] > MOST_BYTES:
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


def _sections(c):
    return [int(s) for s in c['sections'].split(',')]


def _slopes(c):
    """The usual distance slopes: a geometric sequence over the heads from 2^(-8/H) to 2^-8."""
    return [2.0 ** (-8.0 * (i + 1) / c['h']) for i in range(c['h'])] if c['slopes'] else None


def _tensors(c, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed) * 7919 + 13)
    normal = lambda *s: torch.randn(s, generator=gen, device=DEV)  # noqa: E731
    ints = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=gen, device=DEV, dtype=torch.int32)  # noqa: E731
    t = {}
    if c['op'] == 'attention':
        b, tq, tk, d = c['b'], c['tq'], c['tk'], c['d']
        t['q'] = 1.5 * normal(b, c['h'], tq, d)              # scores of the size that trained heads have
        t['k'] = normal(b, c['hk'], tk, d) + 0.5 * normal(1, c['hk'], 1, d)
        t['v'] = normal(b, c['hk'], tk, d)
        if c['documents']:                                   # documents laid end to end, the last places unused (-1)
            starts = (torch.rand(b, tk, generator=gen, device=DEV) < c['documents'] / tk).int()
            ids = torch.cumsum(starts, 1, dtype=torch.int32)
            t['documents'] = torch.where(torch.arange(tk, device=DEV) < tk - tk // 50, ids, -1).int()
        if c['prefix']:
            t['prefix'] = ints(0, tk // 2 + 1, b)
        if c['lengths']:                                     # a cache filled to somewhere in its second half
            t['lengths'] = ints(max(tq, tk // 2), tk + 1, b)
        if c['grad']:
            t['dy'] = normal(b, c['h'], tq, d)
    elif c['op'] == 'rope':
        b, n, axes = c['b'], c['t'], len(_sections(c))
        t['q'], t['k'] = normal(b, c['h'], n, c['d']), normal(b, c['hk'], n, c['d'])
        far = 100000 if n == 1 else 32768
        start = ints(0, far, axes, b, 1)
        side = max(1, int(round(n ** (1 / axes))))
        at = torch.arange(n, device=DEV)                     # a grid of `axes` axes in reading order, from any corner
        grid = torch.stack([(at // side ** (axes - 1 - a)) % (side if a else n) for a in range(axes)])
        t['positions'] = (grid[:, None, :] + start).int()
        if c['grad']:
            t['dq'], t['dk'] = normal(*t['q'].shape), normal(*t['k'].shape)
    else:
        b, n, w = c['b'], c['t'], c['c']
        memory = normal(w) * 1.5 + 2.5                       # channels that forget soon and channels that keep for long
        t['a'] = torch.sigmoid(normal(b, n, w) + memory)
        t['x'] = (1 - t['a']) * normal(b, n, w)
        if c['start']:
            t['h0'] = normal(b, w)
        if c['grad']:
            t['dh'] = normal(b, n, w)
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

    def attention(m, i):
        how = dict(causal=c['causal'], softcap=c['cap'] or None, slopes=_slopes(c), documents=i.get('documents'),
                   prefix=i.get('prefix'), lengths=i.get('lengths'))
        y = O.attention(i['q'], i['k'], i['v'], **how)
        return [y, *O.attention_grad(i['q'], i['k'], i['v'], y, i['dy'], **how)] if c['grad'] else [y]

    def rope(m, i):
        how = dict(positions=i['positions'], sections=_sections(c), per_axis=c['per_axis'])
        y = O.rope_axes(i['q'], i['k'], **how)
        return [*y, *O.rope_axes(i['dq'], i['dk'], inverse=True, **how)] if c['grad'] else [*y]

    def scan(m, i):
        h = O.linear_recurrence(i['a'], i['x'], i.get('h0'))
        return [h, *O.linear_recurrence_grad(i['a'], h, i['dh'], i.get('h0'))] if c['grad'] else [h]

    decl = {n: {'shape': list(x.shape), 'dtype': 'i32' if x.dtype == torch.int32 else 'f32'} for n, x in t.items()}
    return compile_forward(Module(), {'attention': attention, 'rope': rope, 'scan': scan}[c['op']], decl, seed=0)


def _outputs(c, t):
    """Names and tensors that a pass writes."""
    if c['op'] == 'attention':
        return {'y': 'q', 'dq': 'q', 'dk': 'k', 'dv': 'v'} if c['grad'] else {'y': 'q'}
    if c['op'] == 'rope':
        return {'q': 'q', 'k': 'k', 'dq': 'q', 'dk': 'k'} if c['grad'] else {'q': 'q', 'k': 'k'}
    names = {'h': 'x', 'da': 'a', 'dx': 'x', 'dh0': 'h0'} if c['grad'] else {'h': 'x'}
    return {n: like for n, like in names.items() if like in t}


def run(state):
    c, t = state.case, state.t
    if own:
        out = {n: torch.empty_like(t[like]) for n, like in _outputs(c, t).items()}
        r = state.handle.run_device(t, list(out.values()), stream=torch.cuda.current_stream().cuda_stream)
        if r.error is not None:
            raise r.error
        return out
    return {'attention': _attention, 'rope': _rope, 'scan': _scan}[c['op']](c, t)


# ---- plain forms, in 32 bits ------------------------------------------------------------------

def _seen(c, t):
    """[B, 1, Tq, Tk] which key a query sees, and [B, 1, Tq, Tk] their distance."""
    b, tq, tk = c['b'], c['tq'], c['tk']
    n = t['lengths'].long() if c['lengths'] else torch.full((b,), tk, device=DEV)
    p = (n[:, None] - tq + torch.arange(tq, device=DEV))[:, :, None]
    j = torch.arange(tk, device=DEV)[None, None, :]
    seen = (p >= 0) & (j < n[:, None, None])
    if c['causal']:
        before = j <= p
        if c['prefix']:
            before = before | (j < t['prefix'].long()[:, None, None])
        seen = seen & before
    if c['documents']:
        doc = t['documents']
        mine = torch.gather(doc, 1, p[:, :, 0].clamp(min=0))
        seen = seen & (mine[:, :, None] == doc[:, None, :]) & (doc[:, None, :] >= 0)
    return seen[:, None], (p - j).abs()[:, None].float()


def _attention(c, t):
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


def _exponents(c):
    """Axis of each pair, and the exponent of the base in its frequency."""
    sizes = _sections(c)
    axis = [a for a, n in enumerate(sizes) for _ in range(n)]
    at = [p / n for n in sizes for p in range(n)] if c['per_axis'] else [p / sum(sizes) for p in range(sum(sizes))]
    return axis, at


def _rope(c, t):
    axis, at = _exponents(c)
    half = len(axis)
    freq = 10000.0 ** -torch.tensor(at, dtype=torch.float64, device=DEV)
    angle = t['positions'].double()[torch.tensor(axis, device=DEV)].permute(1, 2, 0) * freq      # far positions need 64 bits
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turn(x, sin):
        x1, x2 = x[..., :half], x[..., half:2 * half]
        return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin, x[..., 2 * half:]], -1)
    out = {'q': turn(t['q'], sin), 'k': turn(t['k'], sin)}
    if c['grad']:
        out.update(dq=turn(t['dq'], -sin), dk=turn(t['dk'], -sin))
    return out


def _scanned(a, x, far=1):
    """h[t] = a[t] h[t-1] + x[t] along axis 1 in log2(T) passes: each joins spans of `far` steps with the ones before."""
    if far >= a.shape[1]:
        return x
    joined = torch.cat([x[:, :far], x[:, far:] + a[:, far:] * x[:, :-far]], 1)
    return _scanned(torch.cat([a[:, :far], a[:, far:] * a[:, :-far]], 1), joined, 2 * far)


def _scan(c, t):
    a, x = t['a'], t['x']
    if c['start']:
        x = torch.cat([x[:, :1] + a[:, :1] * t['h0'][:, None], x[:, 1:]], 1)
    h = _scanned(a, x)
    if not c['grad']:
        return {'h': h}
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = _scanned(after.flip(1), t['dh'].flip(1)).flip(1)
    first = t['h0'][:, None] if c['start'] else torch.zeros_like(h[:, :1])
    out = {'h': h, 'da': g * torch.cat([first, h[:, :-1]], 1), 'dx': g}
    if c['start']:
        out['dh0'] = a[:, 0] * g[:, 0]
    return out


# ---- work -------------------------------------------------------------------------------------

def work(case):
    c = case
    if c['op'] == 'attention':
        q, k = c['b'] * c['h'] * c['tq'] * c['d'], c['b'] * c['hk'] * c['tk'] * c['d']
        pairs = c['tq'] * c['tk'] - (c['tq'] * (c['tq'] - 1) // 2 if c['causal'] else 0)      # a causal triangle at the end
        if c['lengths']:
            k, pairs = k * 3 // 4, pairs * 3 // 4            # lengths lie between half and all of the cache
        if c['documents']:
            pairs = pairs // max(1, c['documents'])          # about so many documents a row
        products = 2 * c['b'] * c['h'] * pairs * c['d']
        if c['grad']:
            return {'bytes': 4 * (4 * q + 4 * k), 'flops': 7 * products}
        return {'bytes': 4 * (2 * q + 2 * k), 'flops': 2 * products}
    if c['op'] == 'rope':
        n = c['b'] * (c['h'] + c['hk']) * c['t'] * c['d']
        passes = 2 if c['grad'] else 1
        return {'bytes': passes * 8 * n + 4 * c['b'] * c['t'] * len(_sections(c)), 'flops': passes * 3 * n}
    n, first = c['b'] * c['t'] * c['c'], (c['b'] * c['c'] if c['start'] else 0)
    # h is written once; the backward pass reads it again, as its values do not fit the chip
    return {'bytes': 4 * ((3 + 4) * n + 2 * first) if c['grad'] else 4 * (3 * n + first), 'flops': (2 + 3) * n if c['grad'] else 2 * n}


# ---- the same in 64 bits ----------------------------------------------------------------------

def _exact_attention(c, t):
    out = {n: torch.zeros_like(t[like], dtype=torch.float64) for n, like in _outputs(c, t).items()}
    tq, tk, g = c['tq'], c['tk'], c['h'] // c['hk']
    slopes = _slopes(c)
    for b in range(c['b']):
        n = int(t['lengths'][b]) if c['lengths'] else tk
        pos = torch.arange(n - tq, n, device=DEV)[:, None]
        key = torch.arange(tk, device=DEV)[None, :]
        hidden = (key >= n).expand(tq, tk) | (pos < 0)
        if c['causal']:
            hidden = hidden | ((key > pos) & (key >= (int(t['prefix'][b]) if c['prefix'] else 0)))
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
                s = s - slopes[h] * (pos - key).abs()
            w = torch.softmax(s.masked_fill(hidden, -1e300), 1).masked_fill(hidden | none, 0.0)
            y = torch.mm(w, v)
            out['y'][b, h] = y.detach()
            if c['grad']:
                gq, gk, gv = torch.autograd.grad(y, (q, k, v), t['dy'][b, h].double())
                out['dq'][b, h] = gq
                out['dk'][b, h // g] += gk
                out['dv'][b, h // g] += gv
    return out


def _exact_rope(c, t):
    axis, at = _exponents(c)
    half = len(axis)
    out = {}
    for name, source, sign in (('q', 'q', 1), ('k', 'k', 1), ('dq', 'dq', -1), ('dk', 'dk', -1)):
        if source not in t:
            continue
        x = t[source].double()
        y = x.clone()
        for p in range(half):
            w = sign * t['positions'][axis[p]].double() * math.exp(-at[p] * math.log(10000.0))
            w = w[:, None]
            y[..., p] = x[..., p] * torch.cos(w) - x[..., p + half] * torch.sin(w)
            y[..., p + half] = x[..., p + half] * torch.cos(w) + x[..., p] * torch.sin(w)
        out[name] = y
    return out


def _exact_scan(c, t):
    a, x = t['a'].double(), t['x'].double()
    h = torch.empty_like(x)
    before = t['h0'].double() if c['start'] else torch.zeros_like(x[:, 0])
    first = before
    for i in range(c['t']):
        before = torch.addcmul(x[:, i], a[:, i], before, out=h[:, i])
    if not c['grad']:
        return {'h': h}
    g, dh = torch.empty_like(x), t['dh'].double()
    behind = torch.zeros_like(first)
    for i in reversed(range(c['t'])):
        torch.add(dh[:, i], behind, out=g[:, i])
        behind = a[:, i] * g[:, i]
    out = {'h': h, 'dx': g, 'da': torch.cat([g[:, :1] * first[:, None], g[:, 1:] * h[:, :-1]], 1)}
    if c['start']:
        out['dh0'] = behind
    return out


def exact(case, seed):
    t = _tensors(case, seed)
    return {'attention': _exact_attention, 'rope': _exact_rope, 'scan': _exact_scan}[case['op']](case, t)

"""The sequence operators on the GPU against 64 bits, at the sizes and masks where they can go wrong."""
import numpy as np
import pytest
import torch

import _sequence as R
from tensorgrad_amd import backend, nn
from tensorgrad_amd import ir as IR
from tensorgrad_amd import ops as O
from tensorgrad_amd.compile import compile as tg_compile
from tensorgrad_amd.compile import compile_forward
from tensorgrad_amd.module import Module

pytestmark = pytest.mark.gpu


def rng(*key):
    return np.random.default_rng(list(key))


def f32(a):
    return np.ascontiguousarray(a, np.float32)


def forward(fn, arrays, decl=None, stream=0):
    """The outputs of a traced forward, run in device memory."""
    decl = decl or {n: {'shape': list(a.shape), 'dtype': 'i32' if a.dtype == np.int32 else 'f32'} for n, a in arrays.items()}
    ex = compile_forward(Module(), lambda m, i: fn(i), decl, seed=0)
    g = ex.graph_for(arrays).graph
    dev = {n: torch.from_numpy(a).cuda() for n, a in arrays.items()}
    outs = [torch.full(g.tensors[t].shape, float('nan'), device='cuda') for t in g.outputs]
    torch.cuda.synchronize()
    r = ex.run_device(dev, outs, stream)
    if r.error is not None:
        raise r.error
    torch.cuda.synchronize()
    got = [o.cpu().numpy() for o in outs]
    ex.destroy()
    return got


def attend(q, k, v, dy=None, how=None, masks=None):
    """{'y', ...} of the package for numpy inputs."""
    how, masks = how or {}, masks or {}
    arrays = dict(q=q, k=k, v=v, **masks, **({} if dy is None else {'dy': dy}))

    def fn(i):
        m = {n: i[n] for n in masks}
        y = O.attention(i['q'], i['k'], i['v'], **how, **m)
        return [y] if dy is None else [y, *O.attention_grad(i['q'], i['k'], i['v'], y, i['dy'], **how, **m)]
    return dict(zip(('y', 'dq', 'dk', 'dv'), forward(fn, arrays)))


def check_attention(q, k, v, dy, how, masks, what=''):
    want, tol = R.attention(q, k, v, dy, **how, **masks)
    got = attend(q, k, v, dy, how, masks)
    for n in want:
        R.check(got[n], want[n], tol[n], f'{what} {n}')
    return got


def qkv(B, H, Hk, Tq, Tk, D, Dv, seed, size=1.0):
    r = rng(B, H, Tq, Tk, D, Dv, seed)
    return (f32(size * r.standard_normal((B, H, Tq, D))), f32(r.standard_normal((B, Hk, Tk, D))),
            f32(r.standard_normal((B, Hk, Tk, Dv))), f32(r.standard_normal((B, H, Tq, Dv))))


SHAPES = [  # B, H, Hk, Tq, Tk, D, Dv
    (1, 1, 1, 1, 1, 1, 1), (2, 2, 1, 2, 3, 5, 7), (2, 4, 2, 16, 16, 16, 16), (1, 2, 2, 31, 33, 32, 32), (1, 3, 1, 65, 97, 40, 24),
    (1, 2, 1, 129, 129, 64, 64), (1, 2, 1, 100, 260, 96, 96), (1, 4, 1, 70, 130, 128, 128), (2, 1, 1, 64, 64, 127, 1),
    (1, 7, 1, 3, 300, 80, 80), (3, 2, 2, 1, 517, 64, 64), (1, 16, 2, 1, 1030, 128, 128), (1, 2, 2, 8, 640, 17, 64),
]


@pytest.mark.parametrize('shape', SHAPES)
@pytest.mark.parametrize('how', [dict(), dict(causal=False), dict(softcap=3.0, scale=0.3), dict(slopes=True), dict(softcap=20.0, slopes=True)],
                         ids=['causal', 'full', 'cap', 'slopes', 'cap+slopes'])
def test_attention_shapes_and_scores(shape, how):
    B, H, Hk, Tq, Tk, D, Dv = shape
    how = dict(how)
    if how.get('slopes'):
        how['slopes'] = [2.0 ** (-i - 1) for i in range(H)]
    check_attention(*qkv(*shape, 1, 2.0), how, {}, str(shape))


@pytest.mark.parametrize('shape', [(2, 3, 5, 7), (3, 2, 40, 64), (2, 2, 100, 32), (2, 2, 260, 128)])
@pytest.mark.parametrize('kind', ['documents', 'scattered', 'padding', 'prefix', 'lengths', 'all', 'nothing'])
def test_attention_masks(shape, kind):
    B, H, T, D = shape
    q, k, v, dy = qkv(B, H, 1, T, T, D, D, 2)
    r = rng(T, D, 7)
    how, masks = {}, {}
    if kind in ('documents', 'all'):
        masks['documents'] = np.sort(r.integers(0, 4, (B, T), dtype=np.int32), 1)
    if kind == 'scattered':                              # ids in any order, without a causal mask
        masks['documents'] = r.integers(-1, 3, (B, T), dtype=np.int32)
        how['causal'] = False
    if kind in ('padding', 'all'):
        d = masks.setdefault('documents', np.zeros((B, T), np.int32))
        d[0, T - T // 3:] = -1
        d[1, :T // 3] = -5
    if kind in ('prefix', 'all'):
        masks['prefix'] = np.array([T // 2, 0, T + 9][:B], np.int32)
    if kind in ('lengths', 'all'):                       # fewer places than queries: the first ones lie before position 0
        masks['lengths'] = np.array([T, T // 2, 0][:B], np.int32)
    if kind == 'nothing':
        masks['documents'] = np.full((B, T), -1, np.int32)
    got = check_attention(q, k, v, dy, how, masks, kind)
    if kind == 'nothing':
        assert not any(np.any(x) for x in got.values())


@pytest.mark.parametrize('D', [16, 40, 64, 96, 128])
@pytest.mark.parametrize('scores', [dict(softcap=30.0), dict(softcap=0.5), dict(slopes=[0.5, -0.1]), dict(softcap=5.0, slopes=[0.5, 0.02])],
                         ids=['cap', 'low cap', 'slopes', 'both'])
@pytest.mark.parametrize('T,kind', [(20, 'all'), (90, 'documents'), (150, 'prefix'), (260, 'all'), (130, 'lengths')])
def test_attention_scores_with_masks(T, kind, scores, D):
    """Every variant of the kernels under every kind of mask."""
    q, k, v, dy = qkv(2, 2, 1, T, T, D, D, 27)
    r, masks = rng(T, D, 28), {}
    if kind in ('documents', 'all'):
        masks['documents'] = np.sort(r.integers(-1, 4, (2, T), dtype=np.int32), 1)
    if kind in ('prefix', 'all'):
        masks['prefix'] = np.array([T // 2, 3], np.int32)
    if kind in ('lengths', 'all'):
        masks['lengths'] = np.array([T - 1, T // 2], np.int32)
    check_attention(q, k, v, dy, scores, masks, kind)


@pytest.mark.parametrize('Tq,Tk', [(1, 1), (1, 31), (1, 700), (5, 700), (33, 700), (128, 1000)])
@pytest.mark.parametrize('causal', [True, False])
def test_attention_over_a_part_filled_cache(Tq, Tk, causal):
    """Lengths from none to beyond the cache (clamped); what lies behind them is garbage."""
    q, k, v, dy = qkv(5, 4, 2, Tq, Tk, 64, 64, 3)
    n = np.array([0, 1, Tk // 2, Tk, Tk + 1000], np.int32)
    for b in range(5):
        k[b, :, min(n[b], Tk):], v[b, :, min(n[b], Tk):] = np.nan, np.inf
    check_attention(q, k, v, dy, dict(causal=causal), dict(lengths=n), f'{Tq}x{Tk}')
    check_attention(q, k, v, None, dict(causal=causal), dict(lengths=n), f'{Tq}x{Tk} forward')


@pytest.mark.parametrize('Tq,H,D', [(1, 1, 64), (1, 4, 128), (2, 2, 96), (4, 4, 32), (3, 1, 17)])
@pytest.mark.parametrize('scores', [{}, dict(softcap=4.0), dict(softcap=30.0, slopes=True)], ids=['plain', 'cap', 'both'])
def test_few_rows_with_masks(Tq, H, D, scores):
    """The last tokens against a long cache with documents, a prefix and lengths."""
    q, k, v, _ = qkv(3, H, 1, Tq, 900, D, D, 29)
    r = rng(Tq, D, 30)
    doc = np.sort(r.integers(0, 3, (3, 900), dtype=np.int32), 1)
    doc[1, 870:] = -1
    masks = dict(documents=doc, prefix=np.array([0, 5, 900], np.int32), lengths=np.array([900, 900, 555], np.int32))
    how = dict(scores, slopes=[0.3 / (n + 1) for n in range(H)]) if 'slopes' in scores else scores
    check_attention(q, k, v, None, how, masks)


@pytest.mark.parametrize('bad', [np.nan, np.inf, -np.inf, 3.4e38])
@pytest.mark.parametrize('what', ['padding', 'document', 'future', 'padded query'])
def test_masked_garbage_stays_out(bad, what):
    B, H, T, D = 1, 2, 90, 32
    q, k, v, dy = qkv(B, H, 1, T, T, D, D, 4)
    doc = np.repeat(np.array([[0, 1, 2]], np.int32), 30, 1)
    masks, how = dict(documents=doc), {}
    if what == 'padding':
        doc[:, 60:] = -1
        k[:, :, 60:], v[:, :, 60:] = bad, bad
    elif what == 'document':                             # a whole document of it: its own rows may be anything
        k[:, :, 30:60], v[:, :, 30:60] = bad, bad
        want, tol = R.attention(q, k, v, **masks)
        got = attend(q, k, v, None, how, masks)['y']
        rows = np.r_[0:30, 60:90]
        R.check(got[:, :, rows], want['y'][:, :, rows], tol['y'][:, :, rows], what)
        return
    elif what == 'future':                               # seen by the last query alone
        masks = {}
        k[:, :, -1], v[:, :, -1] = bad, bad
        want, tol = R.attention(q, k, v)
        got = attend(q, k, v)['y']
        R.check(got[:, :, :-1], want['y'][:, :, :-1], tol['y'][:, :, :-1], what)
        return
    else:
        doc[:, 60:] = -1
        q[:, :, 60:], dy[:, :, 60:] = bad, bad
        k[:, :, 60:], v[:, :, 60:] = bad, bad
    got = check_attention(q, k, v, dy, how, masks, what)
    assert not np.any(got['y'][:, :, 60:]) and not np.any(got['dq'][:, :, 60:])
    assert not np.any(got['dk'][:, :, 60:]) and not np.any(got['dv'][:, :, 60:])


def test_visible_infinities_reach_the_result():
    q, k, v, _ = qkv(1, 1, 1, 40, 40, 32, 32, 5)
    v[0, 0, 3, 2] = np.inf
    v[0, 0, 20, 5] = np.nan
    y = attend(q, k, v)['y'][0, 0]
    assert np.all(y[3:, 2] == np.inf) and np.all(np.isfinite(y[:3])) and np.all(np.isfinite(y[:, 3]))
    assert np.all(np.isnan(y[20:, 5])) and np.all(np.isfinite(y[:20, 5]))


@pytest.mark.parametrize('size', [1e-6, 1e-3, 1e3])
def test_attention_keeps_small_and_large_values(size):
    """Scores stay moderate (the scale undoes the size); values and gradients carry it."""
    q, k, v, dy = qkv(1, 2, 1, 70, 70, 64, 64, 6)
    check_attention(f32(q * size), f32(k * size), f32(v * size), f32(dy / size), dict(scale=0.125 / size ** 2), {}, str(size))


def test_columns_of_very_different_size():
    q, k, v, dy = qkv(1, 1, 1, 80, 80, 32, 32, 8)
    v[..., 0] *= 4000
    k[..., 1] *= 300
    q[..., 1] /= 300
    check_attention(q, k, v, dy, {}, {})


def test_large_scores_do_not_overflow():
    q, k, v, dy = qkv(1, 2, 1, 40, 40, 16, 16, 9)
    check_attention(f32(60 * q), f32(10 * k), v, dy, {}, {}, 'plain')
    check_attention(f32(60 * q), f32(10 * k), v, dy, dict(softcap=5.0), {}, 'cap')


def test_attention_gradient_against_differences():
    """Directional differences of the package's own forward, in steps where f32 resolves them: with values of size 1, a
    difference over 2 h at h = 2^-6 is off by h^2 times the third derivative (some 1e-3 here) and 2^-24 / h of rounding."""
    r = rng(11)
    q, k, v, dy = qkv(1, 2, 1, 24, 24, 16, 16, 10)
    how = dict(softcap=4.0, slopes=[0.25, 0.125])
    got = attend(q, k, v, dy, how)
    for name, x in (('dq', q), ('dk', k), ('dv', v)):
        u = f32(r.standard_normal(x.shape) / np.sqrt(x.size))
        h = 2.0 ** -6
        sides = []
        for s in (1, -1):
            args = dict(q=q, k=k, v=v)
            args[name[1]] = f32(x + s * h * u)
            sides.append((attend(args['q'], args['k'], args['v'], None, how)['y'].astype(np.float64) * dy).sum())
        diff = (sides[0] - sides[1]) / (2 * h)
        assert abs(diff - (got[name].astype(np.float64) * u).sum()) <= 1e-3 * np.abs(got[name] * u).sum() + 1e-3


def test_attention_is_deterministic():
    q, k, v, dy = qkv(2, 4, 2, 300, 300, 64, 64, 12)
    a, b = attend(q, k, v, dy), attend(q, k, v, dy)
    assert all(np.array_equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize('T,D', [(30, 16), (150, 64), (600, 128)])
@pytest.mark.parametrize('what', ['q', 'k', 'v', 'dy', 'all'])
def test_rows_of_very_different_size(T, D, what):
    """Neighbouring rows apart by up to 2^24 (2^48 in the products): each keeps its own precision."""
    x = dict(zip(('q', 'k', 'v', 'dy'), qkv(1, 2, 1, T, T, D, D, 13)))
    r = rng(14, T)
    for n in x if what == 'all' else (what,):
        x[n] = f32(x[n] * 2.0 ** r.integers(-24, 1, (1, x[n].shape[1], T, 1)))
    check_attention(*x.values(), dict(softcap=30.0), {}, what)


@pytest.mark.parametrize('Tq,Tk,D', [(20, 5, 16), (130, 33, 64), (700, 300, 128), (3, 1, 8)])
def test_more_queries_than_keys(Tq, Tk, D):
    """Without positions; the second entry's keys are none."""
    q, k, v, dy = qkv(3, 4, 2, Tq, Tk, D, D, 15)
    check_attention(q, k, v, dy, dict(causal=False), {})
    check_attention(q, k, v, dy, dict(causal=False, softcap=2.0), dict(lengths=np.array([Tk, 0, Tk // 2], np.int32)))


@pytest.mark.parametrize('T,D,kind', [(1300, 40, 'documents'), (1100, 96, 'prefix'), (900, 128, 'all'), (1500, 16, 'one document')])
def test_long_rows_in_parts(T, D, kind):
    """Three query heads a key head and walks that are cut into parts, forward and backward; the same bits twice."""
    q, k, v, dy = qkv(1, 3, 1, T, T, D, D, 16)
    r, masks = rng(T, 17), {}
    if kind in ('documents', 'all'):
        masks['documents'] = np.sort(r.integers(0, 5, (1, T), dtype=np.int32), 1)
        masks['documents'][:, T - 37:] = -1
    if kind == 'one document':
        masks['documents'] = np.zeros((1, T), np.int32)
    if kind in ('prefix', 'all'):
        masks['prefix'] = np.array([T // 3], np.int32)
    if kind == 'all':
        masks['lengths'] = np.array([T - 100], np.int32)
    a = check_attention(q, k, v, dy, {}, masks, kind)
    b = attend(q, k, v, dy, {}, masks)
    assert all(np.array_equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize('bad', [np.nan, np.inf, 3.4e38])
@pytest.mark.parametrize('T,D', [(48, 16), (600, 64), (600, 128)])
def test_gradients_beside_a_document_of_garbage(bad, T, D):
    """Of three documents the middle one is not finite: the gradients of the others are as without it."""
    q, k, v, dy = qkv(1, 2, 1, T, T, D, D, 18)
    doc = np.repeat(np.array([[0, 1, 2]], np.int32), T // 3, 1)
    mid, rest = slice(T // 3, 2 * T // 3), np.r_[0:T // 3, 2 * T // 3:T]
    want, tol = R.attention(q, k, v, dy, documents=doc)
    for x in (q, k, v, dy):
        x[:, :, mid] = bad
    got = attend(q, k, v, dy, {}, dict(documents=doc))
    for n in want:
        R.check(got[n][:, :, rest], want[n][:, :, rest], tol[n][:, :, rest], n)


@pytest.mark.parametrize('T,D', [(24, 16), (200, 64)])
def test_one_tensor_in_every_place_and_gradients_asked_twice(T, D):
    x, dy = f32(rng(19, T).standard_normal((2, 2, T, D))), f32(rng(20, T).standard_normal((2, 2, T, D)))

    def fn(i):
        y = O.attention(i['x'], i['x'], i['x'])
        return [y, *O.attention_grad(i['x'], i['x'], i['x'], y, i['dy']), *O.attention_grad(i['x'], i['x'], i['x'], y, i['dy'])]
    got = forward(fn, dict(x=x, dy=dy))
    want, tol = R.attention(x, x, x, dy)
    for n, g in zip(('y', 'dq', 'dk', 'dv', 'dq', 'dk', 'dv'), got):
        R.check(g, want[n], tol[n], n)


@pytest.mark.parametrize('T,D', [(20, 24), (150, 32), (700, 64), (200, 96), (800, 128)])
@pytest.mark.parametrize('which', [0, 1, 2, (0, 1), (2, 0), (1, 2)])
@pytest.mark.parametrize('how', [{}, dict(softcap=10.0)], ids=['plain', 'cap'])
def test_some_of_the_gradients(T, D, which, how):
    """What is not asked for is not computed; what is, is the same."""
    q, k, v, dy = qkv(1, 2, 1, T, T, D, D, 31)
    doc = np.sort(rng(T, 32).integers(0, 3, (1, T), dtype=np.int32), 1)
    which = (which,) if isinstance(which, int) else which

    def fn(i):
        m = dict(how, documents=i['documents'])
        g = O.attention_grad(i['q'], i['k'], i['v'], O.attention(i['q'], i['k'], i['v'], **m), i['dy'], **m)
        return [g[n] for n in which]
    got = forward(fn, dict(q=q, k=k, v=v, dy=dy, documents=doc))
    want, tol = R.attention(q, k, v, dy, documents=doc, **how)
    for n, g in zip(which, got):
        name = ('dq', 'dk', 'dv')[n]
        R.check(g, want[name], tol[name], name)


def test_strided_heads_and_gradients():
    """q, k and v as views of one projection, heads of 40 in rows of 200: read in place, whatever their alignment."""
    B, T, D = 2, 90, 40
    r = rng(33)
    x, dy = f32(r.standard_normal((B, T, 5 * D))), f32(r.standard_normal((B, 3, T, D)))

    def fn(i):
        a, b, c = O.split(i['x'], [3 * D, D, D], -1)
        q, k, v = O.split_heads(a, 3), O.split_heads(b, 1), O.split_heads(c, 1)
        y = O.attention(q, k, v)
        return [y, *O.attention_grad(q, k, v, y, i['dy'])]
    got = forward(fn, dict(x=x, dy=dy))
    heads = lambda z: f32(z.reshape(B, T, -1, D).transpose(0, 2, 1, 3))  # noqa: E731
    want, tol = R.attention(heads(x[..., :3 * D]), heads(x[..., 3 * D:4 * D]), heads(x[..., 4 * D:]), dy)
    for n, g in zip(('y', 'dq', 'dk', 'dv'), got):
        R.check(g, want[n], tol[n], n)


@pytest.mark.parametrize('T', [3, 70])
def test_more_key_heads_than_a_grid_axis_holds(T):
    """70000 key heads, forward: of a few positions, and one token against a longer cache."""
    B, Tq = 70000, 3 if T == 3 else 1
    q, k, v, dy = qkv(B, 1, 1, Tq, T, 4, 4, 21)
    y = attend(q, k, v)['y']
    pick = np.r_[0:20, 65530:65545, B - 20:B]
    want, tol = R.attention(q[pick], k[pick], v[pick])
    R.check(y[pick], want['y'], tol['y'])
    assert np.isfinite(y).all()


# ---- rotary positions -----------------------------------------------------------------------------

@pytest.mark.parametrize('B,H,Hk,T,D,sections', [
    (1, 1, 1, 1, 2, [1]), (2, 3, 1, 7, 10, [2, 1, 2]), (2, 4, 2, 33, 64, [8, 12, 12]), (1, 2, 2, 130, 96, [8, 8]),
    (3, 1, 1, 5, 7, [1, 1]), (1, 2, 1, 64, 128, [16, 24, 24]), (33, 16, 4, 1, 80, [40]), (1, 2, 2, 9, 6, [1, 1, 1])])
@pytest.mark.parametrize('per_axis', [False, True])
@pytest.mark.parametrize('inverse', [False, True])
def test_rope_axes(B, H, Hk, T, D, sections, per_axis, inverse):
    r = rng(T, D, len(sections))
    q, k = f32(r.standard_normal((B, H, T, D))), f32(r.standard_normal((B, Hk, T, D)))
    pos = r.integers(-50, 2000000, (len(sections), B, T), dtype=np.int32)
    pos.flat[:2] = [0, 2 ** 31 - 1][:pos.size]
    got = forward(lambda i: list(O.rope_axes(i['q'], i['k'], i['p'], sections, 5000.0, per_axis, inverse)), dict(q=q, k=k, p=pos))
    for g, x in zip(got, (q, k)):
        want, tol = R.rope_axes(x, pos, sections, 5000.0, per_axis, inverse)
        R.check(g, want, tol)


def test_rope_axes_of_more_heads_than_a_grid_axis_holds():
    r = rng(26)
    q, k = f32(r.standard_normal((1, 200000, 1, 2))), f32(r.standard_normal((1, 1, 1, 2)))
    pos = np.array([[[5]]], np.int32)
    got = forward(lambda i: list(O.rope_axes(i['q'], i['k'], i['p'], [1])), dict(q=q, k=k, p=pos))
    for g, x in zip(got, (q, k)):
        R.check(g, *R.rope_axes(x, pos, [1]))


def test_rope_axes_passes_infinities_of_other_pairs():
    q = f32(rng(1).standard_normal((1, 1, 3, 8)))
    q[0, 0, 1, 6] = np.inf
    y = forward(lambda i: list(O.rope_axes(i['q'], i['q'], i['p'], [2])), dict(q=q, p=np.arange(3, dtype=np.int32).reshape(1, 1, 3)))[0]
    assert y[0, 0, 1, 6] == np.inf and np.isfinite(np.delete(y.ravel(), 14)).all()


# ---- recurrence ------------------------------------------------------------------------------------

@pytest.mark.parametrize('B,T,C', [(1, 1, 1), (2, 2, 3), (3, 17, 64), (2, 63, 65), (1, 128, 256), (2, 257, 33), (1, 1000, 7), (4, 515, 130),
                                   (1, 4097, 12), (300, 3, 5)])
@pytest.mark.parametrize('start', [False, True])
def test_recurrence(B, T, C, start):
    r = rng(B, T, C)
    a = f32(1 / (1 + np.exp(-r.standard_normal((B, T, C)) - 3)))
    a[:, T // 2:T // 2 + 1] = 0                          # a fresh start half way
    x, dh, h0 = (f32(r.standard_normal(s)) for s in ((B, T, C), (B, T, C), (B, C)))
    ins = dict(a=a, x=x, dh=dh, **(dict(h0=h0) if start else {}))

    def fn(i):
        h = O.linear_recurrence(i['a'], i['x'], i.get('h0'))
        return [h, *O.linear_recurrence_grad(i['a'], h, i['dh'], i.get('h0'))]
    got = dict(zip(('h', 'da', 'dx', 'dh0'), forward(fn, ins)))
    want, tol = R.recurrence(a, x, h0 if start else None, dh)
    for n in want:
        R.check(got[n], want[n], tol[n], n)


def test_recurrence_gates_of_any_sign_and_size():
    """Gates beyond 1 grow, negative ones alternate; a zero gate forgets what came before (by its product: only finite
    values)."""
    r = rng(21)
    a = f32(r.uniform(-1.1, 1.1, (2, 300, 40)))
    x, dh = f32(r.standard_normal(a.shape)), f32(r.standard_normal(a.shape))

    def fn(i):
        h = O.linear_recurrence(i['a'], i['x'])
        return [h, *O.linear_recurrence_grad(i['a'], h, i['dh'])]
    got = dict(zip(('h', 'da', 'dx'), forward(fn, dict(a=a, x=x, dh=dh))))
    want, tol = R.recurrence(a, x, None, dh)
    for n in want:
        R.check(got[n], want[n], tol[n], n)


def test_recurrence_does_not_look_ahead_or_across():
    r = rng(22)
    a, x = f32(r.uniform(0.5, 1, (3, 700, 20))), f32(r.standard_normal((3, 700, 20)))
    clean = forward(lambda i: [O.linear_recurrence(i['a'], i['x'])], dict(a=a, x=x))[0]
    a[1, 400:], x[1, 400:] = np.nan, np.inf
    got = forward(lambda i: [O.linear_recurrence(i['a'], i['x'])], dict(a=a, x=x))[0]
    assert np.array_equal(got[[0, 2]], clean[[0, 2]]) and np.array_equal(got[1, :400], clean[1, :400])
    assert np.isnan(got[1, 400:]).all()


def scan_and_gradients(a, x, dh, h0):
    def fn(i):
        h = O.linear_recurrence(i['a'], i['x'], i['h0'])
        return [h, *O.linear_recurrence_grad(i['a'], h, i['dh'], i['h0'])]
    return dict(zip(('h', 'da', 'dx', 'dh0'), forward(fn, dict(a=a, x=x, dh=dh, h0=h0))))


@pytest.mark.parametrize('B,T,C,gate,live', [(1, 700, 5, 4, 40), (2, 900, 70, 1024, 6), (4, 2048, 256, 1.5, 100), (4, 2048, 256, 4, 40),
                                             (1, 60, 3, 1024, 6)])
def test_recurrence_products_of_gates_beyond_the_range_of_values(B, T, C, gate, live):
    """Nothing comes in until the last `live` steps: every state is a finite number, though the gates' product is not. In the
    gradient's direction, dh ends before the first steps."""
    r = rng(23, T)
    a = f32(np.full((B, T, C), gate))
    a[:, :, ::2] *= -1
    x, dh = (f32(r.standard_normal(a.shape)) for _ in range(2))
    x[:, :-live] = 0
    dh[:, live:] = 0
    h0 = f32(np.zeros((B, C)))
    got = scan_and_gradients(a, x, dh, h0)
    want, tol = R.recurrence(a, x, h0, dh)
    for n in want:
        R.check(got[n], want[n], tol[n], n)


def test_recurrence_that_fades_and_comes_back():
    """The state falls by 2^112 and rises again, over and over, at borders that no chunk shares."""
    r = rng(24)
    a = f32(np.where(np.arange(1000) // 56 % 2 == 0, 0.25, 4.0)[None, :, None] * np.ones((2, 1, 70)))
    dh, h0 = f32(r.standard_normal(a.shape)), f32(r.standard_normal((2, 70)))
    got = scan_and_gradients(a, np.zeros_like(a), dh, h0)
    want, tol = R.recurrence(a, np.zeros_like(a), h0, dh)
    for n in want:
        R.check(got[n], want[n], tol[n], n)


def test_recurrence_gates_that_are_not_finite():
    r = rng(25)
    a, x = f32(r.uniform(0.5, 1, (1, 500, 70))), f32(r.standard_normal((1, 500, 70)))
    a[0, 333, 3], a[0, 130, 66] = np.inf, np.nan
    got = forward(lambda i: [O.linear_recurrence(i['a'], i['x'])], dict(a=a, x=x))[0]
    with np.errstate(all='ignore'):
        want, tol = R.recurrence(a, x)
    assert np.isinf(got[0, 333:, 3]).all() and (np.sign(got[0, 333:, 3]) == np.sign(want['h'][0, 333:, 3])).all()
    assert np.isnan(got[0, 130:, 66]).all()
    fine = np.isfinite(want['h'])
    assert (np.isfinite(got) == fine).all()
    R.check(got[fine], want['h'][fine], tol['h'][fine], 'h')


# ---- together, as a model uses them ------------------------------------------------------------------

VOCAB, DIM, HEADS, KV = 29, 32, 4, 2


class Mixed(Module):
    """An attention layer with turned positions and a recurrent layer over a packed batch."""

    def __init__(self):
        self.emb = nn.Embedding(VOCAB, DIM)
        self.q, self.k, self.v, self.o = (nn.Linear(DIM, n, bias=False) for n in (DIM, DIM * KV // HEADS, DIM * KV // HEADS, DIM))
        self.gate, self.val = nn.Linear(DIM, DIM), nn.Linear(DIM, DIM)
        self.head = nn.Linear(DIM, VOCAB)


def mixed_logits(p, i):
    x = p.emb.fwd(i['tokens'])
    q, k, v = (O.split_heads(m.fwd(x), n) for m, n in ((p.q, HEADS), (p.k, KV), (p.v, KV)))
    q, k = O.rope_axes(q, k, i['positions'], [2, 2])
    y = O.attention(q, k, v, softcap=8.0, slopes=[0.5, 0.25, 0.125, 0.0625], documents=i['documents'], prefix=i['prefix'])
    x = O.add(x, p.o.fwd(O.merge_heads(y)))
    a = O.mul(O.sigmoid(p.gate.fwd(x)), O.reshape(i['keep'], [*i['keep'].shape, 1]))
    x = O.add(x, O.linear_recurrence(a, O.tanh(p.val.fwd(x))))
    return p.head.fwd(x)


def mixed_batch(B, T, seed):
    r = rng(B, T, seed)
    doc = np.sort(r.integers(0, 3, (B, T), dtype=np.int32), 1)
    doc[:, T - 2:] = -1
    fresh = np.concatenate([np.ones((B, 1), bool), doc[:, 1:] != doc[:, :-1]], 1)
    at = np.arange(T) - np.maximum.accumulate(np.where(fresh, np.arange(T), 0), 1)
    return {'tokens': r.integers(0, VOCAB, (B, T), dtype=np.int32), 'targets': r.integers(0, VOCAB, (B, T), dtype=np.int32),
            'documents': doc, 'positions': np.ascontiguousarray(np.stack([at, at // 3]).astype(np.int32)),
            'prefix': r.integers(0, T // 2, B, dtype=np.int32), 'keep': f32(~fresh)}


def mixed_torch(w, i, B, T):
    """The same loss in f64 torch, for autograd."""
    t = {n: torch.from_numpy(a) for n, a in i.items()}
    x = w['emb.W'][t['tokens'].long()]
    heads = lambda n, h: (x @ w[n + '.W']).reshape(B, T, h, -1).transpose(1, 2)  # noqa: E731
    q, k, v = heads('q', HEADS), heads('k', KV), heads('v', KV)
    freq = 10000.0 ** -(torch.arange(4, dtype=torch.float64) / 4)
    ang = t['positions'].double()[[0, 0, 1, 1]].permute(1, 2, 0) * freq
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    turn = lambda z: torch.cat([z[..., :4] * c - z[..., 4:] * s, z[..., 4:] * c + z[..., :4] * s], -1)  # noqa: E731
    q, k = turn(q), turn(k).repeat_interleave(HEADS // KV, 1)
    sc = q @ k.transpose(-1, -2) / 8 ** 0.5
    j = torch.arange(T)
    sc = 8 * torch.tanh(sc / 8) - torch.tensor([0.5, 0.25, 0.125, 0.0625]).double()[:, None, None] * (j[:, None] - j).abs()
    d = t['documents']
    ok = ((j <= j[:, None]) | (j < t['prefix'][:, None, None])) & (d[:, :, None] == d[:, None, :]) & (d[:, None, :] >= 0)
    ok = ok[:, None]
    P = torch.softmax(sc.masked_fill(~ok, -1e300), -1).masked_fill(~ok, 0)
    y = (P @ v.repeat_interleave(HEADS // KV, 1)).transpose(1, 2).reshape(B, T, DIM)
    x = x + y @ w['o.W']
    a = torch.sigmoid(x @ w['gate.W'] + w['gate.b']) * t['keep'].double()[..., None]
    z = torch.tanh(x @ w['val.W'] + w['val.b'])
    h, hs = torch.zeros(B, DIM).double(), []
    for n in range(T):
        h = a[:, n] * h + z[:, n]
        hs.append(h)
    x = x + torch.stack(hs, 1)
    logits = x @ w['head.W'] + w['head.b']
    return torch.nn.functional.cross_entropy(logits.reshape(-1, VOCAB), t['targets'].long().reshape(-1)), logits


@pytest.mark.parametrize('B,T', [(2, 12), (3, 65)])
def test_model_of_them_trains_as_in_64_bits(B, T):
    """One SGD step at rate 1 from known weights: what the weights moved by is the gradient. Chains of some ten f32 operations
    and sums over B T positions: 2e-5 of each gradient's norm is about 300 roundings."""
    batch = mixed_batch(B, T, 1)
    decl = {n: {'shape': list(a.shape), 'dtype': 'i32' if a.dtype == np.int32 else 'f32'} for n, a in batch.items()}
    t = tg_compile(Mixed(), lambda p, i: nn.cross_entropy(mixed_logits(p, i), i['targets']), decl, {'kind': 'sgd', 'lr': 1.0}, seed=3)
    before = t.download_params()
    shapes = t.ir.param_shapes()
    r = t.step(batch)
    assert r.kind == 'completed', r.error
    after = t.download_params()
    w = {n: torch.from_numpy(a.reshape(shapes[n])).double().requires_grad_(True) for n, a in before.items()}
    loss, logits = mixed_torch(w, batch, B, T)
    assert abs(r.loss - float(loss)) <= 1e-5 * abs(float(loss))
    grads = dict(zip(w, torch.autograd.grad(loss, list(w.values()))))
    for n, g in grads.items():
        moved = (before[n].astype(np.float64) - after[n]).reshape(shapes[n])
        # the difference of two f32 weights carries their own rounding
        slack = 2e-5 * np.linalg.norm(g) + 2 * R.U * np.linalg.norm(before[n])
        assert np.linalg.norm(moved - g.numpy()) <= slack, n
    kinds = [n['kind'] for n in t._rt.describe()['nodes']]
    assert [kinds.count(k) for k in ('attend', 'attend_grad', 'rope', 'scan', 'scan_grad')] == [1, 1, 2, 1, 1]
    # the trained weights in a forward graph, from host arrays and in device memory
    f = t.attach(lambda p, i: mixed_logits(p, i), {n: d for n, d in decl.items() if n != 'targets'})
    out = f.run(batch).output
    w2 = {n: torch.from_numpy(a.reshape(shapes[n])).double() for n, a in after.items()}
    want = mixed_torch(w2, batch, B, T)[1].numpy()
    assert np.linalg.norm(out - want) <= 1e-5 * np.linalg.norm(want)
    dev = {n: torch.from_numpy(a).cuda() for n, a in batch.items()}
    got = torch.empty(out.shape, device='cuda')
    torch.cuda.synchronize()
    assert f.run_device(dev, [got]).error is None
    torch.cuda.synchronize()
    assert np.array_equal(got.cpu().numpy(), out)
    t.destroy()


def test_model_of_them_steps_alike_captured_and_launched(monkeypatch):
    """Captured steps, replayed with eager work and waits between, against steps launched one by one: the same bits."""
    B, T = 2, 150
    batches = [mixed_batch(B, T, n) for n in range(5)]
    decl = {n: {'shape': list(a.shape), 'dtype': 'i32' if a.dtype == np.int32 else 'f32'} for n, a in batches[0].items()}

    def train(graph):
        monkeypatch.setenv('TG_GRAPH', graph)
        t = tg_compile(Mixed(), lambda p, i: nn.cross_entropy(mixed_logits(p, i), i['targets']), decl, {'kind': 'adam', 'lr': 0.01}, seed=4)
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


# ---- device-resident calls -----------------------------------------------------------------------------

def _scan_executor(B=2, T=100, C=64):
    d = {'a': [B, T, C], 'x': [B, T, C]}
    ex = compile_forward(Module(), lambda m, i: [O.linear_recurrence(i['a'], i['x']), O.mul(i['a'], 2.0), O.reshape(i['x'], [B * T, C])], d, seed=0)
    r = rng(31)
    ins = {n: torch.from_numpy(f32(r.uniform(0.2, 1, s))).cuda() for n, s in d.items()}
    outs = [torch.empty(B, T, C, device='cuda'), torch.empty(B, T, C, device='cuda'), torch.empty(B * T, C, device='cuda')]
    torch.cuda.synchronize()
    return ex, ins, outs


def test_run_device_writes_every_output():
    """A recurrence bound to the caller's tensors beside a fused group (run on the runtime's own buffers) and an output that
    is a view of an input."""
    ex, ins, outs = _scan_executor()
    host = ex.run({n: t.cpu().numpy() for n, t in ins.items()}).output
    for _ in range(3):
        for o in outs:
            o.fill_(float('nan'))
        torch.cuda.synchronize()
        r = ex.run_device(ins, outs)
        assert r.error is None
        torch.cuda.synchronize()
        assert np.array_equal(outs[0].cpu().numpy(), host)
        assert torch.equal(outs[1], ins['a'] * 2) and torch.equal(outs[2], ins['x'].reshape(outs[2].shape))
    ex.destroy()


def test_run_device_follows_the_stream():
    """Producer, call and consumer on one stream, then on several, without the host waiting between."""
    ex, ins, outs = _scan_executor(4, 1000, 256)
    want = ex.run({n: t.cpu().numpy() for n, t in ins.items()}).output
    streams = [torch.cuda.Stream() for _ in range(3)]
    keep = []
    for turn in range(6):
        s = streams[turn % 3]
        with torch.cuda.stream(s):
            scaled = {n: t * 2 for n, t in ins.items()}
            scaled['a'] = scaled['a'] / 2
            o = [torch.empty_like(x) for x in outs]
            assert ex.run_device(scaled, o, s.cuda_stream).error is None
            keep.append((scaled, o, o[0] / 2))
    torch.cuda.synchronize()
    for _, _, half in keep:                             # doubling and halving are exact
        assert np.array_equal(half.cpu().numpy(), want)
    host = ex.run({n: t.cpu().numpy() for n, t in ins.items()}).output      # the host path waits for them
    assert np.array_equal(host, want)
    ex.destroy()


def test_run_device_refusals():
    ex, ins, outs = _scan_executor()
    bad = [
        (dict(ins, a=ins['a'].cpu()), outs, "input 'a': not"),
        (dict(ins, a=ins['a'][:1]), outs, 'elements'),
        (dict(ins, a=ins['a'].double()), outs, 'float32'),
        (dict(ins, a=ins['a'].transpose(0, 1).contiguous().transpose(0, 1)), outs, 'contiguous'),
        ({'a': ins['a']}, outs, 'missing input'),
        (ins, outs[:2], '3 outputs'),
        (ins, [ins['a'], outs[1], outs[2]], 'overlap'),
        (ins, [outs[0], outs[0], outs[2]], 'overlap'),
        (dict(ins, a=torch.empty(2 * 100 * 64 + 1, device='cuda')[1:]), outs, 'aligned'),
        (dict(ins, a=np.zeros((2, 100, 64), np.float32)), outs, 'device memory'),
    ]
    for i, o, what in bad:
        r = ex.run_device(i, o)
        assert r.kind == 'failed' and what in str(r.error), (what, r.error)
    n = 2 * 100 * 64 * 4
    with pytest.raises(backend.BackendError, match='expected'):
        ex._owner[0].run_device(['a', 'x'], [ins['a'].data_ptr(), ins['x'].data_ptr()], [n, n - 4], [o.data_ptr() for o in outs], [n] * 3)
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        graph.capture_begin(capture_error_mode='relaxed')
        r = ex.run_device(ins, outs, s.cuda_stream)
        graph.capture_end()
    assert r.kind == 'failed' and 'captured' in str(r.error)
    torch.cuda.synchronize()
    assert ex.run_device(ins, outs).kind == 'completed'
    ex.destroy()
    assert ex.run_device(ins, outs).kind == 'aborted'


def test_run_device_with_random_numbers_and_parameters():
    """Dropout takes a new seed each call, parameters may be replaced between calls; both as `run` does."""
    class M(Module):
        def __init__(self):
            self.l = nn.Linear(8, 8)
    fwd = lambda m, i: O.dropout(m.l.fwd(i['x']), 0.5)  # noqa: E731
    x = f32(rng(41).standard_normal((16, 8)))
    host, dev = (compile_forward(M(), fwd, {'x': [16, 8]}, seed=1) for _ in range(2))
    p = {n: f32(rng(42).standard_normal(a.shape)) for n, a in host.download_params().items()}
    out = [torch.empty(16, 8, device='cuda') for _ in range(4)]
    xd = torch.from_numpy(x).cuda()
    torch.cuda.synchronize()
    for turn in range(4):
        if turn == 2:
            host.upload_params(p)
            dev.upload_params(p)
        want = host.run({'x': x}).output
        assert dev.run_device({'x': xd}, [out[turn]]).error is None
        torch.cuda.synchronize()
        assert np.array_equal(out[turn].cpu().numpy(), want)
    host.destroy()
    dev.destroy()


def test_parametric_length_and_host_run():
    """One executor over growing caches: a graph per length, the same results as from host arrays."""
    ex = compile_forward(Module(), lambda m, i: O.attention(i['q'], i['k'], i['v'], lengths=i['n']),
                         {'q': [2, 4, 1, 32], 'k': [2, 2, None, 32], 'v': [2, 2, None, 32], 'n': {'shape': [2], 'dtype': 'i32'}}, seed=0)
    for T in (1, 40, 300):
        q, k, v, _ = qkv(2, 4, 2, 1, T, 32, 32, 51)
        n = np.array([T, (T + 1) // 2], np.int32)
        host = ex.run(dict(q=q, k=k, v=v, n=n)).output
        want, tol = R.attention(q, k, v, lengths=n)
        R.check(host, want['y'], tol['y'])
        out = torch.empty(2, 4, 1, 32, device='cuda')
        dev = {m: torch.from_numpy(a).cuda() for m, a in dict(q=q, k=k, v=v, n=n).items()}
        torch.cuda.synchronize()
        assert ex.run_device(dev, [out]).error is None
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy(), host)
    ex.destroy()


# ---- values at the ends of f32's range --------------------------------------------------------------------

@pytest.mark.parametrize('T,D', [(20, 16), (90, 64), (150, 128), (700, 40)])
@pytest.mark.parametrize('kind', ['causal', 'lengths', 'documents', 'prefix'])
@pytest.mark.parametrize('sizes', [(1e-20, 1e-20, None), (1e-35, 1e-3, None), (1e-3, 1e-35, None), (1e-10, 1e-10, 2.0 ** -60)],
                         ids=['both tiny', 'tiny q', 'tiny k', 'small scale'])
def test_scores_too_small_to_tell_apart(T, D, kind, sizes):
    """Products of q, k and the scale near or below f32's least: every key counts alike, hidden ones not at all."""
    q, k, v, dy = qkv(2, 2, 1, T, T, D, D, 61)
    r, how, masks = rng(T, 62), {}, {}
    if kind == 'lengths':
        how['causal'] = False
        masks['lengths'] = np.array([T - 1, T // 2], np.int32)
    if kind == 'documents':
        masks['documents'] = np.sort(r.integers(-1, 3, (2, T), dtype=np.int32), 1)
    if kind == 'prefix':
        masks['prefix'] = np.array([T // 2, 3], np.int32)
    if sizes[2]:
        how['scale'] = sizes[2]
    check_attention(f32(q * sizes[0]), f32(k * sizes[1]), v, dy, how, masks, kind)


def test_one_tiny_query_row_among_others():
    q, k, v, dy = qkv(1, 2, 1, 150, 150, 64, 64, 63)
    q[0, :, 77] *= 1e-36
    check_attention(q, f32(k * 1e-2), v, dy, {}, {})


@pytest.mark.parametrize('T', [40, 150])
@pytest.mark.parametrize('how', [{}, dict(softcap=5.0), dict(slopes=[0.0, 0.0])], ids=['plain', 'cap', 'slopes'])
def test_large_rows_whose_products_vanish(T, how):
    """q has only even features, k only odd ones, of 1e25: all scores are exactly 0, so y is the mean of the seen values, though
    the sizes' product passes f32's range. v and dy likewise: dP is 0. A mean of n values in f32 from weights off by some 20
    roundings: 64 (16 + 4 sqrt n) roundings of the mean absolute value are generous."""
    q, k, v, dy = qkv(1, 2, 1, T, T, 64, 64, 64)
    q, k = f32(q * 1e25), f32(k * 1e25)
    q[..., 1::2], k[..., ::2] = 0, 0
    n = np.arange(1, T + 1)[:, None]
    got = attend(q, k, v, dy, how)
    slack = 64 * (16 + 4 * np.sqrt(T)) * R.U
    for h in range(2):
        want = np.cumsum(v[0, 0].astype(np.float64), 0) / n
        assert np.all(np.abs(got['y'][0, h] - want) <= slack * np.cumsum(np.abs(v[0, 0]), 0) / n)
    P = np.tril(np.ones((T, T))) / n
    G = dy[0].astype(np.float64)
    assert np.all(np.abs(got['dv'][0, 0] - sum(P.T @ G[h] for h in range(2))) <= slack * sum(P.T @ np.abs(G[h]) for h in range(2)))
    assert np.isfinite(got['dq']).all() and np.isfinite(got['dk']).all()


# ---- what is not finite and seen ----------------------------------------------------------------------------

SPLIT = [  # B, H, Hk, Tq, Tk, D: keys in parts, by the kernel of few rows and by tiles, joined by 32 and by 256 threads a row
    (8, 1, 1, 1, 1000, 64), (1, 4, 1, 1, 5000, 128), (1, 2, 2, 100, 600, 64), (1, 2, 1, 64, 5000, 32), (2, 2, 1, 300, 300, 64)]


@pytest.mark.parametrize('shape', SPLIT)
@pytest.mark.parametrize('bad', [np.nan, np.inf])
def test_a_query_that_is_not_finite_shows(shape, bad):
    """Its own row alone: an infinite query's scores are infinite (of either sign: NaN weights) or NaN."""
    B, H, Hk, Tq, Tk, D = shape
    q, k, v, _ = qkv(B, H, Hk, Tq, Tk, D, D, 71)
    want, tol = R.attention(q, k, v)
    q[0, 0, Tq // 2, 3] = bad
    y = attend(q, k, v)['y']
    assert np.isnan(y[0, 0, Tq // 2]).all()
    rest = np.ones((B, H, Tq), bool)
    rest[0, 0, Tq // 2] = False
    R.check(y[rest], want['y'][rest], tol['y'][rest])


@pytest.mark.parametrize('shape', SPLIT)
@pytest.mark.parametrize('at', ['first', 'middle', 'last'])
def test_a_key_that_is_not_a_number_shows_where_it_is_seen(shape, at):
    B, H, Hk, Tq, Tk, D = shape
    q, k, v, _ = qkv(B, H, Hk, Tq, Tk, D, D, 72)
    want, tol = R.attention(q, k, v)
    j = {'first': 0, 'middle': Tk - Tq // 2 - 1, 'last': Tk - 1}[at]
    k[0, 0, j, 5] = np.nan
    y = attend(q, k, v)['y']
    hit = np.zeros((B, H, Tq), bool)
    hit[0, :H // Hk, max(j - (Tk - Tq), 0):] = True
    assert np.isnan(y[hit]).all()
    R.check(y[~hit], want['y'][~hit], tol['y'][~hit])


@pytest.mark.parametrize('T,D', [(20, 16), (90, 64), (600, 64)])
def test_a_gradient_of_a_query_that_is_not_a_number(T, D):
    """dq of its row, and dk and dv of the keys it sees."""
    q, k, v, dy = qkv(1, 1, 1, T, T, D, D, 73)
    want, tol = R.attention(q, k, v, dy)
    at = T // 2
    q[0, 0, at, 3] = np.nan
    got = attend(q, k, v, dy)
    rest = np.arange(T) != at
    assert np.isnan(got['dq'][0, 0, at]).all() and np.isnan(got['y'][0, 0, at]).all()
    R.check(got['dq'][0, 0, rest], want['dq'][0, 0, rest], tol['dq'][0, 0, rest])
    for n in ('dk', 'dv'):
        assert np.isnan(got[n][0, 0, :at + 1]).all()
        R.check(got[n][0, 0, at + 1:], want[n][0, 0, at + 1:], tol[n][0, 0, at + 1:], n)


def check_keys_of_minus_infinity(shape):
    """A row that sees only scores of minus infinity has no softmax (NaN); beside others such a key counts for nothing."""
    B, H, Hk, Tq, Tk, D = shape
    q, k, v, _ = qkv(B, H, Hk, Tq, Tk, D, D, 74)
    q = np.abs(q) + f32(0.1)
    dead = Tk - Tq + 1                       # the first query sees these alone
    k[0, 0, :dead] = -np.inf                 # of one key head
    y = attend(q, k, v)['y']
    assert np.isnan(y[0, :H // Hk, 0]).all() and np.isfinite(y[0, H // Hk:]).all() and np.isfinite(y[1:]).all()
    if Tq > 1:
        doc = np.zeros((B, Tk), np.int32)
        doc[:, :dead] = -1
        want, tol = R.attention(q, np.where(np.isfinite(k), k, f32(0)), v, documents=doc)
        R.check(y[:, :, 1:], want['y'][:, :, 1:], tol['y'][:, :, 1:])


@pytest.mark.parametrize('shape', [(1, 1, 1, 20, 20, 16), (1, 1, 1, 90, 90, 64), (1, 2, 1, 300, 600, 64)])
def test_keys_of_minus_infinity_weigh_nothing(shape):
    check_keys_of_minus_infinity(shape)


@pytest.mark.parametrize('graph', ['0', '1'])
def test_replays_timed_before_the_first_call(graph, monkeypatch):
    """A forward graph's host memory comes with its first replay, whoever asks for it: with dropout, with inputs that go by the
    copy engine, and with none at all."""
    monkeypatch.setenv('TG_GRAPH', graph)

    class M(Module):
        def __init__(self):
            self.l = nn.Linear(8, 8)
    x = f32(rng(61).standard_normal((40000, 8)))
    for fwd, ins in ((lambda m, i: O.dropout(m.l.fwd(i['x']), 0.5), {'x': x}), (lambda m, i: m.l.fwd(i['x']), {'x': x[:4]}),
                     (lambda m, i: O.mul(m.l.W, 2.0), {})):
        a, b = (compile_forward(M(), fwd, {n: list(z.shape) for n, z in ins.items()}, seed=1) for _ in range(2))
        assert a._owner[0].time_replays(3) > 0
        for _ in range(3):
            got, want = a.run(ins), b.run(ins)
            assert got.error is None and np.array_equal(got.output, want.output)
        a.destroy()
        b.destroy()


def test_run_device_beside_a_training_thread():
    """Another thread trains while this one reads the weights, all equal before and after every step: no call sees half of one."""
    import threading

    class M(Module):
        def __init__(self):
            self.w = self.param([4096, 1024])
    n = 4096 * 1024
    t = tg_compile(M(), lambda p, i: O.mean(p.w), {}, {'kind': 'sgd', 'lr': float(n)}, seed=0)
    t.upload_params({'w': np.zeros(n, np.float32)})
    f = t.attach(lambda p, i: O.add(p.w, 0.5), {})
    out = [torch.empty(4096, 1024, device='cuda') for _ in range(60)]
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    failed = []

    def train():
        for _ in range(150):
            r = t.step({})
            if r.kind != 'completed':
                failed.append(r.error)
    th = threading.Thread(target=train)
    th.start()
    for i, o in enumerate(out):
        assert f.run_device({}, [o], s.cuda_stream if i % 2 else 0).error is None
    th.join()
    torch.cuda.synchronize()
    assert not failed
    for o in out:
        assert float(o.min()) == float(o.max())
    assert np.all(f.run({}).output == np.float32(0.5 - 150))
    t.destroy()


def test_siblings_made_while_another_thread_captures():
    """Every new sibling's first host call captures its step; another thread makes siblings of the same parent meanwhile."""
    import threading

    class M(Module):
        def __init__(self):
            self.l = nn.Linear(16, 16)
    t = tg_compile(M(), lambda p, i: O.mean(p.l.fwd(i['x'])), {'x': [4, 16]}, {'kind': 'sgd', 'lr': 0.0}, seed=0)
    x = f32(rng(62).standard_normal((4, 16)))
    xd, out = torch.from_numpy(x).cuda(), torch.empty(15, 4, 16, device='cuda')
    want = t.attach(lambda p, i: O.relu(p.l.fwd(i['x'])), {'x': [4, 16]}).run({'x': x}).output
    torch.cuda.synchronize()
    failed = []

    def host():
        for _ in range(15):
            f = t.attach(lambda p, i: O.relu(p.l.fwd(i['x'])), {'x': [4, 16]})
            for _ in range(2):
                r = f.run({'x': x})
                if r.error is not None or not np.array_equal(r.output, want):
                    failed.append(r.error or 'host output')
            f.destroy()
    th = threading.Thread(target=host)
    th.start()
    for n in range(15):
        f = t.attach(lambda p, i: O.relu(p.l.fwd(i['x'])), {'x': [4, 16]})
        r = f.run_device({'x': xd}, [out[n]])
        if r.error is not None:
            failed.append(r.error)
        f.destroy()                                      # waits for the call
    th.join()
    assert not failed and all(np.array_equal(o, want) for o in out.cpu().numpy())
    t.destroy()


def test_run_device_refuses_the_stream_of_each_thread():
    ex, ins, outs = _scan_executor()
    r = ex.run_device(ins, outs, 2)                      # hipStreamPerThread
    assert r.kind == 'failed' and 'PerThread' in str(r.error)
    want = ex.run({n: t.cpu().numpy() for n, t in ins.items()}).output
    assert ex.run_device(ins, outs, 1).error is None     # hipStreamLegacy: the default stream
    torch.cuda.synchronize()
    assert np.array_equal(outs[0].cpu().numpy(), want)
    ex.destroy()


def test_calls_are_refused_while_the_last_ones_stream_is_captured():
    """They would wait for it, on their stream or on the host; after the capture they run."""
    ex, ins, outs = _scan_executor()
    host = {n: t.cpu().numpy() for n, t in ins.items()}
    want = ex.run(host).output
    s, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    assert ex.run_device(ins, outs, s.cuda_stream).error is None
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    y = torch.zeros(4, device='cuda')
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        graph.capture_begin(capture_error_mode='relaxed')
        y.add_(1)
        refused = [ex.run_device(ins, outs, other.cuda_stream), ex.run(host)]
        graph.capture_end()
    assert all(r.kind == 'failed' and 'captured' in str(r.error) for r in refused)
    for turn in range(3):
        graph.replay()
        for o in outs:
            o.fill_(float('nan'))
        torch.cuda.synchronize()
        assert ex.run_device(ins, outs, other.cuda_stream).error is None
        assert np.array_equal(ex.run(host).output, want)
        assert np.array_equal(outs[0].cpu().numpy(), want) and np.all(y.cpu().numpy() == turn + 1)
    ex.destroy()


@pytest.mark.parametrize('H,D,Tk', [(1, 64, 700), (4, 128, 900), (2, 96, 70), (8, 32, 5000)])
def test_far_negative_scores_after_one_of_minus_infinity(H, D, Tk):
    """Keys 0, 1, 2, .. of every group of lanes are minus infinity, all other scores some -300: the weights are theirs alone."""
    q, k, v, _ = qkv(2, H, 1, 1, Tk, D, D, 81)
    q, k = f32(np.full_like(q, 4)), f32(k / 16 - 300 / 4 / D)
    doc = np.zeros((2, Tk), np.int32)
    doc[:, :60] = -1
    want, tol = R.attention(q, k, v, scale=1.0, documents=doc)
    k[:, :, :60] = -np.inf
    y = attend(q, k, v, None, dict(scale=1.0))['y']
    R.check(y, want['y'], tol['y'])


@pytest.mark.parametrize('shape', [(1, 1, 1, 1, 3000, 64), (1, 1, 1, 4, 900, 128), (8, 4, 4, 1, 70, 96)])
def test_keys_of_minus_infinity_weigh_nothing_for_few_rows(shape):
    check_keys_of_minus_infinity(shape)


@pytest.mark.parametrize('T,D', [(24, 16), (90, 64), (300, 128), (600, 40)])
@pytest.mark.parametrize('sign', [1, -1])
@pytest.mark.parametrize('what', ['q', 'k'])
def test_infinite_rows_under_a_cap(T, D, sign, what):
    """One infinite feature of a query, or of a key: its scores are plus or minus the cap by the other's sign, with a slope of
    0. As with a feature of 1e6, whose tanh is +-1 to the last bit; that reference's bounds are those of its own size, so the
    bounds here are of the rows before. Gradients of y by the row itself are 0 (the cap is flat there)."""
    q, k, v, dy = qkv(1, 2, 1, T, T, D, D, 91)
    how = dict(softcap=5.0)
    x = dict(q=q, k=k)[what]
    tol = R.attention(q, k, v, dy, **how)[1]
    at = T // 3
    x[0, 0, at, 2] = sign * 1e6
    want, _ = R.attention(q, k, v, dy, **how)
    x[0, 0, at, 2] = sign * np.inf
    got = attend(q, k, v, dy, how)
    for n in ('y', 'dv'):
        R.check(got[n], want[n], 4 * tol[n].max() + 0 * tol[n], n)
    own = 'd' + what
    assert np.all(got[own][0, 0, at] == 0)
    rest = np.arange(T) != at
    R.check(got[own][0, 0, rest], want[own][0, 0, rest], 4 * tol[own].max() + 0 * tol[own][0, 0, rest], own)


def test_tiny_weights_of_large_gradients():
    """A key that every query weighs at 2^-100 (the first tile of rows) or 2^-120 (the second), with dy of 2^94 and 2^114: its dv
    is a sum of ordinary size from both."""
    q, k, v, dy = (np.zeros((1, 1, 64, 64), np.float32) for _ in range(4))
    k[0, 0, 5, 0] = 1
    q[0, 0, :32, 0], q[0, 0, 32:, 0] = -94 * np.log(2), -114 * np.log(2)
    dy += f32(rng(95).uniform(1, 2, dy.shape))
    dy[0, 0, :32] *= 2.0 ** 94
    dy[0, 0, 32:] *= 2.0 ** 114
    how = dict(causal=False, scale=1.0)
    check_attention(q, k, v, dy, how, {})


@pytest.mark.parametrize('B,T,C', [(1, 60, 3), (1, 700, 5), (2, 2048, 70), (4, 4096, 256)])
@pytest.mark.parametrize('back', [1.0, 2.0], ids=['stays', 'returns'])
def test_recurrence_of_large_states_that_fade(B, T, C, back):
    """A state of 1e30 falls by 1e-48 (1e-40), in steps of 0.1 side by side, to an ordinary value that nothing else covers (and
    then grows again, from far below): the product of the gates alone is below f32's range. In the gradient's direction, dh is
    1e30 at the end."""
    r = rng(43, T)
    a = f32(np.ones((B, T, C)))
    lo, n = (T // 4, 40) if T < 100 else (T // 3, 48)
    a[:, lo:lo + n] = 0.1
    a[:, lo + n:lo + n + 20, ::2] = back
    dh = np.zeros_like(a)
    dh[:, -1] = 1e30 * r.uniform(1, 2, (B, C))
    h0 = f32(1e30 * r.uniform(1, 2, (B, C)))
    x = np.zeros_like(a)
    got = scan_and_gradients(a, x, dh, h0)
    want, tol = R.recurrence(a, x, h0, dh)
    for n in want:
        R.check(got[n], want[n], tol[n], n)


@pytest.mark.parametrize('gate', [0.02, 0.3])
def test_recurrence_that_forgets_at_once(gate):
    """Products of gates far below f32's range in every span, over ordinary values and none."""
    r = rng(44)
    a = f32(gate * r.uniform(0.5, 1.5, (2, 1500, 70)))
    x, dh, h0 = f32(r.standard_normal(a.shape)), f32(r.standard_normal(a.shape)), f32(1e25 * r.standard_normal((2, 70)))
    x[:, 300:800] = 0
    got = scan_and_gradients(a, x, dh, h0)
    want, tol = R.recurrence(a, x, h0, dh)
    for n in want:
        R.check(got[n], want[n], tol[n], n)


def test_recurrence_of_infinite_states():
    """A state that has left f32's range stays infinite while its gates are positive, also past spans whose gates' products
    leave the range in other channels or vanish."""
    r = rng(45)
    a, x = f32(r.uniform(0.5, 1, (1, 3000, 70))), f32(r.standard_normal((1, 3000, 70)))
    a[0, 333, 3], a[0, 1500, 5] = np.inf, np.inf
    a[0, 700:900] = 1e-3
    a[0, 2000:2060, 9] = 1e30
    a[0, 2200, 11] = np.nan
    got = forward(lambda i: [O.linear_recurrence(i['a'], i['x'])], dict(a=a, x=x))[0]
    h = np.zeros((3000, 70), np.float32)
    with np.errstate(all='ignore'):
        s = np.zeros(70, np.float32)
        for t in range(3000):
            s = a[0, t] * s + x[0, t]
            h[t] = s
    assert np.array_equal(np.isnan(got[0]), np.isnan(h))
    assert np.array_equal(np.isposinf(got[0]), np.isposinf(h)) and np.array_equal(np.isneginf(got[0]), np.isneginf(h))


def test_rope_axes_of_the_least_base():
    """Angles of up to 2^46: the product of position and frequency, rounded in 64 bits, is the angle; 2^-53 of 2^46 is more than
    any bound on cosines, so the positions here are powers of two and the frequencies too, and their product exact."""
    r = rng(27)
    q = f32(r.standard_normal((1, 2, 24, 8)))
    pos = (2 ** (np.arange(24) % 31)).astype(np.int32).reshape(1, 1, 24)
    got = forward(lambda i: list(O.rope_axes(i['q'], i['q'], i['p'], [4], 2.0 ** -16)), dict(q=q, p=pos))
    want, tol = R.rope_axes(q, pos, [4], 2.0 ** -16)
    for g in got:
        R.check(g, want, tol)


@pytest.mark.parametrize('B,H,Hk,Tq,Tk,D', [(2, 2, 1, 20, 20, 16), (1, 2, 1, 90, 90, 64), (1, 2, 1, 300, 300, 128), (1, 1, 1, 64, 3000, 40),
                                            (2, 4, 2, 1, 700, 64)])
@pytest.mark.parametrize('how', [{}, dict(softcap=2.0 ** 50), dict(slopes=1e-3), dict(softcap=2.0 ** 50, slopes=1e-3)],
                         ids=['plain', 'cap', 'slopes', 'both'])
@pytest.mark.parametrize('size', [1e4, 1e6, 1e8, 1e10, 1e14, 1e30])
def test_scores_of_any_size_choose_their_key(B, H, Hk, Tq, Tk, D, how, size):
    """Keys are words of +-1.37 and a query is `size` times the word of one key that it sees: its score leads by `size` / D and
    more, which is hundreds, though f32 holds it to `size` / 2^24 alone. So y is that key's value, dv the sum of dy over the
    queries of a key, and dq and dk are what rounding leaves of dP - D, which cancel: dP and D are each off by (12 + 8 sqrt D)
    roundings of |dy| |v| (the split of both operands, their sums, y's own roundings), in rows that the scale and |k| or |q|
    multiply."""
    if size > 1e14 and 'softcap' in how:
        return                                           # the cap is reached
    r = rng(B, H, Tq, Tk, D, 101)
    how = dict(how, slopes=[how['slopes']] * H) if 'slopes' in how else how
    _, _, v, dy = qkv(B, H, Hk, Tq, Tk, D, D, 102)
    k = f32(1.37 * r.choice([-1, 1], (B, Hk, Tk, D)))
    chosen = (r.random((B, H, Tq)) * (np.arange(Tq) + 1 + Tk - Tq)).astype(int)
    word = np.stack([[k[b, h * Hk // H][chosen[b, h]] for h in range(H)] for b in range(B)])
    q = f32(word * f32(size / 1.7))
    s = np.einsum('bhqd,bhkd->bhqk', q.astype(np.float64), np.repeat(k, H // Hk, 1).astype(np.float64)) / np.sqrt(D)
    np.put_along_axis(s, chosen[..., None], -np.inf, 3)
    lead = size / 1.7 * 1.37 ** 2 * np.sqrt(D) - s.max(3)
    assert lead.min() > 100                              # words are apart
    got = attend(q, k, v, dy, how)
    y = np.stack([[v[b, h * Hk // H][chosen[b, h]] for h in range(H)] for b in range(B)])
    R.check(got['y'], y.astype(np.float64), 16 * R.U * np.abs(y), 'y')
    dv, dva, n = np.zeros(v.shape), np.zeros(v.shape), np.zeros(v.shape[:3] + (1,))
    for b in range(B):
        for h in range(H):
            np.add.at(dv[b, h * Hk // H], chosen[b, h], dy[b, h].astype(np.float64))
            np.add.at(dva[b, h * Hk // H], chosen[b, h], np.abs(dy[b, h]))
            np.add.at(n[b, h * Hk // H], chosen[b, h], 1)
    R.check(got['dv'], dv, (16 + 4 * np.sqrt(n)) * R.U * dva + 1e-30, 'dv')
    norm = lambda z: np.linalg.norm(z, axis=-1, keepdims=True)  # noqa: E731
    noise = 2 * (12 + 8 * np.sqrt(D)) * R.U * norm(dy) * norm(y) / np.sqrt(D)
    R.check(got['dq'], np.zeros(q.shape), noise * 1.37 + 0 * q, 'dq')
    worst = np.zeros(v.shape[:3] + (1,))
    for b in range(B):
        for h in range(H):
            np.add.at(worst[b, h * Hk // H], chosen[b, h], noise[b, h] * np.abs(q).max())
    R.check(got['dk'], np.zeros(k.shape), worst + 1e-30 * size + 0 * k, 'dk')


@pytest.mark.parametrize('H,Tq,Tk,D', [(1, 1, 1000, 64), (4, 1, 3000, 128), (2, 2, 700, 96), (16, 1, 5000, 32), (1, 3, 129, 17)])
@pytest.mark.parametrize('how', [{}, dict(softcap=2.0 ** 50), dict(slopes=1e-3)], ids=['plain', 'cap', 'slopes'])
@pytest.mark.parametrize('size', [1e4, 1e8, 1e14])
def test_few_rows_of_scores_of_any_size(H, Tq, Tk, D, how, size):
    """As above, without gradients: the keys are read as they are. 17 features: words that differ in one alone are 2 / 17 apart."""
    r = rng(H, Tq, Tk, D, 103)
    how = dict(how, slopes=[how['slopes']] * H) if 'slopes' in how else how
    v = f32(r.standard_normal((2, 1, Tk, D)))
    words = np.unique(r.choice([-1, 1], (4 * Tk, D)), axis=0)
    k = f32(1.37 * np.stack([r.permutation(words)[:Tk] for _ in range(2)])[:, None])
    chosen = (r.random((2, H, Tq)) * (np.arange(Tq) + 1 + Tk - Tq)).astype(int)
    q = f32(np.stack([k[b, 0][chosen[b]] for b in range(2)]) * f32(size / 1.7))
    y = attend(q, k, v, None, how)['y']
    want = np.stack([v[b, 0][chosen[b]] for b in range(2)])
    R.check(y, want.astype(np.float64), 16 * R.U * np.abs(want))


@pytest.mark.parametrize('ratio', [2.0 ** 14, 2.0 ** 18, 2.0 ** 22])
def test_features_of_very_different_size(ratio):
    """One feature of k, and of v, `ratio` times the others, q's smaller by as much. A value is held to 2^-22 of itself or 2^-39 of
    its row's (its tile's) largest, whichever is more: f16 parts of values scaled to 2^14 .. 2^15, whose steps end at 2^-24. The
    second part of the bound counts that for the scores and for y; the rest is as everywhere."""
    q, k, v, _ = qkv(1, 2, 1, 150, 150, 64, 64, 104)
    q[..., 3] /= ratio
    k[..., 3] *= ratio
    v[..., 7] *= ratio
    y = attend(q, k, v)['y']
    tri, eps = np.tril(np.ones((150, 150), bool)), 2.0 ** -39
    for h in range(2):
        Q, K, V = (x.astype(np.float64) for x in (q[0, h], k[0, 0], v[0, 0]))
        s = np.where(tri, Q @ K.T / 8, -np.inf)
        P = np.exp(s - s.max(1, keepdims=True))
        P /= P.sum(1, keepdims=True)
        a = np.abs
        e = (17 + 4 * 8) * R.U * a(Q) @ a(K).T + eps * (a(Q).max(1)[:, None] * a(K).sum(1)[None] + a(Q).sum(1)[:, None] * a(K).max())
        E = np.where(tri, e / 8, 0).max(1)[:, None]
        tol = (2 * E + (20 + 8 * np.sqrt(150)) * R.U) * (P @ a(V)) + eps * a(V).max()
        R.check(y[0, h], P @ V, tol, str(ratio))

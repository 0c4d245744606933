"""Windowed attention, linear attention and the choice of a token on the GPU where their inputs are not ordinary: settings that are
no numbers, logits and states near the ends of f32, infinities and NaN under decays that vanish."""
import numpy as np
import pytest
import torch

import _decoders as D
import _sequence as R
from tensorgrad_amd import ops as O
from tensorgrad_amd.compile import compile_forward
from tensorgrad_amd.module import Module
from test_gpu_decoders import check_linear, check_sample, f32, forward, linear_inputs, rng, run_linear

pytestmark = pytest.mark.gpu

# ---- the choice of a token ----------------------------------------------------------------------------

FORMS = [65, 300, 5000, 30011]     # vocabularies of few rows: sorted by a wavefront, 256 threads, 1024 threads, several blocks a row


@pytest.mark.parametrize('V', FORMS)
@pytest.mark.parametrize('how', [dict(), dict(top_k=5), dict(top_p=0.9)], ids=['none', 'k', 'p'])
def test_sample_a_temperature_that_is_no_number_takes_the_largest_logit(V, how):
    r = rng(V, 101)
    heat = f32(np.where(np.arange(8) % 2, np.nan, 0.9))
    heat[6] = -1
    check_sample(f32(r.standard_normal((8, V))), f32(r.uniform(0.5, 1, 8)), temperature=heat, **how)


@pytest.mark.parametrize('V', FORMS)
@pytest.mark.parametrize('temperature', [1e38, 2.0 ** 127, 3e38])
@pytest.mark.parametrize('how', [dict(), dict(top_k=50), dict(top_p=0.8), dict(min_p=0.1)], ids=['none', 'k', 'p', 'm'])
def test_sample_logits_whose_difference_passes_f32(V, temperature, how):
    """Each weighs by its distance to the largest, also where f32 cannot hold that."""
    r = rng(V, 102)
    logits, u = f32(3.4e38 * r.uniform(-1, 1, (8, V))), f32(r.random(8))
    logits[4:6] = np.where(r.random((2, V)) < 0.1, np.float32(2e38), np.float32(-2e38)) * f32(r.uniform(0.9, 1, (2, V)))
    logits[6, ::2] = -np.inf
    check_sample(logits, u, temperature=temperature, **how)


@pytest.mark.parametrize('V', FORMS)
def test_sample_limits_out_of_range_keep_the_first_or_all(V):
    """In tensors. The first of the order is always kept: alone by a min_p above 1 or not a number and by a top_p that is not above
    0, equal logits behind it or not; a min_p below 0 and a top_p that is 1 at least or not a number do not limit."""
    r = rng(V, 103)
    logits = f32(np.round(r.standard_normal((24, V))))       # many equal ones at the top
    p, m = np.ones(24, np.float32), np.zeros(24, np.float32)
    m[:4], m[4:8], m[8:10], m[10:12] = 3.0, np.nan, np.inf, np.nextafter(np.float32(1), np.float32(2))
    p[12:14], p[14:16], p[16:18], p[18:20], m[20:22], p[22:] = 0.0, -0.5, -np.inf, np.nan, -0.5, np.inf
    k = np.where(np.arange(24) % 2, 30, 0).astype(np.int32)
    got = check_sample(logits, f32(r.uniform(0.3, 1, 24)), top_p=p, min_p=m, top_k=k)
    alone = np.arange(24) < 18
    assert (got[alone] == logits[alone].argmax(1)).all() and (got[~alone] != logits[~alone].argmax(1)).any()
    check_sample(logits, f32(r.uniform(0.3, 1, 24)), min_p=m)


@pytest.mark.parametrize('V', FORMS)
def test_sample_random_numbers_out_of_range_take_an_end(V):
    r = rng(V, 108)
    u = f32([0, 1, 2, 3.9, 4.1, 1e30, np.inf, -0.5, -1e30, -np.inf, np.nan, 0.5])
    check_sample(f32(r.standard_normal((len(u), V))), u, top_k=7)


def mixed_rows(rows, V, seed):
    """Rows without a limit, with each limit, all equal, rounded, flat, greedy, empty, masked, side by side."""
    r = rng(rows, V, seed)
    a = dict(logits=f32(2 * r.standard_normal((rows, V))), u=f32(r.random(rows)),
             **{n: np.full(rows, x, t) for n, x, t in (('temperature', 1, np.float32), ('top_k', 0, np.int32), ('top_p', 1, np.float32), ('min_p', 0, np.float32))})
    kinds = [dict(), dict(temperature=0), dict(top_k=40), dict(top_p=0.7), dict(), dict(top_k=5000), dict(top_p=0.9, top_k=3000), dict(min_p=0.2),
             dict(temperature=np.finfo(np.float32).max), dict(top_k=2 ** 31 - 1), dict(top_p=0.99), dict(min_p=3.0), dict(temperature=np.nan),
             dict(temperature=1e-30, top_p=0.5), dict(top_k=7, top_p=0.6, min_p=0.3)]
    for i in range(rows):
        for n, x in kinds[(i + seed) % len(kinds)].items():
            a[n][i] = x
    at = (np.arange(rows) + seed) % len(kinds)
    a['logits'][at == 3] = 1.5
    a['logits'][at == 4] = -np.inf
    a['logits'][at == 5, ::3] = -np.inf
    a['logits'][at == 6] = np.round(4 * a['logits'][at == 6]) / 4
    a['logits'][at == 10] *= f32(0.01)
    return a


# sample_short; sample_one by 256 and by 1024 threads, twice for their two rules; several blocks a row
@pytest.mark.parametrize('rows,V', [(20, 250), (20, 3001), (300, 9000), (30, 9000), (30, 20000), (16, 30011), (16, 70001), (128, 24577)])
def test_sample_mixed_rows_one_batch_after_another(rows, V):
    """Through one compiled graph: what one batch's rows left in the workspace reaches none of the next one's."""
    batches = [mixed_rows(rows, V, s) for s in (0, 4, 9)]
    decl = {n: {'shape': list(x.shape), 'dtype': 'i32' if x.dtype == np.int32 else 'f32'} for n, x in batches[0].items()}
    ex = compile_forward(Module(), lambda m, i: O.sample(i['logits'], i['u'], i['temperature'], i['top_k'], i['top_p'], i['min_p']), decl,
                         output='i32', seed=0)
    want = [[D.sample(a['logits'][r], float(a['u'][r]), *(a[n][r].item() for n in ('temperature', 'top_k', 'top_p', 'min_p'))) for r in range(rows)]
            for a in batches]
    for turn in (0, 1, 2, 1, 0):
        ins = {n: torch.from_numpy(x).cuda() for n, x in batches[turn].items()}
        out = torch.full((rows,), -7, device='cuda', dtype=torch.int32)
        torch.cuda.synchronize()
        r = ex.run_device(ins, [out])
        assert r.error is None, r.error
        torch.cuda.synchronize()
        assert out.tolist() == want[turn], turn
    ex.destroy()


@pytest.mark.parametrize('how', [dict(), dict(top_k=40, top_p=0.9), dict(temperature=1.5, top_p=0.97), dict(top_k=1025), dict(min_p=0.01)],
                         ids=lambda h: '+'.join(f'{n}={x}' for n, x in h.items()) or 'none')
@pytest.mark.parametrize('rows,V', [(5, 256), (5, 257), (5, 4096), (5, 4097), (256, 4097), (257, 4097), (256, 16384), (257, 16384), (257, 16385),
                                    (128, 24576), (128, 24577), (129, 24577)])
def test_sample_sizes_where_the_kernel_changes(rows, V, how):
    r = rng(rows, V, 107)
    check_sample(f32(2 * r.standard_normal((rows, V))), f32(r.random(rows)), **{n: min(x, V) if n == 'top_k' else x for n, x in how.items()})


# ---- linear attention -------------------------------------------------------------------------------

def by_positions(a, decay, scale):
    """The definition position by position in 64 bits, forward and backward, so that what is not finite goes where it goes."""
    q, k, v, dy = (a[n].astype(np.float64) for n in ('q', 'k', 'v', 'dy'))
    B, H, T, _ = q.shape
    G = H // k.shape[1]
    out = dict(y=np.zeros(dy.shape), state=np.zeros(a['state'].shape), dq=np.zeros(q.shape), dk=np.zeros(k.shape), dv=np.zeros(v.shape),
               dstate=np.zeros(a['state'].shape))
    for b in range(B):
        for h in range(H):
            S, states = a['state'][b, h].astype(np.float64), []
            for t in range(T):
                S = decay[h] * S + np.outer(k[b, h // G, t], v[b, h // G, t])
                states.append(S)
                out['y'][b, h, t] = scale * (S * q[b, h, t][:, None]).sum(0)
                out['dq'][b, h, t] = scale * (S * dy[b, h, t]).sum(1)
            out['state'][b, h] = S
            g = a['dstate'][b, h].astype(np.float64)
            for t in reversed(range(T)):
                g = g + scale * np.outer(q[b, h, t], dy[b, h, t])
                out['dk'][b, h // G, t] += (g * v[b, h // G, t]).sum(1)
                out['dv'][b, h // G, t] += (g * k[b, h // G, t][:, None]).sum(0)
                g = decay[h] * g
            out['dstate'][b, h] = g
    return out


@pytest.mark.parametrize('shape', [(2, 2, 1, 5, 32, 32), (1, 2, 2, 100, 64, 64), (1, 4, 2, 300, 64, 32), (1, 2, 1, 420, 15, 19), (1, 2, 1, 300, 128, 96)])
@pytest.mark.parametrize('decay', [0.9, 0.4, 0.003, 1e-30, 5e-324])
@pytest.mark.parametrize('where', ['q', 'k', 'v', 'state', 'dy', 'dstate'])
def test_linear_infinities_go_where_states_carry_them(shape, decay, where):
    """Infinities and NaN in any operand are in the states, results and gradients that they are in by the definition. No
    decay above 0 forgets them, however small its powers have become in 32 bits."""
    a = linear_inputs(*shape, 104, True)
    H, T = shape[1], shape[3]
    lam = [decay] + [0.9] * (H - 1)
    scale = shape[4] ** -0.5
    for n, x in enumerate((np.inf, np.nan, -np.inf)):
        clean = {m: z.copy() for m, z in a.items()}
        bad = {m: z.copy() for m, z in a.items()}
        at = (0, 0, {'q': T - 2, 'dy': T - 2}.get(where, 1), n) if where not in ('state', 'dstate') else (0, 0, n, 2)
        bad[where][at], clean[where][at] = x, 0
        with np.errstate(all='ignore'):
            want = by_positions(bad, lam, scale)
        _, tol = D.linear(**clean, decay=lam)
        got = run_linear(bad, lam)
        for m in want:
            w, fine = want[m], np.isfinite(want[m])
            assert (np.isfinite(got[m]) == fine).all(), (where, x, m)
            assert (np.isnan(got[m]) == np.isnan(w)).all() and (got[m] == w)[np.isinf(w)].all(), (where, x, m)
            R.check(np.where(fine, got[m], 0), np.where(fine, w, 0), np.where(fine, tol[m], 0), f'{where} {x} {m}')


@pytest.mark.parametrize('decay', [1.0, 0.9, 0.4])
def test_linear_products_that_pass_f32_on_the_way(decay):
    """q.k is infinite in 32 bits where no state and no result is."""
    a = linear_inputs(1, 2, 1, 200, 32, 32, 106, True)
    for n, e in (('q', 70), ('k', 60), ('v', -40), ('dy', -50), ('state', 20), ('dstate', 20)):
        a[n] *= f32(2.0 ** e)
    check_linear(a, [decay] * 2)


@pytest.mark.parametrize('shape', [(1, 2, 1, 8, 32, 32), (1, 2, 2, 100, 64, 64), (1, 4, 2, 300, 64, 32), (1, 2, 1, 420, 15, 19)])
@pytest.mark.parametrize('where', ['q', 'k', 'v', 'state', 'dy', 'dstate', 'all states'])
def test_linear_large_values_outlast_small_weights(shape, where):
    """2^116 times a power of the decay below 2^-126 still counts."""
    a = linear_inputs(*shape, 105, True)
    T = shape[3]
    lam = [0.4] + [0.45] * (shape[1] - 1)
    if where == 'all states':
        a['state'] *= f32(2.0 ** 116)
    elif where in ('state', 'dstate'):
        a[where][0, 0, 1] *= f32(2.0 ** 116)
    else:
        a[where][0, 0, T - 2 if where in ('q', 'dy') else 1] *= f32(2.0 ** 116)
    check_linear(a, lam, what=where)


@pytest.mark.parametrize('size', [2.0 ** 20, 2.0 ** 40])
@pytest.mark.parametrize('gone', [None, 'q', 'v'])
def test_linear_large_values_of_one_size(size, gone):
    """Also where rows or columns of zeros are among them."""
    a = linear_inputs(1, 4, 2, 300, 64, 32, 109, True)
    for n in a:
        a[n] *= f32(size)
    a['dy'] /= f32(size)
    if gone == 'q':
        a['q'][:, :, ::3] = 0
    elif gone == 'v':
        a['v'][..., ::3] = 0
        a['state'][..., ::3] = 0
    check_linear(a, [0.4, 0.1, 0.45, 0.9])


def test_linear_one_column_of_early_values_is_large():
    a = linear_inputs(1, 2, 1, 200, 32, 32, 110)
    a['v'][0, 0, 3, 5] *= np.float32(2.0 ** 116)
    a['v'][0, 0, 3, 6] = 2.0 ** 90
    a['v'][0, 0, 4:, 6] *= np.float32(2.0 ** -30)
    check_linear(a, [0.4, 0.45])


@pytest.mark.parametrize('T,Dk', [(6, 32), (100, 64), (300, 64), (420, 20), (300, 96)])
@pytest.mark.parametrize('kind', ['documents', 'lengths', 'both'])
@pytest.mark.parametrize('garbage', [np.inf, np.nan, 3e38])
def test_linear_masks_under_fast_decays(T, Dk, kind, garbage):
    """What is not there is garbage of any size, and no result shows it."""
    a = linear_inputs(3, 4, 2, T, Dk, Dk, 111, True)
    hidden = np.zeros((3, T), bool)
    if kind != 'lengths':
        a['documents'] = np.repeat(np.arange((T + 36) // 37, dtype=np.int32), 37)[:T][None].repeat(3, 0).copy()
        a['documents'][0, T // 2:T // 2 + 5] = -1
        a['documents'][2, :3] = -2
        hidden |= a['documents'] < 0
    if kind != 'documents':
        a['lengths'] = np.array([T, T - T // 3, 0], np.int32)
        hidden |= np.arange(T)[None] >= a['lengths'][:, None]
    clean = {n: x.copy() for n, x in a.items()}
    for b in range(3):
        for n in ('q', 'k', 'v', 'dy'):
            a[n][b, :, hidden[b]] = garbage
            clean[n][b, :, hidden[b]] = 0
    lam = [0.4, 0.003, 1e-30, 0.9]
    want, tol = D.linear(**clean, decay=lam)
    got = run_linear(a, lam)
    for n in got:
        R.check(got[n], want[n], tol[n], n)
    assert not got['y'][np.broadcast_to(hidden[:, None], got['y'].shape[:3])].any()


def test_linear_results_under_fast_decays_repeat():
    """Also those that are computed again: a batch with an infinity, then without, then with it."""
    a = linear_inputs(2, 4, 2, 300, 64, 64, 112, True)
    lam = [0.4, 0.3, 0.9, 0.999]
    bad = {n: x.copy() for n, x in a.items()}
    bad['v'][0, 1, 17, 3] = np.inf
    bad['k'][1, 0, 5] *= np.float32(2.0 ** 100)
    first, clean = run_linear(bad, lam), run_linear(a, lam)
    check_linear(a, lam)
    for n, x in run_linear(bad, lam).items():
        assert np.array_equal(x, first[n], equal_nan=True), n
    for n, x in run_linear(a, lam).items():
        assert np.array_equal(x, clean[n]), n


@pytest.mark.parametrize('T', [1, 8, 9, 128])
def test_linear_states_before_segments_of_one_segment(T):
    """The op that keeps them for the gradients, in a document that asks for it where there is one segment: the first state."""
    a = linear_inputs(2, 4, 2, T, 32, 16, 113, True, grad=False)

    def fn(i):
        out = O.linear_attention(i['q'], i['k'], i['v'], [0.9] * 4, state=i['state'])
        f = O._linear_fields('borders', i['q'], i['k'], i['v'], [0.9] * 4, None, i['state'], None, None)
        return [*out, O.add_op(O.current_graph(), 'linear_attention_borders', (1, 2, 4, 32, 16), 'f32', 'borders', f)]
    y, state, borders = forward(fn, a)
    want, tol = D.linear(**a, decay=[0.9] * 4)
    R.check(y, want['y'], tol['y'], 'y')
    R.check(state, want['state'], tol['state'], 'state')
    assert np.array_equal(borders[0], a['state'])


@pytest.mark.parametrize('start', [1, 4])
@pytest.mark.parametrize('axis', [2, 3])
def test_operands_that_are_parts_of_others(axis, start):
    """Rows and features of larger tensors from an odd or an aligned place on, read where they lie."""
    T, size = 150, 24
    r = rng(axis, start, 114)
    big = {n: f32(r.standard_normal((2, h, T + 7 * (axis == 2), size + 8 * (axis == 3)))) for n, h in (('q', 4), ('k', 2), ('v', 2), ('dy', 4))}
    cut = lambda x: O.narrow(x, axis, start, T if axis == 2 else size)  # noqa: E731
    part = {n: np.ascontiguousarray(x.take(np.arange(start, start + (T if axis == 2 else size)), axis)) for n, x in big.items()}

    def linear(i):
        q, k, v, dy = (cut(i[n]) for n in ('q', 'k', 'v', 'dy'))
        return [*O.linear_attention(q, k, v, [0.9] * 4), *O.linear_attention_grad(q, k, v, dy, [0.9] * 4)]

    def window(i):
        q, k, v, dy = (cut(i[n]) for n in ('q', 'k', 'v', 'dy'))
        y = O.attention(q, k, v, window=40, sinks=3)
        return [y, *O.attention_grad(q, k, v, y, dy, window=40, sinks=3)]
    for fn, (want, tol), names in ((linear, D.linear(part['q'], part['k'], part['v'], [0.9] * 4, dy=part['dy']), ('y', 'state', 'dq', 'dk', 'dv')),
                                   (window, D.attention(part['q'], part['k'], part['v'], part['dy'], window=40, sinks=3), ('y', 'dq', 'dk', 'dv'))):
        for n, x in zip(names, forward(fn, big)):
            R.check(x, want[n], tol[n], n)


@pytest.mark.parametrize('V', FORMS)
def test_sample_of_a_part_of_the_vocabulary(V):
    r = rng(V, 115)
    x, u = f32(r.standard_normal((6, V + 3))), f32(r.random(6))
    got = forward(lambda i: [O.sample(O.narrow(i['x'], 1, 3, V), i['u'], top_p=0.9)], dict(x=x, u=u))[0]
    assert got.tolist() == [D.sample(x[b, 3:], float(u[b]), top_p=0.9) for b in range(6)]

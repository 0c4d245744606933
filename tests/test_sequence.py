"""The sequence operators without a GPU: refusals, shapes, gradients' IR, and the lowered schedule."""
import numpy as np
import pytest

import _sequence as R
from tensorgrad_amd import backend, nn
from tensorgrad_amd import ir as IR
from tensorgrad_amd import ops as O
from tensorgrad_amd.build_ir import build_forward_ir, build_training_ir
from tensorgrad_amd.module import Module
from tensorgrad_amd.shape import ShapeError
from tensorgrad_amd.trace import tensor_input, trace_fn


def t(name, *shape, dtype='f32'):
    return tensor_input(name, list(shape), dtype)


def refuses(fn, match):
    with pytest.raises(ShapeError, match=match):
        trace_fn(fn)


def base(D=8, Tq=4, Tk=4, H=4, Hk=2):
    return t('q', 2, H, Tq, D), t('k', 2, Hk, Tk, D), t('v', 2, Hk, Tk, D)


def test_attention_refusals():
    refuses(lambda: O.attention(t('z', 2, 4, 8), *base()[1:]), 'must be')
    refuses(lambda: O.attention(t('i', 2, 4, 4, 8, dtype='i32'), *base()[1:]), 'f32')
    refuses(lambda: O.attention(*base()[:2], t('w', 2, 2, 5, 8)), 'agree')
    refuses(lambda: O.attention(base()[0], t('w', 2, 2, 4, 9), t('u', 2, 2, 4, 9)), 'agree')
    refuses(lambda: O.attention(*base(H=3)), 'share')
    refuses(lambda: O.attention(*base(D=129)), 'above 128')
    refuses(lambda: O.attention(*base(Tq=5)), 'last of')
    refuses(lambda: O.attention(*base(Tq=5), causal=False, slopes=[1, 1, 1, 1]), 'last of')
    refuses(lambda: O.attention(t('z', 2, 4, 0, 8), *base()[1:]), 'empty')
    for scale in (0, -1, float('nan'), float('inf'), True):
        refuses(lambda: O.attention(*base(), scale=scale), 'scale')
    for cap in (0, -2.0, float('nan'), float('inf')):
        refuses(lambda: O.attention(*base(), softcap=cap), 'softcap')
    for slopes in ([1.0], [1, 2, 3, float('nan')], [1, 2, 3, 4, 5]):
        refuses(lambda: O.attention(*base(), slopes=slopes), 'slopes')
    refuses(lambda: O.attention(*base(), causal=False, prefix=t('p', 2, dtype='i32')), 'prefix')
    refuses(lambda: O.attention(*base(), prefix=t('p', 3, dtype='i32')), 'prefix')
    refuses(lambda: O.attention(*base(), lengths=t('n', 2)), 'lengths')
    refuses(lambda: O.attention(*base(), documents=t('d', 2, 5, dtype='i32')), 'documents')
    refuses(lambda: O.attention_grad(*base(), t('y', 2, 4, 4, 8), t('g', 2, 4, 4, 9)), 'dy')
    trace_fn(lambda: O.attention(*base(Tq=5), causal=False))       # cross attention may have more queries than keys


def test_attention_refuses_constants_beyond_f32():
    for x in (1e-300, 1e-40, 1e30, 1e300):
        refuses(lambda: O.attention(*base(), scale=x), 'scale')
        refuses(lambda: O.attention(*base(), softcap=x), 'softcap')
    refuses(lambda: O.attention(*base(), slopes=[1, 1, 1, -1e39]), 'slopes')
    trace_fn(lambda: O.attention(*base(), scale=2.0 ** -60, softcap=2.0 ** 60, slopes=[0, -1, 1, 2.0 ** 60]))


def test_rope_axes_refusals():
    q, k, p = (lambda: t('q', 2, 4, 3, 8)), (lambda: t('k', 2, 2, 3, 8)), (lambda n=2, dtype='i32': t('p', n, 2, 3, dtype=dtype))
    refuses(lambda: O.rope_axes(t('q', 2, 3, 8), k(), p(), [2, 2]), 'q must be')
    refuses(lambda: O.rope_axes(q(), t('k', 2, 2, 4, 8), p(), [2, 2]), 'agree')
    for sections in ([], [2, 3], [4, 0], [2, -1], [2.0, 2], [True, 2]):
        refuses(lambda: O.rope_axes(q(), k(), p(), sections), 'sections')
    refuses(lambda: O.rope_axes(q(), k(), p(3), [2, 2]), 'positions')
    refuses(lambda: O.rope_axes(q(), k(), p(dtype='f32'), [2, 2]), 'positions')
    for b in (0, -1.0, float('inf'), float('nan')):
        refuses(lambda: O.rope_axes(q(), k(), p(), [2, 2], b), 'base')


def test_linear_recurrence_refusals():
    a = lambda: t('a', 2, 5, 3)  # noqa: E731
    refuses(lambda: O.linear_recurrence(a(), t('x', 2, 5, 4)), 'x must be')
    refuses(lambda: O.linear_recurrence(t('a', 2, 5), t('x', 2, 5)), 'must be')
    refuses(lambda: O.linear_recurrence(a(), t('x', 2, 5, 3, dtype='i32')), 'x must be')
    refuses(lambda: O.linear_recurrence(a(), t('x', 2, 5, 3), t('h', 3, 2)), 'h0')
    refuses(lambda: O.linear_recurrence(t('a', 2, 0, 3), t('x', 2, 0, 3)), 'must be')
    refuses(lambda: O.linear_recurrence_grad(a(), t('x', 2, 5, 3), t('g', 2, 4, 3)), 'dh must be')


class Params(Module):
    def __init__(self, **shapes):
        for n, s in shapes.items():
            setattr(self, n, self.param(list(s)))


def kinds_of(ir):
    return [n['kind'] for n in backend.plan(ir.wire_json())['nodes']]


def test_gradients_reach_every_operand_and_lower_to_one_node_each():
    m = Params(q=(2, 4, 6, 8), k=(2, 2, 6, 8), v=(2, 2, 6, 5))

    def loss(p, i):
        q, k = O.rope_axes(p.q, p.k, i['pos'], [1, 2])
        return O.mean(O.square(O.attention(q, k, p.v, softcap=5.0, documents=i['doc'])))
    ir = build_training_ir(m, loss, {'pos': {'shape': [2, 2, 6], 'dtype': 'i32'}, 'doc': {'shape': [2, 6], 'dtype': 'i32'}},
                           {'kind': 'sgd', 'lr': 0.1})
    assert {n: g.shape for n, g in ir.param_grads.items()} == {'q': (2, 4, 6, 8), 'k': (2, 2, 6, 8), 'v': (2, 2, 6, 5)}
    kinds = kinds_of(ir)
    assert [kinds.count(k) for k in ('attend', 'attend_grad', 'rope')] == [1, 1, 2]

    m = Params(a=(2, 9, 4), x=(2, 9, 4), h0=(2, 4))
    ir = build_training_ir(m, lambda p, i: O.mean(O.square(O.linear_recurrence(O.sigmoid(p.a), p.x, p.h0))), {}, {'kind': 'sgd', 'lr': 0.1})
    assert {n: g.shape for n, g in ir.param_grads.items()} == {'a': (2, 9, 4), 'x': (2, 9, 4), 'h0': (2, 4)}
    kinds = kinds_of(ir)
    assert [kinds.count(k) for k in ('scan', 'scan_grad')] == [1, 1]


def test_only_the_gradients_that_are_needed_are_made():
    m = Params(k=(1, 1, 6, 8))

    def loss(p, i):
        return O.mean(O.square(O.attention(i['q'], p.k, i['v'])))
    ir = build_training_ir(m, loss, {'q': [1, 2, 6, 8], 'v': [1, 1, 6, 8]}, {'kind': 'sgd', 'lr': 0.1})
    node = [n for n in backend.plan(ir.wire_json())['nodes'] if n['kind'] == 'attend_grad']
    assert len(node) == 1 and node[0]['ops'] == 'attention_grad_k'


def test_heads_are_read_in_place():
    """split_heads gives strided views: no copy runs before the attention or its positions."""
    def fwd(m, i):
        q, k, v = (O.split_heads(O.matmul(i['x'], i[n]), 2) for n in ('wq', 'wk', 'wv'))
        q, k = O.rope_axes(q, k, i['p'], [4])
        return O.attention(q, k, v)
    ir = build_forward_ir(Module(), fwd, {'x': [2, 5, 16], 'wq': [16, 16], 'wk': [16, 16], 'wv': [16, 16],
                                          'p': {'shape': [1, 2, 5], 'dtype': 'i32'}})
    kinds = kinds_of(ir)
    assert 'copy' not in kinds and kinds.count('attend') == 1 and kinds.count('rope') == 1


def test_extension_kinds_are_apart_from_the_reference_union():
    assert not set(IR.EXTENSION_KINDS) & set(IR.OP_KINDS)
    g = trace_fn(lambda: O.attention(*base()))
    op = [o for o in g.ops if o['kind'] == 'attention'][0]
    assert len(IR.get_op_inputs(op)) == 3 and op['documents'] is None


def test_bad_documents_are_refused_by_the_runtime():
    """An IR document written by hand gets the shape checks of the traced one."""
    def wire(**change):
        g = trace_fn(lambda: O.attention(*base()))
        doc = {'graph': IR.graph_to_wire(g), 'paramGrads': {}, 'writebacks': [], 'optimizer': None}
        [o for o in doc['graph']['ops'] if o['kind'] == 'attention'][0].update(change)
        return IR.dumps(doc)
    backend.plan(wire())
    for change in (dict(scale=-1.0), dict(softcap=-1.0), dict(slopes=[1.0]), dict(documents=0), dict(k=0)):
        with pytest.raises(backend.BackendError) as e:
            backend.plan(wire(**change))
        assert e.value.status == backend.TG_INVALID_ARGUMENT


def test_the_64_bit_forms_agree_with_differences():
    """The tests' own references: gradients against central differences in f64."""
    r = np.random.default_rng(5)
    q, k, v, dy = (r.standard_normal(s).astype(np.float32) for s in ((1, 2, 5, 4), (1, 1, 7, 4), (1, 1, 7, 3), (1, 2, 5, 3)))
    how = dict(softcap=2.0, slopes=[0.3, 0.1], prefix=np.array([4]), documents=np.array([[0, 0, 0, 1, 1, 1, 1]]))
    got, _ = R.attention(q, k, v, dy, **how)
    for name, x in (('dq', q), ('dk', k), ('dv', v)):
        u = r.standard_normal(x.shape).astype(np.float32)
        side = []
        for s in (1, -1):
            a = dict(q=q.astype(np.float64), k=k.astype(np.float64), v=v.astype(np.float64))
            a[name[1]] = a[name[1]] + s * 1e-5 * u
            side.append((R.attention(a['q'], a['k'], a['v'], **how)[0]['y'] * dy).sum())
        assert abs((side[0] - side[1]) / 2e-5 - (got[name] * u).sum()) < 1e-7
    a, x, dh = (r.uniform(0.1, 1, (2, 9, 3)) for _ in range(3))
    h0 = r.standard_normal((2, 3))
    got, _ = R.recurrence(a, x, h0, dh)
    for name, z in (('da', a), ('dx', x), ('dh0', h0)):
        u = r.standard_normal(z.shape)
        side = []
        for s in (1, -1):
            p = dict(da=a, dx=x, dh0=h0)
            p[name] = z + s * 1e-6 * u
            side.append((R.recurrence(p['da'], p['dx'], p['dh0'])[0]['h'] * dh).sum())
        assert abs((side[0] - side[1]) / 2e-6 - (got[name] * u).sum()) < 1e-6


def test_rope_axes_refuses_a_base_whose_angles_cannot_be_reduced():
    def turn(base):
        return O.rope_axes(t('q', 2, 4, 3, 8), t('k', 2, 2, 3, 8), t('p', 2, 2, 3, dtype='i32'), [2, 2], base)
    for base in (1e-5, 1e-9, 1e-300):
        refuses(lambda: turn(base), 'base')
    g = trace_fn(lambda: turn(2.0 ** -16))
    doc = {'graph': IR.graph_to_wire(g), 'paramGrads': {}, 'writebacks': [], 'optimizer': None}
    backend.plan(IR.dumps(doc))
    for op in doc['graph']['ops']:
        if op['kind'] == 'rope_axes':
            op['base'] = 1e-9
    with pytest.raises(backend.BackendError, match='base'):
        backend.plan(IR.dumps(doc))

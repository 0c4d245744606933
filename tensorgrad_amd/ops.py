"""User-facing op surface: each call validates shapes and appends IR (reference
`src/ops.ts`). Composite ops decompose into the same primitive kinds, in the same
emission order, as the reference — the IR this produces is what the backend executes
and what the oracle evaluates, so the order of `add_op` calls below is load-bearing
(salts, tensor ids, DCE renumbering).
"""
from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple, Union

from . import shape as S
from .ir import Graph, Tensor, add_op
from .shape import ShapeError
from .trace import current_graph, tensor_input

Number = Union[int, float]

PRNG_SEED_INPUT = '__prngSeed'   # ops.ts:191


def _num(x) -> bool:
    return isinstance(x, (int, float)) and not isinstance(x, bool)


# ---- Element-wise binops (ops.ts:21-101) -------------------------------------------

def _binop(name: str, kind: str, a: Tensor, b: Tensor, out_dtype: Optional[str] = None) -> Tensor:
    if a.dtype != b.dtype:
        raise ShapeError(f'{name}: dtype mismatch ({a.dtype} vs {b.dtype})', name)
    out_shape = S.infer_elementwise_binop(name, a.shape, b.shape, name)
    return add_op(current_graph(), kind, out_shape, out_dtype or a.dtype, name, {'a': a.id, 'b': b.id})


def add(a, b) -> Tensor:
    if _num(a):
        return add_scalar(b, a)
    if _num(b):
        return add_scalar(a, b)
    return _binop('add', 'add', a, b)


def sub(a, b) -> Tensor:
    if _num(b):
        return add_scalar(a, -b)
    if _num(a):
        return _binop('sub', 'sub', const_scalar(a, b.dtype), b)
    return _binop('sub', 'sub', a, b)


def mul(a, b) -> Tensor:
    if _num(a):
        return mul_scalar(b, a)
    if _num(b):
        return mul_scalar(a, b)
    return _binop('mul', 'mul', a, b)


def div(a, b) -> Tensor:
    if _num(b):
        if b == 0:
            raise ShapeError('div: scalar divisor cannot be zero', 'div')
        return mul_scalar(a, 1 / b)
    if _num(a):
        return _binop('div', 'div', const_scalar(a, b.dtype), b)
    return _binop('div', 'div', a, b)


def minimum(a, b) -> Tensor:
    if _num(a):
        return minimum(b, a)
    rhs = const_scalar(b, a.dtype) if _num(b) else b
    return _binop('min', 'min', a, rhs)


def maximum(a, b) -> Tensor:
    if _num(a):
        return maximum(b, a)
    rhs = const_scalar(b, a.dtype) if _num(b) else b
    return _binop('max', 'max', a, rhs)


def clamp(a: Tensor, lo: Number, hi: Number) -> Tensor:
    return minimum(maximum(a, lo), hi)


def mul_scalar(a: Tensor, scalar: Number) -> Tensor:
    return add_op(current_graph(), 'mul_scalar', a.shape, a.dtype, 'mulScalar', {'a': a.id, 'scalar': scalar})


def add_scalar(a: Tensor, scalar: Number) -> Tensor:
    return add_op(current_graph(), 'add_scalar', a.shape, a.dtype, 'addScalar', {'a': a.id, 'scalar': scalar})


# ---- Unary (ops.ts:121-184) ----------------------------------------------------------

def _unary(name: str, a: Tensor) -> Tensor:
    if a.dtype != 'f32':
        raise ShapeError(f'{name}: requires f32, got {a.dtype}', name)
    return add_op(current_graph(), name, a.shape, 'f32', name, {'a': a.id})


def sqrt(a): return _unary('sqrt', a)
def rsqrt(a): return _unary('rsqrt', a)
def log(a): return _unary('log', a)
def exp(a): return _unary('exp', a)
def relu(a): return _unary('relu', a)
def neg(a): return _unary('neg', a)
def abs_(a): return _unary('abs', a)
def tanh(a): return _unary('tanh', a)
def sigmoid(a): return _unary('sigmoid', a)
def erf(a): return _unary('erf', a)
def sin(a): return _unary('sin', a)
def cos(a): return _unary('cos', a)


def square(a: Tensor) -> Tensor:
    return mul(a, a)


def stop_gradient(a: Tensor) -> Tensor:
    return add_op(current_graph(), 'stop_gradient', a.shape, a.dtype, 'stopGradient', {'a': a.id})


def silu(a: Tensor) -> Tensor:
    return mul(a, sigmoid(a))


# ---- Stochastic ops (ops.ts:193-310) ---------------------------------------------------

def _find_or_create_prng_seed(g: Graph) -> Tensor:
    for op in g.ops:
        if op['kind'] == 'tensor_input' and op['name'] == PRNG_SEED_INPUT:
            return g.tensors[op['out']]
    return tensor_input(PRNG_SEED_INPUT, [], 'i32')


def _count_stochastic_ops(g: Graph) -> int:
    return sum(1 for op in g.ops if op['kind'] in ('dropout', 'randn', 'categorical_last'))


def dropout(x: Tensor, p: float) -> Tensor:
    if p == 0:
        return x
    if p < 0 or p >= 1:
        raise ShapeError(f'dropout: p must be in [0, 1), got {p}', 'dropout')
    if x.dtype != 'f32':
        raise ShapeError(f'dropout: requires f32, got {x.dtype}', 'dropout')
    g = current_graph()
    seed = _find_or_create_prng_seed(g)
    salt = _count_stochastic_ops(g)
    return add_op(g, 'dropout', x.shape, 'f32', 'dropout', {'a': x.id, 'seed': seed.id, 'p': p, 'salt': salt})


def randn(shape: Sequence[int]) -> Tensor:
    for d in shape:
        if not isinstance(d, int) or d <= 0:
            raise ShapeError(f'randn: shape must be positive integers, got {S.show(shape)}', 'randn')
    g = current_graph()
    seed = _find_or_create_prng_seed(g)
    salt = _count_stochastic_ops(g)
    return add_op(g, 'randn', shape, 'f32', 'randn', {'seed': seed.id, 'salt': salt, 'shape': list(shape)})


def dropout_with_salt(dy: Tensor, p: float, salt: int, seed_id: int) -> Tensor:
    """Backward dropout sharing the forward's (seed, salt, p) (ops.ts:255-258)."""
    return add_op(current_graph(), 'dropout', dy.shape, 'f32', 'dropout', {'a': dy.id, 'seed': seed_id, 'p': p, 'salt': salt})


def _categorical_last(a: Tensor) -> Tensor:
    if a.dtype != 'f32':
        raise ShapeError(f'categorical: requires f32 logits, got {a.dtype}', 'categorical')
    out_shape = S.infer_sum_last('categorical', a.shape, 'categorical')
    g = current_graph()
    seed = _find_or_create_prng_seed(g)
    salt = _count_stochastic_ops(g)
    return add_op(g, 'categorical_last', out_shape, 'i32', 'categorical', {'a': a.id, 'seed': seed.id, 'salt': salt})


def categorical(logits: Tensor, axis: int = -1) -> Tensor:
    return _axis_reducing(logits, axis, 'categorical', _categorical_last)


def gelu(a: Tensor, approximate: str = 'none') -> Tensor:
    """Exact GELU `0.5*x*(1+erf(x/sqrt2))`, or the tanh form (ops.ts:319-327)."""
    if approximate == 'tanh':
        c = 0.7978845608028654
        x3 = mul(mul(a, a), a)
        inner = mul(add(a, mul(x3, 0.044715)), c)
        return mul(mul(a, 0.5), add(tanh(inner), 1))
    return mul(mul(a, 0.5), add(erf(mul(a, 1 / math.sqrt(2))), 1))


def leaky_relu(a: Tensor, alpha: float = 0.01) -> Tensor:
    return where(greater(a, 0), a, mul(a, alpha))


def softplus(a: Tensor) -> Tensor:
    return add(maximum(a, 0), log(add(exp(neg(abs_(a))), 1)))


# ---- Reductions (ops.ts:358-457) ---------------------------------------------------------

def _mean_last(a: Tensor) -> Tensor:
    if a.dtype != 'f32':
        raise ShapeError(f'mean: requires f32, got {a.dtype}', 'mean')
    return add_op(current_graph(), 'mean_last', S.infer_mean_last('mean', a.shape, 'mean'), a.dtype, 'mean', {'a': a.id})


def _sum_last(a: Tensor) -> Tensor:
    if a.dtype != 'f32':
        raise ShapeError(f'sum: requires f32, got {a.dtype}', 'sum')
    return add_op(current_graph(), 'sum_last', S.infer_sum_last('sum', a.shape, 'sum'), a.dtype, 'sum', {'a': a.id})


def _argmax_last(a: Tensor) -> Tensor:
    if a.dtype != 'f32':
        raise ShapeError(f'argmax: requires f32, got {a.dtype}', 'argmax')
    return add_op(current_graph(), 'argmax_last', S.infer_sum_last('argmax', a.shape, 'argmax'), 'i32', 'argmax', {'a': a.id})


def argmax(a: Tensor, axis: Optional[int] = None) -> Tensor:
    if axis is None:
        return _argmax_last(reshape(a, [-1]))
    return _axis_reducing(a, axis, 'argmax', _argmax_last)


def argmin(a: Tensor, axis: Optional[int] = None) -> Tensor:
    return argmax(neg(a), axis)


def mean(a: Tensor, axis: Optional[int] = None, keep_dims: bool = False) -> Tensor:
    if axis is None:
        n = S.shape_size(a.shape)
        if n == 0:
            raise ShapeError('mean: cannot mean over zero elements', 'mean')
        return mul_scalar(_sum_last(reshape(a, [-1])), 1 / n)
    return _reduce_axis(a, axis, keep_dims, 'mean')


def sum_(a: Tensor, axis: Optional[int] = None, keep_dims: bool = False) -> Tensor:
    if axis is None:
        return _sum_last(reshape(a, [-1]))
    return _reduce_axis(a, axis, keep_dims, 'sum')


def _reduce_axis(a: Tensor, axis_arg: int, keep_dims: bool, kind: str) -> Tensor:
    r = len(a.shape)
    k = r + axis_arg if axis_arg < 0 else axis_arg
    if k < 0 or k >= r:
        raise ShapeError(f"{kind}: axis {axis_arg} out of range for shape [{','.join(map(str, a.shape))}]", kind)
    is_last = k == r - 1
    inp = a if is_last else permute(a, [i for i in range(r) if i != k] + [k])
    if kind == 'mean':
        reduced = _mean_last(inp)
        if is_last:
            return reduced if keep_dims else reshape(reduced, reduced.shape[:-1])
        if not keep_dims:
            return reshape(reduced, reduced.shape[:-1])
        return permute(reduced, _back_perm(k, r))
    dropped = _sum_last(inp)
    if is_last:
        return reshape(dropped, list(dropped.shape) + [1]) if keep_dims else dropped
    if not keep_dims:
        return dropped
    return permute(reshape(dropped, list(dropped.shape) + [1]), _back_perm(k, r))


def _back_perm(k: int, r: int) -> List[int]:
    return list(range(k)) + [r - 1] + list(range(k, r - 1))


# ---- Shape ops (ops.ts:468-502) -----------------------------------------------------------

def reshape(a: Tensor, new_shape: Sequence[int]) -> Tensor:
    out = S.infer_reshape('reshape', a.shape, list(new_shape), 'reshape')
    return add_op(current_graph(), 'reshape', out, a.dtype, 'reshape', {'a': a.id, 'newShape': list(out)})


def permute(a: Tensor, perm: Sequence[int]) -> Tensor:
    out = S.infer_permute('permute', a.shape, perm, 'permute')
    return add_op(current_graph(), 'permute', out, a.dtype, 'permute', {'a': a.id, 'perm': list(perm)})


def swap_axes(a: Tensor, axis1: int, axis2: int) -> Tensor:
    r = len(a.shape)
    i1 = r + axis1 if axis1 < 0 else axis1
    i2 = r + axis2 if axis2 < 0 else axis2
    if i1 < 0 or i1 >= r or i2 < 0 or i2 >= r:
        raise ShapeError(f'swapAxes: axis out of range — got ({axis1}, {axis2}) for rank-{r} tensor', 'swapAxes')
    if i1 == i2:
        return a
    perm = list(range(r))
    perm[i1], perm[i2] = i2, i1
    return permute(a, perm)


# ---- Linear algebra (ops.ts:513-538) ----------------------------------------------------------

def matmul(a: Tensor, b: Tensor) -> Tensor:
    if a.dtype != 'f32' or b.dtype != 'f32':
        raise ShapeError(f'matmul: requires f32, got {a.dtype} and {b.dtype}', 'matmul')
    if len(a.shape) < 2:
        raise ShapeError(f'matmul: lhs must have rank >= 2, got {S.show(a.shape)}', 'matmul')
    if len(b.shape) < 2:
        raise ShapeError(f'matmul: rhs must have rank >= 2, got {S.show(b.shape)}', 'matmul')
    if len(b.shape) == 2:
        out = S.infer_matmul('matmul', a.shape, b.shape, 'matmul')
        return add_op(current_graph(), 'matmul', out, 'f32', 'matmul', {'a': a.id, 'b': b.id})
    if len(a.shape) != len(b.shape):
        raise ShapeError(f'matmul: rank mismatch — lhs {S.show(a.shape)} vs rhs {S.show(b.shape)}. When rhs is '
                         f'batched (rank > 2), lhs must have the same rank. Reshape explicitly if needed.', 'matmul')
    out = S.infer_matmul_batched('matmul', a.shape, b.shape, 'matmul')
    return add_op(current_graph(), 'matmul_batched', out, 'f32', 'matmul', {'a': a.id, 'b': b.id})


# ---- Indexing / casting (ops.ts:545-671) ---------------------------------------------------------

def one_hot(indices: Tensor, depth: int, dtype: str = 'f32') -> Tensor:
    if indices.dtype != 'i32':
        raise ShapeError(f'oneHot: indices must be i32, got {indices.dtype}', 'oneHot')
    out = S.infer_one_hot('oneHot', indices.shape, depth, 'oneHot')
    return add_op(current_graph(), 'one_hot', out, dtype, 'oneHot', {'indices': indices.id, 'depth': depth, 'dtype': dtype})


def take_along_axis(inp: Tensor, indices: Tensor, axis: int) -> Tensor:
    if inp.dtype != 'f32':
        raise ShapeError(f'takeAlongAxis: input must be f32, got {inp.dtype}', 'takeAlongAxis')
    if indices.dtype != 'i32':
        raise ShapeError(f'takeAlongAxis: indices must be i32, got {indices.dtype}', 'takeAlongAxis')
    N = len(inp.shape)
    if len(indices.shape) != N:
        raise ShapeError('takeAlongAxis: input and indices must have the same rank', 'takeAlongAxis')
    k = N + axis if axis < 0 else axis
    if k < 0 or k >= N:
        raise ShapeError(f'takeAlongAxis: axis {axis} out of range for rank-{N} input', 'takeAlongAxis')
    for i in range(N):
        if i != k and inp.shape[i] != indices.shape[i]:
            raise ShapeError(f'takeAlongAxis: input and indices must match on every axis except {k}', 'takeAlongAxis')
    permuted = permute(inp, [i for i in range(N) if i != k] + [k])
    sA = inp.shape[k]
    expanded = reshape(permuted, [1 if i == k else inp.shape[i] for i in range(N)] + [sA])
    oh = one_hot(indices, sA, 'f32')
    return sum_(mul(expanded, oh), -1)


def embedding(table: Tensor, indices: Tensor) -> Tensor:
    """`matmul(oneHot(indices, V), table)` (ops.ts:626-635). The backend recognises this
    pattern and runs a gather forward / segmented scatter-add backward."""
    if len(table.shape) != 2:
        raise ShapeError(f'embedding: table must be 2-d [vocab, dim], got {S.show(table.shape)}', 'embedding')
    if indices.dtype != 'i32':
        raise ShapeError(f'embedding: indices must be i32, got {indices.dtype}', 'embedding')
    return matmul(one_hot(indices, table.shape[0], 'f32'), table)


def arange(n: int, dtype: str = 'i32') -> Tensor:
    if not isinstance(n, int) or n <= 0:
        raise ShapeError(f'arange: n must be a positive integer, got {n}', 'arange')
    return add_op(current_graph(), 'arange', [n], dtype, 'arange', {'n': n, 'dtype': dtype})


def _const_fill(name: str, shape: Sequence[int], dtype: str, value: Number) -> Tensor:
    for d in shape:
        if not isinstance(d, int) or d <= 0:
            raise ShapeError(f'{name}: shape must be positive integers, got {S.show(shape)}', name)
    return add_op(current_graph(), 'const_fill', shape, dtype, name, {'value': value, 'dtype': dtype})


def zeros(shape, dtype='f32'): return _const_fill('zeros', shape, dtype, 0)
def ones(shape, dtype='f32'): return _const_fill('ones', shape, dtype, 1)


# ---- ML primitives (ops.ts:675-760) ----------------------------------------------------------------

def _softmax_causal_last(a: Tensor) -> Tensor:
    if a.dtype != 'f32':
        raise ShapeError(f'softmaxCausal: requires f32, got {a.dtype}', 'softmaxCausal')
    S.infer_where_causal('softmaxCausal', a.shape, 'softmaxCausal')
    return add_op(current_graph(), 'softmax_causal_last', a.shape, 'f32', 'softmaxCausal', {'a': a.id})


def softmax_causal(a: Tensor, axis: int = -1) -> Tensor:
    return _axis_preserving(a, axis, 'softmaxCausal', _softmax_causal_last)


def _log_softmax_last(a: Tensor) -> Tensor:
    if a.dtype != 'f32':
        raise ShapeError(f'logSoftmax: requires f32, got {a.dtype}', 'logSoftmax')
    return add_op(current_graph(), 'log_softmax_last', a.shape, 'f32', 'logSoftmax', {'a': a.id})


def log_softmax(a: Tensor, axis: int = -1) -> Tensor:
    return _axis_preserving(a, axis, 'logSoftmax', _log_softmax_last)


def softmax(a: Tensor, axis: int = -1) -> Tensor:
    return exp(log_softmax(a, axis))


def _axis_preserving(a: Tensor, axis_arg: int, name: str, apply_last) -> Tensor:
    r = len(a.shape)
    if r == 0:
        raise ShapeError(f'{name}: cannot apply to 0-d tensor', name)
    k = r + axis_arg if axis_arg < 0 else axis_arg
    if k < 0 or k >= r:
        raise ShapeError(f'{name}: axis {axis_arg} out of range', name)
    if k == r - 1:
        return apply_last(a)
    perm = [i for i in range(r) if i != k] + [k]
    return permute(apply_last(permute(a, perm)), _back_perm(k, r))


def _axis_reducing(a: Tensor, axis_arg: int, name: str, apply_last) -> Tensor:
    r = len(a.shape)
    if r == 0:
        raise ShapeError(f'{name}: cannot reduce a 0-d tensor', name)
    k = r + axis_arg if axis_arg < 0 else axis_arg
    if k < 0 or k >= r:
        raise ShapeError(f'{name}: axis {axis_arg} out of range', name)
    if k == r - 1:
        return apply_last(a)
    return apply_last(permute(a, [i for i in range(r) if i != k] + [k]))


def where_causal(a: Tensor, fill_value: Number) -> Tensor:
    if a.dtype != 'f32':
        raise ShapeError(f'whereCausal: requires f32, got {a.dtype}', 'whereCausal')
    S.infer_where_causal('whereCausal', a.shape, 'whereCausal')
    return add_op(current_graph(), 'where_causal', a.shape, 'f32', 'whereCausal', {'a': a.id, 'fillValue': fill_value})


# ---- Slicing / concat (ops.ts:766-857) -------------------------------------------------------------

def narrow(a: Tensor, axis: int, start: int, length: int) -> Tensor:
    ax = len(a.shape) + axis if axis < 0 else axis
    end = start + length
    out = S.infer_slice_range('narrow', a.shape, ax, start, end, 'narrow')
    return add_op(current_graph(), 'slice_range', out, a.dtype, 'narrow', {'a': a.id, 'axis': ax, 'start': start, 'end': end})


def scatter_axis(a: Tensor, out_shape: Sequence[int], axis: int, start: int, end: int) -> Tensor:
    out = S.infer_scatter_axis('scatterAxis', a.shape, out_shape, axis, start, end, 'scatterAxis')
    return add_op(current_graph(), 'scatter_axis', out, a.dtype, 'scatterAxis',
                  {'a': a.id, 'outShape': list(out_shape), 'axis': axis, 'start': start, 'end': end})


CONCAT_INPUT_CAP = 7   # ops.ts:788 (kept: it shapes the emitted IR)


def concat(tensors: Sequence[Tensor], axis: int) -> Tensor:
    if len(tensors) == 0:
        raise ShapeError('concat: needs at least one input', 'concat')
    if len(tensors) == 1:
        return tensors[0]
    dtype = tensors[0].dtype
    for t in tensors:
        if t.dtype != dtype:
            raise ShapeError(f'concat: dtype mismatch ({dtype} vs {t.dtype})', 'concat')
    ax = len(tensors[0].shape) + axis if axis < 0 else axis
    layer = list(tensors)
    while len(layer) > CONCAT_INPUT_CAP:
        nxt = []
        for i in range(0, len(layer), CONCAT_INPUT_CAP):
            chunk = layer[i:i + CONCAT_INPUT_CAP]
            nxt.append(chunk[0] if len(chunk) == 1 else _concat_one(chunk, ax))
        layer = nxt
    return _concat_one(layer, ax)


def _concat_one(tensors: Sequence[Tensor], ax: int) -> Tensor:
    out = S.infer_concat('concat', [t.shape for t in tensors], ax, 'concat')
    return add_op(current_graph(), 'concat', out, tensors[0].dtype, 'concat', {'inputs': [t.id for t in tensors], 'axis': ax})


def stack(tensors: Sequence[Tensor], axis: int) -> Tensor:
    if len(tensors) == 0:
        raise ShapeError('stack: needs at least one input', 'stack')
    t0 = tensors[0]
    ax = len(t0.shape) + 1 + axis if axis < 0 else axis
    new_shape = list(t0.shape[:ax]) + [1] + list(t0.shape[ax:])
    return concat([reshape(t, new_shape) for t in tensors], ax)


def split_heads(x: Tensor, n_heads: int) -> Tensor:
    r = len(x.shape)
    if r < 2:
        raise ShapeError(f'splitHeads: requires rank >= 2, got {r}', 'splitHeads')
    T, D = x.shape[r - 2], x.shape[r - 1]
    if D % n_heads != 0:
        raise ShapeError(f'splitHeads: last dim {D} not divisible by nHeads {n_heads}', 'splitHeads')
    lead = list(x.shape[:r - 2])
    reshaped = reshape(x, lead + [T, n_heads, D // n_heads])
    return swap_axes(reshaped, len(lead), len(lead) + 1)


def merge_heads(x: Tensor) -> Tensor:
    r = len(x.shape)
    if r < 3:
        raise ShapeError(f'mergeHeads: requires rank >= 3, got {r}', 'mergeHeads')
    H, T, d = x.shape[r - 3], x.shape[r - 2], x.shape[r - 1]
    lead = list(x.shape[:r - 3])
    swapped = swap_axes(x, r - 3, r - 2)
    return reshape(swapped, lead + [T, H * d])


def split(t: Tensor, sizes: Sequence[int], axis: int) -> List[Tensor]:
    ax = len(t.shape) + axis if axis < 0 else axis
    if ax < 0 or ax >= len(t.shape):
        raise ShapeError(f'split: axis {axis} out of range', 'split')
    if sum(sizes) != t.shape[ax]:
        raise ShapeError(f'split: sizes sum to {sum(sizes)}, but axis {ax} has size {t.shape[ax]}', 'split')
    out, cursor = [], 0
    for s in sizes:
        out.append(narrow(t, ax, cursor, s))
        cursor += s
    return out


def rope(q: Tensor, k: Tensor, base: float = 10000) -> Tuple[Tensor, Tensor]:
    """Rotary embedding, rotate-half convention (ops.ts:878-919)."""
    if q.dtype != 'f32' or k.dtype != 'f32':
        raise ShapeError('rope: q and k must be f32', 'rope')
    T, D = q.shape[-2], q.shape[-1]
    if k.shape[-2] != T or k.shape[-1] != D:
        raise ShapeError('rope: q and k must share sequence and feature dims', 'rope')
    if D % 2 != 0:
        raise ShapeError(f'rope: rotation dim must be even (rotates pairs), got {D}', 'rope')
    half = D // 2
    idx = arange(half, 'f32')
    freqs = exp(mul(idx, -math.log(base) / half))
    positions = arange(T, 'f32')
    angles = mul(reshape(positions, [T, 1]), reshape(freqs, [1, half]))
    cos_half, sin_half = cos(angles), sin(angles)
    cos_full = concat([cos_half, cos_half], -1)
    sin_full = concat([sin_half, sin_half], -1)

    def apply_rot(x: Tensor) -> Tensor:
        x1, x2 = split(x, [half, half], -1)
        rotated = concat([neg(x2), x1], -1)
        return add(mul(x, cos_full), mul(rotated, sin_full))
    return apply_rot(q), apply_rot(k)


# ---- Sequence operators (no reference counterpart) ---------------------------------------------------

ATTENTION_MAX_HEAD = 128   # the kernels' tiles hold whole heads
ATTENTION_RANGE = 2.0 ** 60   # of constants that the kernels multiply in f32
ROPE_LEAST_BASE = 2.0 ** -16   # angles below 2^47, which 64 bits reduce to a quarter turn


def _finite(x) -> bool:
    return _num(x) and math.isfinite(x)


def _count(x) -> bool:
    return isinstance(x, int) and not isinstance(x, bool)


def _attention_fields(site: str, q: Tensor, k: Tensor, v: Tensor, causal, scale, softcap, slopes, documents, prefix,
                      lengths, window, sinks) -> dict:
    for name, t in (('q', q), ('k', k), ('v', v)):
        if t.dtype != 'f32':
            raise ShapeError(f'{site}: {name} must be f32, got {t.dtype}', site)
        if len(t.shape) != 4:
            raise ShapeError(f'{site}: {name} must be [batch, heads, length, head size], got {S.show(t.shape)}', site)
    B, H, Tq, D = q.shape
    _, Hk, Tk, Dv = v.shape
    if min(B, H, Tq, D, Hk, Tk, Dv) < 1:
        raise ShapeError(f'{site}: empty operand', site)
    if k.shape != (B, Hk, Tk, D) or v.shape[0] != B:
        raise ShapeError(f'{site}: q {S.show(q.shape)}, k {S.show(k.shape)} and v {S.show(v.shape)} must agree in batch, '
                         'q and k in head size, k and v in heads and length', site)
    if H % Hk != 0:
        raise ShapeError(f'{site}: {H} query heads cannot share {Hk} key heads evenly', site)
    if D > ATTENTION_MAX_HEAD or Dv > ATTENTION_MAX_HEAD:
        raise ShapeError(f'{site}: head sizes above {ATTENTION_MAX_HEAD} are not supported, got {D} and {Dv}', site)
    positional = causal or slopes is not None or documents is not None
    if positional and Tq > Tk:
        raise ShapeError(f'{site}: {Tq} queries are not the last of {Tk} positions', site)
    if scale is None:
        scale = 1 / math.sqrt(D)
    for name, x in (('scale', scale), ('softcap', softcap)):
        if x is not None and (not _finite(x) or not 1 / ATTENTION_RANGE <= x <= ATTENTION_RANGE):
            raise ShapeError(f'{site}: {name} must be positive, between 2^-60 and 2^60, got {x}', site)
    if slopes is not None:
        slopes = [float(x) for x in slopes] if all(_finite(x) and abs(x) <= ATTENTION_RANGE for x in slopes) else None
        if slopes is None or len(slopes) != H:
            raise ShapeError(f'{site}: slopes must be {H} finite numbers, one per query head, of 2^60 at most', site)
    if prefix is not None and not causal:
        raise ShapeError(f'{site}: a prefix needs a causal mask', site)
    if window is not None and (not _count(window) or not 1 <= window < 2 ** 31):
        raise ShapeError(f'{site}: window must be a whole number of positions, 1 at least, got {window}', site)
    if not _count(sinks) or not 0 <= sinks < 2 ** 31:
        raise ShapeError(f'{site}: sinks must be a whole number of positions, got {sinks}', site)
    if window is not None and not causal:
        raise ShapeError(f'{site}: a window needs a causal mask', site)
    if sinks and window is None:
        raise ShapeError(f'{site}: sinks need a window', site)
    if sinks and documents is not None:
        raise ShapeError(f'{site}: sinks are the first positions of a sequence, which documents end', site)
    for name, t, shape in (('documents', documents, (B, Tk)), ('prefix', prefix, (B,)), ('lengths', lengths, (B,))):
        if t is not None and (t.dtype != 'i32' or t.shape != shape):
            raise ShapeError(f'{site}: {name} must be i32 {S.show(shape)}, got {t.dtype} {S.show(t.shape)}', site)
    ids = {n: None if t is None else t.id for n, t in (('documents', documents), ('prefix', prefix), ('lengths', lengths))}
    return {'q': q.id, 'k': k.id, 'v': v.id, **ids, 'causal': bool(causal), 'scale': scale, 'softcap': softcap, 'slopes': slopes,
            'window': window, 'sinks': sinks}


def attention(q: Tensor, k: Tensor, v: Tensor, causal: bool = True, scale: Optional[float] = None,
              softcap: Optional[float] = None, slopes: Optional[Sequence[float]] = None, documents: Optional[Tensor] = None,
              prefix: Optional[Tensor] = None, lengths: Optional[Tensor] = None, window: Optional[int] = None,
              sinks: int = 0) -> Tensor:
    """Attention of q [B, H, Tq, D] over k [B, Hk, Tk, D], v [B, Hk, Tk, Dv] -> [B, H, Tq, Dv]. Query head h reads key head
    h // (H / Hk). With x = scale q.k (scale: 1 / sqrt(D)), the score of key j for a query at position p is

        softcap tanh(x / softcap) - slopes[h] |p - j|        (each part where it is given)

    `lengths` i32 [B]: only the first lengths[b] keys are there (clamped to 0..Tk; without it all Tk). The queries are the
    last Tq of those positions, so one new token against a filled cache is Tq = 1. `causal` hides keys after p, except those
    below `prefix` i32 [B], which every query sees. `window` leaves a query the last `window` keys up to its own, p - window < j,
    beside the first `sinks` positions (not with documents) and those of a prefix; both need the causal mask. `documents` i32
    [B, Tk]: a query sees the keys of its own document (that at its position); negative ids are padding, which sees and is seen by nothing. A query that sees no key (or, where
    positions matter, lies before position 0) gives zeros and takes and gives no gradient. What a mask hides has no
    influence, whatever its values (infinities and NaN included)."""
    f = _attention_fields('attention', q, k, v, causal, scale, softcap, slopes, documents, prefix, lengths, window, sinks)
    return add_op(current_graph(), 'attention', (*q.shape[:3], v.shape[3]), 'f32', 'attention', f)


def attention_grad(q: Tensor, k: Tensor, v: Tensor, y: Tensor, dy: Tensor, causal: bool = True, scale: Optional[float] = None,
                   softcap: Optional[float] = None, slopes: Optional[Sequence[float]] = None,
                   documents: Optional[Tensor] = None, prefix: Optional[Tensor] = None,
                   lengths: Optional[Tensor] = None, window: Optional[int] = None, sinks: int = 0) -> Tuple[Tensor, Tensor, Tensor]:
    """(dq, dk, dv) of y = attention(q, k, v, ...) for the gradient dy of y; the other arguments as given there."""
    site = 'attentionGrad'
    f = _attention_fields(site, q, k, v, causal, scale, softcap, slopes, documents, prefix, lengths, window, sinks)
    shape = (*q.shape[:3], v.shape[3])
    for name, t in (('y', y), ('dy', dy)):
        if t.dtype != 'f32' or t.shape != shape:
            raise ShapeError(f'{site}: {name} must be f32 {S.show(shape)}, got {t.dtype} {S.show(t.shape)}', site)
    g = current_graph()
    stats = add_op(g, 'attention_stats', (*q.shape[:3], 2), 'f32', site, f)
    f = dict(f, y=y.id, stats=stats.id, dy=dy.id)
    return tuple(add_op(g, f'attention_grad_{n}', t.shape, 'f32', site, f) for n, t in (('q', q), ('k', k), ('v', v)))


def rope_axes(q: Tensor, k: Tensor, positions: Tensor, sections: Sequence[int], base: float = 10000, per_axis: bool = False,
              inverse: bool = False) -> Tuple[Tensor, Tensor]:
    """Rotary embedding by positions of several axes (time, height, width; one axis: given positions), rotate-half
    convention as `rope`. q [B, H, T, D], k [B, Hk, T, D], positions i32 [A, B, T]; `sections` gives each axis its number of
    pairs, laid end to end: with half = sum(sections), pair p is (x[p], x[p + half]), features from 2 half on pass
    unchanged. A pair of axis a turns by positions[a] * base^(-p / half), with `per_axis` by
    positions[a] * base^(-(p - first pair of a) / sections[a]). `inverse` turns back (the gradient)."""
    site = 'ropeAxes'
    for name, t in (('q', q), ('k', k)):
        if t.dtype != 'f32' or len(t.shape) != 4 or min(t.shape) < 1:
            raise ShapeError(f'{site}: {name} must be f32 [batch, heads, length, head size], got {t.dtype} {S.show(t.shape)}', site)
    B, _, T, D = q.shape
    if (k.shape[0], k.shape[2], k.shape[3]) != (B, T, D):
        raise ShapeError(f'{site}: q {S.show(q.shape)} and k {S.show(k.shape)} must agree in batch, length and head size', site)
    sections = list(sections)
    if not sections or not all(isinstance(n, int) and not isinstance(n, bool) and n > 0 for n in sections) or 2 * sum(sections) > D:
        raise ShapeError(f'{site}: sections must be positive pair counts of at most {D // 2} in all, got {sections}', site)
    if positions.dtype != 'i32' or positions.shape != (len(sections), B, T):
        raise ShapeError(f'{site}: positions must be i32 {S.show((len(sections), B, T))}, got {positions.dtype} '
                         f'{S.show(positions.shape)}', site)
    if not _finite(base) or base < ROPE_LEAST_BASE:
        raise ShapeError(f'{site}: base must be positive, at least 2^-16, got {base}', site)
    return tuple(_rope_axes(x, positions, sections, base, bool(per_axis), bool(inverse)) for x in (q, k))


def _rope_axes(x: Tensor, positions: Tensor, sections, base, per_axis: bool, inverse: bool) -> Tensor:
    return add_op(current_graph(), 'rope_axes', x.shape, 'f32', 'ropeAxes', {
        'a': x.id, 'positions': positions.id, 'sections': list(sections), 'base': base, 'perAxis': per_axis, 'inverse': inverse})


def _recurrence_check(site: str, a: Tensor, h0: Optional[Tensor], **others: Tensor) -> None:
    for name, t in (('a', a), *others.items()):
        if t.dtype != 'f32' or len(t.shape) != 3 or min(t.shape) < 1 or t.shape != a.shape:
            raise ShapeError(f'{site}: {name} must be f32 [batch, length, channels] like a {S.show(a.shape)}, got {t.dtype} '
                             f'{S.show(t.shape)}', site)
    if h0 is not None and (h0.dtype != 'f32' or h0.shape != (a.shape[0], a.shape[2])):
        raise ShapeError(f'{site}: h0 must be f32 [batch, channels] for a {S.show(a.shape)}, got {h0.dtype} {S.show(h0.shape)}', site)


def linear_recurrence(a: Tensor, x: Tensor, h0: Optional[Tensor] = None) -> Tensor:
    """Gated linear recurrence h[:, t] = a[:, t] h[:, t-1] + x[:, t] over [B, T, C], each channel by itself, from h0 [B, C]
    (zeros without it). A gate of 0 starts afresh (the first position of a packed document)."""
    _recurrence_check('linearRecurrence', a, h0, x=x)
    return add_op(current_graph(), 'linear_recurrence', a.shape, 'f32', 'linearRecurrence',
                  {'a': a.id, 'x': x.id, 'h0': None if h0 is None else h0.id})


def linear_recurrence_grad(a: Tensor, h: Tensor, dh: Tensor, h0: Optional[Tensor] = None) -> Tuple[Tensor, ...]:
    """(da, dx), with h0 (da, dx, dh0), of h = linear_recurrence(a, x, h0) for the gradient dh of h."""
    site = 'linearRecurrenceGrad'
    _recurrence_check(site, a, h0, h=h, dh=dh)
    f = {'a': a.id, 'h': h.id, 'dh': dh.id, 'h0': None if h0 is None else h0.id}
    outs = (('a', a.shape), ('x', a.shape)) + ((('h0', h0.shape),) if h0 is not None else ())
    return tuple(add_op(current_graph(), f'linear_recurrence_grad_{n}', s, 'f32', site, f) for n, s in outs)


LINEAR_MAX_HEAD = 128      # the kernels' tiles hold whole heads
LINEAR_SEGMENT = 128       # positions between the states that the gradients take from the forward pass


def _linear_fields(site: str, q: Tensor, k: Tensor, v: Tensor, decay, scale, state, documents, lengths) -> dict:
    for name, t in (('q', q), ('k', k), ('v', v)):
        if t.dtype != 'f32' or len(t.shape) != 4 or min(t.shape) < 1:
            raise ShapeError(f'{site}: {name} must be f32 [batch, heads, length, head size], got {t.dtype} {S.show(t.shape)}', site)
    B, H, T, D = q.shape
    Hk, Dv = v.shape[1], v.shape[3]
    if k.shape != (B, Hk, T, D) or v.shape != (B, Hk, T, Dv):
        raise ShapeError(f'{site}: q {S.show(q.shape)}, k {S.show(k.shape)} and v {S.show(v.shape)} must agree in batch and length, '
                         'q and k in head size, k and v in heads', site)
    if H % Hk != 0:
        raise ShapeError(f'{site}: {H} query heads cannot share {Hk} key heads evenly', site)
    if max(D, Dv) > LINEAR_MAX_HEAD:
        raise ShapeError(f'{site}: head sizes above {LINEAR_MAX_HEAD} are not supported, got {D} and {Dv}', site)
    decay = [float(x) for x in decay] if all(_finite(x) and 0 < x <= 1 for x in decay) else None
    if decay is None or len(decay) != H:
        raise ShapeError(f'{site}: decay must be {H} numbers above 0, of 1 at most, one per query head', site)
    if scale is None:
        scale = 1 / math.sqrt(D)
    if not _finite(scale) or not 1 / ATTENTION_RANGE <= scale <= ATTENTION_RANGE:
        raise ShapeError(f'{site}: scale must be positive, between 2^-60 and 2^60, got {scale}', site)
    if state is not None and (state.dtype != 'f32' or state.shape != (B, H, D, Dv)):
        raise ShapeError(f'{site}: state must be f32 {S.show((B, H, D, Dv))}, got {state.dtype} {S.show(state.shape)}', site)
    for name, t, shape in (('documents', documents, (B, T)), ('lengths', lengths, (B,))):
        if t is not None and (t.dtype != 'i32' or t.shape != shape):
            raise ShapeError(f'{site}: {name} must be i32 {S.show(shape)}, got {t.dtype} {S.show(t.shape)}', site)
    ids = {n: None if t is None else t.id for n, t in (('state', state), ('documents', documents), ('lengths', lengths))}
    return {'q': q.id, 'k': k.id, 'v': v.id, **ids, 'decay': decay, 'scale': scale}


def linear_attention(q: Tensor, k: Tensor, v: Tensor, decay: Sequence[float], scale: Optional[float] = None,
                     state: Optional[Tensor] = None, documents: Optional[Tensor] = None,
                     lengths: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """Linear attention with a decay for each head: (y, last state) of q [B, H, T, D], k [B, Hk, T, D], v [B, Hk, T, Dv]. Query
    head h reads key head h // (H / Hk) and has the state S [D, Dv], from `state` [B, H, D, Dv] (zeros without it):

        S[t] = decay[h] S[t-1] + k[t] v[t]^T,   y[t] = scale S[t]^T q[t]        (scale: 1 / sqrt(D))

    which is y[t] = scale sum over s <= t of decay^(t - s) (q[t].k[s]) v[s] beside what `state` adds. The last state [B, H, D, Dv]
    is what the next positions start from: a prompt is read in one call, or in pieces, and answered with T = 1. `lengths` i32 [B]:
    only the first lengths[b] positions are there (clamped to 0..T), y is 0 behind them and the last state that after them.
    `documents` i32 [B, T]: the state starts from zeros where an id differs from the one before (position 0 goes on from `state`);
    negative ids are padding, where y and the state are 0. What is not there has no influence, whatever its values; infinities and
    NaN that are there stay in the state, whatever the decay."""
    f = _linear_fields('linearAttention', q, k, v, decay, scale, state, documents, lengths)
    B, H, T, D = q.shape
    g = current_graph()
    return (add_op(g, 'linear_attention', (B, H, T, v.shape[3]), 'f32', 'linearAttention', f),
            add_op(g, 'linear_attention_state', (B, H, D, v.shape[3]), 'f32', 'linearAttention', f))


def linear_attention_grad(q: Tensor, k: Tensor, v: Tensor, dy: Optional[Tensor], decay: Sequence[float],
                          scale: Optional[float] = None, state: Optional[Tensor] = None, documents: Optional[Tensor] = None,
                          lengths: Optional[Tensor] = None, dstate: Optional[Tensor] = None) -> Tuple[Tensor, ...]:
    """(dq, dk, dv), with `state` (dq, dk, dv, its gradient), of linear_attention(q, k, v, decay, ...) for the gradients dy of y
    and dstate of the last state, one of which may be absent (None)."""
    site = 'linearAttentionGrad'
    f = _linear_fields(site, q, k, v, decay, scale, state, documents, lengths)
    B, H, T, D = q.shape
    if dy is None and dstate is None:
        raise ShapeError(f'{site}: needs the gradient of y or of the last state', site)
    for name, t, shape in (('dy', dy, (B, H, T, v.shape[3])), ('dstate', dstate, (B, H, D, v.shape[3]))):
        if t is not None and (t.dtype != 'f32' or t.shape != shape):
            raise ShapeError(f'{site}: {name} must be f32 {S.show(shape)}, got {t.dtype} {S.show(t.shape)}', site)
    g = current_graph()
    segments = -(-T // LINEAR_SEGMENT)
    borders = None if segments == 1 else add_op(g, 'linear_attention_borders', (segments, B, H, D, v.shape[3]), 'f32', site, f)
    f = dict(f, dy=None if dy is None else dy.id, dstate=None if dstate is None else dstate.id)
    outs = (('q', q), ('k', k), ('v', v)) + ((('state', state),) if state is not None else ())
    more = {'q': {'borders': None if borders is None else borders.id}}
    return tuple(add_op(g, f'linear_attention_grad_{n}', t.shape, 'f32', site, dict(f, **more.get(n, {}))) for n, t in outs)


# ---- Choice of the next token (no reference counterpart) ---------------------------------------------

SAMPLE_MAX_VOCAB = 1 << 24   # weights are whole numbers of 62 bits in all


def sample(logits: Tensor, u: Tensor, temperature=1.0, top_k=None, top_p=None, min_p=None) -> Tensor:
    """The next token of each row: i32 [...] for logits f32 [..., V] and random numbers u f32 [...] from [0, 1).

    Tokens are ordered by falling logit, equal ones by rising index, and weigh exp((logit - largest) / temperature). Each limit
    keeps a first part of that order: `top_k` tokens; of those the fewest whose weights reach `top_p` of their sum; and of those
    the ones of at least `min_p` times the largest weight. The token is the first kept one, in the vocabulary's order, where the
    kept weights' running sum passes u of them all; a u below 0 (or NaN) counts as 0, one from 1 on takes the last.

    A limit is one number for all rows, or a tensor of u's shape with a number for each (f32, `top_k` i32); None, a top_k below 1
    or a top_p from 1 on do not limit, and a temperature of 0 takes the largest logit. In tensors, a temperature that is not above 0
    does so too (NaN with it); the first of the order is always kept, alone where top_p is not above 0, min_p above 1 or min_p NaN; a
    top_p of NaN and a min_p below 0 do not limit. Minus infinity and NaN are never chosen; a row without any other logit gives -1.

    Weights are computed in 64 bits, 2^-50 of the largest off at most, and rounded to whole multiples of 2^(b - 62) of it for a
    vocabulary of b bits (less than half of that counts as 0); sums of these are exact."""
    site = 'sample'
    if logits.dtype != 'f32' or len(logits.shape) < 1 or min(logits.shape) < 1:
        raise ShapeError(f'{site}: logits must be f32 [..., vocabulary], got {logits.dtype} {S.show(logits.shape)}', site)
    rows = logits.shape[:-1]
    if logits.shape[-1] > SAMPLE_MAX_VOCAB:
        raise ShapeError(f'{site}: vocabularies above {SAMPLE_MAX_VOCAB} are not supported, got {logits.shape[-1]}', site)
    if u.dtype != 'f32' or u.shape != rows:
        raise ShapeError(f'{site}: u must be f32 {S.show(rows)}, got {u.dtype} {S.show(u.shape)}', site)
    f = {'logits': logits.id, 'u': u.id}
    values = []
    for name, x, none, ok in (('temperature', temperature, 1.0, lambda x: x >= 0), ('topK', top_k, 0, lambda x: _count(x) and 0 <= x < 2 ** 31),
                              ('topP', top_p, 1.0, lambda x: x > 0), ('minP', min_p, 0.0, lambda x: 0 <= x <= 1)):
        dtype = 'i32' if name == 'topK' else 'f32'
        f[name] = None
        if isinstance(x, Tensor):
            if x.dtype != dtype or x.shape != rows:
                raise ShapeError(f'{site}: {name} must be a number or {dtype} {S.show(rows)}, got {x.dtype} {S.show(x.shape)}', site)
            f[name] = x.id
            x = none
        elif x is None:
            x = none
        elif not _finite(x) or not ok(x):
            raise ShapeError(f'{site}: {name} out of range, got {x}', site)
        values.append(x)
    return add_op(current_graph(), 'sample', rows, 'i32', site, dict(f, values=values))


# ---- Broadcast / constants / comparisons (ops.ts:943-1008) -----------------------------------------

def broadcast_to(a: Tensor, target: Sequence[int]) -> Tensor:
    S.infer_broadcast_to('broadcastTo', a.shape, target, 'broadcastTo')
    return add_op(current_graph(), 'broadcast_to', target, a.dtype, 'broadcastTo', {'a': a.id, 'targetShape': list(target)})


def sum_to_shape(a: Tensor, target: Sequence[int]) -> Tensor:
    S.infer_sum_to_shape('sumToShape', a.shape, target, 'sumToShape')
    return add_op(current_graph(), 'sum_to_shape', target, a.dtype, 'sumToShape', {'a': a.id, 'targetShape': list(target)})


def const_scalar(value: Number, dtype: str = 'f32') -> Tensor:
    return add_op(current_graph(), 'const_scalar', [], dtype, 'constScalar', {'value': value, 'dtype': dtype})


def less(a, b) -> Tensor:
    if _num(a):
        return greater(b, a)
    rhs = const_scalar(b, a.dtype) if _num(b) else b
    return _binop('less', 'less', a, rhs, 'bool')


def greater(a, b) -> Tensor:
    if _num(a):
        return less(b, a)
    rhs = const_scalar(b, a.dtype) if _num(b) else b
    return _binop('greater', 'greater', a, rhs, 'bool')


def where(cond: Tensor, a: Tensor, b: Tensor) -> Tensor:
    if cond.dtype != 'bool':
        raise ShapeError(f'where: cond must be bool, got {cond.dtype}', 'where')
    if a.dtype != b.dtype:
        raise ShapeError(f'where: a/b dtype mismatch ({a.dtype} vs {b.dtype})', 'where')
    out = S.infer_where('where', cond.shape, a.shape, b.shape, 'where')
    return add_op(current_graph(), 'where', out, a.dtype, 'where', {'cond': cond.id, 'a': a.id, 'b': b.id})


def relu_grad(x: Tensor, dy: Tensor) -> Tensor:
    if x.dtype != 'f32' or dy.dtype != 'f32':
        raise ShapeError(f'reluGrad: requires f32, got {x.dtype} and {dy.dtype}', 'reluGrad')
    out = S.infer_relu_grad('reluGrad', x.shape, dy.shape, 'reluGrad')
    return add_op(current_graph(), 'relu_grad', out, 'f32', 'reluGrad', {'x': x.id, 'dy': dy.id})


# ---- Adam-fused ops (ops.ts:1014-1065) -----------------------------------------------------------------

def adam_update_m(m: Tensor, g: Tensor, beta1: float) -> Tensor:
    if m.dtype != 'f32' or g.dtype != 'f32':
        raise ShapeError('adamUpdateM: requires f32', 'adamUpdateM')
    if m.shape != g.shape:
        raise ShapeError('adamUpdateM: shape mismatch', 'adamUpdateM')
    return add_op(current_graph(), 'adam_update_m', m.shape, 'f32', 'adamUpdateM', {'m': m.id, 'g': g.id, 'beta1': beta1})


def adam_update_v(v: Tensor, g: Tensor, beta2: float) -> Tensor:
    if v.dtype != 'f32' or g.dtype != 'f32':
        raise ShapeError('adamUpdateV: requires f32', 'adamUpdateV')
    if v.shape != g.shape:
        raise ShapeError('adamUpdateV: shape mismatch', 'adamUpdateV')
    return add_op(current_graph(), 'adam_update_v', v.shape, 'f32', 'adamUpdateV', {'v': v.id, 'g': g.id, 'beta2': beta2})


def adam_update_p(p: Tensor, m_new: Tensor, v_new: Tensor, lrt: Tensor, eps: float, decay_shrink=1) -> Tensor:
    if p.dtype != 'f32':
        raise ShapeError('adamUpdateP: requires f32', 'adamUpdateP')
    if lrt.dtype != 'f32' or len(lrt.shape) != 0:
        raise ShapeError('adamUpdateP: lrt must be a 0-d f32 scalar', 'adamUpdateP')
    if p.shape != m_new.shape:
        raise ShapeError('adamUpdateP: p/mNew shape mismatch', 'adamUpdateP')
    is_tensor = isinstance(decay_shrink, Tensor)
    if is_tensor and (decay_shrink.dtype != 'f32' or len(decay_shrink.shape) != 0):
        raise ShapeError('adamUpdateP: decayShrink tensor must be a 0-d f32 scalar', 'adamUpdateP')
    return add_op(current_graph(), 'adam_update_p', p.shape, 'f32', 'adamUpdateP', {
        'p': p.id, 'mNew': m_new.id, 'vNew': v_new.id, 'lrt': lrt.id, 'eps': eps,
        'decayShrink': 1 if is_tensor else decay_shrink,
        'decayShrinkTensor': decay_shrink.id if is_tensor else None,
    })


# ---- Conv / pool (ops.ts:1084-1197) ----------------------------------------------------------------------

def pair_opt(v, default: int) -> Tuple[int, int]:
    if v is None:
        return (default, default)
    if isinstance(v, int):
        return (v, v)
    return (v[0], v[1])


def conv2d(inp: Tensor, weight: Tensor, stride=None, padding=None, groups: int = 1) -> Tensor:
    if inp.dtype != 'f32':
        raise ShapeError(f'conv2d: input must be f32, got {inp.dtype}', 'conv2d')
    if weight.dtype != 'f32':
        raise ShapeError(f'conv2d: weight must be f32, got {weight.dtype}', 'conv2d')
    sH, sW = pair_opt(stride, 1)
    pH, pW = pair_opt(padding, 0)
    out = S.infer_conv2d('conv2d', inp.shape, weight.shape, sH, sW, pH, pW, groups, 'conv2d')
    return add_op(current_graph(), 'conv2d', out, 'f32', 'conv2d', {
        'input': inp.id, 'weight': weight.id, 'strideH': sH, 'strideW': sW, 'padH': pH, 'padW': pW, 'groups': groups})


def conv2d_input_grad(weight: Tensor, dy: Tensor, inH, inW, strideH, strideW, padH, padW, groups) -> Tensor:
    cOut, wInC = weight.shape[0], weight.shape[1]
    B = dy.shape[0]
    if dy.shape[1] != cOut:
        raise ShapeError(f"conv2dInputGrad: dy's C={dy.shape[1]} doesn't match weight C_out={cOut}", 'conv2dInputGrad')
    return add_op(current_graph(), 'conv2d_input_grad', [B, wInC * groups, inH, inW], 'f32', 'conv2dInputGrad', {
        'weight': weight.id, 'dy': dy.id, 'inH': inH, 'inW': inW, 'strideH': strideH, 'strideW': strideW,
        'padH': padH, 'padW': padW, 'groups': groups})


def conv2d_weight_grad(inp: Tensor, dy: Tensor, kH, kW, strideH, strideW, padH, padW, groups) -> Tensor:
    cIn, cOut = inp.shape[1], dy.shape[1]
    return add_op(current_graph(), 'conv2d_weight_grad', [cOut, cIn // groups, kH, kW], 'f32', 'conv2dWeightGrad', {
        'input': inp.id, 'dy': dy.id, 'kH': kH, 'kW': kW, 'strideH': strideH, 'strideW': strideW,
        'padH': padH, 'padW': padW, 'groups': groups})


def max_pool2d(inp: Tensor, kernel_size, stride=None, padding=None) -> Tensor:
    if inp.dtype != 'f32':
        raise ShapeError(f'maxPool2d: input must be f32, got {inp.dtype}', 'maxPool2d')
    kH, kW = (kernel_size, kernel_size) if isinstance(kernel_size, int) else (kernel_size[0], kernel_size[1])
    if stride is None:
        sH, sW = kH, kW
    elif isinstance(stride, int):
        sH, sW = stride, stride
    else:
        sH, sW = stride[0], stride[1]
    pH, pW = pair_opt(padding, 0)
    out = S.infer_max_pool2d('maxPool2d', inp.shape, kH, kW, sH, sW, pH, pW, 'maxPool2d')
    return add_op(current_graph(), 'max_pool_2d', out, 'f32', 'maxPool2d', {
        'input': inp.id, 'kH': kH, 'kW': kW, 'strideH': sH, 'strideW': sW, 'padH': pH, 'padW': pW})


def max_pool2d_grad(inp: Tensor, dy: Tensor, kH, kW, strideH, strideW, padH, padW) -> Tensor:
    return add_op(current_graph(), 'max_pool_2d_grad', inp.shape, 'f32', 'maxPool2dGrad', {
        'input': inp.id, 'dy': dy.id, 'kH': kH, 'kW': kW, 'strideH': strideH, 'strideW': strideW,
        'padH': padH, 'padW': padW})


def nearest_upsample2d(x: Tensor, factor: int) -> Tensor:
    if len(x.shape) != 4:
        raise ShapeError('nearestUpsample2d: input must be rank-4 [B, C, H, W]', 'nearestUpsample2d')
    if factor == 1:
        return x
    B, C, H, W = x.shape
    expanded = broadcast_to(reshape(x, [B, C, H, 1, W, 1]), [B, C, H, factor, W, factor])
    return reshape(expanded, [B, C, H * factor, W * factor])

"""Windowed attention, linear attention and the choice of a token in 64 bits, straight from their definitions, with bounds on
what f32 arithmetic may differ by (counted as in _sequence.py, in units U = 2^-24)."""
import numpy as np

import _sequence as R

U = R.U


def attention(q, k, v, dy=None, window=None, sinks=0, **how):
    """_sequence.attention with the mask of a window and of sinks beside the others."""
    plain = R.seen_mask

    def seen_mask(B, Tq, Tk, causal, slopes, documents, prefix, lengths):
        seen, p = plain(B, Tq, Tk, causal, slopes, documents, prefix, lengths)
        if window is not None:
            j = np.arange(Tk)
            near = (j[None, None, :] > p[:, :, None] - window) | (j < sinks)
            if prefix is not None:
                near = near | (j[None, None, :] < prefix[:, None, None])
            seen = seen & near
        return seen, p
    R.seen_mask = seen_mask
    try:
        return R.attention(q, k, v, dy, **how)
    finally:
        R.seen_mask = plain


def _runs(n, T, doc):
    """Which positions are there, and the first position of each one's document."""
    live = np.arange(T) < n
    since = np.zeros(T, int)
    for t in range(1, T):
        since[t] = since[t - 1] if doc is None or doc[t] == doc[t - 1] else t
    return (live if doc is None else live & (doc >= 0)), since


def linear(q, k, v, decay, scale=None, state=None, documents=None, lengths=None, dy=None, dstate=None):
    """{'y', 'state'}, with dy or dstate {'dq', 'dk', 'dv', 'dstate'} beside them, and bounds. Each result is a sum over pairs of
    weight times dot product times value: the dot product is off by (12 + 4 sqrt(D)) U of its operands' norms, the weight
    lam^n by its exponent's roundings, 2 n |ln lam| U, and 4 U of its own; sums of T terms by 4 sqrt(T) U. Taking a pair through
    the states of the positions between rounds a dozen times more, and a dot product more: twice the counts."""
    f64 = lambda x: None if x is None else x.astype(np.float64)  # noqa: E731
    q, k, v, state, dy, dstate = map(f64, (q, k, v, state, dy, dstate))
    B, H, T, D = q.shape
    Hk, Dv = v.shape[1], v.shape[3]
    G = H // Hk
    scale = 1 / np.sqrt(D) if scale is None else scale
    shapes = {'y': (B, H, T, Dv), 'state': (B, H, D, Dv)}
    if dy is not None or dstate is not None:
        shapes.update(dq=q.shape, dk=k.shape, dv=v.shape, dstate=(B, H, D, Dv))
    out = {n: np.zeros(s) for n, s in shapes.items()}
    tol = {n: np.zeros(s) for n, s in shapes.items()}
    at = np.arange(T)
    base = 48 + 8 * np.sqrt(max(D, Dv)) + 8 * np.sqrt(T * G)
    norm = lambda x: np.linalg.norm(x, axis=-1)  # noqa: E731
    for b in range(B):
        n = T if lengths is None else int(np.clip(lengths[b], 0, T))
        live, since = _runs(n, T, None if documents is None else documents[b])
        z = lambda x: np.where(live[:, None], x, 0.0)  # noqa: E731
        far = at[:, None] - at[None, :]
        pairs = (far >= 0) & (at[None, :] >= since[:, None]) & live[:, None] & live[None, :]
        opens = live & (since == 0)
        ends = n > 0 and live[n - 1]
        for h in range(H):
            lam, ln = decay[h], abs(np.log(decay[h]))
            Q, K, V = z(q[b, h]), z(k[b, h // G]), z(v[b, h // G])
            S0 = np.zeros((D, Dv)) if state is None else state[b, h]
            power = lambda e: lam ** np.maximum(e, 0).astype(float)  # noqa: E731
            roundings = lambda e: (base + 4 * ln * np.maximum(e, 0)) * U  # noqa: E731
            W = np.where(pairs, power(far), 0.0)
            c = np.where(opens, power(at + 1), 0.0)
            e = np.where(live & (at >= since[n - 1]) & ends, power(n - 1 - at), 0.0) if n else np.zeros(T)
            f = (lam ** n if opens[n - 1] else 0.0) if n else 1.0
            We, ce, ee, fe = W * roundings(far), c * roundings(at + 1), e * roundings(n - 1 - at), f * roundings(np.array(n))
            out['y'][b, h] = scale * ((W * (Q @ K.T)) @ V + c[:, None] * (Q @ S0))
            tol['y'][b, h] = scale * ((We * np.outer(norm(Q), norm(K))) @ np.abs(V) + ce[:, None] * np.outer(norm(Q), norm(S0.T)))
            out['state'][b, h] = (K * e[:, None]).T @ V + f * S0
            tol['state'][b, h] = np.abs(K * ee[:, None]).T @ np.abs(V) + fe * np.abs(S0)
            if 'dq' not in shapes:
                continue
            Y = np.zeros((T, Dv)) if dy is None else z(dy[b, h])
            G1 = np.zeros((D, Dv)) if dstate is None else dstate[b, h]
            P, X = W * (Q @ K.T), W * (Y @ V.T)
            Pe, Xe = We * np.outer(norm(Q), norm(K)), We * np.outer(norm(Y), norm(V))
            out['dq'][b, h] = scale * (X @ K + c[:, None] * (Y @ S0.T))
            tol['dq'][b, h] = scale * (Xe @ np.abs(K) + ce[:, None] * np.outer(norm(Y), norm(S0)))
            out['dk'][b, h // G] += scale * X.T @ Q + e[:, None] * (V @ G1.T)
            tol['dk'][b, h // G] += scale * Xe.T @ np.abs(Q) + ee[:, None] * np.outer(norm(V), norm(G1))
            out['dv'][b, h // G] += scale * P.T @ Y + e[:, None] * (K @ G1)
            tol['dv'][b, h // G] += scale * Pe.T @ np.abs(Y) + ee[:, None] * np.outer(norm(K), norm(G1.T))
            out['dstate'][b, h] = scale * (Q * c[:, None]).T @ Y + f * G1
            tol['dstate'][b, h] = scale * np.abs(Q * ce[:, None]).T @ np.abs(Y) + fe * np.abs(G1)
    return out, tol


def recurrence(q, k, v, decay, scale, state, documents, lengths):
    """y and the last state of one head, position by position: the definition itself."""
    T, D = q.shape
    S = np.zeros((D, v.shape[1])) if state is None else state.copy()
    y = np.zeros((T, v.shape[1]))
    for t in range(T if lengths is None else min(max(lengths, 0), T)):
        if documents is not None and (documents[t] < 0 or (t > 0 and documents[t] != documents[t - 1])):
            S = np.zeros_like(S)
        if documents is None or documents[t] >= 0:
            S = decay * S + np.outer(k[t], v[t])
            y[t] = scale * S.T @ q[t]
    return y, S


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The token of one row, by its definition, in 64 bits."""
    x = logits.astype(np.float64)
    there = np.flatnonzero(x > -np.inf)
    if len(there) == 0:
        return -1
    order = there[np.argsort(-x[there], kind='stable')]
    if not temperature > 0:
        return int(order[0])
    top = x[order[0]]
    with np.errstate(invalid='ignore'):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / temperature))
    n = len(order)
    if top_k > 0:
        n = min(n, top_k)
    if top_p < 1:
        sums = np.cumsum(w[:n])
        n = 1 + int((sums[:n - 1] < top_p * sums[n - 1]).sum())
    n = max(1, min(n, int((w[:n] >= min_p).sum())))
    kept = np.sort(order[:n])
    weight = dict(zip(order[:n].tolist(), w[:n].tolist()))
    sums = np.cumsum([weight[i] for i in kept.tolist()])
    return int(kept[min(int((sums <= u * sums[-1]).sum()), n - 1)])

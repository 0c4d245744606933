"""The sequence operators in 64 bits, straight from their definitions, with bounds on what f32 arithmetic may differ by.

Bounds count roundings in units U = 2^-24, half a step of f32. A product of two values may be taken from operands split
into two 11-bit parts with the product of the low parts left out: each operand then keeps 22 bits (2^-22 = 4 U off at most)
and the lost product is another 4 U, 12 U in all. A sum of n terms in f32 is off by about sqrt(n) U of its terms' absolute
sum; 4 sqrt(n) U is allowed. A value's own last roundings (exp, log, tanh, a division) are 2 to 4 U each. A probability
below 2^-126, the smallest normal f32, may count as zero (the hardware's exp2 gives no subnormals): each pair may be off by
TINY = 2^-126, whatever its relative bound says."""
import numpy as np

U = 2.0 ** -24
TINY = 2.0 ** -126


def seen_mask(B, Tq, Tk, causal, slopes, documents, prefix, lengths):
    """[B, Tq, Tk] which keys a query sees, and the queries' positions [B, Tq]."""
    n = np.full(B, Tk) if lengths is None else np.clip(lengths, 0, Tk)
    p = n[:, None] - Tq + np.arange(Tq)
    j = np.arange(Tk)
    seen = np.broadcast_to(j < n[:, None, None], (B, Tq, Tk)).copy()
    if causal or slopes is not None or documents is not None:
        seen &= (p >= 0)[:, :, None]
    if causal:
        before = j[None, None, :] <= p[:, :, None]
        if prefix is not None:
            before = before | (j[None, None, :] < prefix[:, None, None])
        seen &= before
    if documents is not None:
        mine = np.take_along_axis(documents, np.maximum(p, 0), 1)
        seen &= (mine[:, :, None] == documents[:, None, :]) & (documents[:, None, :] >= 0)
    return seen, p


def attention(q, k, v, dy=None, causal=True, scale=None, softcap=None, slopes=None, documents=None, prefix=None, lengths=None):
    """{'y', 'dq', 'dk', 'dv'} and their bounds, of f32 inputs, in f64. Hidden pairs are left out by selection, so that
    nothing of them gets in."""
    with np.errstate(all='ignore'):
        return _attention(*(None if x is None else x.astype(np.float64) for x in (q, k, v, dy)), causal, scale, softcap, slopes,
                          documents, prefix, lengths)


def _attention(q, k, v, dy, causal, scale, softcap, slopes, documents, prefix, lengths):
    B, H, Tq, D = q.shape
    Hk, Tk, Dv = k.shape[1], k.shape[2], v.shape[3]
    g = H // Hk
    scale = 1 / np.sqrt(D) if scale is None else scale
    seen, p = seen_mask(B, Tq, Tk, causal, slopes, documents, prefix, lengths)
    names = ('y',) if dy is None else ('y', 'dq', 'dk', 'dv')
    like = {'y': (B, H, Tq, Dv), 'dq': q.shape, 'dk': k.shape, 'dv': v.shape}
    out = {n: np.zeros(like[n]) for n in names}
    tol = {n: np.zeros(like[n]) for n in names}
    pick = lambda m, x: np.where(m, x, 0.0)  # noqa: E731
    for b in range(B):
        m = seen[b]
        rows, cols = m.any(1), m.any(0)          # a row or column that takes no part is left out whole
        for h in range(H):
            Q, K, V = pick(rows[:, None], q[b, h]), pick(cols[:, None], k[b, h // g]), pick(cols[:, None], v[b, h // g])
            # pairs that are not seen may still hold what must not get in: every sum below selects by m
            x = pick(m, (Q @ K.T if np.isfinite(Q).all() and np.isfinite(K).all()
                         else np.stack([(Q[i] * K).sum(1) for i in range(Tq)]))) * scale
            t = np.tanh(x / softcap) if softcap else np.zeros_like(x)
            s = softcap * t if softcap else x
            far = np.abs(p[b][:, None] - np.arange(Tk))
            if slopes is not None:
                s = s - slopes[h] * far
            s = np.where(m, s, -np.inf)
            top = np.where(rows, s.max(1, initial=-np.inf), 0.0)[:, None]
            e = pick(m, np.exp(s - top))
            P = e / np.where(rows, e.sum(1), 1.0)[:, None]
            norm = lambda z: np.linalg.norm(z, axis=1)  # noqa: E731
            e_s = pick(m, (12 + 4 * np.sqrt(D)) * U * scale * norm(Q)[:, None] * norm(K)[None]
                       + 6 * U * np.abs(pick(m, s)) + (0 if slopes is None else 4 * U * abs(slopes[h]) * far)
                       + (4 * U * softcap * np.abs(t) if softcap else 0))
            R = (2 * e_s.max(1) + (20 + 8 * np.sqrt(Tk)) * U)[:, None]
            vis = lambda w, z: np.stack([(w[i][m[i], None] * z[m[i]]).sum(0) for i in range(w.shape[0])])  # noqa: E731
            y = vis(P, V)
            out['y'][b, h] = y
            tol['y'][b, h] = R * vis(P, np.abs(V)) + TINY * vis(m, np.abs(V))
            if dy is None:
                continue
            G = pick(rows[:, None], dy[b, h])
            dP = pick(m, np.stack([(G[i] * V).sum(1) for i in range(Tq)]))
            Di = (G * y).sum(1)[:, None]
            fac = 1 - t * t
            ds = pick(m, P * (dP - Di) * fac)
            e_dp = (pick(m, (12 + 4 * np.sqrt(Dv)) * U * norm(G)[:, None] * norm(V)[None])
                    + ((np.abs(G) * tol['y'][b, h]).sum(1) + 4 * np.sqrt(Dv) * U * norm(G) * norm(y))[:, None])
            e_ds = pick(m, TINY * np.abs(dP - Di) * fac + P * ((R + 8 * U) * np.abs(dP - Di) * fac + e_dp * fac
                                + (np.abs(dP - Di) * (4 * U + 2 * np.abs(t) * (e_s / softcap if softcap else 0)))))
            out['dq'][b, h] = scale * vis(ds, K)
            tol['dq'][b, h] = scale * (vis(e_ds, np.abs(K)) + (16 + 4 * np.sqrt(Tk)) * U * vis(np.abs(ds), np.abs(K)))
            mt = m.T
            visT = lambda w, z: np.stack([(w[mt[j], j][:, None] * z[mt[j]]).sum(0) for j in range(Tk)])  # noqa: E731
            n = (16 + 4 * np.sqrt(Tq * g)) * U
            out['dk'][b, h // g] += scale * visT(ds, Q)
            tol['dk'][b, h // g] += scale * (visT(e_ds, np.abs(Q)) + n * visT(np.abs(ds), np.abs(Q)))
            out['dv'][b, h // g] += visT(P, G)
            tol['dv'][b, h // g] += (R.max() + n) * visT(P, np.abs(G)) + TINY * visT(m, np.abs(G))
    return out, tol


def rope_axes(x, positions, sections, base=10000.0, per_axis=False, inverse=False):
    """y and its bound: the angle is exact to 64 bits, cosine and sine are 4 U off at most (their range reduction included),
    the two products and their sum 3 U."""
    half = sum(sections)
    y = x.astype(np.float64).copy()
    tol = np.zeros_like(y)
    p = 0
    for a, n in enumerate(sections):
        for r in range(n):
            w = positions[a].astype(np.float64) * base ** -(r / n if per_axis else p / half)
            c, s = np.cos(w)[:, None], np.sin(w)[:, None] * (-1 if inverse else 1)
            x1, x2 = x[..., p].astype(np.float64), x[..., p + half].astype(np.float64)
            y[..., p], y[..., p + half] = x1 * c - x2 * s, x2 * c + x1 * s
            tol[..., p] = tol[..., p + half] = 7 * U * (np.abs(x1) + np.abs(x2))
            p += 1
    return y, tol


def recurrence(a, x, h0=None, dh=None):
    """{'h', 'da', 'dx', 'dh0'} and bounds. A step rounds its product and its sum (2 U of each); an error made at t reaches
    t' through the gates between, as the value does, so the bound follows the recurrence itself on absolute values. Joining
    spans (products of gates) rounds each span's gates again: 4 U a step more, counted by the same recurrence."""
    a, x = a.astype(np.float64), x.astype(np.float64)
    B, T, C = a.shape
    first = np.zeros((B, C)) if h0 is None else h0.astype(np.float64)
    h, mag = np.zeros_like(a), np.zeros_like(a)
    err = np.zeros_like(a)
    b, e, w = first, np.zeros((B, C)), np.abs(first)
    for t in range(T):
        w = np.abs(a[:, t]) * w + np.abs(x[:, t])
        b = a[:, t] * b + x[:, t]
        e = np.abs(a[:, t]) * e + 8 * U * w
        h[:, t], err[:, t], mag[:, t] = b, e, w
    out, tol = {'h': h}, {'h': err}
    if dh is None:
        return out, tol
    dh = dh.astype(np.float64)
    g, ge = np.zeros_like(a), np.zeros_like(a)
    c, e, w = np.zeros((B, C)), np.zeros((B, C)), np.zeros((B, C))
    for t in reversed(range(T)):
        w = w + np.abs(dh[:, t])
        g[:, t] = dh[:, t] + c
        e = e + 8 * U * w
        ge[:, t] = e
        c, w, e = a[:, t] * g[:, t], np.abs(a[:, t]) * w, np.abs(a[:, t]) * e
    before = np.concatenate([first[:, None], h[:, :-1]], 1)
    berr = np.concatenate([np.zeros((B, 1, C)), err[:, :-1]], 1)
    out.update(dx=g, da=g * before)
    tol.update(dx=ge, da=ge * np.abs(before) + np.abs(g) * berr + 2 * U * np.abs(g * before))
    if h0 is not None:
        out['dh0'], tol['dh0'] = c, e + 2 * U * np.abs(c)
    return out, tol


def check(got, want, tol, what=''):
    """Every element within its bound (and a hair for results next to zero); none of it NaN."""
    assert got.shape == want.shape, what
    off = np.abs(got.astype(np.float64) - want)
    bad = ~(off <= tol + 1e-37)
    if bad.any():
        at = tuple(int(i) for i in np.argwhere(bad)[0])
        raise AssertionError(f'{what}: {int(bad.sum())} of {bad.size} values out of bounds, first at {at}: {got[at]} for '
                             f'{want[at]}, off {off[at]:.3g}, bound {tol[at]:.3g}')

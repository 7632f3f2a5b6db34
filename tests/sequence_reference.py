"""Plain 64-bit forms of the sequence-block operators, token by token and row by row, for the tests."""
import numpy as np


def lengths_of(lengths, T, B):
    if lengths is None:
        return np.full(B, T)
    f = np.asarray(lengths, np.float64)
    f = np.where(np.isnan(f), 0, f)
    return np.clip(np.trunc(f), 0, T).astype(int)


def attention(q, k, v, decay, scale=1.0, state=None, lengths=None):
    """(out, state_out) of the recurrence."""
    q, k, v, decay = (np.asarray(a, np.float64) for a in (q, k, v, decay))
    T, B, H, dk = q.shape
    g, dv = H // k.shape[2], v.shape[-1]
    k, v = np.repeat(k, g, 2), np.repeat(v, g, 2)
    S = np.zeros((B, H, dk, dv)) if state is None else np.asarray(state, np.float64).copy()
    out = np.zeros((T, B, H, dv))
    n = lengths_of(lengths, T, B)
    for b in range(B):
        for t in range(n[b]):
            S[b] = decay[:, None, None] * S[b] + k[t, b][:, :, None] * v[t, b][:, None, :]
            out[t, b] = scale * np.einsum('hd,hde->he', q[t, b], S[b])
    return out, S


def attention_backward(q, k, v, decay, dout, scale=1.0, state=None, dstate_out=None, lengths=None):
    """(dq, dk, dv, dstate) by going through the recurrence backwards."""
    q, k, v, decay, dout = (np.asarray(a, np.float64) for a in (q, k, v, decay, dout))
    T, B, H, dk = q.shape
    K = k.shape[2]
    g, dv = H // K, v.shape[-1]
    k, v = np.repeat(k, g, 2), np.repeat(v, g, 2)
    n = lengths_of(lengths, T, B)
    dq, dkk, dvv = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
    R = np.zeros((B, H, dk, dv)) if dstate_out is None else np.asarray(dstate_out, np.float64).copy()
    for b in range(B):
        S = np.zeros((H, dk, dv)) if state is None else np.asarray(state, np.float64)[b].copy()
        for t in range(n[b]):
            S = decay[:, None, None] * S + k[t, b][:, :, None] * v[t, b][:, None, :]
            dq[t, b] = scale * np.einsum('he,hde->hd', dout[t, b], S)
        for t in reversed(range(n[b])):
            M = R[b] + scale * q[t, b][:, :, None] * dout[t, b][:, None, :]
            dkk[t, b] = np.einsum('hde,he->hd', M, v[t, b])
            dvv[t, b] = np.einsum('hde,hd->he', M, k[t, b])
            R[b] = decay[:, None, None] * M
    shared = lambda a: a.reshape(T, B, K, g, a.shape[-1]).sum(3)  # noqa: E731
    return dq, shared(dkk), shared(dvv), R


ACT = {'sigmoid': lambda x: 1 / (1 + np.exp(-x)), 'tanh': np.tanh, 'rel': lambda x: np.maximum(x, 0),
       'el': lambda x: np.where(x > 0, x, np.expm1(np.minimum(x, 0))), 'linear': lambda x: x}
ACT_DERIV = {'sigmoid': lambda a: a * (1 - a), 'tanh': lambda a: 1 - a * a, 'rel': lambda a: (a > 0) * 1.0,
             'el': lambda a: np.where(a > 0, 1.0, a + 1), 'linear': np.ones_like}


def gated_norm(x, y, gate, w_post, scale, w_pre, eps=1e-6, act='sigmoid', want_h=True):
    """dict of x_out, h_out, r_post, r_pre."""
    d = lambda a: None if a is None else np.asarray(a, np.float64)  # noqa: E731
    x, y, gate, w_post, scale, w_pre = map(d, (x, y, gate, w_post, scale, w_pre))
    o = {'x_out': x}
    if y is not None:
        o['r_post'] = 1 / np.sqrt((y * y).mean(1) + eps)
        n = y * o['r_post'][:, None] * (1 if w_post is None else w_post)
        o['x_out'] = x + (1 if scale is None else scale) * (1 if gate is None else ACT[act](gate)) * n
    if want_h:
        o['r_pre'] = 1 / np.sqrt((o['x_out'] ** 2).mean(1) + eps)
        o['h_out'] = o['x_out'] * o['r_pre'][:, None] * (1 if w_pre is None else w_pre)
    return o


def gated_norm_backward(x_out, y, gate, w_post, scale, w_pre, r_post, r_pre, dx_out, dh, act='sigmoid'):
    """dict of dx, dy, dgate, dw_post, dscale, dw_pre (those that exist)."""
    d = lambda a: None if a is None else np.asarray(a, np.float64)  # noqa: E731
    x_out, y, gate, w_post, scale, w_pre, r_post, r_pre, dx_out, dh = map(
        d, (x_out, y, gate, w_post, scale, w_pre, r_post, r_pre, dx_out, dh))
    G, o = (0 if dx_out is None else dx_out), {}
    if dh is not None:
        r = r_pre[:, None]
        xh, e = x_out * r, dh * (1 if w_pre is None else w_pre)
        G = G + r * (e - xh * (e * xh).mean(1, keepdims=True))
        o['dw_pre'] = (dh * xh).sum(0)
    o['dx'] = G
    if y is not None:
        r, w, s = r_post[:, None], 1 if w_post is None else w_post, 1 if scale is None else scale
        yh, a = y * r, 1 if gate is None else ACT[act](gate)
        o['dscale'] = (G * a * yh * w).sum(0)
        if gate is not None:
            o['dgate'] = G * s * yh * w * ACT_DERIV[act](a)
        o['dw_post'] = (G * s * a * yh).sum(0)
        e = G * s * a * w
        o['dy'] = r * (e - yh * (e * yh).mean(1, keepdims=True))
    return o


def muon(param, grad, momentum, rate, beta, nesterov, weight_decay, steps):
    """(param, momentum, update)."""
    param, grad, momentum = (np.asarray(a, np.float64) for a in (param, grad, momentum))
    momentum = beta * momentum + grad
    u = grad + beta * momentum if nesterov else momentum
    update = np.empty_like(u)
    for i in np.ndindex(u.shape[:-2]):
        X = u[i] / (np.sqrt((u[i] ** 2).sum()) + 1e-7)
        for _ in range(steps):
            A = X @ X.T if X.shape[0] <= X.shape[1] else None
            if A is not None:
                X = 3.4445 * X + (-4.7750 * A + 2.0315 * A @ A) @ X
            else:
                A = X.T @ X
                X = 3.4445 * X + X @ (-4.7750 * A + 2.0315 * A @ A)
        update[i] = X
    return (1 - rate * weight_decay) * param - rate * update, momentum, update

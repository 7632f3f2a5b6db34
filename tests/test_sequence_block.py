"""The sequence-block operators together, as a model would use them: the norm before a block, projections, decayed linear
attention, the projection back, gate, residual and the norms around it, the gradients of all of it, and the
orthogonalised update of the weight matrices; then the same weights answer token by token.

The yardstick is the same step in 64 bits.  Tolerance: the operators' own errors are below 1e-6 of the sums of absolute
values they form (see their tests), the projections' below 1e-5 (the GEMM's bar); a chain of ten of them, each with a
gain near one, stays below 1e-4 of the largest value of the array compared.  The update's singular values amplify what
reaches them by up to 3.4445^5 in the directions the gradient hardly has, against sqrt(m) in its norm: 1e-2.
"""
import numpy as np
import pytest

import sequence_reference as ref

T, B, H, DK, DV, D = 70, 3, 4, 16, 24, 48
SCALE, EPS, RATE = DK ** -0.5, 1e-6, 0.05


def _weights(rs):
    f = lambda *s: (rs.standard_normal(s) / np.sqrt(s[-1])).astype(np.float32)  # noqa: E731
    w = {'q': f(H * DK, D), 'k': f(H * DK, D), 'v': f(H * DV, D), 'g': f(D, D), 'o': f(D, H * DV)}
    w |= {n: (1 + 0.1 * rs.standard_normal(D)).astype(np.float32) for n in ('pre', 'post', 'next')}
    w['scale'] = (0.5 + 0.1 * rs.standard_normal(D)).astype(np.float32)
    return w


def _step64(x, w, decay, state, lengths, dx2, dh2):
    """Outputs and gradients of one block in 64 bits."""
    x, w = x.astype(np.float64), {k: v.astype(np.float64) for k, v in w.items()}
    N = T * B
    first = ref.gated_norm(x, None, None, None, None, w['pre'], EPS)
    h = first['h_out']
    q, k, v, g = (h @ w[n].T for n in 'qkvg')
    q4, k4, v4 = q.reshape(T, B, H, DK), k.reshape(T, B, H, DK), v.reshape(T, B, H, DV)
    out, s_out = ref.attention(q4, k4, v4, decay, SCALE, state, lengths)
    a = out.reshape(N, H * DV)
    y = a @ w['o'].T
    post = ref.gated_norm(x, y, g, w['post'], w['scale'], w['next'], EPS, 'sigmoid')
    b = ref.gated_norm_backward(post['x_out'], y, g, w['post'], w['scale'], w['next'], post['r_post'], post['r_pre'], dx2, dh2, 'sigmoid')
    da = b['dy'] @ w['o']
    dq, dk, dv, _ = ref.attention_backward(q4, k4, v4, decay, da.reshape(T, B, H, DV), SCALE, state, None, lengths)
    dq, dk, dv = dq.reshape(N, -1), dk.reshape(N, -1), dv.reshape(N, -1)
    dh = dq @ w['q'] + dk @ w['k'] + dv @ w['v'] + b['dgate'] @ w['g']
    f = ref.gated_norm_backward(x, None, None, None, None, w['pre'], None, first['r_pre'], b['dx'], dh)
    grads = {'q': dq.T @ h, 'k': dk.T @ h, 'v': dv.T @ h, 'g': b['dgate'].T @ h, 'o': b['dy'].T @ a, 'pre': f['dw_pre'], 'post': b['dw_post'],
             'next': b['dw_pre'], 'scale': b['dscale'], 'x': f['dx']}
    return {'x_out': post['x_out'], 'h_out': post['h_out'], 'state': s_out}, grads


class _Block(object):
    """The same with handler calls on arrays that stay where they are."""

    def __init__(self, h, w, decay, state, lengths):
        self.h, N = h, T * B
        self.w = {k: h.create_from_numpy(v) for k, v in w.items()}
        self.decay, self.state, self.lengths = (h.create_from_numpy(a) for a in (decay, state, lengths))
        z = lambda *s: h.zeros(s)  # noqa: E731
        self.x, self.dx2, self.dh2 = z(N, D), z(N, D), z(N, D)
        self.h1, self.r1, self.r2, self.r3 = z(N, D), z(N), z(N), z(N)
        self.qkv = z(N, H * (2 * DK + DV))           # one hub, three views
        cols = [0, H * DK, 2 * H * DK, H * (2 * DK + DV)]
        self.parts = {n: self.qkv[:, a:b] for n, a, b in zip('qkv', cols, cols[1:])}
        self.dqkv = z(N, H * (2 * DK + DV))
        self.dparts = {n: self.dqkv[:, a:b] for n, a, b in zip('qkv', cols, cols[1:])}
        self.g, self.a, self.y, self.s_out = z(N, D), z(N, H * DV), z(N, D), z(B, H, DK, DV)
        self.x_out, self.h_out = z(N, D), z(N, D)
        self.dx, self.dy, self.dg, self.da, self.dh1 = z(N, D), z(N, D), z(N, D), z(N, H * DV), z(N, D)
        self.grad = {k: z(*v.shape) for k, v in w.items()}
        self.momentum = {k: z(*v.shape) for k, v in w.items() if v.ndim == 2}
        self.update = {k: z(*v.shape) for k, v in w.items() if v.ndim == 2}

    def heads(self, a, d):
        return a.reshape((T, B, H, d))

    def gradients(self):
        h, w, p, dp = self.h, self.w, self.parts, self.dparts
        h.gated_norm_forward(self.x, None, None, None, None, w['pre'], None, self.h1, None, self.r1, epsilon=EPS)
        for n in 'qkv':
            h.dot_mm(self.h1, w[n], p[n], transb=True)
        h.dot_mm(self.h1, w['g'], self.g, transb=True)
        q, k, v = self.heads(p['q'], DK), self.heads(p['k'], DK), self.heads(p['v'], DV)
        h.linear_attention_forward(q, k, v, self.decay, self.heads(self.a, DV), scale=SCALE, state=self.state, state_out=self.s_out,
                                   lengths=self.lengths)
        h.dot_mm(self.a, w['o'], self.y, transb=True)
        h.gated_norm_forward(self.x, self.y, self.g, w['post'], w['scale'], w['next'], self.x_out, self.h_out, self.r2, self.r3, epsilon=EPS)
        for a in list(self.grad.values()) + [self.dx, self.dy, self.dg, self.dqkv, self.dh1]:
            h.fill(a, 0.0)
        G = self.grad
        h.gated_norm_backward(self.x_out, self.y, self.g, w['post'], w['scale'], w['next'], self.r2, self.r3, self.dx2, self.dh2, self.dx, self.dy,
                              self.dg, G['post'], G['scale'], G['next'])
        h.dot_mm(self.dy, w['o'], self.da)
        h.linear_attention_backward(q, k, v, self.decay, self.heads(self.da, DV), self.heads(dp['q'], DK), self.heads(dp['k'], DK),
                                    self.heads(dp['v'], DV), scale=SCALE, state=self.state, lengths=self.lengths)
        for n in 'qkv':
            h.dot_add_mm(dp[n], w[n], self.dh1)
            h.dot_mm(dp[n], self.h1, G[n], transa=True)
        h.dot_add_mm(self.dg, w['g'], self.dh1)
        h.dot_mm(self.dg, self.h1, G['g'], transa=True)
        h.dot_mm(self.dy, self.a, G['o'], transa=True)
        # the residual's gradient is in dx already: the norm before the block adds its own
        h.gated_norm_backward(self.x, None, None, None, None, w['pre'], None, self.r1, None, self.dh1, self.dx, None, None, None, None, G['pre'])

    def train(self):
        self.gradients()
        for n in self.momentum:
            self.h.muon_update(self.w[n], self.grad[n], self.momentum[n], self.update[n], RATE)
        for n in ('pre', 'post', 'next', 'scale'):
            self.h.mult_add_st(-RATE, self.grad[n], self.w[n])


def _close(got, want, rel, what):
    assert np.abs(got - want).max() <= rel * np.abs(want).max(), (what, float(np.abs(got - want).max() / np.abs(want).max()))


@pytest.fixture(scope='module')
def setting():
    from brainstorm_b200 import B200Handler
    rs = np.random.RandomState(3)
    w = _weights(rs)
    f = lambda *s: rs.standard_normal(s).astype(np.float32)  # noqa: E731
    return {'h': B200Handler(seed=0), 'w': w, 'x': f(T * B, D), 'dx2': f(T * B, D), 'dh2': f(T * B, D), 'state': f(B, H, DK, DV),
            'decay': np.float32([0.5, 0.9, 0.97, 0.999]), 'lengths': np.float32([T, 41, 0])}


def _block(s):
    b = _Block(s['h'], s['w'], s['decay'], s['state'], s['lengths'])
    for n in ('x', 'dx2', 'dh2'):
        s['h'].set_from_numpy(getattr(b, n), s[n])
    return b


@pytest.mark.gpu
def test_outputs_and_all_gradients(setting):
    s, b = setting, _block(setting)
    b.gradients()
    outs, grads = _step64(s['x'], s['w'], s['decay'], s['state'], s['lengths'], s['dx2'], s['dh2'])
    get = s['h'].get_numpy_copy
    for n, a in (('x_out', b.x_out), ('h_out', b.h_out), ('state', b.s_out)):
        _close(get(a), outs[n], 1e-4, n)
    for n, want in grads.items():
        _close(get(b.dx if n == 'x' else b.grad[n]), want, 1e-4, n)


@pytest.mark.gpu
def test_training_steps_recorded_and_not(setting):
    """Two updates call by call and two replays of a recording give the same bits, and the first is the 64-bit one."""
    s = setting
    get = s['h'].get_numpy_copy
    plain = _block(s)
    plain.train()
    _, grads = _step64(s['x'], s['w'], s['decay'], s['state'], s['lengths'], s['dx2'], s['dh2'])
    for n in plain.momentum:
        want, _, update = ref.muon(s['w'][n], grads[n], np.zeros_like(s['w'][n]), float(np.float32(RATE)), float(np.float32(0.95)), True, 0.0, 5)
        assert np.linalg.norm(get(plain.update[n]) - update) <= 1e-2 * np.linalg.norm(update), n
    plain.train()
    replayed = _block(s)
    replayed.train()                                   # once the ordinary way, which makes the library's own buffers
    replayed2 = _block(s)
    step = s['h'].record(replayed2.train)
    step.launch()
    step.launch()
    replayed.train()
    for n in s['w']:
        assert np.array_equal(get(plain.w[n]), get(replayed.w[n])), n
        assert np.array_equal(get(plain.w[n]), get(replayed2.w[n])), n
    step.release()


@pytest.mark.gpu
def test_answering_token_by_token_agrees_with_the_prompt(setting):
    s = setting
    h, get = s['h'], s['h'].get_numpy_copy
    b = _block(s)
    b.lengths = None
    b.gradients()
    want_x, want_s = get(b.x_out).reshape(T, B, D), get(b.s_out)
    z = lambda *shape: h.zeros(shape)  # noqa: E731
    state = h.create_from_numpy(s['state'])
    h1, q, k, v, g, a, y, x_out, h_out, r = z(B, D), z(B, H * DK), z(B, H * DK), z(B, H * DV), z(B, D), z(B, H * DV), z(B, D), z(B, D), z(B, D), z(B)
    x = b.x.reshape((T, B, D))
    r2 = z(B)
    for t in range(T):
        h.gated_norm_forward(x[t], None, None, None, None, b.w['pre'], None, h1, None, r, epsilon=EPS)
        for n, o in (('q', q), ('k', k), ('v', v), ('g', g)):
            h.dot_mm(h1, b.w[n], o, transb=True)
        h.linear_attention_step(q.reshape((B, H, DK)), k.reshape((B, H, DK)), v.reshape((B, H, DV)), b.decay, state, a.reshape((B, H, DV)), scale=SCALE)
        h.dot_mm(a, b.w['o'], y, transb=True)
        h.gated_norm_forward(x[t], y, g, b.w['post'], b.w['scale'], b.w['next'], x_out, h_out, r, r2, epsilon=EPS)
        _close(get(x_out), want_x[t], 1e-4, 'token %d' % t)
    _close(get(state), want_s, 1e-4, 'state')

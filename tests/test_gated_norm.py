"""The norms, gate and residual around a block through the handler against the plain form in 64 bits.

Tolerance.  With U = 2^-24: a mean of D squares rounds each square once and adds them up in at most D / threads + 10
steps, so 1 / rms is off by at most (E + 12) U of itself with E = 16 values for each thread; an output is a sum of
products of at most six factors, each of which is rounded once (activations: at most 4 U and, through the argument of
exp and the subtraction in 1 - a^2, 4 U of one), with at most four sums, and the two means enter once each.  So
|error| <= 80 U (the same sum with absolute values).  r_pre is a function of the x_out that was formed: where x and the
gated norm nearly cancel, x_out is off by far more than its own rounding, by e = 80 U (|x| + |x_out - x|) as any output
is, and r(x_out) = (mean(x_out^2) + eps)^(-1/2) has the derivative -r^3 mean(x_out dx_out): r_pre is off by at most r^3
mean((|x_out| + e) e) more (e^2 bounds the second order), and h_out by |x_out w_pre| times that.  A column sum over N rows adds to that at most N / blocks + blocks
roundings: (80 + N) U of the sum of absolute values.
"""
import numpy as np
import pytest

import sequence_reference as ref

U = 2.0 ** -24


def _case(N, D, seed=0, gate=True, weights=True):
    rs = np.random.RandomState(seed)
    f = lambda *s: rs.standard_normal(s).astype(np.float32)  # noqa: E731
    d = {'x': f(N, D), 'y': 3 * f(N, D), 'gate': f(N, D), 'w_post': 1 + f(D) / 4, 'scale': f(D), 'w_pre': 1 + f(D) / 4, 'dx_out': f(N, D), 'dh': f(N, D)}
    if not gate:
        d['gate'] = None
    if not weights:
        d['w_post'] = d['scale'] = d['w_pre'] = None
    return d


def _forward(h, d, act, eps=1e-6, post=True, pre=True):
    N, D = d['x'].shape
    up = {k: None if v is None else h.create_from_numpy(v) for k, v in d.items()}
    o = {'x_out': h.zeros((N, D)), 'h_out': h.zeros((N, D)), 'r_post': h.zeros((N,)), 'r_pre': h.zeros((N,))}
    h.gated_norm_forward(up['x'], up['y'] if post else None, up['gate'] if post else None, up['w_post'], up['scale'], up['w_pre'],
                         o['x_out'] if post else None, o['h_out'] if pre else None, o['r_post'], o['r_pre'], epsilon=eps, activation=act)
    return up, o


def _backward(h, up, o, act, post=True, pre=True, accumulate=False, fill=0.0):
    N, D = up['x'].shape
    g = {n: h.zeros((N, D)) for n in ('dx', 'dy', 'dgate')}
    g |= {n: h.zeros((D,)) for n in ('dw_post', 'dscale', 'dw_pre')}
    for a in g.values():
        h.fill(a, fill)
    gated = post and up['gate'] is not None
    h.gated_norm_backward((o['x_out'] if post else up['x']) if pre else None, up['y'] if post else None, up['gate'] if gated else None, up['w_post'], up['scale'],
                          up['w_pre'], o['r_post'] if post else None, o['r_pre'] if pre else None, up['dx_out'], up['dh'] if pre else None, g['dx'],
                          g['dy'] if post else None, g['dgate'] if gated else None, g['dw_post'] if post else None, g['dscale'] if post else None,
                          g['dw_pre'] if pre else None, activation=act, accumulate=accumulate)
    return g


def _magnitudes(d, o, act, post, pre):
    """Sums of absolute values along the formulas."""
    a = lambda v: None if v is None else np.abs(np.asarray(v, np.float64))  # noqa: E731
    one = lambda v: 1 if v is None else a(v)  # noqa: E731
    m, G = {}, a(d['dx_out'])
    if pre:
        r, xh = o['r_pre'][:, None], a(o['x_out']) * o['r_pre'][:, None]
        e = a(d['dh']) * one(d['w_pre'])
        G = G + r * (e + xh * (e * xh).mean(1, keepdims=True))
        m['dw_pre'] = (a(d['dh']) * xh).sum(0)
    m['dx'] = G
    if post:
        r, yh = o['r_post'][:, None], a(d['y']) * o['r_post'][:, None]
        act_a = 1 if d['gate'] is None else np.abs(ref.ACT[act](d['gate'].astype(np.float64))) + 0.05
        m['dscale'] = (G * act_a * yh * one(d['w_post'])).sum(0)
        if d['gate'] is not None:
            m['dgate'] = G * one(d['scale']) * yh * one(d['w_post'])
        m['dw_post'] = (G * one(d['scale']) * act_a * yh).sum(0)
        e = G * one(d['scale']) * act_a * one(d['w_post'])
        m['dy'] = r * (e + yh * (e * yh).mean(1, keepdims=True))
    return m


def _check(h, d, act, post=True, pre=True, eps=1e-6):
    up, o = _forward(h, d, act, eps, post, pre)
    got = {k: h.get_numpy_copy(v).astype(np.float64) for k, v in o.items()}
    want = ref.gated_norm(d['x'], d['y'] if post else None, d['gate'], d['w_post'], d['scale'], d['w_pre'], eps, act, pre)
    size = {k: np.abs(v) for k, v in want.items()}
    size['x_out'] = np.abs(d['x']).astype(np.float64)
    if post:
        size['x_out'] = size['x_out'] + np.abs(want['x_out'] - d['x'])
    if pre:
        w, e = 1 if d['w_pre'] is None else np.abs(d['w_pre']), 80 * U * size['x_out']
        size['h_out'] = size['x_out'] * want['r_pre'][:, None] * w
    bound = {k: 80 * U * v for k, v in size.items()}
    if pre and post:
        x = np.abs(want['x_out'])
        off = want['r_pre'] ** 3 * ((x + e) * e).mean(1)
        bound['r_pre'] = bound['r_pre'] + off
        bound['h_out'] = bound['h_out'] + x * w * off[:, None]
    for k in want:
        if k == 'x_out' and not post:
            continue
        assert (np.abs(got[k] - want[k]) <= bound[k] + 1e-37).all(), k
    g = {k: h.get_numpy_copy(v).astype(np.float64) for k, v in _backward(h, up, o, act, post, pre).items()}
    # the backward formula at the forward pass's own float32 results
    f = {k: got[k] for k in ('x_out', 'r_post', 'r_pre')}
    if not post:
        f['x_out'] = d['x'].astype(np.float64)
    wants = ref.gated_norm_backward(f['x_out'] if pre else None, d['y'] if post else None, d['gate'], d['w_post'], d['scale'], d['w_pre'], f['r_post'],
                                    f['r_pre'], d['dx_out'], d['dh'] if pre else None, act)
    sizes = _magnitudes(d, f, act, post, pre)
    N = d['x'].shape[0]
    for k, m in sizes.items():
        terms = 80 + (N if k in ('dw_post', 'dscale', 'dw_pre') else 0)
        err = np.abs(g[k] - wants[k])
        assert (err <= terms * U * m + 1e-37).all(), (k, float((err / (terms * U * m + 1e-37)).max()))


# one value, one row, widths at and off the vector and thread borders, the widest row, more rows than blocks
SHAPES = [(1, 1), (3, 2), (1, 31), (7, 32), (5, 33), (4, 127), (9, 128), (2, 129), (300, 130), (3, 256), (3, 260), (17, 511), (700, 512), (11, 513), (33, 1000),
          (5, 1024), (6, 1537), (400, 2048), (3, 4096), (2, 4097), (2, 8191), (3, 12000), (2, 16384), (310, 16383),
          (3000, 125), (3000, 126), (4000, 128), (5000, 33), (2500, 129), (2500, 253), (2500, 254), (1300, 509), (1300, 1021), (900, 1022), (900, 2045), (700, 2047), (700, 4093), (301, 4094)]


@pytest.fixture(scope='module')
def handler():
    from brainstorm_b200 import B200Handler
    return B200Handler(seed=0)


@pytest.mark.gpu
@pytest.mark.parametrize('shape', SHAPES)
def test_forward_and_gradients(handler, shape):
    _check(handler, _case(*shape, seed=shape[1]), 'sigmoid')


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(700, 1000), (593, 1000), (600, 1021), (1190, 510), (1300, 333), (610, 1537), (300, 2044), (300, 2045), (3, 2046), (3, 4093), (3, 4094), (3, 4799),
                                   (3, 4801), (160, 5001), (2, 8189), (2, 8190), (3, 4096), (600, 4096), (2500, 129), (3000, 17), (6000, 64), (2500, 50), (700, 32),
                                   (4000, 1)])
def test_around_the_limits_of_the_forms(handler, shape):
    """Few rows and many, widths that fill 256, 512 or 1024 threads."""
    _check(handler, _case(*shape, seed=shape[0]), 'sigmoid')


@pytest.mark.gpu
@pytest.mark.parametrize('act', sorted(ref.ACT))
@pytest.mark.parametrize('shape', [(13, 40), (5, 555)])
def test_activations(handler, act, shape):
    _check(handler, _case(*shape, seed=1), act)


@pytest.mark.gpu
@pytest.mark.parametrize('post, pre', [(True, False), (False, True)])
@pytest.mark.parametrize('gate', [True, False])
@pytest.mark.parametrize('weights', [True, False])
@pytest.mark.parametrize('shape', [(9, 64), (5, 301)])
def test_first_and_last_norm_and_parts_left_out(handler, shape, post, pre, gate, weights):
    _check(handler, _case(*shape, seed=2, gate=gate and post, weights=weights), 'tanh', post, pre)


@pytest.mark.gpu
@pytest.mark.parametrize('weights', [True, False])
@pytest.mark.parametrize('gate', [True, False])
def test_parts_left_out(handler, gate, weights):
    _check(handler, _case(21, 200, seed=3, gate=gate, weights=weights), 'sigmoid')


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(6, 48), (5, 37)])
def test_strided_rows_and_in_place(handler, shape):
    h, (N, D) = handler, shape
    d = _case(N, D, seed=4)
    up, o = _forward(h, d, 'sigmoid')
    want = {k: h.get_numpy_copy(v) for k, v in o.items()}
    g = {k: h.get_numpy_copy(v) for k, v in _backward(h, up, o, 'sigmoid').items()}
    hub = h.zeros((N, 3 * D + 5))
    views = {k: hub[:, i * D + i:(i + 1) * D + i] for i, k in enumerate(('x', 'y', 'gate'))}
    for k, a in views.items():
        h.set_from_numpy(a, d[k])
    res = h.zeros((N, 2 * D + 1))
    h.gated_norm_forward(views['x'], views['y'], views['gate'], up['w_post'], up['scale'], up['w_pre'], res[:, :D], res[:, D + 1:], o['r_post'], o['r_pre'])
    close = lambda a, b: (np.abs(a.astype(np.float64) - b) <= 160 * U * (np.abs(b) + np.abs(b).max())).all()  # noqa: E731  (sums in another order)
    assert close(h.get_numpy_copy(res[:, :D]), want['x_out']) and close(h.get_numpy_copy(res[:, D + 1:]), want['h_out'])
    assert not h.get_numpy_copy(res[:, D:D + 1]).any()
    # x_out over x, h_out over y; dx over dx_out
    h.gated_norm_forward(up['x'], up['y'], up['gate'], up['w_post'], up['scale'], up['w_pre'], up['x'], up['y'], o['r_post'], o['r_pre'])
    assert np.array_equal(h.get_numpy_copy(up['x']), want['x_out']) and np.array_equal(h.get_numpy_copy(up['y']), want['h_out'])
    y, dy, dgate = h.create_from_numpy(d['y']), h.zeros((N, D)), h.zeros((N, D))
    h.gated_norm_backward(up['x'], y, up['gate'], up['w_post'], up['scale'], up['w_pre'], o['r_post'], o['r_pre'], up['dx_out'], up['dh'], up['dx_out'], dy,
                          dgate, None, None, None, accumulate=False)
    for a, k in ((up['dx_out'], 'dx'), (dy, 'dy'), (dgate, 'dgate')):
        assert np.array_equal(h.get_numpy_copy(a), g[k]), k


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(40, 64), (7, 99)])
def test_gradients_are_added(handler, shape):
    h, d = handler, _case(*shape, seed=5)
    up, o = _forward(h, d, 'sigmoid')
    once = {k: h.get_numpy_copy(v) for k, v in _backward(h, up, o, 'sigmoid').items()}
    more = {k: h.get_numpy_copy(v) for k, v in _backward(h, up, o, 'sigmoid', accumulate=True, fill=1.0).items()}
    for k in once:
        assert np.abs(more[k] - (once[k].astype(np.float64) + 1)).max() <= U * (np.abs(once[k]).max() + 1), k


@pytest.mark.gpu
def test_gradients_against_differences(handler):
    """Central differences of the 64-bit forward pass."""
    h, act = handler, 'sigmoid'
    d = _case(6, 24, seed=6)
    up, o = _forward(h, d, act)
    g = {k: h.get_numpy_copy(v).astype(np.float64) for k, v in _backward(h, up, o, act).items()}
    rs = np.random.RandomState(7)
    for name in ('x', 'y', 'gate', 'w_post', 'scale', 'w_pre'):
        way = rs.standard_normal(d[name].shape)

        def loss(e):
            x = dict(d)
            x[name] = d[name] + e * way
            f = ref.gated_norm(x['x'], x['y'], x['gate'], x['w_post'], x['scale'], x['w_pre'], 1e-6, act)
            return (f['x_out'] * d['dx_out']).sum() + (f['h_out'] * d['dh']).sum()
        e = 1e-4       # the difference is off by about e^2 of the terms, the gradients by 100 U
        slope = (loss(e) - loss(-e)) / (2 * e)
        terms = g['d' + name] * way
        assert abs(terms.sum() - slope) <= 1e-5 * np.abs(terms).sum() + 1e-5, name


@pytest.mark.gpu
def test_zero_rows_values_that_are_not_finite_and_no_rows(handler):
    h = handler
    d = _case(8, 70, seed=8)
    d['x'][1] = d['y'][1] = 0
    up, o = _forward(h, d, 'sigmoid')
    clean = {k: h.get_numpy_copy(v) for k, v in o.items()}
    assert np.isfinite(clean['h_out']).all() and not clean['h_out'][1].any()
    g = {k: h.get_numpy_copy(v) for k, v in _backward(h, up, o, 'sigmoid').items()}
    assert all(np.isfinite(v).all() for v in g.values())
    d['y'][3, 4] = np.nan
    d['x'][5, 6] = np.inf
    _, o = _forward(h, d, 'sigmoid')
    keep = [0, 1, 2, 4, 6, 7]
    assert np.array_equal(h.get_numpy_copy(o['h_out'])[keep], clean['h_out'][keep])
    z = lambda *s: h.ones(s)  # noqa: E731
    h.gated_norm_forward(z(0, 8), z(0, 8), None, None, None, None, z(0, 8), z(0, 8), z(0,), z(0,))
    sums = [z(8) for _ in range(3)]
    h.gated_norm_backward(z(0, 8), z(0, 8), None, None, None, None, z(0,), z(0,), None, z(0, 8), z(0, 8), z(0, 8), None, *sums, accumulate=True)
    assert all((h.get_numpy_copy(s) == 1).all() for s in sums)
    h.gated_norm_backward(z(0, 8), z(0, 8), None, None, None, None, z(0,), z(0,), None, z(0, 8), z(0, 8), z(0, 8), None, *sums, accumulate=False)
    assert all((h.get_numpy_copy(s) == 0).all() for s in sums)


@pytest.mark.gpu
def test_same_bits_every_time_and_when_replayed(handler):
    h = handler
    d = _case(900, 520, seed=9)
    up, o = _forward(h, d, 'sigmoid')
    first = {k: h.get_numpy_copy(v) for k, v in _backward(h, up, o, 'sigmoid').items()}
    g = {k: h.zeros(v.shape) for k, v in first.items()}

    def step():
        h.gated_norm_backward(o['x_out'], up['y'], up['gate'], up['w_post'], up['scale'], up['w_pre'], o['r_post'], o['r_pre'], up['dx_out'], up['dh'],
                              g['dx'], g['dy'], g['dgate'], g['dw_post'], g['dscale'], g['dw_pre'], accumulate=False)
    step()
    a, b = h.record(step), h.record(step)
    for r in (a, b, a):
        r.launch()
        step()
        r.launch()
        for k in first:
            assert np.array_equal(h.get_numpy_copy(g[k]), first[k]), k
    a.release()
    b.release()


def _shape(i, *shape):
    from brainstorm_b200 import B200Array
    return B200Array(None, (i + 1) << 20, tuple(shape))


def test_refusals():
    from brainstorm_b200.sequence_ops import SequenceOps
    h = SequenceOps()
    x, y, g, xo, ho = (_shape(i, 4, 8) for i in range(5))
    w, r, r2 = _shape(5, 8), _shape(6, 4), _shape(7, 4)
    def fwd(x=x, y=y, gate=g, w=w, xo=xo, ho=ho, r=r, **kw):  # noqa: E306
        return h.gated_norm_forward(x, y, gate, w, None, None, xo, ho, r, r2, **kw)
    for kw, text in (({'activation': 'relu'}, 'unknown activation'), ({'epsilon': -1.0}, 'epsilon'), ({'epsilon': float('nan')}, 'epsilon'),
                     ({'w': _shape(9, 7)}, 'w_post has 7'), ({'y': _shape(9, 4, 9)}, 'y has shape'), ({'r': _shape(9, 3)}, 'r_post has 3'),
                     ({'xo': None}, 'needs x_out'), ({'y': None}, 'nothing to gate'), ({'y': None, 'gate': None, 'ho': None}, 'h_out has to be given'),
                     ({'xo': y}, 'x_out overlaps y'), ({'ho': xo}, 'h_out overlaps x_out'), ({'x': _shape(9, 2, 4, 8)}, 'expected 2-D')):
        with pytest.raises(ValueError, match=text):
            fwd(**kw)
    with pytest.raises(NotImplementedError, match='column stride'):
        fwd(y=_shape(9, 4, 16)[:, ::2])
    def bwd(y=y, gate=g, xo=xo, dh=_shape(9, 4, 8), dgate=_shape(10, 4, 8), dy=_shape(11, 4, 8), dw_pre=None, r=r, dx=_shape(12, 4, 8)):  # noqa: E306
        return h.gated_norm_backward(xo, y, gate, w, None, None, r, r2, None, dh, dx, dy, dgate, None, None, dw_pre)
    for kw, text in (({'dgate': None}, 'needs dgate'), ({'dy': None}, 'needs r_post and dy'), ({'r': None}, 'needs r_post and dy'), ({'xo': None}, 'needs x_out'),
                     ({'dh': None, 'dw_pre': w}, 'dw_pre needs dh'), ({'y': None, 'dh': None}, 'nothing to differentiate'), ({'y': None}, 'there is no gate'),
                     ({'dx': y}, 'dx overlaps y'), ({'dx': _shape(11, 4, 8)}, 'dy overlaps dx')):
        with pytest.raises(ValueError, match=text):
            bwd(**kw)


@pytest.mark.gpu
def test_refusals_of_the_library(handler):
    from brainstorm_b200 import B200Error
    h, z = handler, lambda *s: handler.zeros(s)
    with pytest.raises(B200Error, match='16384'):
        h.gated_norm_forward(z(1, 16385), None, None, None, None, None, None, z(1, 16385), None, None)

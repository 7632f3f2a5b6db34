"""The gated norm's three ways through memory (single loads, 128-bit, 128-bit from the boundary before the row), each with
added gradients, in place and with row pitches, against the plain form in 64 bits.

Bounds: those of ``test_gated_norm`` for an overwritten gradient; adding it to what was there rounds the sum once more."""
import numpy as np
import pytest

import sequence_reference as ref
from test_gated_norm import U, _backward, _case, _forward, _magnitudes

# rows, width: up to 64 and 128 columns single, then multiples of four 128-bit and others from the boundary (widths near 4096 that
# leave too many threads idle are single again); few rows and more than the GPU holds at once, 256, 512 and 1024 threads a row
FORMS = [(40, 50), (700, 64), (30, 99), (900, 128), (30, 132), (3000, 256), (40, 1000), (900, 1000), (20, 2048), (300, 3000), (700, 4096), (12, 4096), (8, 8192), (5, 12000),
         (30, 129), (3000, 131), (40, 1021), (900, 1022), (20, 2045), (300, 2999), (700, 4093), (12, 5001), (160, 8189), (12, 4095), (6, 8191), (4, 16383)]


@pytest.fixture(scope='module')
def handler():
    from brainstorm_b200 import B200Handler
    return B200Handler(seed=0)


def _wants(d, o, act='sigmoid'):
    """(gradients in 64 bits at the forward pass's float32 results, bounds)."""
    f = {k: o[k].astype(np.float64) for k in ('x_out', 'r_post', 'r_pre')}
    want = ref.gated_norm_backward(f['x_out'], d['y'], d['gate'], d['w_post'], d['scale'], d['w_pre'], f['r_post'], f['r_pre'], d['dx_out'], d['dh'], act)
    N = d['x'].shape[0]
    bound = {k: (80 + (N if k in ('dw_post', 'dscale', 'dw_pre') else 0)) * U * m + 1e-37 for k, m in _magnitudes(d, f, act, True, True).items()}
    return want, bound


@pytest.mark.gpu
@pytest.mark.parametrize('accumulate', [False, True])
@pytest.mark.parametrize('shape', FORMS)
def test_dx_in_the_place_of_dx_out(handler, shape, accumulate):
    """The incoming gradient counts once, whether the other gradients are added or not."""
    h, (N, D) = handler, shape
    d = _case(N, D, seed=D)
    up, o = _forward(h, d, 'sigmoid')
    want, bound = _wants(d, {k: h.get_numpy_copy(v) for k, v in o.items()})
    dx, dy, dgate = up['dx_out'], h.ones((N, D)), h.ones((N, D))
    h.gated_norm_backward(o['x_out'], up['y'], up['gate'], up['w_post'], up['scale'], up['w_pre'], o['r_post'], o['r_pre'], dx, up['dh'], dx, dy, dgate, None, None,
                          None, accumulate=accumulate)
    assert (np.abs(h.get_numpy_copy(dx) - want['dx']) <= bound['dx']).all()
    for k, a in (('dy', dy), ('dgate', dgate)):
        whole = want[k] + (1 if accumulate else 0)
        assert (np.abs(h.get_numpy_copy(a) - whole) <= bound[k] + (U * (np.abs(whole) + bound[k]) if accumulate else 0)).all(), k


@pytest.mark.gpu
def test_dx_in_the_place_of_dx_out_without_a_norm_before_the_next_block(handler):
    """Then the gradient of x is that of x_out: added by default it would be doubled."""
    h, d = handler, _case(20, 260, seed=1)
    up, o = _forward(h, d, 'sigmoid', pre=False)
    dy, dgate = h.zeros((20, 260)), h.zeros((20, 260))
    h.gated_norm_backward(None, up['y'], up['gate'], up['w_post'], up['scale'], None, o['r_post'], None, up['dx_out'], None, up['dx_out'], dy, dgate, None, None, None)
    assert np.array_equal(h.get_numpy_copy(up['dx_out']), d['dx_out'])


@pytest.mark.gpu
@pytest.mark.parametrize('shape', FORMS)
def test_gradients_are_added(handler, shape):
    """The default: onto ones, vectors included."""
    h, d = handler, _case(*shape, seed=shape[0])
    up, o = _forward(h, d, 'sigmoid')
    want, bound = _wants(d, {k: h.get_numpy_copy(v) for k, v in o.items()})
    got = {k: h.get_numpy_copy(v) for k, v in _backward(h, up, o, 'sigmoid', accumulate=True, fill=1.0).items()}
    for k in want:
        assert (np.abs(got[k] - (want[k] + 1)) <= bound[k] + U * (np.abs(want[k] + 1) + bound[k])).all(), k


def _hub(h, rows, width, names, gap, start):
    """(hub full of sevens, views): column ranges with `gap` columns between them, from column `start` on."""
    pitch = start + len(names) * (width + gap)
    hub = h.zeros((rows, pitch))
    h.fill(hub, 7.0)
    return hub, {k: hub[:, start + i * (width + gap):start + i * (width + gap) + width] for i, k in enumerate(names)}


def _untouched(h, hub, views):
    """Whether the columns that no view holds are still sevens."""
    whole, free = h.get_numpy_copy(hub), np.ones(hub.shape[1], bool)
    for v in views.values():
        first = (v.ptr - hub.ptr) // 4
        free[first:first + v.shape[1]] = False
    return (whole[:, free] == 7).all()


def _check_forward(d, got):
    want = ref.gated_norm(d['x'], d['y'], d['gate'], d['w_post'], d['scale'], d['w_pre'])
    assert (np.abs(got['x_out'] - want['x_out']) <= 80 * U * (np.abs(d['x']) + np.abs(want['x_out'] - d['x']))).all()
    assert (np.abs(got['r_post'] - want['r_post']) <= 80 * U * want['r_post']).all()
    # the second norm as a function of the x_out that was formed
    again = ref.gated_norm(got['x_out'], None, None, None, None, d['w_pre'])
    for k in ('r_pre', 'h_out'):
        assert (np.abs(got[k] - again[k]) <= 80 * U * np.abs(again[k])).all(), k


# hubs whose columns let the 128-bit form through (start, gap and width multiples of four), the shifted one (all ranges start alike,
# with a pitch that is a multiple of four off the width), and neither
@pytest.mark.gpu
@pytest.mark.parametrize('accumulate', [False, True])
@pytest.mark.parametrize('shape, start, gap', [((40, 50), 3, 2), ((30, 128), 4, 8), ((30, 132), 8, 4), ((700, 1000), 4, 4), ((20, 4096), 4, 4), ((7, 8192), 0, 4),
                                               ((30, 129), 1, 3), ((600, 1021), 2, 3), ((700, 1021), 0, 7), ((12, 5001), 3, 3), ((30, 1000), 1, 4), ((25, 2045), 2, 3),
                                               ((30, 129), 0, 2), ((30, 132), 0, 1), ((12, 4095), 0, 1), ((300, 1021), 1, 1), ((4, 12000), 0, 3)])
def test_rows_with_a_pitch(handler, shape, start, gap, accumulate):
    h, (N, D) = handler, shape
    d = _case(N, D, seed=D + start)
    hub, v = _hub(h, N, D, ('x', 'y', 'gate', 'dx_out', 'dh'), gap, start)
    for k, a in v.items():
        h.set_from_numpy(a, d[k])
    w = {k: h.create_from_numpy(d[k]) for k in ('w_post', 'scale', 'w_pre')}
    res, out = _hub(h, N, D, ('x_out', 'h_out'), gap, start)
    r = {k: h.zeros((N,)) for k in ('r_post', 'r_pre')}
    h.gated_norm_forward(v['x'], v['y'], v['gate'], w['w_post'], w['scale'], w['w_pre'], out['x_out'], out['h_out'], r['r_post'], r['r_pre'])
    got = {k: h.get_numpy_copy(a) for k, a in {**out, **r}.items()}
    assert _untouched(h, res, out)
    _check_forward(d, got)
    grads, g = _hub(h, N, D, ('dx', 'dy', 'dgate'), gap, start)
    for a in g.values():
        h.fill(a, 1.0)
    g |= {k: h.ones((D,)) for k in ('dw_post', 'dscale', 'dw_pre')}
    h.gated_norm_backward(out['x_out'], v['y'], v['gate'], w['w_post'], w['scale'], w['w_pre'], r['r_post'], r['r_pre'], v['dx_out'], v['dh'], g['dx'], g['dy'],
                          g['dgate'], g['dw_post'], g['dscale'], g['dw_pre'], accumulate=accumulate)
    want, bound = _wants(d, got)
    one = 1.0 if accumulate else 0.0
    for k in want:
        whole = want[k] + one
        assert (np.abs(h.get_numpy_copy(g[k]) - whole) <= bound[k] + one * U * (np.abs(whole) + bound[k])).all(), k
    assert _untouched(h, grads, {k: g[k] for k in ('dx', 'dy', 'dgate')}) and _untouched(h, hub, v)


@pytest.mark.gpu
@pytest.mark.parametrize('pitched', [False, True])
@pytest.mark.parametrize('shape', FORMS)
def test_in_place(handler, shape, pitched):
    """x_out over x and h_out over y: the bits that other arrays get, or in a hub whose columns start alike the results to rounding."""
    h, (N, D) = handler, shape
    d = _case(N, D, seed=D)
    up, o = _forward(h, d, 'sigmoid')
    x, y, gate = up['x'], up['y'], up['gate']
    if pitched:
        _, v = _hub(h, N, D, ('x', 'y', 'gate'), 4 - D % 4, 1 if D % 4 else 0)
        for k, a in v.items():
            h.set_from_numpy(a, d[k])
        x, y, gate = v['x'], v['y'], v['gate']
    h.gated_norm_forward(x, y, gate, up['w_post'], up['scale'], up['w_pre'], x, y, o['r_post'], o['r_pre'])
    got = {k: h.get_numpy_copy(a) for k, a in (('x_out', x), ('h_out', y), ('r_post', o['r_post']), ('r_pre', o['r_pre']))}
    if pitched:
        _check_forward(d, got)
    else:
        _, apart = _forward(h, d, 'sigmoid')
        for k, a in apart.items():
            assert np.array_equal(got[k], h.get_numpy_copy(a)), k

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

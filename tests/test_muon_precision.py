"""The orthogonalised update to the precision of its products, in every form that they take.

Tolerance.  A product of two matrices that are held in 22 bits (each value off by at most 2^-22 of itself, and twice that
little for the product of the low parts that is left out) is off by at most d = 3 * 2^-22 of its size, with errors
of independent entries; the sums of a chunk truncate, a few steps of 2^-23 more: d <= 4 * 2^-22.  A step forms D = A + b / 2c I, whose
eigenvalues are within 1.18, then P = c D D + .. I, which is off by c (2 * 1.18 d + 1.18^2 d) <= 8 d beside eigenvalues between 0.64
and 3.45, then P X: 2-norm errors of about 8 d + d that the independence of the entries divides by more than the four by which the
bound takes them: 2.5 d = 10 * 2^-22 a step, of |update|_F.  An error grows by at most 3.4445 in a later step, as the small
singular values and with them |X|_F do, until most of them are near one: the bound for `steps` steps is steps * 10 * 2^-22, 1.2e-5 for
five.  Without one of the two cross products, or with half precision alone, the error is 1e-4 to 2e-3: twenty times the bound or more
(test_the_bound_needs_every_product).

X is held to 2^-25 / 4096 = 2^-37 at least, however small it is (where |u| is small beside the 1e-7 it is divided by: the update is small
then too).  Each of the steps + 1 times that it is formed, its rows x cols values are off by that much, which grows by at most 3.4445
a step: sqrt(rows cols) 2^-37 (1 + 3.4445 + .. + 3.4445^steps) <= FLOOR = 1.41 sqrt(rows cols) 2^-37 3.4445^steps more in all, 4e-8 to 1e-6 for the
shapes here beside updates of norm 1 to 30.
"""
import numpy as np
import pytest

import sequence_reference as ref

STEP = 10 * 2.0 ** -22
A, B, C = 3.4445, -4.7750, 2.0315


def _case(shape, seed=0, size=1.0):
    rs = np.random.RandomState(seed)
    f = lambda: (rs.standard_normal(shape) * size).astype(np.float32)  # noqa: E731
    return {'param': f(), 'grad': f(), 'momentum': f()}


def _update(h, d, steps):
    up = {k: h.create_from_numpy(v) for k, v in d.items()}
    update = h.ones(d['param'].shape)
    h.muon_update(up['param'], up['grad'], up['momentum'], update, 0.02, steps=steps)
    return h.get_numpy_copy(update).astype(np.float64)


def _errors(got, d, steps):
    """(Frobenius norm of the error, of the update, FLOOR), each matrix."""
    beta = float(np.float32(0.95))
    want = ref.muon(d['param'], d['grad'], d['momentum'], 0.02, beta, True, 0.0, steps)[2]
    norm = lambda a: np.sqrt((a ** 2).sum((-2, -1)))  # noqa: E731
    return norm(got - want), norm(want), 1.41 * np.sqrt(want.shape[-2] * want.shape[-1]) * 2.0 ** -37 * 3.4445 ** steps


def _check(got, d, steps):
    error, size, floor = _errors(got, d, steps)
    assert (error <= steps * STEP * size + floor).all(), float((error / (steps * STEP * size + floor)).max())


@pytest.fixture(scope='module')
def handler():
    from brainstorm_b200 import B200Handler
    return B200Handler(seed=0)


# The products D, P and X of a step each run in the form with the least waves on 148 SMs: tiles of 128 x 64, of 128 x 128, or of 256 x 256
# on pairs of SMs; symmetric ones are stored in blocks of 128 or 256.  Wide and tall, sizes off the tiles, one value along K
# behind a chunk.
SHAPES = [(1, 1), (3, 7), (16, 40), (65, 129), (205, 256), (256, 205), (1000, 17), (4, 130, 130),                      # one launch
          (17, 1000), (129, 700), (700, 129), (321, 450), (513, 640), (640, 513), (2, 300, 260),                      # 128 x 64 all
          (30, 210, 215), (40, 301, 163),                                                                             # 128 x 128 all
          (40, 165, 170), (40, 215, 165), (30, 193, 257), (4, 1000, 1000),                                            # 128 x 128, then pairs
          (20, 165, 390), (20, 395, 165),                                                                             # 128 x 64, then pairs
          (20, 165, 210), (40, 165, 120), (1500, 1290),                                                               # 128 x 64, then 128 x 128
          (20, 390, 395), (20, 435, 390), (20, 385, 513),                                                             # pairs all
          (6, 795, 800), (6, 840, 795)]                                                                               # pairs, then 128 x 128


@pytest.mark.gpu
@pytest.mark.parametrize('steps', [1, 5])
@pytest.mark.parametrize('shape', SHAPES)
def test_the_update_has_the_precision_of_float32(handler, shape, steps):
    d = _case(shape, seed=sum(shape))
    _check(_update(handler, d, steps), d, steps)


@pytest.mark.gpu
@pytest.mark.parametrize('steps', [1, 5])
@pytest.mark.parametrize('size', [1e-30, 1e-15, 1e-4, 1e25, 3e37])
@pytest.mark.parametrize('shape', [(20, 30), (200, 150), (2, 300, 260)])
def test_whatever_the_size_of_the_gradient(handler, shape, size, steps):
    """Down to where the 1e-7 beside the norm makes the update small, and nothing, up to where float32 ends."""
    d = _case(shape, seed=1, size=size)
    if size > 1e37:
        d['momentum'][:] = 0           # the sum of the two would not be finite
    _check(_update(handler, d, steps), d, steps)


def _halves(x):
    x = x.astype(np.float32) * np.float32(4096)
    hi = x.astype(np.float16)
    lo = (x - hi.astype(np.float32)).astype(np.float16)
    return hi.astype(np.float64) / 4096, lo.astype(np.float64) / 4096


@pytest.mark.parametrize('terms, holds', [('hl lh', True), ('hl', False), ('lh', False), ('', False)])
@pytest.mark.parametrize('steps', [1, 5])
@pytest.mark.parametrize('shape', [(3, 7), (16, 40), (64, 64), (205, 256), (300, 129)])
def test_the_bound_needs_every_product(shape, steps, terms, holds):
    """The iteration on the CPU from two half-precision parts: with all three products the bound holds, without one it does not."""
    d = _case(shape, seed=sum(shape))
    beta = float(np.float32(0.95))
    momentum = beta * d['momentum'].astype(np.float64) + d['grad']
    u = d['grad'] + beta * momentum

    def product(a, b):
        (ah, al), (bh, bl) = _halves(a), _halves(b)
        return (ah @ bh + (ah @ bl if 'hl' in terms else 0) + (al @ bh if 'lh' in terms else 0)).astype(np.float32)
    X = (u / (np.linalg.norm(u) + 1e-7)).astype(np.float32)
    tall, eye = shape[0] > shape[1], np.eye(min(shape), dtype=np.float32)
    for _ in range(steps):
        D = (product(X.T, X) if tall else product(X, X.T)) + np.float32(B / (2 * C)) * eye
        P = np.float32(C) * product(D, D) + np.float32(A - B * B / (4 * C)) * eye
        X = product(X, P) if tall else product(P, X)
    error, size, _ = _errors(X.astype(np.float64), d, steps)
    assert error <= steps * STEP * size if holds else error > 10 * steps * STEP * size

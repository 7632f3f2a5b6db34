"""Momentum with an orthogonalised update through the handler against the plain form in 64 bits.

Tolerance.  The momentum is two products and a sum: 2 U of the absolute values, U = 2^-24.  A Newton-Schulz step maps a
singular value s to p(s) = 3.4445 s - 4.7750 s^3 + 2.0315 s^5, whose slope is at most 3.4445 for s in [0, 1.21], where all
of them stay; an error made before a step is thus at most 3.4445 times as large after it, so errors of relative size d in
each step grow to at most d (1 + 3.4445 + ... ) <= 3.4445^steps / 2.4445 d, while the norm of X itself grows from 1 towards
sqrt(m).  One step's products (operands split in two parts, 12 U, sums that truncate every 16 terms and are rounded
every 256 or fewer, 40 U) are each off by at most 60 U of the norms' product, with factors 4.775 * 1.21^2 and
2.0315 * 1.21^4 and three products on a path: d <= 60 U * (3.4445 + 2 * 4.775 * 1.47 + 3 * 2.0315 * 2.15) <= 1900 U in the
2-norm, and the errors of the many entries are independent, which divides their 2-norm against the Frobenius norm by far
more than the ten by which the bound here is taken: |error|_F <= 190 U * 3.4445^steps / 2.4445 * max(1, |update|_F) for
steps > 0, and 4 U |update|_F without a step.
"""
import numpy as np
import pytest

import sequence_reference as ref

U = 2.0 ** -24


def _case(shape, seed=0, rank=None):
    rs = np.random.RandomState(seed)
    f = lambda *s: rs.standard_normal(s).astype(np.float32)  # noqa: E731
    grad = f(*shape) * 1e-3
    if rank:
        grad = (f(*shape[:-1], rank) @ f(*shape[:-2], rank, shape[-1]) * 1e-3 + 0.1 * grad).astype(np.float32)
    return {'param': f(*shape), 'grad': grad, 'momentum': f(*shape) * 2e-3}


def _run(h, d, rate=0.02, beta=0.95, nesterov=True, weight_decay=0.01, steps=5):
    up = {k: h.create_from_numpy(v) for k, v in d.items()}
    update = h.ones(d['param'].shape)
    h.muon_update(up['param'], up['grad'], up['momentum'], update, rate, beta=beta, nesterov=nesterov, weight_decay=weight_decay, steps=steps)
    return [h.get_numpy_copy(a) for a in (up['param'], up['momentum'], update)]


def _check(h, d, rate=0.02, beta=0.95, nesterov=True, weight_decay=0.01, steps=5):
    f = lambda v: float(np.float32(v))  # noqa: E731  (the library takes float32 scalars)
    param, momentum, update = (a.astype(np.float64) for a in _run(h, d, rate, beta, nesterov, weight_decay, steps))
    w_param, w_momentum, w_update = ref.muon(d['param'], d['grad'], d['momentum'], f(rate), f(beta), nesterov, f(weight_decay), steps)
    assert (np.abs(momentum - w_momentum) <= 2 * U * (np.abs(beta * d['momentum']) + np.abs(d['grad'])) + 1e-44).all()
    for i in np.ndindex(update.shape[:-2]):
        size = np.linalg.norm(w_update[i])
        bound = 190 * U * 3.4445 ** steps / 2.4445 * max(1.0, size) if steps else 4 * U * size
        assert np.linalg.norm(update[i] - w_update[i]) <= bound, i
    # the parameters follow from the update that was returned
    want = (1 - f(rate) * f(weight_decay)) * d['param'] - f(rate) * update
    assert (np.abs(param - want) <= 4 * U * (np.abs(d['param']) + abs(rate) * np.abs(update))).all()


# one value, vectors, wide and tall, at and off the tiles, stacks
SHAPES = [(1, 1), (1, 7), (9, 1), (2, 3), (16, 16), (31, 33), (64, 64), (65, 127), (127, 65), (128, 128), (129, 300), (300, 129), (205, 256), (17, 1000), (1000, 17),
          (513, 640), (3, 40, 24), (2, 24, 40), (4, 130, 130), (2, 1, 5), (3, 128, 64), (2, 300, 260)]


@pytest.fixture(scope='module')
def handler():
    from brainstorm_b200 import B200Handler
    return B200Handler(seed=0)


@pytest.mark.gpu
@pytest.mark.parametrize('shape', SHAPES)
def test_update(handler, shape):
    _check(handler, _case(shape, seed=sum(shape)))


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(256, 256), (1000, 60), (60, 512), (128, 513), (1, 1), (129, 250), (8, 250, 65), (64, 17, 30), (65, 17, 30), (3, 40, 1)])
def test_around_the_limits_of_a_single_launch(handler, shape):
    """Up to eight tiles of 128 x 64 a matrix and 64 in all run as one launch, more product by product."""
    _check(handler, _case(shape, seed=sum(shape)))


@pytest.mark.gpu
@pytest.mark.parametrize('steps', [0, 1, 2, 3, 8])
@pytest.mark.parametrize('shape', [(30, 50), (200, 150)])
def test_steps(handler, shape, steps):
    _check(handler, _case(shape, seed=1), steps=steps)


@pytest.mark.gpu
@pytest.mark.parametrize('nesterov', [True, False])
@pytest.mark.parametrize('beta', [0.0, 0.5])
def test_momentum_forms(handler, nesterov, beta):
    _check(handler, _case((60, 70), seed=2), beta=beta, nesterov=nesterov, weight_decay=0.0, rate=0.5)


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(96, 160), (2, 300, 200)])
def test_singular_values_come_near_one(handler, shape):
    """A direction of low rank with noise: what the iteration is for."""
    d = _case(shape, seed=3, rank=8)
    update = _run(handler, d)[2].astype(np.float64)
    want = ref.muon(d['param'], d['grad'], d['momentum'], 0.02, 0.95, True, 0.01, 5)[2]
    got, exact = np.linalg.svd(update, compute_uv=False), np.linalg.svd(want, compute_uv=False)
    assert np.abs(got - exact).max() <= 190 * U * 3.4445 ** 5 / 2.4445 * np.sqrt(min(shape[-2:]))
    assert got[..., 0].max() < 1.25 and got[..., :8].min() > 0.65


@pytest.mark.gpu
@pytest.mark.parametrize('size', [1e-12, 1e-30, 1e12, 3e18])
@pytest.mark.parametrize('shape', [(20, 30), (200, 150)])
def test_magnitudes(handler, shape, size):
    """1e-12 is near the 1e-7 in the norm's denominator, the squares of 3e18 overflow in float32, those of 1e-30 vanish."""
    d = _case(shape, seed=4)
    for k in ('grad', 'momentum'):
        d[k] = (d[k] * np.float64(size) * 1e3).astype(np.float32)
    _check(handler, d)


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(12, 20), (150, 140), (2, 40, 70)])
def test_zero_and_values_that_are_not_finite(handler, shape):
    d = _case(shape, seed=5)
    for k in ('grad', 'momentum'):
        d[k][:] = 0
    param, momentum, update = _run(handler, d)
    assert not update.any() and not momentum.any()
    d = _case(shape, seed=5)
    clean = _run(handler, d)[2]
    d['grad'][(0,) * (len(shape) - 2) + (1, 2)] = np.nan
    update = _run(handler, d)[2]
    assert np.isnan(update[0] if len(shape) == 3 else update).all()
    if len(shape) == 3:
        assert np.array_equal(update[1], clean[1])


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(70, 90), (3, 64, 64), (300, 200)])
def test_same_bits_every_time_and_when_replayed(handler, shape):
    h, d = handler, _case(shape, seed=6)
    first = _run(h, d)
    assert all(np.array_equal(a, b) for a, b in zip(first, _run(h, d)))
    up = {k: h.create_from_numpy(v) for k, v in d.items()}
    update = h.zeros(shape)

    def step():
        h.muon_update(up['param'], up['grad'], up['momentum'], update, 0.02, weight_decay=0.01)
    step()
    recorded = h.record(step)
    for r in (recorded, recorded):
        for k in up:
            h.set_from_numpy(up[k], d[k])
        r.launch()
        for a, b in zip((up['param'], up['momentum'], update), first):
            assert np.array_equal(h.get_numpy_copy(a), b)
        step()
    recorded.release()


@pytest.mark.gpu
def test_a_stack_is_its_matrices(handler):
    d = _case((3, 50, 80), seed=7)
    whole = _run(handler, d)
    for i in range(3):
        one = _run(handler, {k: v[i] for k, v in d.items()})
        assert all(np.allclose(a, b[i], rtol=0, atol=1e-5) for a, b in zip(one, whole))


@pytest.mark.gpu
def test_empty(handler):
    h = handler
    for shape in ((0, 4), (4, 0), (0, 3, 3)):
        h.muon_update(*[h.zeros(shape) for _ in range(4)], 0.1)


def test_refusals():
    from brainstorm_b200 import B200Array
    from brainstorm_b200.sequence_ops import SequenceOps
    a = lambda i, *s: B200Array(None, (i + 1) << 20, tuple(s))  # noqa: E731
    h, args = SequenceOps(), [a(i, 4, 8) for i in range(4)]
    for change, text in (((1, a(9, 4, 9)), 'grad has shape'), ((3, args[0]), 'update overlaps param'), ((2, args[1]), 'momentum overlaps grad')):
        bad = list(args)
        bad[change[0]] = change[1]
        with pytest.raises(ValueError, match=text):
            h.muon_update(*bad, 0.1)
    with pytest.raises(ValueError, match='matrices'):
        h.muon_update(*[a(i, 8) for i in range(4)], 0.1)
    for steps in (-1, 101, 2.5):
        with pytest.raises(ValueError, match='steps'):
            h.muon_update(*args, 0.1, steps=steps)
    with pytest.raises(NotImplementedError, match='contiguous'):
        h.muon_update(a(0, 4, 16)[:, :8], *args[1:], 0.1)

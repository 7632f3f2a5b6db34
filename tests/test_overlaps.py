"""Calls of the sequence operators whose arrays share memory: in place where that is allowed, refused elsewhere.

The checks come before any launch, so they are tested on views of addresses that nothing is read from."""
import numpy as np
import pytest


def _array(i, *shape):
    from brainstorm_b200 import B200Array
    return B200Array(None, (i + 1) << 20, tuple(shape))


class _Reached(Exception):
    """The call passed all checks and came to the library."""


@pytest.fixture
def ops(monkeypatch):
    import brainstorm_b200.sequence_ops as so

    class Library(object):
        def __getattr__(self, name):
            if name.endswith('floats'):
                return lambda *args: 0
            raise _Reached
    monkeypatch.setattr(so, 'lib', Library())
    return so.SequenceOps()


ROWS, W = 8, 6


def _norm_forward(ops, x, y, x_out, h_out):
    ops.gated_norm_forward(x, y, None, None, None, None, x_out, h_out, _array(8, ROWS), _array(9, ROWS))


def _norm_backward(ops, dx_out, dx, accumulate=False):
    a = lambda i: _array(i, ROWS, W)  # noqa: E731
    ops.gated_norm_backward(a(10), a(11), None, None, None, None, _array(8, ROWS), _array(9, ROWS), dx_out, a(12), dx, a(13), None, None, None, None,
                            accumulate=accumulate)


# views of one address: contiguous, and with a row pitch
@pytest.mark.parametrize('first, second, allowed', [(W, W, True), (2 * W, 2 * W, True), (2 * W, W, False), (W, 2 * W, False), (W + 1, W, False), (W + 2, 2 * W, False)])
def test_in_place_takes_the_same_rows(ops, first, second, allowed):
    view = lambda pitch: _array(0, ROWS, pitch)[:, :W]  # noqa: E731
    a, b, c, d = view(first), view(second), _array(1, ROWS, W), _array(2, ROWS, W)
    for call, text in ((lambda: _norm_forward(ops, a, c, b, d), 'x_out overlaps x'), (lambda: _norm_forward(ops, c, a, d, b), 'h_out overlaps y'),
                       (lambda: _norm_backward(ops, a, b), 'dx overlaps dx_out')):
        if allowed:
            with pytest.raises(_Reached):
                call()
        else:
            with pytest.raises(ValueError, match=text):
                call()


@pytest.mark.gpu
def test_the_library_takes_the_same_rows_in_place():
    """The same refusals of the C entries, which check before they launch."""
    from brainstorm_b200 import B200Handler, B200Error
    from brainstorm_b200._lib import lib, check
    from brainstorm_b200.sequence_ops import _norm_args
    h = B200Handler(seed=0)
    a, b, c, r = h.zeros((ROWS, 2 * W)), h.zeros((ROWS, 2 * W)), h.zeros((ROWS, 2 * W)), h.zeros((ROWS,))

    def forward(x_out, h_out, ld_x_out, ld_h_out):
        check(lib.b200_gated_norm_forward(_norm_args(a.ptr, b.ptr, 0, 0, 0, 0, x_out, h_out, r.ptr, r.ptr + 4 * ROWS // 2, ROWS // 2, W, 2 * W, 2 * W, 0, ld_x_out,
                                                     ld_h_out, 1e-6, 0)))
    forward(a.ptr, b.ptr, 2 * W, 2 * W)
    for args in ((a.ptr, c.ptr, W, W), (c.ptr, b.ptr, W, W)):
        with pytest.raises(B200Error, match='row pitch'):
            forward(*args)

    def backward(ld_dx):
        check(lib.b200_gated_norm_backward(0, b.ptr, 0, 0, 0, 0, r.ptr, 0, a.ptr, 0, a.ptr, c.ptr, 0, 0, 0, 0, ROWS // 2, W, 0, 2 * W, 0, 2 * W, 0, ld_dx, 2 * W, 0, 0,
                                           0, 0, 0))
    backward(2 * W)
    with pytest.raises(B200Error, match='row pitch'):
        backward(W)


# column ranges of one hub, as (first column, columns), and row ranges
@pytest.mark.parametrize('x_out, overlaps', [((0, W), True), ((2, W), True), ((1 + W, W), False), ((1, W), False)])
def test_column_ranges_of_a_hub(ops, x_out, overlaps):
    hub = _array(0, ROWS, 2 * W + 1)
    x, out = hub[:, 1:W + 1], hub[:, x_out[0]:sum(x_out)]
    with pytest.raises(ValueError if overlaps else _Reached, match='x_out overlaps x' if overlaps else None):
        _norm_forward(ops, x, _array(1, ROWS, W), out, _array(2, ROWS, W))
    with pytest.raises(ValueError if overlaps else _Reached, match='dx overlaps dx_out' if overlaps else None):
        _norm_backward(ops, x, out)


@pytest.mark.parametrize('shift, overlaps', [(8, True), (-8, True), (31, True), (32, False), (96, False), (-32, False)])
@pytest.mark.parametrize('T', [1, 4])
def test_attention_outputs_in_a_hub(ops, T, shift, overlaps):
    """q in columns 32 to 63 of a hub of 160, the output `shift` columns further on."""
    hub, start = _array(0, T, 2, 160), 32
    part = lambda c: hub[:, :, c:c + 32].reshape((T, 2, 4, 8))  # noqa: E731
    q, out, k, v, decay = part(start), part(start + shift), _array(1, T, 2, 4, 8), _array(2, T, 2, 4, 8), _array(3, 4)
    error, text = (ValueError, 'overlaps q') if overlaps else (_Reached, None)
    with pytest.raises(error, match=text and 'out ' + text):
        ops.linear_attention_forward(q, k, v, decay, out)
    with pytest.raises(error, match=text and 'dq ' + text):
        ops.linear_attention_backward(q, k, v, decay, _array(4, T, 2, 4, 8), out, _array(5, T, 2, 4, 8), _array(6, T, 2, 4, 8))
    with pytest.raises(error, match=text and 'out ' + text):
        ops.linear_attention_step(q[0], k[0], v[0], decay, _array(7, 2, 4, 8, 8), out[0])


def test_rows_of_a_hub(ops):
    """Alternate rows do not meet, nor do earlier and later ones; rows that both views hold do."""
    hub = _array(0, 3 * ROWS, 2 * W)
    y, h_out = _array(1, ROWS, W), _array(2, ROWS, W)
    for x, x_out in ((hub[0:2 * ROWS:2, :W], hub[1:2 * ROWS + 1:2, :W]), (hub[:ROWS, :W], hub[ROWS:2 * ROWS, :W]), (hub[:ROWS, :W], hub[1:ROWS + 1, W:])):
        with pytest.raises(_Reached):
            _norm_forward(ops, x, y, x_out, h_out)
    for x, x_out in ((hub[:ROWS, :W], hub[1:ROWS + 1, :W]), (hub[0:2 * ROWS:2, :W], hub[2:2 * ROWS + 2:2, :W]), (hub[:ROWS, :W], hub[1:2 * ROWS + 1:2, :W]),
                     (hub[:ROWS, :W], hub[1:ROWS + 1, W - 1:2 * W - 1])):
        with pytest.raises(ValueError, match='x_out overlaps x'):
            _norm_forward(ops, x, y, x_out, h_out)


def _places(offset, shape, strides):
    return {offset + sum(i * s for i, s in zip(index, strides)) for index in np.ndindex(*shape)}


def test_the_rule_against_enumeration():
    """Small views of up to three dimensions, nested, interleaved and folded, against the sets of their elements."""
    from brainstorm_b200.sequence_ops import _overlap
    rs = np.random.RandomState(0)
    met = 0
    for _ in range(4000):
        (a_shape, a_strides), (b_shape, b_strides) = [
            (tuple(int(i) for i in rs.randint(1, 5, n)), tuple(int(i) for i in rs.choice([0, 1, 1, 2, 3, 4, 6, 7, 12, 24, 25], n))) for n in rs.randint(1, 4, 2)]
        delta = int(rs.randint(-40, 41))
        want = bool(_places(0, a_shape, a_strides) & _places(delta, b_shape, b_strides))
        assert _overlap(delta, a_shape, a_strides, b_shape, b_strides) == want, (delta, a_shape, a_strides, b_shape, b_strides)
        met += want
    assert 500 < met < 3500


def test_views_that_cannot_be_told_apart_in_time_are_refused():
    """Strides without any nesting make the search long: it gives up and says that they may overlap."""
    from brainstorm_b200.sequence_ops import _overlap
    shape, strides = (997, 991, 983, 977), (9973, 9967, 9949, 9941)
    assert _overlap(3, shape, strides, shape, tuple(s + 2 for s in strides))


def test_outputs_that_fold_onto_themselves(ops):
    """Views built with a stride of zero, or rows that run into one another: read, but not written."""
    from brainstorm_b200 import B200Array
    T, B, H, d = 4, 2, 3, 8
    a = lambda i, heads=H: _array(i, T, B, heads, d)  # noqa: E731
    shared = lambda i: B200Array(None, (i + 1) << 20, (T, B, H, d), (B * d, d, 0, 1))  # noqa: E731
    close = lambda i: B200Array(None, (i + 1) << 20, (T, B, H, d), (B * (H * d - 1), H * d - 1, d, 1))  # noqa: E731
    turned = B200Array(None, 9 << 20, (T, B, H, d), (d, T * d, B * T * d, 1))      # batch and heads before time
    decay = _array(20, H)
    for out in (shared(1), close(1)):
        with pytest.raises(ValueError, match='out overlaps itself'):
            ops.linear_attention_forward(a(2), a(3), a(4), decay, out)
        with pytest.raises(ValueError, match='out overlaps itself'):
            ops.linear_attention_step(a(2)[0], a(3)[0], a(4)[0], decay, _array(5, B, H, d, d), out[0])
        for i, name in enumerate(('dq', 'dk', 'dv')):
            grads = [a(6), a(7), a(8)]
            grads[i] = out
            with pytest.raises(ValueError, match=name + ' overlaps itself'):
                ops.linear_attention_backward(a(2), a(3), a(4), decay, a(5), *grads)
    with pytest.raises(_Reached):
        ops.linear_attention_forward(shared(1), close(2), shared(3), decay, turned)
    with pytest.raises(_Reached):
        ops.linear_attention_backward(shared(1), close(2), shared(3), decay, shared(4), turned, a(10), a(11))

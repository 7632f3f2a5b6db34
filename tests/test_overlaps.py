"""Calls of the sequence operators whose arrays share memory: in place where that is allowed, refused elsewhere.

The checks come before any launch, so they are tested on views of addresses that nothing is read from."""
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

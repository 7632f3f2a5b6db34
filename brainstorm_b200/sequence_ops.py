"""Handler methods for sequence blocks: decayed linear attention, the norms, gate and residual around a
block, and the momentum update of a weight matrix whose direction is orthogonalised.

The reference has none of them; they stand beside its LSTM (brainstorm/layers/lstm_layer.py:21), Highway
(highway_layer.py:21) and BatchNorm (batch_normalization_layer.py:23) layers and its steppers
(training/steppers.py:46-145), and follow the conventions of its handlers: outputs are arguments, sequence
arrays have time first and batch second, whole numbers travel as float32, and backward methods add to
their gradients (``accumulate=False`` overwrites).  As everywhere in the backend, this file only turns views
into pointers and extents; the kernels are in ``csrc/linear_attention*.cu``, ``gated_norm.cu`` and ``muon.cu``.
"""
from __future__ import annotations

import ctypes
import functools
import struct
from operator import gt

from ._lib import lib, check
from .array import B200Array

_ACTIVATIONS = {'sigmoid': 0, 'tanh': 1, 'rel': 2, 'el': 3, 'linear': 4}


def _activation(name):
    try:
        return _ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError('unknown activation %r (one of %s)' % (name, ', '.join(sorted(_ACTIVATIONS))))


def _ptr(a):
    return 0 if a is None else a.ptr


def _rows(a, shape, what):
    """Row pitch of a 2-D array of the given shape."""
    if a is None:
        return 0
    if a.shape != shape:
        raise ValueError('%s has shape %r, expected %r' % (what, a.shape, shape))
    if a._contig:
        return shape[1]
    if shape[1] > 1 and a.strides[1] != 1:
        raise NotImplementedError('%s: matrix view with a non-unit column stride' % what)
    return a.strides[0] if shape[0] > 1 else shape[1]


def _vector(a, n, what):
    if a is None:
        return 0
    if a.size != n:
        raise ValueError('%s has %d values, expected %d' % (what, a.size, n))
    if not a._contig:
        raise NotImplementedError('%s must be contiguous' % what)
    return a.ptr


def _whole(a, shape, what):
    """Address of a contiguous array of the given shape (0 for None)."""
    if a is None:
        return 0
    if a.shape != shape:
        raise ValueError('%s has shape %r, expected %r' % (what, a.shape, shape))
    if not a._contig:
        raise NotImplementedError('%s must be contiguous' % what)
    return a.ptr


def _heads(a, what):
    """(t, b, h) strides of a (T, B, heads, d) or (B, heads, d) array with contiguous d."""
    if a.shape[-1] > 1 and a.strides[-1] != 1:
        raise NotImplementedError('%s: the last dimension must be contiguous' % what)
    return tuple(a.strides[:3]) if len(a.shape) == 4 else (0,) + tuple(a.strides[:2])


@functools.lru_cache(maxsize=4096)
def _folds(shape, strides):
    """Whether a view may hold one element twice: a stride that does not reach past the smaller ones together."""
    past = 0
    for s, n in sorted((s, n) for n, s in zip(shape, strides) if n > 1):
        if s <= past:
            return True
        past += s * (n - 1)
    return False


def _result_heads(a, what):
    """_heads of an array that is written."""
    if a.size and _folds(a.shape, a.strides):
        raise ValueError('%s overlaps itself' % what)
    return _heads(a, what)


def _expect(a, shape, what):
    if a.shape != shape:
        raise ValueError('%s has shape %r, expected %r' % (what, a.shape, shape))


def _span(a):
    """[first, last) address of a view."""
    if a._contig:
        return a.ptr, a.ptr + 4 * a.size
    return a.ptr, a.ptr + 4 * (sum((n - 1) * s for n, s in zip(a.shape, a.strides)) + 1)


def _meet(arrays):
    """Whether the address ranges of any two of the arrays overlap: if none do, the k-th end in order is no later than
    start k + 1; where two do, one more range has begun than that before some end."""
    arrays = [a for a in arrays if a is not None and a.size]
    starts = [a.ptr for a in arrays]
    ends = [a.ptr + 4 * a.size if a._contig else _span(a)[1] for a in arrays]
    starts.sort()
    ends.sort()
    return any(map(gt, ends, starts[1:]))


def _same(a, b):
    """Whether two views have every element in the same place."""
    return a.ptr == b.ptr and a.shape == b.shape and (a._contig and b._contig or
                                                      all(s == t for n, s, t in zip(a.shape, a.strides, b.strides) if n > 1))


def _folded(shape, strides):
    """A view's (stride, extent) pairs: adjacent dimensions that follow one another in memory as one."""
    dims = []
    for n, s in zip(reversed(shape), reversed(strides)):
        if n > 1 and dims and s == dims[-1][0] * dims[-1][1]:
            dims[-1] = (dims[-1][0], dims[-1][1] * n)
        elif n > 1:
            dims.append((s, n))
    return dims


@functools.lru_cache(maxsize=4096)
def _overlap(delta, a_shape, a_strides, b_shape, b_strides):
    """Whether two views, b starting ``delta`` elements behind a, have an element in common: whole numbers i within a's
    extents and j within b's with sum i * a's strides - sum j * b's strides == delta.  Dimensions with the same
    stride count together; going from the largest stride down, a number is tried only where the smaller strides
    can still make up the rest, which leaves one or two for the views of a hub.  A search that does not end soon
    counts as an overlap."""
    reach = {}
    for dims, sign in ((_folded(a_shape, a_strides), 1), (_folded(b_shape, b_strides), -1)):
        for s, n in dims:
            if s == 0:
                continue
            lo, hi = reach.get(abs(s), (0, 0))
            step = sign * (n - 1) * (1 if s > 0 else -1)
            reach[abs(s)] = (lo + min(step, 0), hi + max(step, 0))
    terms = sorted(((s, lo, hi) for s, (lo, hi) in reach.items()), reverse=True)
    below = [(0, 0)]                                   # what the strides behind a place in the order can make up
    for s, lo, hi in reversed(terms):
        below.insert(0, (below[0][0] + s * lo, below[0][1] + s * hi))
    tries = 10000

    def search(i, rest):
        nonlocal tries
        if i == len(terms):
            return rest == 0
        s, lo, hi = terms[i]
        least, most = below[i + 1]
        for x in range(max(lo, -((most - rest) // s)), min(hi, (rest - least) // s) + 1):
            tries -= 1
            if tries < 0 or search(i + 1, rest - s * x):
                return True
        return False
    return search(0, delta)


def _apart(outputs, inputs, allowed=()):
    """Refuse an output that has an element in common with another operand (row-pitched views may interleave in one
    buffer, as the columns of a hub do).  An output that may be an input has to be the same view: with another row
    pitch it would write rows that are still to be read.  Called when operands meet (``_meet``)."""
    seen = [(n, a) + _span(a) for n, a in inputs if a is not None and a.size]
    for name, a in outputs:
        if a is None or not a.size:
            continue
        lo, hi = _span(a)
        for other, b, b_lo, b_hi in seen:
            if lo >= b_hi or b_lo >= hi or (name, other) in allowed and _same(a, b):
                continue
            delta = b_lo - lo
            if delta % 4 or _overlap(delta // 4, a.shape, a.strides, b.shape, b.strides):
                raise ValueError('%s overlaps %s' % (name, other))
        seen.append((name, a, lo, hi))


_Strides12, _Strides21 = ctypes.c_int64 * 12, ctypes.c_int64 * 21
# The calls that serve single tokens pass their arguments as one packed struct: converted one by one, those of a step
# cost 2.4 us, packed 0.5.
_attention_args = struct.Struct('@17qf').pack
_norm_args = struct.Struct('@17qfi').pack


class SequenceOps(object):
    """Mixin of ``B200Handler``."""

    # ------------------------------------------------------------ decayed linear attention
    def linear_attention_forward(self, q, k, v, decay, out, scale=1.0, state=None, state_out=None, lengths=None):
        """``S[t] = decay[h] * S[t-1] + outer(k[t], v[t])``, ``out[t] = scale * q[t] . S[t]``.

        Args:
            q, out: (T, B, H, dk) and (T, B, H, dv).
            k, v: (T, B, K, dk) and (T, B, K, dv); K divides H, head h of q reads head ``h // (H // K)``.
                The last dimension of all four must be contiguous; the others may be strided (for results: without an
                element that lies in two places).
            decay: (H,), a constant factor for each head.
            state, state_out: (B, H, dk, dv) before the first and after the last token; ``state=None`` starts
                from zero.  ``state_out`` may be ``state``.
            lengths: (B,) float32 values that hold whole numbers, truncated like labels and held to [0, T]:
                ``out`` is zero behind the end of a sequence and the state stays as it was there.  What the
                inputs hold behind the end is not read.

        dk, dv: 1 to 128.  A non-finite value of a token spreads to later tokens of its sequence and head, and may
        spread to up to 15 tokens before it.  Up to 8 tokens everything is float32.  From 9 on operands have 22 bits and sums on
        the tensor core truncate (errors are two to three times those of float32 sums), and a value more than 2^17 below the largest of its row (one token and head of ``q``, ``k``, ``v`` or
        ``dout``, and the state) keeps fewer bits: it is held to 2^-38 of that largest value, and so is a token's part in an output
        beside the largest part.  Later tokens do not matter."""
        T, B, H, K, dk, dv = self._attention_shapes(q, k, v, 4)
        _expect(out, (T, B, H, dv), 'out')
        strides = 0
        if not (q._contig and k._contig and v._contig and out._contig):
            strides = _Strides12(*(_heads(q, 'q') + _heads(k, 'k') + _heads(v, 'v') + _result_heads(out, 'out')))
        if _meet((q, k, v, out, decay, state, state_out, lengths)):
            _apart((('out', out), ('state_out', state_out)), (('q', q), ('k', k), ('v', v), ('decay', decay), ('state', state), ('lengths', lengths)),
                   (('state_out', 'state'),))
        need = lib.b200_linear_attention_forward_scratch_floats(T, B, H, dk, dv)
        # stream-ordered and released with the call: calls on two streams, and recorded graphs, have their own
        work = B200Array.empty((need,), zero=False) if need else None
        states = (B, H, dk, dv)
        check(lib.b200_linear_attention_forward(_attention_args(
            q.ptr, k.ptr, v.ptr, _vector(decay, H, 'decay'), out.ptr, _whole(state, states, 'state'), _whole(state_out, states, 'state_out'),
            _vector(lengths, B, 'lengths'), strides and ctypes.addressof(strides), _ptr(work), need, T, B, H, K, dk, dv, scale)))

    def linear_attention_backward(self, q, k, v, decay, dout, dq, dk, dv, scale=1.0, state=None, dstate_out=None, dstate=None, lengths=None,
                                  accumulate=True):
        """Gradients of ``linear_attention_forward``: adds to ``dq``, ``dk``, ``dv`` (overwrites them without
        ``accumulate``) and writes ``dstate``, the gradient of ``state``.  ``dstate_out`` is the gradient of
        ``state_out`` (None: zero).  Gradients are zero behind the end of a
        sequence; ``dout`` is not read there."""
        T, B, H, K, d_k, d_v = self._attention_shapes(q, k, v, 4)
        for a, shape, what in ((dout, (T, B, H, d_v), 'dout'), (dq, q.shape, 'dq'), (dk, k.shape, 'dk'), (dv, v.shape, 'dv')):
            _expect(a, shape, what)
        arrays = (('q', q), ('k', k), ('v', v), ('dout', dout), ('dq', dq), ('dk', dk), ('dv', dv))
        strides = 0
        if not all(a._contig for _, a in arrays):
            strides = _Strides21(*[s for i, (what, a) in enumerate(arrays) for s in (_result_heads if i > 3 else _heads)(a, what)])
        if _meet((q, k, v, dout, dq, dk, dv, decay, state, dstate_out, dstate, lengths)):
            _apart(arrays[4:] + (('dstate', dstate),),
                   arrays[:4] + (('decay', decay), ('state', state), ('dstate_out', dstate_out), ('lengths', lengths)))
        states = (B, H, d_k, d_v)
        need = lib.b200_linear_attention_backward_scratch_floats(T, B, H, K, d_k, d_v)
        work = B200Array.empty((need,), zero=False) if need else None
        check(lib.b200_linear_attention_backward(
            q.ptr, k.ptr, v.ptr, _vector(decay, H, 'decay'), dout.ptr, dq.ptr, dk.ptr, dv.ptr, _whole(state, states, 'state'),
            _whole(dstate_out, states, 'dstate_out'), _whole(dstate, states, 'dstate'), _vector(lengths, B, 'lengths'), T, B, H, K, d_k, d_v,
            strides, scale, 1 if accumulate else 0, _ptr(work), need))

    def linear_attention_step(self, q, k, v, decay, state, out, scale=1.0):
        """One token for every sequence: q (B, H, dk), k (B, K, dk), v (B, K, dv), out (B, H, dv); ``state``
        (B, H, dk, dv) is updated in place.  The recurrence of ``linear_attention_forward``."""
        B, H, K, dk, dv = self._attention_shapes(q, k, v, 3)
        _expect(out, (B, H, dv), 'out')
        strides = 0
        if not (q._contig and k._contig and v._contig and out._contig):
            strides = _Strides12(*(_heads(q, 'q') + _heads(k, 'k') + _heads(v, 'v') + _result_heads(out, 'out')))
        if _meet((q, k, v, out, decay, state)):
            _apart((('out', out), ('state', state)), (('q', q), ('k', k), ('v', v), ('decay', decay)))
        s = _whole(state, (B, H, dk, dv), 'state')
        check(lib.b200_linear_attention_forward(_attention_args(q.ptr, k.ptr, v.ptr, _vector(decay, H, 'decay'), out.ptr, s, s, 0,
                                                                strides and ctypes.addressof(strides), 0, 0, 1, B, H, K, dk, dv, scale)))

    @staticmethod
    def _attention_shapes(q, k, v, ndim):
        if len(q.shape) != ndim or len(k.shape) != ndim or len(v.shape) != ndim:
            raise ValueError('q, k and v must have %d dimensions, got %r, %r, %r' % (ndim, q.shape, k.shape, v.shape))
        *lead, H, dk = q.shape
        K, dv = k.shape[-2], v.shape[-1]
        if k.shape != (*lead, K, dk) or v.shape != (*lead, K, dv):
            raise ValueError('shapes %r, %r, %r of q, k, v do not agree' % (q.shape, k.shape, v.shape))
        if (K == 0) != (H == 0) or K and H % K:
            raise ValueError('%d heads cannot share %d key/value heads' % (H, K))
        return (*lead, H, K, dk, dv)

    # ------------------------------------------------------- norms, gate and residual of a block
    def gated_norm_forward(self, x, y, gate, w_post, scale, w_pre, x_out, h_out, r_post, r_pre, epsilon=1e-6, activation='sigmoid'):
        """The norms after a block and before the next one, with the gate and residual scale between them::

            x_out = x + scale * activation(gate) * (y / rms(y) * w_post)
            h_out = x_out / rms(x_out) * w_pre

        Args:
            x, y, gate, x_out, h_out: (rows, width) residual stream, block output, gate before its activation,
                and the results; rows may be strided.  ``y=None`` leaves out the first line (``x_out`` is then
                not written; the norm before the first block), ``h_out=None`` the second (after the last
                block), ``gate=None`` the gate.
            w_post, scale, w_pre: vectors of ``width`` values, or None for ones.
            r_post, r_pre: (rows,) receive ``1 / rms`` of ``y`` and ``x_out``, which the backward pass needs.
            epsilon: added to the mean squares, which are float32: values from 1.8e19 on leave its range, and a row that holds one
                is normalised to zeros.
            activation: 'sigmoid', 'tanh', 'rel', 'el' or 'linear'.

        width: up to 16384.  ``x_out`` may be ``x`` and ``h_out`` may be ``y``, the same view; no other output may overlap
        another operand."""
        act = _activation(activation)
        if len(x.shape) != 2:
            raise ValueError('expected 2-D arrays, got shape %r' % (x.shape,))
        if y is None and (gate is not None or h_out is None):
            raise ValueError('without a block output there is nothing to gate, and h_out has to be given')
        if y is not None and x_out is None:
            raise ValueError('a block output needs x_out')
        if not epsilon >= 0:
            raise ValueError('epsilon must not be negative')
        shape = rows, width = x.shape
        if y is None:
            x_out = None
        lds = [width if a is not None and a._contig and a.shape == shape else _rows(a, shape, what)
               for a, what in ((x, 'x'), (y, 'y'), (gate, 'gate'), (x_out, 'x_out'), (h_out, 'h_out'))]
        if _meet((x, y, gate, x_out, h_out, w_post, scale, w_pre, r_post, r_pre)):
            _apart((('x_out', x_out), ('h_out', h_out), ('r_post', r_post), ('r_pre', r_pre)),
                   (('x', x), ('y', y), ('gate', gate), ('w_post', w_post), ('scale', scale), ('w_pre', w_pre)), (('x_out', 'x'), ('h_out', 'y')))
        check(lib.b200_gated_norm_forward(_norm_args(
            x.ptr, _ptr(y), _ptr(gate), _vector(w_post, width, 'w_post'), _vector(scale, width, 'scale'), _vector(w_pre, width, 'w_pre'), _ptr(x_out),
            _ptr(h_out), _vector(r_post, rows, 'r_post') if y is not None else 0, _vector(r_pre, rows, 'r_pre') if h_out is not None else 0, rows,
            width, *lds, epsilon, act)))

    def gated_norm_backward(self, x_out, y, gate, w_post, scale, w_pre, r_post, r_pre, dx_out, dh, dx, dy, dgate, dw_post, dscale, dw_pre,
                            activation='sigmoid', accumulate=True):
        """Gradients of ``gated_norm_forward`` from those of ``x_out`` (``dx_out``, None: zero) and ``h_out`` (``dh``,
        None: it was not taken).  ``y``, ``gate`` and the weights are None where they were in the forward pass; a
        vector gradient that is None is not computed.  Adds to all gradients, or overwrites them without
        ``accumulate``.  Without a block output ``x_out`` is the forward pass's ``x``.  ``dx`` may be ``dx_out``, the same view:
        it becomes the gradient of ``x``, in which ``dx_out`` counts once, with ``accumulate`` or without."""
        act = _activation(activation)
        if len(dx.shape) != 2:
            raise ValueError('expected 2-D arrays, got shape %r' % (dx.shape,))
        shape = rows, width = dx.shape
        if y is None and dh is None:
            raise ValueError('there is nothing to differentiate')
        if y is None and (gate is not None or dw_post is not None or dscale is not None):
            raise ValueError('without a block output there is no gate, w_post or scale')
        if y is not None and (r_post is None or dy is None):
            raise ValueError('a block output needs r_post and dy')
        if gate is not None and dgate is None:
            raise ValueError('a gate needs dgate')
        if dh is not None and (x_out is None or r_pre is None):
            raise ValueError('dh needs x_out and r_pre')
        if dh is None and dw_pre is not None:
            raise ValueError('dw_pre needs dh')
        if dh is None:
            x_out = None
        if y is None:
            dy = None
        if gate is None:
            dgate = None
        named = (('x_out', x_out), ('y', y), ('gate', gate), ('dx_out', dx_out), ('dh', dh), ('dx', dx), ('dy', dy), ('dgate', dgate))
        lds = [_rows(a, shape, what) for what, a in named]
        if _meet((x_out, y, gate, dx_out, dh, dx, dy, dgate, dw_post, dscale, dw_pre, w_post, scale, w_pre, r_post, r_pre)):
            _apart(named[5:] + (('dw_post', dw_post), ('dscale', dscale), ('dw_pre', dw_pre)),
                   named[:5] + (('w_post', w_post), ('scale', scale), ('w_pre', w_pre), ('r_post', r_post), ('r_pre', r_pre)), (('dx', 'dx_out'),))
        need = lib.b200_gated_norm_scratch_floats(rows, width) if not (dw_post is None and dscale is None and dw_pre is None) else 0
        work = B200Array.empty((need,), zero=False) if need else None
        check(lib.b200_gated_norm_backward(
            _ptr(x_out), _ptr(y), _ptr(gate), _vector(w_post, width, 'w_post'), _vector(scale, width, 'scale'), _vector(w_pre, width, 'w_pre'),
            _vector(r_post, rows, 'r_post') if y is not None else 0, _vector(r_pre, rows, 'r_pre') if dh is not None else 0, _ptr(dx_out), _ptr(dh),
            dx.ptr, _ptr(dy), _ptr(dgate), _vector(dw_post, width, 'dw_post'), _vector(dscale, width, 'dscale'), _vector(dw_pre, width, 'dw_pre'),
            rows, width, *lds, act, 1 if accumulate else 0, _ptr(work), need))

    # ---------------------------------------------------- momentum with an orthogonalised update
    def muon_update(self, param, grad, momentum, update, learning_rate, beta=0.95, nesterov=True, weight_decay=0.0, steps=5):
        """One update of a weight matrix, or of a stack of equally shaped ones ((rows, cols) or (n, rows, cols),
        contiguous)::

            momentum = beta * momentum + grad
            update   = orthogonalised(grad + beta * momentum if nesterov else momentum)
            param    = (1 - learning_rate * weight_decay) * param - learning_rate * update

        ``orthogonalised(u)`` is ``steps`` Newton-Schulz iterations ``X = 3.4445 X + (-4.7750 A + 2.0315 A A) X`` with
        ``A = X X^T`` from ``u / (|u| + 1e-7)``: the singular values of ``u`` are all brought near one, each matrix of
        a stack on its own.  A zero direction gives a zero update.  Values of ``X`` have 22 bits and are held to 2^-37 at
        least: where ``|u|`` is below 1e-7 so is the update's precision, relative to its then small size."""
        if len(param.shape) not in (2, 3):
            raise ValueError('expected matrices, got shape %r' % (param.shape,))
        if not 0 <= steps <= 100 or int(steps) != steps:
            raise ValueError('steps must be a whole number from 0 to 100')
        shape = param.shape
        arrays = (('param', param), ('grad', grad), ('momentum', momentum), ('update', update))
        ptrs = [_whole(a, shape, what) for what, a in arrays]
        if _meet((param, grad, momentum, update)):
            _apart((arrays[0],) + arrays[2:], arrays[1:2])
        n, rows, cols = shape if len(shape) == 3 else (1,) + shape
        need = lib.b200_muon_scratch_floats(n, rows, cols)
        work = B200Array.empty((need,), zero=False) if need else None
        check(lib.b200_muon_update(*ptrs, n, rows, cols, learning_rate, beta, 1 if nesterov else 0, weight_decay, int(steps), _ptr(work), need))

"""Decayed linear attention through the handler against the recurrence in 64 bits.

Tolerance.  Every output is a sum of products of operands; with U = 2^-24 (half a float32 step) a product that is
formed from two operands, each split into two 11-bit parts with the product of the two low parts left out, is off by
at most 3 * 2^-22 = 12 U of itself; a power of the decay and its factors round a few times more (8 U); adding up
dk products, a chunk of 64 tokens and one state for each chunk before it rounds at most dk + 64 + T / 64 times, each by
at most 2 U (tensor-core sums truncate).  So |error| <= TERMS * U * (the same sum with absolute values), TERMS =
2 * (dk + dv + 64 + T / 64) + 40 with room for dk and dv changing places in the gradients.  The few sums over shared heads add
less than the spare.
"""
import numpy as np
import pytest

import sequence_reference as ref

U = 2.0 ** -24


def _case(T, B, H, K, dk, dv, seed=0, ragged=False, decays=None):
    rs = np.random.RandomState(seed)
    f = lambda *s: rs.standard_normal(s).astype(np.float32)  # noqa: E731
    d = {'q': f(T, B, H, dk), 'k': f(T, B, K, dk), 'v': f(T, B, K, dv), 'state': f(B, H, dk, dv), 'dout': f(T, B, H, dv),
         'dstate_out': f(B, H, dk, dv)}
    d['decay'] = (1 - 2.0 ** -rs.uniform(1, 9, H)).astype(np.float32) if decays is None else np.resize(np.float32(decays), H)
    d['lengths'] = None
    if ragged:
        n = rs.randint(0, T + 1, B)
        n[0] = T
        if B > 1:
            n[1] = 0
        if B > 2:
            n[2] = 1
        d['lengths'] = n.astype(np.float32)
    return d


def _bound(d, scale, backward):
    a = {k: None if d[k] is None else np.abs(d[k]) for k in ('q', 'k', 'v', 'decay', 'dout', 'state', 'dstate_out')}
    T, _, _, dk = d['q'].shape
    terms = 2 * (dk + d['v'].shape[-1] + 64 + T / 64) + 40
    if backward:
        sums = ref.attention_backward(a['q'], a['k'], a['v'], a['decay'], a['dout'], abs(scale), a['state'], a['dstate_out'], d['lengths'])
    else:
        sums = ref.attention(a['q'], a['k'], a['v'], a['decay'], abs(scale), a['state'], d['lengths'])
    return [terms * U * s + 1e-30 for s in sums]


def _check(got, want, bound, what):
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= bound).all(), '%s: %g of the bound' % (what, float((err / bound).max()))


def _poison(d):
    """NaN and infinities behind the end of every sequence: padding is not read."""
    if d['lengths'] is None:
        return d
    d = {k: None if v is None else v.copy() for k, v in d.items()}
    for b, n in enumerate(d['lengths'].astype(int)):
        for i, name in enumerate(('q', 'k', 'v', 'dout')):
            d[name][n:, b] = (np.nan, np.inf)[i % 2]
    return d


def _run(h, d, scale=1.0, backward=True, use_state=True, accumulate=False, start=None):
    up = lambda a: None if a is None else h.create_from_numpy(a)  # noqa: E731
    p = {k: up(v) for k, v in _poison(d).items()}
    if not use_state:
        p['state'] = p['dstate_out'] = None
    T, B, H, dk = d['q'].shape
    dv = d['v'].shape[-1]
    out, state_out = h.ones((T, B, H, dv)), h.ones((B, H, dk, dv))
    h.linear_attention_forward(p['q'], p['k'], p['v'], p['decay'], out, scale=scale, state=p['state'], state_out=state_out, lengths=p['lengths'])
    got = {'out': out, 'state_out': state_out}
    if backward:
        g = {n: h.ones(d[n[1:]].shape) for n in ('dq', 'dk', 'dv')}
        got['dstate'] = h.ones((B, H, dk, dv))
        h.linear_attention_backward(p['q'], p['k'], p['v'], p['decay'], p['dout'], g['dq'], g['dk'], g['dv'], scale=scale, state=p['state'],
                                    dstate_out=p['dstate_out'], dstate=got['dstate'], lengths=p['lengths'], accumulate=accumulate)
        got |= g
    return {k: h.get_numpy_copy(v) for k, v in got.items()}


# time, batch, heads, key/value heads, dk, dv: one token, chunk borders, lengths off every tile, many chunks, all head
# sizes of the tiles and between them, shared heads, more blocks than the GPU holds at once
SHAPES = [(1, 1, 1, 1, 1, 1), (3, 300, 4, 2, 16, 96), (4, 300, 2, 1, 30, 64), (8, 400, 2, 2, 64, 40), (7, 200, 4, 2, 128, 124), (5, 90, 3, 3, 52, 15), (8, 3, 2, 2, 127, 126), (1, 3, 4, 2, 64, 64), (2, 2, 2, 2, 8, 8), (15, 1, 2, 1, 16, 16), (16, 2, 2, 2, 32, 32), (17, 2, 3, 3, 33, 31),
          (63, 2, 2, 2, 64, 64), (64, 2, 2, 2, 64, 64), (65, 2, 2, 2, 64, 64), (128, 3, 4, 4, 128, 128), (129, 2, 6, 2, 40, 72),
          (200, 3, 4, 1, 128, 17), (200, 3, 2, 2, 5, 128), (333, 2, 2, 2, 96, 64), (700, 1, 2, 2, 64, 128), (31, 40, 8, 8, 16, 16),
          (1100, 1, 1, 1, 48, 48), (2500, 1, 2, 1, 32, 64)]


@pytest.fixture(scope='module')
def handler():
    from brainstorm_b200 import B200Handler
    return B200Handler(seed=0)


@pytest.mark.gpu
@pytest.mark.parametrize('ragged', [False, True])
@pytest.mark.parametrize('shape', SHAPES)
def test_forward_and_gradients(handler, shape, ragged):
    d = _case(*shape, seed=sum(shape), ragged=ragged)
    scale = shape[4] ** -0.5
    got = _run(handler, d, scale)
    out, state = ref.attention(d['q'], d['k'], d['v'], d['decay'], scale, d['state'], d['lengths'])
    for name, want, bound in zip(('out', 'state_out'), (out, state), _bound(d, scale, False)):
        _check(got[name], want, bound, name)
    wants = ref.attention_backward(d['q'], d['k'], d['v'], d['decay'], d['dout'], scale, d['state'], d['dstate_out'], d['lengths'])
    for name, want, bound in zip(('dq', 'dk', 'dv', 'dstate'), wants, _bound(d, scale, True)):
        _check(got[name], want, bound, name)


@pytest.mark.gpu
@pytest.mark.parametrize('decays', [[0.0], [1.0], [0.5, 0.0, 1.0, 0.999], [-0.75, 0.25]])
@pytest.mark.parametrize('T', [5, 150])
def test_decays_at_the_ends_of_their_range(handler, decays, T):
    d = _case(T, 2, 4, 4, 24, 40, seed=3, decays=decays)
    got = _run(handler, d)
    out, state = ref.attention(d['q'], d['k'], d['v'], d['decay'], 1.0, d['state'])
    for name, want, bound in zip(('out', 'state_out'), (out, state), _bound(d, 1.0, False)):
        _check(got[name], want, bound, name)
    wants = ref.attention_backward(d['q'], d['k'], d['v'], d['decay'], d['dout'], 1.0, d['state'], d['dstate_out'])
    for name, want, bound in zip(('dq', 'dk', 'dv', 'dstate'), wants, _bound(d, 1.0, True)):
        _check(got[name], want, bound, name)


@pytest.mark.gpu
@pytest.mark.parametrize('T', [3, 100])
def test_without_states(handler, T):
    d = _case(T, 2, 2, 2, 32, 32, seed=4)
    got = _run(handler, d, use_state=False)
    d['state'] = d['dstate_out'] = None
    out, state = ref.attention(d['q'], d['k'], d['v'], d['decay'])
    for name, want, bound in zip(('out', 'state_out'), (out, state), _bound(d, 1.0, False)):
        _check(got[name], want, bound, name)
    wants = ref.attention_backward(d['q'], d['k'], d['v'], d['decay'], d['dout'])
    for name, want, bound in zip(('dq', 'dk', 'dv', 'dstate'), wants, _bound(d, 1.0, True)):
        _check(got[name], want, bound, name)


@pytest.mark.gpu
@pytest.mark.parametrize('K', [2, 4])
@pytest.mark.parametrize('T', [3, 100])
def test_gradients_are_added_by_default(handler, T, K):
    d = _case(T, 3, 4, K, 32, 24, seed=5, ragged=True)
    once, more = _run(handler, d), _run(handler, d, accumulate=True)
    for n in ('dq', 'dk', 'dv'):          # onto ones: one more rounding
        assert np.abs(more[n] - (once[n].astype(np.float64) + 1)).max() <= 2 * U * (np.abs(once[n]).max() + 1)
    assert np.array_equal(more['dstate'], once['dstate'])


@pytest.mark.gpu
@pytest.mark.parametrize('T', [4, 130])
def test_strided_views_and_row_order(handler, T):
    """q, k, v as column ranges of one hub, results into another; and arrays with batch before time."""
    h, (B, H, dk, dv) = handler, (2, 3, 32, 20)
    d = _case(T, B, H, H, dk, dv, seed=6)
    want = _run(h, d)
    hub = h.zeros((T, B, H * (2 * dk + dv)))
    views = {'q': hub[:, :, :H * dk], 'k': hub[:, :, H * dk:2 * H * dk], 'v': hub[:, :, 2 * H * dk:]}
    for n, a in views.items():
        h.set_from_numpy(a, d[n].reshape(T, B, -1))
    v4 = {n: a.reshape((T, B, H, a.shape[-1] // H)) for n, a in views.items()}
    res = h.zeros((T, B, H * dv + 7))
    out = res[:, :, 3:3 + H * dv].reshape((T, B, H, dv))
    up = lambda n: h.create_from_numpy(d[n])  # noqa: E731
    h.linear_attention_forward(v4['q'], v4['k'], v4['v'], up('decay'), out, state=up('state'))
    whole = h.get_numpy_copy(res)
    assert np.array_equal(whole[:, :, 3:3 + H * dv].reshape(T, B, H, dv), want['out'])
    assert not whole[:, :, :3].any() and not whole[:, :, 3 + H * dv:].any()
    grads = h.zeros((T, B, H * (2 * dk + dv)))
    g = [grads[:, :, a:b].reshape((T, B, H, -1)) for a, b in ((0, H * dk), (H * dk, 2 * H * dk), (2 * H * dk, H * (2 * dk + dv)))]
    h.linear_attention_backward(v4['q'], v4['k'], v4['v'], up('decay'), up('dout'), *g, state=up('state'), dstate_out=up('dstate_out'))
    got = h.get_numpy_copy(grads)
    for n, (a, b) in (('dq', (0, H * dk)), ('dk', (H * dk, 2 * H * dk)), ('dv', (2 * H * dk, H * (2 * dk + dv)))):
        assert np.array_equal(got[:, :, a:b].reshape(want[n].shape), want[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(1, 1, 1, 1, 1), (1, 16, 16, 64, 64), (5, 6, 2, 33, 18), (300, 4, 4, 128, 128), (7, 8, 4, 16, 128), (64, 3, 1, 96, 50),
                                   (700, 2, 2, 16, 96), (700, 3, 1, 12, 12), (350, 4, 2, 24, 64), (350, 2, 2, 30, 20), (400, 3, 3, 64, 32), (300, 4, 2, 57, 68),
                                   (90, 8, 4, 52, 15), (5, 2, 2, 127, 127), (200, 4, 4, 97, 64)])
def test_steps_are_the_recurrence(handler, shape):
    """Token by token with the state in place, against the whole sequence in 64 bits."""
    h, (B, H, K, dk, dv), T = handler, shape, 4
    d = _case(T, B, H, K, dk, dv, seed=7)
    state, out = h.create_from_numpy(d['state']), h.zeros((T, B, H, dv))
    q, k, v, decay = (h.create_from_numpy(d[n]) for n in ('q', 'k', 'v', 'decay'))
    for t in range(T):
        h.linear_attention_step(q[t], k[t], v[t], decay, state, out[t], scale=0.25)
    want = ref.attention(d['q'], d['k'], d['v'], d['decay'], 0.25, d['state'])
    for got, w, bound, name in zip((out, state), want, _bound(d, 0.25, False), ('out', 'state')):
        _check(h.get_numpy_copy(got), w, bound, name)


@pytest.mark.gpu
@pytest.mark.parametrize('T', [0, 1, 40, 300, 2000])
def test_state_in_place(handler, T):
    h = handler
    d = _case(T, 2, 2, 2, 32, 32, seed=8)
    apart = _run(h, d)
    p = {n: h.create_from_numpy(a) for n, a in d.items() if a is not None}
    out = h.zeros((T, 2, 2, 32))
    h.linear_attention_forward(p['q'], p['k'], p['v'], p['decay'], out, state=p['state'], state_out=p['state'])
    assert np.array_equal(h.get_numpy_copy(p['state']), apart['state_out'])
    assert np.array_equal(h.get_numpy_copy(out), apart['out'])


@pytest.mark.gpu
def test_pieces_of_a_sequence_equal_the_whole(handler):
    """A prompt in two calls that hand the state on, then single steps: the same stream of outputs."""
    h, T = handler, 150
    d = _case(T, 2, 4, 2, 64, 48, seed=9)
    p = {n: h.create_from_numpy(a) for n, a in d.items() if a is not None}
    out, state = h.zeros((T, 2, 4, 48)), h.create_from_numpy(d['state'])
    for a, b in ((0, 70), (70, 147)):
        h.linear_attention_forward(p['q'][a:b], p['k'][a:b], p['v'][a:b], p['decay'], out[a:b], state=state, state_out=state)
    for t in range(147, T):
        h.linear_attention_step(p['q'][t], p['k'][t], p['v'][t], p['decay'], state, out[t])
    want = ref.attention(d['q'], d['k'], d['v'], d['decay'], 1.0, d['state'])
    for got, w, bound, name in zip((out, state), want, _bound(d, 1.0, False), ('out', 'state')):
        _check(h.get_numpy_copy(got), w, bound, name)


@pytest.mark.gpu
@pytest.mark.parametrize('T', [6, 140])
def test_gradients_against_differences(handler, T):
    """Directional derivatives of the 64-bit forward pass along the kernel's gradients' own inputs."""
    d = _case(T, 2, 2, 1, 16, 24, seed=10, ragged=True)
    got = _run(handler, d, 0.3)
    rs = np.random.RandomState(11)

    def loss(e):
        x = {n: d[n].astype(np.float64) + e * way[n] for n in ('q', 'k', 'v', 'state')}
        out, state = ref.attention(x['q'], x['k'], x['v'], d['decay'], 0.3, x['state'], d['lengths'])
        return (out * d['dout']).sum() + (state * d['dstate_out']).sum()
    for name in ('q', 'k', 'v', 'state'):
        way = {n: rs.standard_normal(d[n].shape) * (n == name) for n in ('q', 'k', 'v', 'state')}
        # the loss is linear in each operand: a difference over any distance is its derivative, to rounding in 64 bits
        slope = (loss(1.0) - loss(-1.0)) / 2
        terms = got['d' + name].astype(np.float64) * way[name]
        bound = (np.abs(way[name]) * dict(zip(('q', 'k', 'v', 'state'), _bound(d, 0.3, True)))[name]).sum()
        assert abs(terms.sum() - slope) <= bound + 1e-9 * np.abs(terms).sum(), name


@pytest.mark.gpu
@pytest.mark.parametrize('T', [20, 200])
def test_extreme_magnitudes(handler, T):
    """Operands around 1e-15 and 1e15, and a head that is all zero."""
    d = _case(T, 2, 3, 3, 32, 32, seed=12)
    d['q'] *= np.float32(1e-15)
    d['k'] *= np.float32(1e15)
    d['v'] *= np.float32(1e-12)
    d['dout'] *= np.float32(1e10)
    d['k'][:, :, 1] = 0
    d['state'] *= 1000
    got = _run(handler, d)
    out, state = ref.attention(d['q'], d['k'], d['v'], d['decay'], 1.0, d['state'])
    for name, want, bound in zip(('out', 'state_out'), (out, state), _bound(d, 1.0, False)):
        _check(got[name], want, bound, name)
    wants = ref.attention_backward(d['q'], d['k'], d['v'], d['decay'], d['dout'], 1.0, d['state'], d['dstate_out'])
    for name, want, bound in zip(('dq', 'dk', 'dv', 'dstate'), wants, _bound(d, 1.0, True)):
        _check(got[name], want, bound, name)


@pytest.mark.gpu
@pytest.mark.parametrize('value', [np.nan, np.inf])
def test_a_value_that_is_not_finite_stays_in_its_sequence_head_and_future(handler, value):
    T, at = 200, 130
    d = _case(T, 2, 2, 2, 32, 32, seed=13)
    want = _run(handler, d, backward=False)
    d['v'][at, 0, 1, 5] = value
    got = _run(handler, d, backward=False)['out']
    assert np.array_equal(got[:, 1], want['out'][:, 1]) and np.array_equal(got[:, 0, 0], want['out'][:, 0, 0])
    assert np.array_equal(got[:at - 15, 0, 1], want['out'][:at - 15, 0, 1])     # up to 15 tokens before it may be lost
    assert not np.isfinite(got[at:, 0, 1, 5]).any()
    rest = np.arange(32) != 5
    assert np.isfinite(got[:, 0, 1][:, rest]).all()


@pytest.mark.gpu
def test_same_bits_every_time_and_when_replayed(handler):
    h = handler
    d = _case(300, 2, 4, 2, 64, 64, seed=14, ragged=True)
    first = _run(h, d, 0.125)
    for _ in range(3):
        again = _run(h, d, 0.125)
        assert all(np.array_equal(first[n], again[n]) for n in first)
    p = {n: None if a is None else h.create_from_numpy(a) for n, a in d.items()}
    o = {n: h.zeros(a.shape) for n, a in first.items()}

    def step():
        h.linear_attention_forward(p['q'], p['k'], p['v'], p['decay'], o['out'], scale=0.125, state=p['state'], state_out=o['state_out'],
                                   lengths=p['lengths'])
        h.linear_attention_backward(p['q'], p['k'], p['v'], p['decay'], p['dout'], o['dq'], o['dk'], o['dv'], scale=0.125, state=p['state'],
                                    dstate_out=p['dstate_out'], dstate=o['dstate'], lengths=p['lengths'], accumulate=False)
    step()
    recorded, second = h.record(step), h.record(step)     # two recordings, their workspaces apart
    for r in (recorded, second, recorded):
        for a in o.values():
            h.fill(a, np.nan)
        r.launch()
        step()                                            # an ordinary call between replays
        r.launch()
        for n in first:
            assert np.array_equal(h.get_numpy_copy(o[n]), first[n]), n
    recorded.release()
    second.release()


@pytest.mark.gpu
def test_on_the_side_stream(handler):
    from brainstorm_b200 import lib
    from brainstorm_b200._lib import check
    import ctypes
    h = handler
    d = _case(400, 2, 4, 4, 64, 64, seed=15)
    want = _run(h, d)
    p = {n: h.create_from_numpy(a) for n, a in d.items() if a is not None}
    out = [h.zeros((400, 2, 4, 64)) for _ in range(2)]
    mark = ctypes.c_uint64()
    check(lib.b200_mark_create(ctypes.byref(mark)))
    check(lib.b200_mark(mark.value))
    check(lib.b200_use_stream(1))
    try:
        check(lib.b200_wait_mark(mark.value))
        h.linear_attention_forward(p['q'], p['k'], p['v'], p['decay'], out[0], state=p['state'])
        check(lib.b200_mark(mark.value))
    finally:
        check(lib.b200_use_stream(0))
    h.linear_attention_forward(p['q'], p['k'], p['v'], p['decay'], out[1], state=p['state'])     # at the same time on the main stream
    check(lib.b200_wait_mark(mark.value))
    for o in out:
        assert np.array_equal(h.get_numpy_copy(o), want['out'])
    check(lib.b200_mark_destroy(mark.value))


@pytest.mark.gpu
def test_lengths_are_truncated_and_held_to_the_sequence(handler):
    d = _case(30, 5, 2, 2, 16, 16, seed=16)
    d['lengths'] = np.float32([7.9, -3, 1e9, np.nan, 0.5])
    got = _run(handler, d, backward=False)
    out, state = ref.attention(d['q'], d['k'], d['v'], d['decay'], 1.0, d['state'], d['lengths'])
    for name, want, bound in zip(('out', 'state_out'), (out, state), _bound(d, 1.0, False)):
        _check(got[name], want, bound, name)


@pytest.mark.gpu
def test_empty_extents(handler):
    h = handler
    for T, B, H in ((0, 2, 2), (5, 0, 2), (5, 2, 0)):
        z = lambda *s: h.ones(s)  # noqa: E731
        state_out, grads = z(B, H, 8, 8), [z(T, B, H, 8) for _ in range(3)]
        h.linear_attention_forward(z(T, B, H, 8), z(T, B, H, 8), z(T, B, H, 8), z(H), z(T, B, H, 8), state=z(B, H, 8, 8), state_out=state_out)
        assert (h.get_numpy_copy(state_out) == 1).all()
        h.linear_attention_backward(z(T, B, H, 8), z(T, B, H, 8), z(T, B, H, 8), z(H), z(T, B, H, 8), *grads)


class _Shape(object):
    """Enough of an array for the checks, which come before any launch."""
    _contig, ptr = True, 0

    def __new__(cls, *shape, at=0):
        from brainstorm_b200 import B200Array
        return B200Array(None, at, tuple(shape))


def _calls():
    from brainstorm_b200.sequence_ops import SequenceOps
    return SequenceOps()


@pytest.mark.parametrize('change, error', [
    ({'k': (4, 2, 3, 8), 'v': (4, 2, 3, 8)}, 'cannot share'), ({'k': (4, 2, 2, 9)}, 'do not agree'), ({'v': (5, 2, 2, 8)}, 'do not agree'), ({'q': (4, 2, 8)}, '4 dimensions'),
    ({'out': (4, 2, 4, 9)}, 'out has shape'), ({'state': (2, 4, 8, 9)}, 'state has shape'), ({'state_out': (1, 4, 8, 8)}, 'state_out has shape'),
    ({'decay': (3,)}, 'decay has 3'), ({'lengths': (3,)}, 'lengths has 3')])
def test_refusals(change, error):
    shapes = {'q': (4, 2, 4, 8), 'k': (4, 2, 2, 8), 'v': (4, 2, 2, 8), 'decay': (4,), 'out': (4, 2, 4, 8), 'state': (2, 4, 8, 8),
              'state_out': (2, 4, 8, 8), 'lengths': (2,)}
    shapes.update(change)
    a = {n: _Shape(*s, at=(i + 1) << 20) for i, (n, s) in enumerate(shapes.items())}
    with pytest.raises(ValueError, match=error):
        _calls().linear_attention_forward(a['q'], a['k'], a['v'], a['decay'], a['out'], state=a['state'], state_out=a['state_out'], lengths=a['lengths'])


def test_refusals_of_overlaps_and_strides():
    s = lambda i, *shape: _Shape(*shape, at=(i + 1) << 20)  # noqa: E731
    q, k, v, decay, out = s(0, 4, 2, 4, 8), s(1, 4, 2, 2, 8), s(2, 4, 2, 2, 8), s(3, 4), s(4, 4, 2, 4, 8)
    with pytest.raises(ValueError, match='out overlaps q'):
        _calls().linear_attention_forward(q, k, v, decay, q)
    with pytest.raises(ValueError, match='out overlaps q'):
        _calls().linear_attention_forward(q, k, v, decay, _Shape(4, 2, 4, 8, at=q.ptr + 64))
    with pytest.raises(NotImplementedError, match='contiguous'):
        _calls().linear_attention_forward(s(0, 4, 2, 4, 16)[:, :, :, ::2], k, v, decay, out)
    with pytest.raises(ValueError, match='dq overlaps dout'):
        _calls().linear_attention_backward(q, k, v, decay, out, out, s(5, 4, 2, 2, 8), s(6, 4, 2, 2, 8))
    with pytest.raises(ValueError, match='dv overlaps dk'):
        _calls().linear_attention_backward(q, k, v, decay, out, s(5, 4, 2, 4, 8), s(6, 4, 2, 2, 8), s(6, 4, 2, 2, 8))
    state = s(9, 2, 4, 8, 8)
    with pytest.raises(ValueError, match='dstate overlaps dstate_out'):
        _calls().linear_attention_backward(q, k, v, decay, out, s(5, 4, 2, 4, 8), s(6, 4, 2, 2, 8), s(7, 4, 2, 2, 8), dstate_out=state, dstate=state)
    with pytest.raises(ValueError, match='3 dimensions'):
        _calls().linear_attention_step(q, k, v, decay, s(5, 2, 4, 8, 8), out)


@pytest.mark.gpu
def test_refusals_of_the_library(handler):
    from brainstorm_b200 import B200Error
    h, z = handler, lambda *s: handler.zeros(s)
    for dk, dv in ((129, 8), (8, 200), (0, 8), (8, 0)):
        with pytest.raises(B200Error, match='values'):
            h.linear_attention_forward(z(2, 1, 1, dk), z(2, 1, 1, dk), z(2, 1, 1, dv), z(1), z(2, 1, 1, dv))


@pytest.mark.gpu
@pytest.mark.parametrize('dv', [128, 127])
def test_states_beyond_32_bit_offsets(handler, dv):
    """8.7 GB of states, of which the last one is not zero: the address of a state does not fit 32 bits."""
    h, (B, H, dk) = handler, (33300, 4, 128)
    rng = np.random.RandomState(21)
    q, k, v, s = rng.randn(dk), rng.randn(dk), rng.randn(dv), rng.randn(dk, dv)
    up = {n: h.zeros(shape) for n, shape in (('q', (B, H, dk)), ('k', (B, H, dk)), ('v', (B, H, dv)), ('out', (B, H, dv)), ('state', (B, H, dk, dv)))}
    assert up['state'].size > 2 ** 31
    for n, x in (('q', q), ('k', k), ('v', v), ('state', s)):
        h.set_from_numpy(up[n][B - 1, H - 1], x.astype(np.float32))
    h.linear_attention_step(up['q'], up['k'], up['v'], h.create_from_numpy(np.full(H, 0.5, np.float32)), up['state'], up['out'])
    q, k, v, s = (x.astype(np.float32).astype(np.float64) for x in (q, k, v, s))
    want = 0.5 * s + np.outer(k, v)
    # a state: two products and a sum, three half steps; an output: those, a product and a sum of 128 terms
    assert (np.abs(h.get_numpy_copy(up['state'][B - 1, H - 1]) - want) <= 3 * U * (0.5 * np.abs(s) + np.abs(np.outer(k, v)))).all()
    bound = 132 * U * (np.abs(q) @ (0.5 * np.abs(s) + np.abs(np.outer(k, v))))
    assert (np.abs(h.get_numpy_copy(up['out'][B - 1, H - 1]) - q @ want) <= bound).all()
    assert not h.get_numpy_copy(up['out'][:B - 1]).any() and not h.get_numpy_copy(up['state'][0]).any()


# more blocks than the GPU has SMs: four warps a block instead of eight
@pytest.mark.gpu
@pytest.mark.parametrize('shape, ragged, decays', [((70, 40, 8, 4, 64, 64), True, None), ((129, 20, 8, 2, 48, 80), True, None), ((100, 20, 8, 8, 128, 128), False, None),
                                                   ((65, 26, 6, 3, 33, 31), True, None), ((80, 40, 4, 4, 127, 126), True, None), ((150, 40, 4, 2, 96, 64), True, [1.0, 0.0, 0.5]),
                                                   ((40, 100, 2, 2, 5, 128), True, [-0.75, 1.0]), ((9, 200, 1, 1, 17, 20), True, None), ((600, 38, 2, 1, 80, 48), True, None)])
def test_many_sequences(handler, shape, ragged, decays):
    d = _case(*shape, seed=sum(shape), ragged=ragged, decays=decays)
    scale = shape[4] ** -0.5
    got = _run(handler, d, scale)
    out, state = ref.attention(d['q'], d['k'], d['v'], d['decay'], scale, d['state'], d['lengths'])
    for name, want, bound in zip(('out', 'state_out'), (out, state), _bound(d, scale, False)):
        _check(got[name], want, bound, name)
    wants = ref.attention_backward(d['q'], d['k'], d['v'], d['decay'], d['dout'], scale, d['state'], d['dstate_out'], d['lengths'])
    for name, want, bound in zip(('dq', 'dk', 'dv', 'dstate'), wants, _bound(d, scale, True)):
        _check(got[name], want, bound, name)
    more = _run(handler, d, scale, accumulate=True)       # onto ones
    for name in ('dq', 'dk', 'dv'):
        # rounding the sum with one, and the one or two sums in between
        assert (np.abs(more[name] - (got[name].astype(np.float64) + 1)) <= 4 * U * (np.abs(got[name]) + 1)).all(), name


@pytest.mark.gpu
@pytest.mark.parametrize('dk', [32, 96])
@pytest.mark.parametrize('name', ['q', 'k', 'v'])
@pytest.mark.parametrize('value', [np.nan, np.inf])
def test_a_value_that_is_not_finite_among_many_sequences(handler, value, name, dk):
    T, at = 140, 90
    d = _case(T, 90, 2, 2, dk, 32, seed=17)
    want = _run(handler, d, backward=False)
    d[name][at, 50, 1, 5] = value
    got = _run(handler, d, backward=False)['out']
    same = np.ones(got.shape[1:3], bool)
    same[50, 1] = False
    assert np.array_equal(got[:, same], want['out'][:, same])
    assert np.array_equal(got[:at - 15, 50, 1], want['out'][:at - 15, 50, 1])
    assert not np.isfinite(got[at, 50, 1, 5])
    if name == 'q':
        assert np.array_equal(got[at + 1:, 50, 1], want['out'][at + 1:, 50, 1])
    else:
        assert not np.isfinite(got[at:, 50, 1, 5]).any()


@pytest.mark.gpu
@pytest.mark.parametrize('lengths', [False, True])
@pytest.mark.parametrize('shift, shift_out', [(0, None), (1, None), (0, 2), (3, 3)])
@pytest.mark.parametrize('dk, dv', [(52, 15), (127, 126), (16, 17), (5, 3), (90, 97), (64, 64), (1, 1), (1, 3), (128, 1), (3, 128), (30, 50)])
def test_a_token_for_many_streams(handler, dk, dv, shift, shift_out, lengths):
    """States that start `shift` floats behind a 16-byte boundary; in place, or into another array that starts elsewhere."""
    h, (B, H, K) = handler, (307, 4, 2)
    d = _case(1, B, H, K, dk, dv, seed=dk + dv)
    if lengths:
        d['lengths'] = (np.arange(B) % 3 > 0).astype(np.float32)
    p = {n: None if a is None else h.create_from_numpy(a) for n, a in _poison(d).items()}
    size = B * H * dk * dv

    def at(offset):
        flat = h.create_from_numpy(np.full(size + 8, 7.0, np.float32))
        return flat, flat[offset:offset + size].reshape((B, H, dk, dv))
    flat, state = at(shift)
    flat_out, state_out = (flat, state) if shift_out is None else at(shift_out)
    h.set_from_numpy(state, d['state'])
    out = h.ones((1, B, H, dv))
    h.linear_attention_forward(p['q'], p['k'], p['v'], p['decay'], out, scale=0.5, state=state, state_out=state_out, lengths=p['lengths'])
    want, want_state = ref.attention(d['q'], d['k'], d['v'], d['decay'], 0.5, d['state'], d['lengths'])
    for got, w, bound, what in zip((out, state_out), (want, want_state), _bound(d, 0.5, False), ('out', 'state')):
        _check(h.get_numpy_copy(got), w, bound, what)
    if lengths:
        assert np.array_equal(h.get_numpy_copy(state_out)[::3], d['state'][::3]) and not h.get_numpy_copy(out)[0, ::3].any()
    offset = shift if shift_out is None else shift_out
    around = h.get_numpy_copy(flat_out)
    assert (around[:offset] == 7).all() and (around[offset + size:] == 7).all()

"""Decayed linear attention over tokens of very different size.  A token's output does not depend on later tokens at all.

Tolerance.  That of ``test_linear_attention``, TERMS * U * the same sum with absolute values, holds while both halves of
every operand are normal numbers.  The chunked form scales a token's row of q, k, v or dout, a row of scores, the weighted
keys of a chunk and the state by the power of two that takes the largest value into [2^13, 2^14); its two
half-precision parts end at 2^-24, so an operand is also off by up to 2^-25 / 2^13 = 2^-38 of that largest value,
whatever its own size.  With every row replaced by its largest value, and states by theirs, let M be the same sum of absolute
values.  The rows of q, k, v and the state enter once each: their part is at most 4 * 2^-38 M.  A score is off by 2^-38 of the largest of its
row, which with its v is at most M / dk; up to 64 tokens of a chunk have one: 64 * 2^-38 M.  A weighted key is off by 2^-38 of
the chunk's largest, up to 64 tokens again, and ends in the state: 64 * 2^-38 M.  Together less than 2^-30 M, with room for the
products of two of these errors and the scores' way through them.
"""
import numpy as np
import pytest

import sequence_reference as ref
from test_linear_attention import _bound, _case, _check, _run

# time, batch, heads, key/value heads, dk, dv: the recurrent form; few and many blocks of both widths; segments; sizes off the tiles
SHAPES = [(8, 2, 4, 2, 64, 48), (64, 2, 4, 2, 64, 64), (100, 1, 4, 4, 128, 128), (150, 2, 4, 2, 48, 80), (90, 40, 4, 4, 64, 64), (90, 40, 4, 2, 40, 72), (80, 40, 4, 4, 127, 126),
          (1100, 1, 4, 4, 48, 48), (1030, 1, 4, 2, 128, 96), (1000, 1, 4, 2, 33, 70)]
DECAYS = [0.99, 0.0, 1.0, 0.3]


@pytest.fixture(scope='module')
def handler():
    from brainstorm_b200 import B200Handler
    return B200Handler(seed=0)


def _all(d, scale):
    out = ref.attention(d['q'], d['k'], d['v'], d['decay'], scale, d['state'], d['lengths'])
    grads = ref.attention_backward(d['q'], d['k'], d['v'], d['decay'], d['dout'], scale, d['state'], d['dstate_out'], d['lengths'])
    return dict(zip(('out', 'state_out', 'dq', 'dk', 'dv', 'dstate'), out + grads))


def _bounds(d, scale):
    rows = dict(d)
    for name in ('q', 'k', 'v', 'dout', 'state', 'dstate_out'):
        over = (-2, -1) if 'state' in name else -1
        rows[name] = np.broadcast_to(np.abs(d[name]).max(over, keepdims=True), d[name].shape)
    rows['decay'] = np.abs(d['decay'])
    return {name: a + 2.0 ** -30 * m for (name, m), a in zip(_all(rows, scale).items(), _bound(d, scale, False) + _bound(d, scale, True))}


def _check_all(h, d, scale=0.125):
    got, want, bound = _run(h, d, scale), _all(d, scale), _bounds(d, scale)
    for name in want:
        _check(got[name], want[name], bound[name], name)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize('power', [20, 40, -40])
@pytest.mark.parametrize('name', ['q', 'k', 'v', 'dout'])
@pytest.mark.parametrize('shape', SHAPES)
def test_one_token_of_another_size(handler, shape, name, power):
    d = _case(*shape, seed=sum(shape), decays=DECAYS)
    at = shape[0] * 3 // 5
    plain = _run(handler, d, 0.125)
    d[name][at] *= np.float32(2.0 ** power)
    got = _check_all(handler, d)
    if name in ('k', 'v'):      # what comes before the token, seen in the direction of each result, keeps its bits
        assert np.array_equal(got['out'][:at], plain['out'][:at]) and np.array_equal(got['dq'][:at], plain['dq'][:at])
    if name in ('q', 'dout'):
        assert np.array_equal(got['dk'][at + 1:], plain['dk'][at + 1:]) and np.array_equal(got['dv'][at + 1:], plain['dv'][at + 1:])


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(100, 2, 4, 2, 64, 64), (130, 1, 4, 4, 128, 128), (90, 40, 4, 2, 40, 72), (1100, 1, 4, 4, 48, 48)])
def test_every_token_of_its_own_size(handler, shape):
    """Sizes from 2^-30 to 2^30, drawn for each token, head and operand."""
    d = _case(*shape, seed=sum(shape), decays=DECAYS)
    rs = np.random.RandomState(1)
    for name in ('q', 'k', 'v', 'dout'):
        d[name] *= np.exp2(rs.randint(-30, 31, d[name].shape[:3]))[..., None].astype(np.float32)
    _check_all(handler, d, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize('T', [70, 700])
def test_keys_and_values_whose_product_is_outside_the_range_of_their_scales(handler, T):
    """Keys near 2^100 with values near 2^-100 and the other way round, and queries that bring the scores back."""
    d = _case(T, 2, 4, 4, 32, 32, seed=2, decays=DECAYS)
    for b, power in enumerate((100, -100)):
        d['q'][:, b] *= np.float32(2.0 ** -power)
        d['k'][:, b] *= np.float32(2.0 ** power)
        d['v'][:, b] *= np.float32(2.0 ** -power)
        d['dout'][:, b] *= np.float32(2.0 ** power)
        d['state'][b] *= np.float32(2.0 ** 20)
    got, want, bound = _run(handler, d), _all(d, 1.0), _bounds(d, 1.0)
    for name in ('out', 'state_out'):
        _check(got[name], want[name], bound[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize('T', [9, 70, 700])
def test_queries_near_the_end_of_float32(handler, T):
    """Queries near 2^112 with keys near 2^-112, and the other way round: the scores are of ordinary size."""
    d = _case(T, 2, 4, 2, 32, 32, seed=6, decays=DECAYS)
    for b, power in enumerate((112, -112)):
        d['q'][:, b] *= np.float32(2.0 ** power)
        d['k'][:, b] *= np.float32(2.0 ** -power)
        d['state'][b] *= np.float32(2.0 ** -power)
    _check_all(handler, d, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize('T', [8, 60])
def test_a_prompt_agrees_with_answering_token_by_token(handler, T):
    """The two forms, on tokens of which the last is by far the largest."""
    h, (B, H, dk, dv) = handler, (2, 4, 64, 64)
    d = _case(T, B, H, H, dk, dv, seed=3, decays=DECAYS)
    d['k'][T - 1] *= np.float32(2.0 ** 40)
    whole = _run(h, d, backward=False)
    p = {n: h.create_from_numpy(a) for n, a in d.items() if a is not None}
    out = h.zeros((T, B, H, dv))
    for t in range(T):
        h.linear_attention_step(p['q'][t], p['k'][t], p['v'][t], p['decay'], p['state'], out[t])
    bound = _bounds(d, 1.0)
    for name, a in (('out', out), ('state_out', p['state'])):
        _check(whole[name], h.get_numpy_copy(a).astype(np.float64), 2 * bound[name], 'two forms')


@pytest.mark.gpu
@pytest.mark.parametrize('scale', [1.0, 4.0])
@pytest.mark.parametrize('decay', [30.0, -1e6])
@pytest.mark.parametrize('T, B', [(8, 2), (60, 2), (200, 40), (700, 1)])
def test_powers_of_a_large_decay_beyond_float32_meet_zeros(handler, T, B, decay, scale):
    """Keys before the last four tokens, or gradients behind the first four, are zero: powers of the decay that leave the range
    of float32 multiply nothing else."""
    d = _case(T, B, 2, 2, 32, 40, seed=4, decays=[decay, 0.5])
    d['k'][:T - 4], d['state'][:] = 0, 0
    with np.errstate(all='ignore'):
        got, want, bound = _run(handler, d, scale, backward=False), _all(d, scale), _bounds(d, scale)
    for name in ('out', 'state_out'):
        _check(got[name], want[name], bound[name], name)
    d = _case(T, B, 2, 2, 32, 40, seed=5, decays=[decay, 0.5])
    for name in ('dout', 'k', 'v'):
        d[name][4:] = 0
    d['state'][:], d['dstate_out'][:] = 0, 0
    with np.errstate(all='ignore'):                       # the states behind the first tokens do overflow
        got, want, bound = _run(handler, d, scale), _all(d, scale), _bounds(d, scale)
    for name in ('dk', 'dv', 'dstate', 'dq'):
        n = 4 if name == 'dq' else None
        _check(got[name][:n], want[name][:n], bound[name][:n], name)

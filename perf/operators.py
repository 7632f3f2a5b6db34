"""Cases of the sequence-block operators: decayed linear attention (whole prompts, training, single steps), the
norms, gate and residual around a block, and the update of a weight matrix with orthogonalised momentum.

``run`` computes the plain form with elementary torch operations in 32 bits, or, where ``own`` is true, makes the
handler calls a program makes.  Arrays are laid out as the framework lays out its sequence buffers: time first,
then batch, features last, float32 throughout; lengths are float32 values that hold whole numbers, like labels.
"""
import math

import torch

own = False

F32, F64 = torch.float32, torch.float64
DEVICE = 'cuda'


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the first words of one stream: a call that is all latency
        {'name': 'prompt_words', 'kind': 'prompt', 'time': 24, 'batch': 1, 'heads': 8, 'kv_heads': 8, 'dk': 64, 'dv': 64, 'ragged': False},
        # long documents read before an answer; few streams, so the time axis has to be shared out
        {'name': 'prompt_long', 'kind': 'prompt', 'time': 8192, 'batch': 2, 'heads': 16, 'kv_heads': 16, 'dk': 128, 'dv': 128, 'ragged': False},
        # the time and batch extents of the character-model benchmark, with 16 heads of 64 for its 1000 units
        {'name': 'train_characters', 'kind': 'train', 'time': 100, 'batch': 128, 'heads': 16, 'kv_heads': 16, 'dk': 64, 'dv': 64, 'ragged': False},
        # a padded batch of documents with carried state, shared key/value heads and head sizes off every tile
        {'name': 'train_ragged', 'kind': 'train', 'time': 1999, 'batch': 6, 'heads': 12, 'kv_heads': 4, 'dk': 48, 'dv': 80, 'ragged': True},
        # one token of one stream
        {'name': 'step_one', 'kind': 'step', 'batch': 1, 'heads': 16, 'kv_heads': 16, 'dk': 64, 'dv': 64},
        # one token of many streams: the state is all there is to move
        {'name': 'step_streams', 'kind': 'step', 'batch': 512, 'heads': 16, 'kv_heads': 16, 'dk': 128, 'dv': 128},
        # one time step of the character model's batch, forward only (answering)
        {'name': 'norm_step', 'kind': 'norm', 'rows': 128, 'width': 1000, 'act': 'sigmoid', 'backward': False},
        # the batch and width of the Highway benchmark, forward and backward
        {'name': 'norm_train', 'kind': 'norm', 'rows': 8192, 'width': 4096, 'act': 'sigmoid', 'backward': True},
        # a width no vector access divides, a last batch that is not full
        {'name': 'norm_odd', 'kind': 'norm', 'rows': 3001, 'width': 1537, 'act': 'tanh', 'backward': True},
        # the projection of a small model's classes
        {'name': 'muon_small', 'kind': 'muon', 'batch': 1, 'rows': 205, 'cols': 256, 'nesterov': True},
        # the four recurrent matrices of the character model's layer, updated together
        {'name': 'muon_gates', 'kind': 'muon', 'batch': 4, 'rows': 1000, 'cols': 1000, 'nesterov': True},
        # a weight matrix of the Highway benchmark's width
        {'name': 'muon_wide', 'kind': 'muon', 'batch': 1, 'rows': 4096, 'cols': 4096, 'nesterov': True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(['prompt', 'train', 'step', 'norm', 'muon'])
    if kind == 'norm':
        width = _log(rng, 17, 8192)
        return {'kind': kind, 'rows': _log(rng, 1, max(1, 33554432 // width)), 'width': width,
                'act': rng.choice(['sigmoid', 'tanh', 'linear', 'rel', 'el']), 'backward': rng.random() < 0.6}
    if kind == 'muon':
        rows, cols = _log(rng, 16, 4096), _log(rng, 16, 4096)
        return {'kind': kind, 'batch': min(_log(rng, 1, 6), max(1, 16777216 // (rows * cols))), 'rows': rows, 'cols': cols,
                'nesterov': rng.random() < 0.7}
    kv = rng.choice([1, 2, 3, 4, 6, 8])
    heads = kv * rng.choice([1, 1, 1, 2, 4])
    dk, dv = (rng.choice([16, 32, 48, 64, 96, 128]) if rng.random() < 0.6 else rng.randint(8, 128) for _ in range(2))
    if kind == 'step':
        return {'kind': kind, 'batch': _log(rng, 1, max(1, 134217728 // (heads * dk * dv))), 'heads': heads, 'kv_heads': kv, 'dk': dk, 'dv': dv}
    most = (67108864 if kind == 'prompt' else 18000000) // (heads * (dk + dv))
    time = _log(rng, 2, min(8192, most))
    return {'kind': kind, 'time': time, 'batch': _log(rng, 1, max(1, min(256, most // time))), 'heads': heads, 'kv_heads': kv,
            'dk': dk, 'dv': dv, 'ragged': rng.random() < 0.5}


# ---------------------------------------------------------------------------------------------------- inputs
def _inputs(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    n = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE, dtype=F32)  # noqa: E731
    u = lambda *shape: torch.rand(*shape, generator=g, device=DEVICE, dtype=F32)   # noqa: E731
    kind = case['kind']
    if kind == 'norm':
        N, D = case['rows'], case['width']
        t = {'x': n(N, D) * 2, 'y': n(N, D) * (0.5 + u(N, 1)), 'gate': n(N, D), 'w_post': 1 + 0.1 * n(D), 'scale': 0.1 + 0.05 * n(D),
             'w_pre': 1 + 0.1 * n(D)}
        if case['backward']:
            t |= {'dx_out': n(N, D), 'dh': n(N, D)}
        return t
    if kind == 'muon':
        b, r, c = case['batch'], case['rows'], case['cols']
        k = max(1, min(r, c) // 8)
        # gradients of a layer: a few strong directions (errors times activations) and noise over all of them
        grad = 1e-3 * (n(b, r, k) @ n(b, k, c) / math.sqrt(k) + 0.5 * n(b, r, c))
        return {'param': n(b, r, c) / math.sqrt(c), 'grad': grad, 'momentum': 5e-3 * n(b, r, c)}
    B, H, K, dk, dv = (case[k] for k in ('batch', 'heads', 'kv_heads', 'dk', 'dv'))
    decay = (1 - torch.exp2(-2 - 8 * u(H))).to(F32)
    if kind == 'step':
        return {'q': n(B, H, dk), 'k': n(B, K, dk), 'v': n(B, K, dv), 'decay': decay, 'state': 3 * n(B, H, dk, dv)}
    T = case['time']
    t = {'q': n(T, B, H, dk), 'k': n(T, B, K, dk), 'v': n(T, B, K, dv), 'decay': decay, 'state': n(B, H, dk, dv)}
    if case['ragged']:   # a padded batch: one full row, one that ended before it began, the rest anywhere
        lengths = torch.floor(u(B) * (T + 1)).clamp_(max=T)
        lengths[0] = T
        lengths[1:2] = 0
        t['lengths'] = lengths
    if kind == 'train':
        t |= {'dout': n(T, B, H, dv), 'dstate_out': n(B, H, dk, dv)}
    return t


def _outputs(case, t):
    like = torch.empty_like
    if case['kind'] == 'norm':
        rows = t['x'].new_empty(case['rows'])
        o = {'x_out': like(t['x']), 'h_out': like(t['x']), 'r_post': rows, 'r_pre': like(rows)}
        if case['backward']:
            o |= {'dx': like(t['x']), 'dy': like(t['x']), 'dgate': like(t['x']), 'dw_post': like(t['w_post']), 'dscale': like(t['scale']),
                  'dw_pre': like(t['w_pre'])}
        return o
    if case['kind'] == 'muon':
        return {'update': like(t['param'])}
    o = {'out': t['q'].new_empty(tuple(t['q'].shape[:-1]) + (case['dv'],))}
    if case['kind'] != 'step':
        o['state_out'] = like(t['state'])
    if case['kind'] == 'train':
        o |= {'dq': like(t['q']), 'dk': like(t['k']), 'dv': like(t['v']), 'dstate': like(t['state'])}
    return o


_the_handler = []


def _handler():
    if not _the_handler:
        from brainstorm_b200 import B200Handler
        _the_handler.append(B200Handler(seed=0, device=torch.cuda.current_device()))
    return _the_handler[0]


def prepare(case, seed):
    t = _inputs(case, seed)
    state = {'case': dict(case), 'in': t, 'out': _outputs(case, t)}
    if own:   # the same memory as the framework's arrays
        from brainstorm_b200 import B200Array
        state['handler'] = _handler()
        state['arrays'] = {k: B200Array(x, x.data_ptr(), tuple(x.shape)) for k, x in (t | state['out']).items()}
        torch.cuda.synchronize()     # made on torch's stream, used on the handler's
    return state


# ---------------------------------------------------------------------------------------------------- plain forms
CHUNK = 64


def _power(decay, exponent, ndim):
    """decay[h] ** exponent in 64 bits, rounded once; exponent (...,) -> (..., H)."""
    e = exponent.to(F64).unsqueeze(-1)
    return (decay.to(F64) ** e).to(F32)


def _decayed(q, k, v, decay, reverse=False):
    """out[t] = sum over s <= t (s >= t in reverse) of decay^|t-s| (q[t].k[s]) v[s]; (T, B, H, d) arrays."""
    T, B, H, dk = q.shape
    dv = v.shape[-1]
    if reverse:
        q, k, v = q.flip(0), k.flip(0), v.flip(0)
    N = -(-T // CHUNK)

    def chunks(x):
        x = torch.cat([x, x.new_zeros((N * CHUNK - T,) + tuple(x.shape[1:]))])
        return x.reshape(N, CHUNK, B, H, x.shape[-1]).permute(2, 3, 0, 1, 4)     # (B, H, N, C, d)
    q, k, v = chunks(q), chunks(k), chunks(v)
    i = torch.arange(CHUNK, device=q.device)
    apart = (i[:, None] - i[None, :])
    weight = _power(decay, apart.clamp(min=0), 3).permute(2, 0, 1) * (apart >= 0)            # (H, C, C)
    out = (q @ k.transpose(-1, -2) * weight[None, :, None]) @ v
    to_end = _power(decay, CHUNK - 1 - i, 2).t()[None, :, None, :, None]
    added = (k * to_end).transpose(-1, -2) @ v                                              # (B, H, N, dk, dv)
    n = torch.arange(N, device=q.device)
    before = n[:, None] - 1 - n[None, :]
    carry = _power(decay, before.clamp(min=0) * CHUNK, 3).permute(2, 0, 1) * (before >= 0)   # (H, N, N)
    state = (carry[None] @ added.reshape(B, H, N, dk * dv)).reshape(B, H, N, dk, dv)
    from_start = _power(decay, i + 1, 2).t()[None, :, None, :, None]
    out = out + (q * from_start) @ state
    out = out.permute(2, 3, 0, 1, 4).reshape(N * CHUNK, B, H, dv)[:T]
    return out.flip(0) if reverse else out


def _attend(case, t, o):
    T, B, H, K = case['time'], case['batch'], case['heads'], case['kv_heads']
    scale, decay, S0 = case['dk'] ** -0.5, t['decay'], t['state']
    at = torch.arange(T, device=S0.device)[:, None].expand(T, B)
    n = t['lengths'].long() if 'lengths' in t else torch.full((B,), T, device=S0.device)
    live = (at < n)[..., None, None]
    q = torch.where(live, t['q'] * scale, 0)
    k, v = (torch.where(live, t[x], 0).repeat_interleave(H // K, dim=2) for x in 'kv')
    since = _power(decay, at + 1, 3)[..., None]                                  # (T, B, H, 1)
    until = torch.where(live, _power(decay, (n - 1 - at).clamp(min=0), 3)[..., None], 0)
    whole = _power(decay, n, 2)[..., None, None]
    o['out'] = torch.where(live, _decayed(q, k, v, decay) + torch.einsum('tbhd,bhde->tbhe', q * since, S0), 0)
    o['state_out'] = whole * S0 + torch.einsum('tbhd,tbhe->bhde', k * until, v)
    if case['kind'] == 'train':
        do, dS = torch.where(live, t['dout'], 0), t['dstate_out']
        shared = lambda x: x.reshape(T, B, K, H // K, x.shape[-1]).sum(3)  # noqa: E731
        dq = _decayed(do, v, k, decay) + torch.einsum('tbhe,bhde->tbhd', do * since, S0)
        o['dq'] = torch.where(live, dq * scale, 0)
        o['dk'] = shared(_decayed(v, do, q, decay, True) + torch.einsum('tbhe,bhde->tbhd', v * until, dS))
        o['dv'] = shared(_decayed(k, q, do, decay, True) + torch.einsum('tbhd,bhde->tbhe', k * until, dS))
        o['dstate'] = whole * dS + torch.einsum('tbhd,tbhe->bhde', q * since, do)
    return o


def _step(case, t, o):
    g = case['heads'] // case['kv_heads']
    k, v = (t[x].repeat_interleave(g, dim=1) for x in 'kv')
    t['state'].copy_(t['decay'][None, :, None, None] * t['state'] + k[..., :, None] * v[..., None, :])
    o['out'] = torch.einsum('bhd,bhde->bhe', t['q'] * case['dk'] ** -0.5, t['state'])
    return {'out': o['out'], 'state': t['state']}


_ACT = {'sigmoid': (lambda x: 1 / (1 + torch.exp(-x)), lambda y: y * (1 - y)), 'tanh': (torch.tanh, lambda y: 1 - y * y),
        'rel': (lambda x: x * (x > 0), lambda y: (y > 0).to(y.dtype)), 'el': (lambda x: torch.where(x > 0, x, torch.exp(x.clamp(max=0)) - 1), lambda y: torch.where(y > 0, 1.0, y + 1)),
        'linear': (lambda x: x, torch.ones_like)}
EPSILON = 1e-6


def _norm(case, t, o):
    f, df = _ACT[case['act']]
    gate = f(t['gate'])
    o['r_post'] = (t['y'].square().mean(1) + EPSILON).rsqrt()
    y_hat = t['y'] * o['r_post'][:, None]
    o['x_out'] = t['x'] + t['scale'] * gate * (y_hat * t['w_post'])
    o['r_pre'] = (o['x_out'].square().mean(1) + EPSILON).rsqrt()
    x_hat = o['x_out'] * o['r_pre'][:, None]
    o['h_out'] = x_hat * t['w_pre']
    if case['backward']:
        o['dw_pre'] = (t['dh'] * x_hat).sum(0)
        e = t['dh'] * t['w_pre']
        o['dx'] = t['dx_out'] + o['r_pre'][:, None] * (e - x_hat * (e * x_hat).mean(1, keepdim=True))
        d = o['dx'] * t['scale']
        n = y_hat * t['w_post']
        o['dscale'] = (o['dx'] * gate * n).sum(0)
        o['dgate'] = d * n * df(gate)
        d = d * gate
        o['dw_post'] = (d * y_hat).sum(0)
        e = d * t['w_post']
        o['dy'] = o['r_post'][:, None] * (e - y_hat * (e * y_hat).mean(1, keepdim=True))
    return o


RATE, BETA, DECAY, STEPS = 0.02, 0.95, 0.01, 5
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _muon(case, t, o):
    t['momentum'].mul_(BETA).add_(t['grad'])
    X = t['grad'] + BETA * t['momentum'] if case['nesterov'] else t['momentum']
    flat = case['rows'] > case['cols']
    X = X.transpose(1, 2) if flat else X
    X = X / (X.square().sum((1, 2), keepdim=True).sqrt() + 1e-7)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        A = X @ X.transpose(1, 2)
        X = a * X + (b * A + c * (A @ A)) @ X
    o['update'] = X.transpose(1, 2).contiguous() if flat else X
    t['param'].mul_(1 - RATE * DECAY).sub_(RATE * o['update'])
    return {'param': t['param'], 'momentum': t['momentum'], 'update': o['update']}


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    case, kind = state['case'], state['case']['kind']
    if not own:
        o = dict(state['out'])
        return {'prompt': _attend, 'train': _attend, 'step': _step, 'norm': _norm, 'muon': _muon}[kind](case, state['in'], o)
    h, a, out = state['handler'], state['arrays'], state['out']
    if kind in ('prompt', 'train'):
        scale, lengths = case['dk'] ** -0.5, a.get('lengths')
        h.linear_attention_forward(a['q'], a['k'], a['v'], a['decay'], a['out'], scale=scale, state=a['state'], state_out=a['state_out'],
                                   lengths=lengths)
        if kind == 'train':
            h.linear_attention_backward(a['q'], a['k'], a['v'], a['decay'], a['dout'], a['dq'], a['dk'], a['dv'], scale=scale,
                                        state=a['state'], dstate_out=a['dstate_out'], dstate=a['dstate'], lengths=lengths, accumulate=False)
        return out
    if kind == 'step':
        h.linear_attention_step(a['q'], a['k'], a['v'], a['decay'], a['state'], a['out'], scale=case['dk'] ** -0.5)
        return {'out': out['out'], 'state': state['in']['state']}
    if kind == 'norm':
        h.gated_norm_forward(a['x'], a['y'], a['gate'], a['w_post'], a['scale'], a['w_pre'], a['x_out'], a['h_out'], a['r_post'], a['r_pre'],
                             epsilon=EPSILON, activation=case['act'])
        if case['backward']:
            h.gated_norm_backward(a['x_out'], a['y'], a['gate'], a['w_post'], a['scale'], a['w_pre'], a['r_post'], a['r_pre'], a['dx_out'],
                                  a['dh'], a['dx'], a['dy'], a['dgate'], a['dw_post'], a['dscale'], a['dw_pre'], activation=case['act'],
                                  accumulate=False)
        return out
    h.muon_update(a['param'], a['grad'], a['momentum'], a['update'], learning_rate=RATE, beta=BETA, nesterov=case['nesterov'],
                  weight_decay=DECAY, steps=STEPS)
    return {'param': state['in']['param'], 'momentum': state['in']['momentum'], 'update': out['update']}


def work(case):
    kind = case['kind']
    if kind == 'norm':
        # forward: x, y, gate in, x_out, h_out out.  The rest of the network lies between the two calls, so the backward
        # call reads x_out, y, gate again, beside dx_out and dh, and writes three gradients.
        arrays = 13 if case['backward'] else 5
        return {'bytes': 4.0 * arrays * case['rows'] * case['width'], 'flops': (60.0 if case['backward'] else 20.0) * case['rows'] * case['width']}
    if kind == 'muon':
        b, r, c = case['batch'], case['rows'], case['cols']
        m, n = min(r, c), max(r, c)
        # a step: two symmetric products, of which half is enough, and a full one
        return {'bytes': 4.0 * 6 * b * r * c, 'flops': b * STEPS * (m * m * n + m ** 3 + 2.0 * m * m * n)}
    B, H, K, dk, dv = (case[k] for k in ('batch', 'heads', 'kv_heads', 'dk', 'dv'))
    states = 4.0 * B * H * dk * dv
    if kind == 'step':
        return {'bytes': 2 * states + 4.0 * B * (H + K) * (dk + dv), 'flops': 5.0 * B * H * dk * dv}
    rows = case['time'] * B
    # the recurrence itself: a state update and a read for each token; with gradients a second state and three reads more
    forward, backward = 4.0 * rows * (H + K) * (dk + dv), 4.0 * rows * (2 * H * dk + H * dv + 2 * K * (dk + dv))
    if kind == 'prompt':
        return {'bytes': forward + 2 * states, 'flops': 4.0 * rows * H * dk * dv}
    return {'bytes': forward + backward + 5 * states, 'flops': 12.0 * rows * H * dk * dv}


# ---------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    t = {k: x.to(F64) for k, x in _inputs(case, seed).items()}
    kind = case['kind']
    if kind == 'muon':
        # the same polynomial of the other Gram matrix, in Horner's form
        momentum = BETA * t['momentum'] + t['grad']
        X = t['grad'] + BETA * momentum if case['nesterov'] else momentum
        X = X / (torch.linalg.vector_norm(X, dim=(1, 2), keepdim=True) + 1e-7)
        a, b, c = COEFFICIENTS
        tall = case['rows'] > case['cols']
        for _ in range(STEPS):
            G = X.mT @ X if tall else X @ X.mT
            P = torch.diag_embed(G.new_full(G.shape[:2], a)) + b * G + c * (G @ G)
            X = X @ P if tall else P @ X
        return {'param': (1 - RATE * DECAY) * t['param'] - RATE * X, 'momentum': momentum, 'update': X}
    if kind == 'norm':
        f = {'sigmoid': torch.sigmoid, 'tanh': torch.tanh, 'rel': torch.relu, 'el': torch.nn.functional.elu, 'linear': lambda x: x}[case['act']]
        names = ('x', 'y', 'gate', 'w_post', 'scale', 'w_pre')
        p = [t[k].requires_grad_(case['backward']) for k in names]
        x, y, gate, w_post, scale, w_pre = p
        r_post = 1 / torch.sqrt(torch.mean(y * y, 1) + EPSILON)
        x_out = x + f(gate) * scale * w_post * y * r_post[:, None]
        r_pre = 1 / torch.sqrt(torch.mean(x_out * x_out, 1) + EPSILON)
        h_out = w_pre * x_out * r_pre[:, None]
        o = {'x_out': x_out, 'h_out': h_out, 'r_post': r_post, 'r_pre': r_pre}
        if case['backward']:
            grads = torch.autograd.grad([x_out, h_out], p, [t['dx_out'], t['dh']])
            o |= {'d' + k: d for k, d in zip(names, grads)}
        return {k: v.detach() for k, v in o.items()}
    g, scale, decay = case['heads'] // case['kv_heads'], case['dk'] ** -0.5, t['decay'][None, :, None, None]
    wide = lambda x: x.repeat_interleave(g, dim=-2)  # noqa: E731
    S = t['state'].clone()
    if kind == 'step':
        S = decay * S + wide(t['k'])[..., None] * wide(t['v'])[..., None, :]
        return {'out': ((t['q'] * scale)[..., None] * S).sum(-2), 'state': S}
    # the recurrence, token by token; backwards the same with the gradient of the state
    T, B, H = case['time'], case['batch'], case['heads']
    n = t['lengths'].long() if 'lengths' in t else torch.full((B,), T, device=DEVICE)
    o = {'out': t['q'].new_zeros(T, B, H, case['dv'])}
    if kind == 'train':
        o |= {'dq': torch.zeros_like(t['q']), 'dk': torch.zeros_like(t['k']), 'dv': torch.zeros_like(t['v'])}
    for s in range(T):
        live = (s < n)[:, None, None]
        S = torch.where(live[..., None], decay * S + wide(t['k'][s])[..., None] * wide(t['v'][s])[..., None, :], S)
        o['out'][s] = live * torch.matmul(scale * t['q'][s][:, :, None], S)[:, :, 0]
        if kind == 'train':
            o['dq'][s] = live * scale * torch.matmul(S, t['dout'][s][..., None])[..., 0]
    o['state_out'] = S
    if kind == 'train':
        R = t['dstate_out'].clone()
        for s in range(T - 1, -1, -1):
            live = (s < n)[:, None, None]
            M = R + scale * t['q'][s][..., None] * t['dout'][s][..., None, :]
            dk = live * torch.matmul(M, wide(t['v'][s])[..., None])[..., 0]
            dv = live * torch.matmul(wide(t['k'][s])[:, :, None], M)[:, :, 0]
            o['dk'][s] = dk.reshape(B, -1, g, dk.shape[-1]).sum(2)
            o['dv'][s] = dv.reshape(B, -1, g, dv.shape[-1]).sum(2)
            R = torch.where(live[..., None], decay * M, R)
        o['dstate'] = R
    return o

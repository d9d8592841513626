"""Cases for the operators of a deployed W8A8 decoder block: the 8-bit integer linear (per-token quantisation of
the activations and the product with per-channel weights), the gated activation that feeds one, the residual add
with the norms on both sides of it, and the rotary embedding from positions.

Hidden sizes, MLP widths, head counts and sequence lengths are those of the Llama-7B block that the benchmark
quantises (4096, 11008, 32 heads of 128, 2048 tokens a sequence) or generic."""
import math

import torch

own = False

_TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def listed():
    return [
        # one decoding step of one sequence through an attention projection: latency
        {'name': 'linear_token', 'op': 'linear', 'm': 1, 'n': 4096, 'k': 4096, 'type': 'bf16', 'sym': True, 'bias': False},
        # a decoding step of a batch through an MLP projection, activations with a zero point
        {'name': 'linear_batch', 'op': 'linear', 'm': 24, 'n': 11008, 'k': 4096, 'type': 'bf16', 'sym': False, 'bias': True},
        # sizes that divide by nothing, in fp32
        {'name': 'linear_ragged', 'op': 'linear', 'm': 333, 'n': 1001, 'k': 1399, 'type': 'fp32', 'sym': False, 'bias': True},
        # one calibration sequence through an MLP projection
        {'name': 'linear_sequence', 'op': 'linear', 'm': 2048, 'n': 11008, 'k': 4096, 'type': 'bf16', 'sym': True, 'bias': False},
        # eight sequences through the down projection: the largest product
        {'name': 'linear_large', 'op': 'linear', 'm': 16384, 'n': 4096, 'k': 11008, 'type': 'fp16', 'sym': True, 'bias': False},
        # the MLP's second half: gated activation and down projection, a few tokens and one sequence
        {'name': 'down_tokens', 'op': 'down', 'm': 4, 'n': 4096, 'k': 11008, 'type': 'bf16', 'act': 'silu'},
        {'name': 'down_sequence', 'op': 'down', 'm': 2048, 'n': 4096, 'k': 11008, 'type': 'bf16', 'act': 'silu'},
        # residual add between two norms of one token; of sixteen sequences
        {'name': 'norm_token', 'op': 'norm', 'b': 1, 't': 1, 'c': 4096, 'type': 'bf16', 'post': True, 'gate': 'none', 'next': 0},
        {'name': 'norm_large', 'op': 'norm', 'b': 16, 't': 2048, 'c': 4096, 'type': 'bf16', 'post': True, 'gate': 'channel', 'next': 0},
        # residual add, norm and quantisation in front of an attention projection
        {'name': 'norm_into_linear', 'op': 'norm', 'b': 2, 't': 1024, 'c': 4096, 'type': 'bf16', 'post': False, 'gate': 'none', 'next': 4096},
        # rotary positions of one decoding step far into a long context, interleaved pairs on half of each head
        {'name': 'rotary_token', 'op': 'rotary', 'b': 16, 't': 1, 'h': 32, 'g': 8, 'd': 128, 'r': 64, 'far': 1000000, 'inter': True, 'type': 'bf16'},
        # rotary positions of eight sequences, halves of whole heads
        {'name': 'rotary_large', 'op': 'rotary', 'b': 8, 't': 2048, 'h': 32, 'g': 32, 'd': 128, 'r': 128, 'far': 30000, 'inter': False, 'type': 'bf16'},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['linear', 'linear', 'down', 'norm', 'norm', 'rotary'])
    kind = rng.choice(['bf16', 'bf16', 'fp16', 'fp32'])
    if op in ('linear', 'down'):
        m, n, k = _spread(rng, 1, 6000), _spread(rng, 64, 11008), _spread(rng, 64, 11008)
        if rng.random() < 0.6:
            n, k = -(-n // 128) * 128, -(-k // 128) * 128
        if op == 'down':
            kind = rng.choice(['bf16', 'fp16'])  # in fp32 the last bit of exp moves codes: nothing to hold 32 bits to
            return {'op': op, 'm': m, 'n': n, 'k': k, 'type': kind, 'act': rng.choice(['silu', 'gelu_tanh'])}
        return {'op': op, 'm': m, 'n': n, 'k': k, 'type': kind, 'sym': rng.random() < 0.6, 'bias': rng.random() < 0.5}
    if op == 'norm':
        b, t, c = rng.choice([1, 2, 5, 16]), _spread(rng, 1, 2048), _spread(rng, 64, 8192)
        if rng.random() < 0.6:
            c = -(-c // 64) * 64
        follow = 0 if kind == 'fp32' or rng.random() < 0.6 else _spread(rng, 64, 8192)
        t = min(t, 512) if follow else t
        return {'op': op, 'b': b, 't': t, 'c': c, 'type': kind, 'post': rng.random() < 0.5,
                'gate': rng.choice(['none', 'channel', 'sequence', 'full']), 'next': follow}
    d = 2 * rng.randint(16, 128)
    if rng.random() < 0.6:
        d = -(-d // 32) * 32
    r = d if rng.random() < 0.6 else 2 * rng.randint(1, d // 2)
    g = rng.choice([1, 4, 8])
    return {'op': op, 'b': rng.choice([1, 3, 8]), 't': _spread(rng, 1, 2048), 'h': g * rng.choice([1, 2, 4]), 'g': g, 'd': d, 'r': r,
            'far': _spread(rng, 100, 1000000), 'inter': rng.random() < 0.5, 'type': kind}


def _rows_apart_by_16(codes):
    """The same codes with rows that begin at multiples of 16 bytes, as the products read them."""
    n, k = codes.shape
    room = torch.zeros((n, -(-k // 16) * 16), dtype=torch.int8, device=codes.device)
    room[:, :k] = codes
    return room[:, :k]


def _weights(g, n, k):
    """A linear's weights in 8 bits with a scale for each output channel."""
    w = torch.randn((n, k), generator=g, device='cuda') * 0.02
    scale = w.abs().amax(1) / 127
    return _rows_apart_by_16(torch.round(w / scale[:, None]).to(torch.int8)), scale


def _activations(g, shape, dtype, shift=0.0):
    """Activations of a decoder block: some channels are much larger than the others."""
    x = torch.randn(shape, generator=g, device='cuda') + shift
    x *= 1 + 8 * (torch.rand(shape[-1], generator=g, device='cuda') < 0.01)
    return x.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    op, dtype = case['op'], _TYPES[case['type']]
    state = {'op': op, 'type': dtype}
    if op == 'linear':
        state['x'] = _activations(g, (case['m'], case['k']), dtype, 0.0 if case['sym'] else 0.7)
        state['w'], state['w_scale'] = _weights(g, case['n'], case['k'])
        state['bias'] = torch.randn(case['n'], generator=g, device='cuda').to(dtype) if case['bias'] else None
        state['w_sum'] = None if case['sym'] else state['w'].sum(1, dtype=torch.int32)
    elif op == 'down':
        state['gate'] = _activations(g, (case['m'], case['k']), dtype)
        state['up'] = _activations(g, (case['m'], case['k']), dtype)
        state['w'], state['w_scale'] = _weights(g, case['n'], case['k'])
        state['act'] = case['act']
    elif op == 'norm':
        b, t, c = case['b'], case['t'], case['c']
        state['x'] = _activations(g, (b, t, c), dtype)
        state['residual'] = _activations(g, (b, t, c), dtype)
        state['weight'] = (1 + 0.3 * torch.randn(c, generator=g, device='cuda')).to(dtype)
        state['post'] = (1 + 0.3 * torch.randn(c, generator=g, device='cuda')).to(dtype) if case['post'] else None
        shape = {'none': None, 'channel': (c,), 'sequence': (b, 1, c), 'full': (b, t, c)}[case['gate']]
        state['gate'] = None if shape is None else torch.randn(shape, generator=g, device='cuda').to(dtype)
        state['scale'] = 0.5 if case['post'] else 1.0
        state['eps'] = 1e-6
        state['next'] = _weights(g, case['next'], c) if case['next'] else None
    else:
        b, t, h, kv, d = case['b'], case['t'], case['h'], case['g'], case['d']
        # projections' outputs seen as heads: (batch, heads, tokens, head size) over (batch, tokens, heads, head size)
        state['q'] = torch.randn((b, t, h, d), generator=g, device='cuda').to(dtype).transpose(1, 2)
        state['k'] = torch.randn((b, t, kv, d), generator=g, device='cuda').to(dtype).transpose(1, 2)
        first = torch.randint(0, max(1, case['far'] - t), (b, 1), generator=g, device='cuda')
        state['positions'] = first + torch.arange(t, device='cuda')
        turn = torch.arange(0, case['r'], 2, device='cuda', dtype=torch.float64) / case['r']
        state['inv_freq'] = (10000.0 ** -turn).float()
        state['inter'] = case['inter']
    return state


# ---- plain forms --------------------------------------------------------------------------------------------

def _codes(v, sym):
    """Codes, scale and zero point of each row of v (fp32). Products next to a rounding border are formed in 64
    bits: scale and reciprocal are fp32 numbers, the product is rounded once."""
    if sym:
        top = v.abs().amax(-1, keepdim=True).clamp(min=1e-5)
        return torch.round(v.double() * (127.0 / top).double()), top / 127.0, None
    low, high = v.amin(-1, keepdim=True).clamp(max=0.0), v.amax(-1, keepdim=True).clamp(min=0.0)
    wide = (high - low).clamp(min=1e-5)
    per = (255.0 / wide).double()
    zero = -128 - torch.round(low.double() * per)
    return (torch.round(v.double() * per) + zero).clamp(-128, 127), wide / 255.0, zero


def _product(v, sym, w, w_scale, bias, dtype):
    codes, scale, zero = _codes(v, sym)
    whole = w.double()
    total = codes @ whole.t()  # sums of whole numbers, over what 32 bits hold
    if zero is not None:
        total = total - zero * whole.sum(1)
    y = total.float() * scale * w_scale
    if bias is not None:
        y = y + bias.float()
    return y.to(dtype)


def _act(x, kind):
    if kind == 'silu':
        return x / (1 + torch.exp(-x))
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))


def _rms(v, weight, eps):
    return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps) * weight.float()


def _turned(x, cos, sin, inter):
    v, r = x.float(), 2 * cos.shape[-1]
    one, two = (v[..., 0:r:2], v[..., 1:r:2]) if inter else (v[..., : r // 2], v[..., r // 2: r])
    a, b = one * cos - two * sin, two * cos + one * sin
    first = torch.stack((a, b), -1).flatten(-2) if inter else torch.cat((a, b), -1)
    return torch.cat((first, v[..., r:]), -1).to(x.dtype)


def _run_plain(s):
    op, dtype = s['op'], s['type']
    if op == 'linear':
        return _product(s['x'].float(), s['w_sum'] is None, s['w'], s['w_scale'], s['bias'], dtype)
    if op == 'down':
        return _product(_act(s['gate'].float(), s['act']) * s['up'].float(), True, s['w'], s['w_scale'], None, dtype)
    if op == 'norm':
        t = s['x'].float()
        if s['post'] is not None:
            t = _rms(t, s['post'], s['eps'])
        if s['gate'] is not None:
            t = t * s['gate'].float()
        h = (s['residual'].float() + s['scale'] * t).to(dtype)
        y = _rms(h.float(), s['weight'], s['eps'])
        return h, y.to(dtype) if s['next'] is None else _product(y, True, *s['next'], None, dtype)
    angle = (s['positions'].double()[:, None, :, None] * s['inv_freq'].double())
    cos, sin = angle.cos().float(), angle.sin().float()
    return _turned(s['q'], cos, sin, s['inter']), _turned(s['k'], cos, sin, s['inter'])


def _run_own(s):
    from lightcompress_b200 import block_ops, int8_linear
    op = s['op']
    if op == 'linear':
        return int8_linear.int8_dynamic_forward_func(s['x'], s['w'], s['w_scale'], s['bias'], w_sum=s['w_sum'])
    if op == 'down':
        codes, scale = int8_linear.gated_act_quant(s['gate'], s['up'], s['act'])
        return int8_linear.int8_gemm(codes, scale, s['w'], s['w_scale'], out_dtype=s['type'])
    if op == 'norm':
        h, y = block_ops.residual_norm(s['x'], s['residual'], weight=s['weight'], post_weight=s['post'], gate=s['gate'],
                                       scale=s['scale'], eps=s['eps'], quant=s['next'] is not None)
        if s['next'] is not None:
            y = int8_linear.int8_gemm(*y, *s['next'], out_dtype=s['type'])
        return h, y
    return block_ops.rotary_embed(s['q'], s['k'], s['positions'], s['inv_freq'], interleaved=s['inter'])


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


def work(case):
    size = 4 if case['type'] == 'fp32' else 2
    op = case['op']
    if op in ('linear', 'down'):
        m, n, k = case['m'], case['n'], case['k']
        inputs = 2 if op == 'down' else 1
        return {'bytes': inputs * m * k * size + n * k + 4 * n + m * n * size, 'flops': 2 * m * n * k}
    if op == 'norm':
        rows, c, n = case['b'] * case['t'], case['c'], case['next']
        gate = {'none': 0, 'channel': c, 'sequence': case['b'] * c, 'full': rows * c}[case['gate']]
        out = rows * n * size + n * c + 4 * n if n else rows * c * size
        return {'bytes': (3 * rows * c + gate + c * (2 if case['post'] else 1)) * size + out, 'flops': 2 * rows * n * c + 10 * rows * c}
    values = case['b'] * case['t'] * (case['h'] + case['g']) * case['d']
    return {'bytes': 2 * values * size + 8 * case['b'] * case['t'], 'flops': 3 * values}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------

def _exact_product(v, sym, w, w_scale, bias):
    """sum over k of (q - z) w, times both scales. Scales are kept in fp32, so they are fp32 numbers here too."""
    if sym:
        span, low = torch.maximum(v.max(1).values, -v.min(1).values), torch.zeros_like(v[:, 0])
        steps, least, shift = 127.0, -127, 0
    else:
        low = torch.minimum(v.min(1).values, torch.zeros_like(v[:, 0]))
        span = torch.maximum(v.max(1).values, torch.zeros_like(low)).float() - low.float()
        steps, least, shift = 255.0, -128, -128
    span = torch.maximum(span.float(), torch.tensor(1e-5, device=v.device))
    ratio, scale = (steps / span).double(), (span / steps).double()
    zero = shift - (low * ratio).round()
    q = ((v * ratio[:, None]).round() + zero[:, None]).clip(least, 127) - zero[:, None]
    y = torch.einsum('mk,nk->mn', q, w.double()) * torch.outer(scale, w_scale.double())
    return y if bias is None else y + bias.double()


def exact(case, seed):
    s = prepare(case, seed)
    op = s['op']
    if op == 'linear':
        return _exact_product(s['x'].double(), case['sym'], s['w'], s['w_scale'], s['bias'])
    if op == 'down':
        x = s['gate'].double()
        if s['act'] == 'silu':
            x = x * torch.sigmoid(x)
        else:
            x = x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))  # (1 + tanh u) / 2 is the sigmoid of 2u
        return _exact_product(x * s['up'].double(), True, s['w'], s['w_scale'], None)
    if op == 'norm':
        c = case['c']
        t = s['x'].double()
        if s['post'] is not None:
            t = t / ((t ** 2).sum(-1, keepdim=True) / c + s['eps']).sqrt() * s['post'].double()
        if s['gate'] is not None:
            t = s['gate'].double() * t
        h = s['residual'].double() + t * s['scale']
        kept = h.to(s['type']).double()  # the second norm is of the sum as it is kept
        y = kept / ((kept ** 2).sum(-1, keepdim=True) / c + s['eps']).sqrt() * s['weight'].double()
        if s['next'] is not None:
            y = _exact_product(y.reshape(-1, c), True, *s['next'], None).reshape(case['b'], case['t'], case['next'])
        return h, y
    outs = []
    turn = torch.polar(torch.ones((), dtype=torch.float64, device='cuda'),
                       s['positions'].double()[:, None, :, None] * s['inv_freq'].double())
    for x in (s['q'], s['k']):
        v, r = x.double(), case['r']
        if case['inter']:
            pairs = torch.view_as_complex(v[..., :r].reshape(*v.shape[:-1], r // 2, 2).contiguous())
            first = torch.view_as_real(pairs * turn).flatten(-2)
        else:
            pairs = torch.complex(v[..., : r // 2].contiguous(), v[..., r // 2: r].contiguous()) * turn
            first = torch.cat((pairs.real, pairs.imag), -1)
        outs.append(torch.cat((first, v[..., r:]), -1))
    return tuple(outs)

"""A decoder block as it is deployed in W8A8: int8 linears for q, k, v, o, gate, up and down, the norms fused with the
residual adds and the quantisation in front of each group of linears, rotary positions, the gated quantisation in front of
the down projection -- against the same block with 64-bit arithmetic everywhere, the same codes of the weights, and the
quantisation of the activations as documented."""
import pytest
import torch

from oracle import w8a8_ref as ref

pytestmark = pytest.mark.gpu


class Block:
    """Weights of one block: hidden c, h heads and g key / value heads of d, MLP width f."""

    def __init__(self, c, h, g, d, f, dtype, sandwich, seed=0):
        gen = torch.Generator().manual_seed(seed)
        self.c, self.h, self.g, self.d, self.dtype, self.sandwich = c, h, g, d, dtype, sandwich
        self.lin = {}
        for name, n, k in (('q', h * d, c), ('k', g * d, c), ('v', g * d, c), ('o', c, h * d), ('gate', f, c), ('up', f, c),
                           ('down', c, f)):
            w = torch.randn(n, k, generator=gen) / k ** 0.5
            s = w.abs().amax(1) / 127
            bias = torch.randn(n, generator=gen).to(dtype) * 0.1 if name in 'qkv' else None
            self.lin[name] = (torch.round(w / s[:, None]).to(torch.int8), s, bias)
        self.norm = {n: (1 + 0.1 * torch.randn(c, generator=gen)).to(dtype) for n in ('in', 'attn', 'mlp', 'post')}


def attention(q, k, v, past):
    """q (B, H, T, D) against k, v (B, G, S, D), causal from position `past` on, in q's precision."""
    b, h, t, d = q.shape
    k, v = (x.repeat_interleave(h // x.shape[1], 1) for x in (k, v))
    s = q @ k.transpose(-1, -2) / d ** 0.5
    mask = torch.arange(k.shape[2], device=q.device)[None] > torch.arange(t, device=q.device)[:, None] + past
    return torch.softmax(s.masked_fill(mask, float('-inf')), -1) @ v


def deployed(blk, x, pos, freq, cache=None):
    """The block through the library; returns (output, this step's keys and values)."""
    from lightcompress_b200 import block_ops, int8_linear
    lin = {n: int8_linear.Int8Linear(w.cuda(), s.cuda(), None if bias is None else bias.cuda()) for n, (w, s, bias) in
           blk.lin.items()}
    norm = {n: w.cuda() for n, w in blk.norm.items()}
    b, t, _ = x.shape

    def mul(name, q):
        m = lin[name]
        return int8_linear.int8_gemm(*q, m.weight, m.weight_scale, m.bias, out_dtype=blk.dtype)
    h, qx = block_ops.residual_norm(x, weight=norm['in'], quant=True)
    q, k, v = (mul(n, qx).unflatten(-1, (-1, blk.d)).transpose(1, 2) for n in 'qkv')
    q, k = block_ops.rotary_embed(q, k, pos, freq)
    past = 0
    if cache is not None:
        past = cache[0].shape[2]
        k, v = torch.cat((cache[0], k), 2), torch.cat((cache[1], v), 2)
    ctx = attention(q.double(), k.double(), v.double(), past).to(blk.dtype).transpose(1, 2).flatten(2)
    attn = lin['o'](ctx)
    h, qy = block_ops.residual_norm(attn, h, weight=norm['mlp'], post_weight=norm['attn'] if blk.sandwich else None,
                                    scale=0.7 if blk.sandwich else 1.0, quant=True)
    z = int8_linear.gated_act_quant(mul('gate', qy), mul('up', qy), 'silu')
    out, _ = block_ops.residual_norm(mul('down', z), h, post_weight=norm['post'] if blk.sandwich else None,
                                     scale=0.7 if blk.sandwich else 1.0)
    return out, (k, v)


def definition(blk, x, pos, freq):
    """The same block in fp64; activations are quantised by the documented formula where the block quantises them, and
    rounded to the tensor type where it keeps them."""
    keep = lambda v: v.to(blk.dtype).double()  # noqa: E731
    b, t, _ = x.shape

    def mul(name, v):
        w, s, bias = blk.lin[name]
        q, a_s, _ = ref.quant_rows(v.reshape(-1, v.shape[-1]))
        y = (q.double() @ w.double().t()) * a_s.double()[:, None] * s.double()
        return keep((y if bias is None else y + bias.double()).reshape(b, t, -1))
    y = ref.rms(x, blk.norm['in'], 1e-6)
    q, k, v = (mul(n, y).unflatten(-1, (-1, blk.d)).transpose(1, 2) for n in 'qkv')
    q, k = keep(ref.rotary(q, pos, freq)), keep(ref.rotary(k, pos, freq))
    ctx = keep(attention(q, k, v, 0).transpose(1, 2).flatten(2))
    scale = 0.7 if blk.sandwich else 1.0
    h = keep(ref.residual(mul('o', ctx), x, blk.norm['attn'] if blk.sandwich else None, None, scale))
    y = ref.rms(h, blk.norm['mlp'], 1e-6)
    z = ref.act(mul('gate', y), 'silu') * mul('up', y)
    return keep(ref.residual(mul('down', z), h, blk.norm['post'] if blk.sandwich else None, None, scale))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('sandwich', [False, True])
@pytest.mark.parametrize('c,h,g,d,f,b,t', [(256, 4, 2, 64, 640, 2, 33), (1024, 8, 8, 128, 2752, 1, 300), (200, 5, 1, 40, 328, 3, 7)])
def test_block(dtype, sandwich, c, h, g, d, f, b, t):
    """Tolerance, in the 2-norm of the block's change of the stream (output less input): values are rounded to the type some
    ten times on the way (eps/2 each, ten in quadrature: 3 eps/2), and a value that lies next to a border of its rounding or
    of its code falls to either side, a step of 1/127 of the row's largest in a share of the codes that is the relative
    error times 127, under 1 %: 0.1 / 127 of a row's largest, about 4 sigma: 0.3 %. Twice the sum for the four quantisations
    that follow one another."""
    from lightcompress_b200.block_ops import rope_frequencies
    blk = Block(c, h, g, d, f, dtype, sandwich)
    x = torch.randn(b, t, c, generator=torch.Generator().manual_seed(9)).to(dtype)
    freq, _ = rope_frequencies(d, device='cpu')
    pos = torch.arange(t)[None] + 17
    got, _ = deployed(blk, x.cuda(), pos.cuda(), freq.cuda())
    want = definition(blk, x, pos, freq)
    change = (want - x.double()).norm()
    off = float((got.cpu().double() - want).norm() / change)
    assert off < 2 * (3 * torch.finfo(dtype).eps / 2 + 0.003), off


@pytest.mark.parametrize('dtype', [torch.bfloat16])
def test_one_token_at_a_time_continues_the_prompt(dtype):
    """Each token's row of every linear depends on that token alone (scales per token), so the block applied to a prompt
    and then token by token gives each token the same values as the block applied to all of them, to the last bit: the
    products are exact whatever tile they run in, and the other operators work on rows."""
    from lightcompress_b200.block_ops import rope_frequencies
    blk = Block(256, 4, 2, 64, 640, dtype, True)
    freq, _ = rope_frequencies(64)
    x = torch.randn(2, 40, 256, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    pos = torch.arange(40, device='cuda')[None]
    whole, (k, v) = deployed(blk, x, pos, freq)
    _, cache = deployed(blk, x[:, :36], pos[:, :36], freq)
    assert torch.equal(cache[0], k[:, :, :36]) and torch.equal(cache[1], v[:, :, :36])
    for t in range(36, 40):
        out, cache = deployed(blk, x[:, t:t + 1], pos[:, t:t + 1], freq, cache)
        assert torch.equal(cache[0], k[:, :, :t + 1]) and torch.equal(cache[1], v[:, :, :t + 1])
        # attention itself is torch's, in fp64: its sums may be associated otherwise for one query, 2^-50 before rounding
        assert float((out - whole[:, t:t + 1]).float().abs().max()) <= float(torch.finfo(dtype).eps * whole.float().abs().max())


def test_block_captured_into_a_graph():
    from lightcompress_b200.block_ops import residual_norm, rope_frequencies, rotary_embed
    from lightcompress_b200.int8_linear import Int8Linear, gated_act_quant, int8_gemm
    blk = Block(256, 4, 4, 64, 640, torch.bfloat16, False)
    lin = {n: Int8Linear(w.cuda(), s.cuda(), None if b is None else b.cuda()) for n, (w, s, b) in blk.lin.items()}
    nw = blk.norm['in'].cuda()
    freq, _ = rope_frequencies(64)
    pos = torch.zeros(3, 1, dtype=torch.int64, device='cuda')

    def step(x):
        h, q = residual_norm(x, weight=nw, quant=True)
        a = int8_gemm(*q, lin['q'].weight, lin['q'].weight_scale, lin['q'].bias).unflatten(-1, (-1, 64)).transpose(1, 2)
        a, _ = rotary_embed(a, None, pos, freq)
        h, q = residual_norm(lin['o'](a.transpose(1, 2).flatten(2)), h, weight=nw, quant=True)
        z = gated_act_quant(lin['gate'](h), lin['up'](h))
        return residual_norm(int8_gemm(*z, lin['down'].weight, lin['down'].weight_scale), h)[0]
    xs = [torch.randn(3, 1, 256, generator=torch.Generator().manual_seed(i)).bfloat16().cuda() for i in range(3)]
    held = xs[0].clone()
    step(held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(held)
    for i, x in enumerate(xs):
        held.copy_(x)
        pos.fill_(100 * i)
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        assert torch.equal(got, step(x))


@pytest.mark.parametrize('tokens', [1, 5, 300])
def test_branches_on_two_streams(tokens):
    """gate and up side by side on two streams, joined by the gated quantisation: eagerly, and captured with the fork and
    the join in the graph, where the joining kernel depends on two of the library's kernels at once."""
    from lightcompress_b200.block_ops import residual_norm
    from lightcompress_b200.int8_linear import Int8Linear, gated_act_quant, int8_gemm
    blk = Block(256, 4, 4, 64, 1408, torch.bfloat16, False)
    lin = {n: Int8Linear(w.cuda(), s.cuda(), None if b is None else b.cuda()) for n, (w, s, b) in blk.lin.items()}
    nw = blk.norm['in'].cuda()
    xs = [torch.randn(1, tokens, 256, generator=torch.Generator().manual_seed(i)).bfloat16().cuda() for i in range(4)]

    def mul(name, q):
        return int8_gemm(*q, lin[name].weight, lin[name].weight_scale)

    def in_turn(x):
        h, q = residual_norm(x, x, weight=nw, quant=True)
        z = gated_act_quant(mul('gate', q), mul('up', q))
        return residual_norm(mul('down', z), h, weight=nw)
    want = [in_turn(x) for x in xs]
    side = torch.cuda.Stream()

    def side_by_side(x):
        h, q = residual_norm(x, x, weight=nw, quant=True)
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            up = mul('up', q)
        gate = mul('gate', q)
        here.wait_stream(side)
        z = gated_act_quant(gate, up)
        y = residual_norm(mul('down', z), h, weight=nw)
        for t in q:
            t.record_stream(side)
        up.record_stream(here)
        return y
    for rep in range(5):
        for x, w in zip(xs, want):
            assert all(map(torch.equal, side_by_side(x), w))
    held = xs[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ys = side_by_side(held)
    for rep in range(5):
        for x, w in zip(xs, want):
            held.copy_(x)
            graph.replay()
            torch.cuda.synchronize()
            assert all(map(torch.equal, ys, w))

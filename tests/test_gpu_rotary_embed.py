"""rotary_embed against its 64-bit restatement (oracle/w8a8_ref.py).

Tolerance: one rounding to the tensor type (eps/2 of the value); the remainder of the angle modulo 2 pi is rounded to
fp32 (2^-24 of at most pi), the fp64 angle of positions under 2^31 is off by under 2^-21, sine and cosine by 2 steps, the two
products and their sum by a rounding each: in all under 2^-20 of (|x1| + |x2|) * |scale|, 2^-21 without far positions."""
import pytest
import torch

from oracle import w8a8_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _heads(b, h, t, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + 7 * h + d)
    return torch.randn(b, t, h, d, generator=g).to(dtype).transpose(1, 2)


def _check(got, x, pos, freq, inter, scale):
    want = ref.rotary(x, pos, freq, inter, scale)
    r = 2 * freq.numel()
    size = x.double().abs()
    pair = torch.zeros_like(size)
    if inter:
        pair[..., :r] = (size[..., 0:r:2] + size[..., 1:r:2]).repeat_interleave(2, -1)
    else:
        pair[..., :r] = (size[..., :r // 2] + size[..., r // 2:r]).repeat(1, 1, 1, 2)
    tol = torch.finfo(x.dtype).eps / 2 * want.abs() * (1 + 2.0 ** -16) + 2.0 ** -20 * abs(scale) * pair \
        + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    assert got.shape == x.shape and got.dtype == x.dtype
    assert bool(((got.cpu().double() - want).abs() <= tol).all())
    assert torch.equal(got.cpu()[..., r:], x[..., r:])                # what is not turned is kept to the bit


CASES = [(1, 1, 1, 1, 2, 2), (2, 4, 2, 3, 64, 64), (2, 32, 8, 5, 128, 128), (1, 32, 32, 70, 128, 64), (3, 5, 1, 2, 80, 32),
         (2, 3, 3, 9, 34, 20), (1, 2, 1, 300, 256, 256), (16, 32, 8, 1, 128, 64), (1, 7, 0, 4, 96, 96), (2, 1, 1, 11, 33, 6),
         (1, 1, 1, 3, 1024, 1024), (2, 6, 2, 4, 72, 8), (1, 4, 4, 2, 40, 24), (1, 64, 8, 33, 64, 32)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('inter', [False, True])
@pytest.mark.parametrize('b,h,g,t,d,r', CASES)
def test_rotary(dtype, inter, b, h, g, t, d, r):
    from lightcompress_b200.block_ops import rope_frequencies, rotary_embed
    q = _heads(b, h, t, d, dtype)
    k = _heads(b, g, t, d, dtype, 5) if g else None
    freq, _ = rope_frequencies(r, device='cpu')
    pos = torch.randint(0, 5000, (b, 1), generator=torch.Generator().manual_seed(t)) + torch.arange(t)
    for p, scale in ((pos, 1.0), (pos[:1], 1.3), (pos[0], 1.0)):
        oq, ok = rotary_embed(q.cuda(), None if k is None else k.cuda(), p.cuda(), freq.cuda(), inter, scale)
        _check(oq, q, p, freq, inter, scale)
        if k is None:
            assert ok is None
        else:
            _check(ok, k, p, freq, inter, scale)
        assert oq.transpose(1, 2).is_contiguous()


@pytest.mark.parametrize('inter', [False, True])
def test_far_and_odd_positions(inter):
    from lightcompress_b200.block_ops import rotary_embed
    pos = torch.tensor([0, 1, -1, -70000, 131071, 10 ** 6, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31 + 1, 2 ** 31 - 2], dtype=torch.int64)
    freq = torch.cat((torch.tensor([1.0, 0.999999, 3.14159265, 0.5]), 10000.0 ** -(torch.arange(12) / 12.0)))
    q = _heads(1, 3, pos.numel(), 32, torch.float32)
    oq, _ = rotary_embed(q.cuda(), None, pos.cuda(), freq.cuda(), inter)
    _check(oq, q, pos, freq, inter, 1.0)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('inter', [False, True])
def test_views_of_one_projection_and_in_place(dtype, inter):
    from lightcompress_b200.block_ops import rope_frequencies, rotary_embed
    b, t, h, g, d = 2, 6, 8, 2, 64
    freq, _ = rope_frequencies(48, device='cpu')
    qkv = torch.randn(b, t, (h + 2 * g) * d + 3, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    pos = torch.arange(t)[None] + 100
    for first in (0, 3):                                   # the second lies off 16 bytes
        whole = qkv.clone()
        v = whole[..., first:first + (h + 2 * g) * d]
        q = v[..., :h * d].unflatten(-1, (h, d)).transpose(1, 2)
        k = v[..., h * d:(h + g) * d].unflatten(-1, (g, d)).transpose(1, 2)
        q0, k0 = q.cpu().clone(), k.cpu().clone()
        oq, ok = rotary_embed(q, k, pos.cuda(), freq.cuda(), inter)
        _check(oq, q0, pos, freq, inter, 1.0)
        _check(ok, k0, pos, freq, inter, 1.0)
        assert torch.equal(whole, qkv)
        iq, ik = rotary_embed(q, k, pos.cuda(), freq.cuda(), inter, inplace=True)
        assert iq is q and ik is k and torch.equal(q, oq) and torch.equal(k, ok)
        used = slice(first, first + (h + g) * d)
        rest = qkv.clone()
        rest[..., used] = whole[..., used]
        assert torch.equal(whole, rest)                    # values and neighbours are untouched
    contiguous = torch.randn(b, h, t, d, device='cuda').to(dtype)   # heads before tokens in memory
    oq, _ = rotary_embed(contiguous, None, pos.cuda(), freq.cuda(), inter)
    _check(oq, contiguous.cpu(), pos, freq, inter, 1.0)
    with pytest.raises(ValueError, match='one tensor'):
        rotary_embed(contiguous, contiguous[:, :1], pos.cuda(), freq.cuda(), inter, inplace=True)
    with pytest.raises(ValueError, match='expanded'):
        rotary_embed(contiguous[:1].expand(2, h, t, d), None, pos.cuda(), freq.cuda(), inter, inplace=True)


def test_agrees_with_the_table_kernel_and_empty_and_captured():
    from lightcompress_b200.block_ops import rope_apply_one, rope_frequencies, rotary_embed
    b, h, t, d = 2, 4, 50, 128
    freq, _ = rope_frequencies(d)
    q = _heads(b, h, t, d, torch.float32).cuda()
    pos = torch.arange(t, device='cuda')
    angle = torch.cat((pos.double()[:, None] * freq.double(),) * 2, -1)[None]
    table = rope_apply_one(q, angle.cos().float().contiguous(), angle.sin().float().contiguous())
    oq, _ = rotary_embed(q, None, pos, freq)
    # the same two products and sum of fp32 values a few steps apart
    assert torch.allclose(oq, table, rtol=1e-5, atol=1e-5)
    e = q[:, :, :0]
    assert rotary_embed(e, e[:, :1], pos[:0], freq)[0].shape == e.shape
    xs = [_heads(b, h, t, d, torch.float32, s).cuda() for s in range(2)]
    held, at = xs[0].clone(), pos.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = rotary_embed(held, held[:, :1], at, freq)
    for i, x in enumerate(xs):
        held.copy_(x)
        at.copy_(pos + 1000 * i)
        g.replay()
        want = rotary_embed(x, x[:, :1], pos + 1000 * i, freq)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


# Heads whose halves lie at multiples of 1, 2, 4 and 8 values, with pieces that do not fill their items, and batches whose
# tokens share a block or have several
NARROW = [(1, 16, 4, 61, 192, 142), (4, 16, 4, 27, 160, 44), (3, 8, 4, 19, 220, 220), (2, 16, 8, 9, 166, 150), (3, 4, 1, 101, 168, 140),
          (8, 1, 1, 26, 214, 214), (5, 2, 1, 500, 24, 8), (3, 1, 1, 8, 192, 192), (2, 3, 1, 700, 14, 2), (4, 5, 5, 3, 98, 98),
          (1, 1, 1, 5000, 64, 12), (2, 900, 100, 2, 12, 4), (1, 3, 2, 2, 1023, 1022), (7, 2, 2, 350, 22, 20)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('inter', [False, True])
@pytest.mark.parametrize('b,h,g,t,d,r', NARROW)
def test_heads_that_lie_anyhow(dtype, inter, b, h, g, t, d, r):
    from lightcompress_b200.block_ops import rope_frequencies, rotary_embed
    test_rotary(dtype, inter, b, h, g, t, d, r)
    # in place, and as parts of one projection's output
    freq, _ = rope_frequencies(r, device='cpu')
    pos = torch.arange(t) + 3
    qk = _heads(b, h + g, t, d, dtype, 9)
    on = qk.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    oq, ok = rotary_embed(on[:, :h], on[:, h:], pos.cuda(), freq.cuda(), inter, inplace=True)
    _check(oq, qk[:, :h], pos, freq, inter, 1.0)
    _check(ok, qk[:, h:], pos, freq, inter, 1.0)

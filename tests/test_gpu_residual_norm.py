"""residual_norm against its 64-bit restatement (oracle/w8a8_ref.py).

Tolerances: a rounding to the tensor type is off by half a step, eps/2 of the value.  In fp32, a sum of C squares
in any order of partial sums of at most 64 terms a thread is off by under 100 roundings, 2^-17 relative, and half of
that in the root; the products and sums behind it add a few roundings of the terms they work on.  So h is within
eps/2 |h| + 2^-18 (|residual| + |scale gate t|), and y, formed from the kept h, within (eps/2 + 2^-17) |y|."""
import pytest
import torch

from oracle import w8a8_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
FINE = 2.0 ** -17


def _data(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + shape[-1])
    x = torch.randn(*shape, generator=g)
    x[..., ::13] *= 6
    x = x * (torch.rand(*shape[:-1], 1, generator=g) * 4 + 0.01)
    return x.to(dtype)


def _check(h, y, x, res, w, post, gate, scale, eps, offset):
    dtype = x.dtype
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * half * 2          # half a step below the normal range
    want = ref.residual(x, res, post, gate, scale, eps, offset)
    term = ref.residual(x, None, post, gate, scale, eps, offset).abs() + (0 if res is None else res.double().abs())
    got = h.cpu().double()
    assert bool(((got - want).abs() <= half * want.abs() * (1 + FINE) + FINE / 2 * term + tiny).all())
    if y is not None:
        wy = ref.rms(h.cpu(), w, eps, offset)
        assert bool(((y.cpu().double() - wy).abs() <= (half * (1 + FINE) + FINE) * wy.abs() + tiny).all())


SHAPES = [(1, 1), (1, 4096), (3, 7), (2, 5, 64), (2, 3, 1399), (4, 11, 4096), (2, 2, 2, 200), (3, 8192), (5, 8200), (2, 20000),
          (1, 16384), (2, 40001), (600, 512), (2000, 128), (37, 1024), (3, 2056)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', SHAPES)
def test_residual_norm(dtype, shape):
    from lightcompress_b200.block_ops import residual_norm
    c = shape[-1]
    x, res = _data(shape, dtype, 1), _data(shape, dtype, 2)
    w, post = _data((c,), dtype, 3), _data((c,), dtype, 4)
    gates = {None: None, 'channel': _data((c,), dtype, 5), 'full': _data(shape, dtype, 6)}
    if len(shape) > 2:
        gates['sequence'] = _data((shape[0], *([1] * (len(shape) - 2)), c), dtype, 7)
    cu = lambda t: None if t is None else t.cuda()  # noqa: E731
    cases = [(res, w, None, None, 1.0, 1e-6, 0.0), (None, w, None, None, 1.0, 1e-5, 1.0), (res, None, post, None, 0.22, 1e-6, 0.0)]
    cases += [(res, w, post, gate, 0.5, 1e-6, float(i % 2)) for i, gate in enumerate(gates.values())]
    cases += [(None, w, None, gates['channel'], -2.0, 1e-6, 0.0)]
    for r, wt, p, gate, scale, eps, offset in cases:
        h, y = residual_norm(x.cuda(), cu(r), weight=cu(wt), post_weight=cu(p), gate=cu(gate), scale=scale, eps=eps,
                             weight_offset=offset)
        assert h.shape == x.shape and h.dtype == dtype and (y is None) == (wt is None)
        _check(h, y, x, r, wt, p, gate, scale, eps, offset)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('sym', [True, False])
@pytest.mark.parametrize('shape', [(1, 1), (1, 4096), (5, 1399), (2, 6, 64), (3, 8192), (2, 20000), (300, 512), (3, 40001)])
def test_quantised_form(dtype, sym, shape):
    """The codes against y / s with y in 64 bits: half a step, and 255 steps times the 2^-17 that y may be off."""
    from lightcompress_b200.block_ops import residual_norm
    x, res, w = _data(shape, dtype, 1), _data(shape, dtype, 2), _data((shape[-1],), dtype, 3)
    plain_h, _ = residual_norm(x.cuda(), res.cuda(), weight=w.cuda())
    h, q = residual_norm(x.cuda(), res.cuda(), weight=w.cuda(), quant=True, sym=sym)
    assert torch.equal(h, plain_h) and q[0].shape == x.shape and q[0].dtype == torch.int8 and len(q) == (2 if sym else 3)
    y = ref.rms(h.cpu(), w, 1e-6)
    _, s, z = ref.quant_rows(y.reshape(-1, shape[-1]), sym)
    assert q[1].shape == (*shape[:-1], 1)
    assert torch.allclose(q[1].cpu().reshape(-1).double(), s.double(), rtol=2 * FINE, atol=0)
    codes = q[0].cpu().double()
    limit = torch.full_like(codes, 0.5 + 256 * FINE)
    if not sym:
        assert float((q[2].cpu().reshape(-1).double() - z).abs().max()) <= 1
        limit[(q[0].cpu() == 127) | (q[0].cpu() == -128)] += 0.5
        codes = codes - q[2].cpu().double()
    assert bool(((codes - y / q[1].cpu().double()).abs() <= limit).all())


def test_nothing_to_add_keeps_the_tensor():
    from lightcompress_b200.block_ops import residual_norm
    x = _data((4, 256), torch.bfloat16).cuda()
    h, y = residual_norm(x)
    assert h is x and y is None
    h, y = residual_norm(x, weight=torch.ones_like(x[0]))
    assert h is x and y.shape == x.shape


@pytest.mark.parametrize('dtype', TYPES)
def test_strides_alignment_and_neighbours(dtype):
    from lightcompress_b200.block_ops import residual_norm
    big = _data((40, 700), dtype).cuda()
    w = _data((512,), dtype, 3).cuda()
    for x, r in ((big[:, 3:515], big[:, 100:612]), (big[::2, :512], big[1::2, 8:520]), (big[:, 16:528], big[:, 32:544]),
                 (big[:1, :512].expand(40, 512), big[:, :512])):
        h, y = residual_norm(x, r, weight=w)
        _check(h, y, x.cpu(), r.cpu(), w.cpu(), None, None, 1.0, 1e-6, 0.0)
        h2, y2 = residual_norm(x.contiguous(), r.contiguous(), weight=w)
        assert torch.allclose(h, h2, rtol=2 * torch.finfo(dtype).eps, atol=1e-6)
    odd = _data((513,), dtype, 3).cuda()[1:]                 # weights off 16 bytes
    h, y = residual_norm(big[:, :512], big[:, 8:520], weight=odd, post_weight=odd, gate=odd)
    _check(h, y, big[:, :512].cpu(), big[:, 8:520].cpu(), odd.cpu(), odd.cpu(), odd.cpu(), 1.0, 1e-6, 0.0)


def test_rows_that_are_not_finite_and_rows_of_zeros():
    from lightcompress_b200.block_ops import residual_norm
    x = _data((6, 1024), torch.bfloat16)
    x[1] = 0
    x[2, 5] = float('inf')
    x[3, 7] = float('nan')
    w = _data((1024,), torch.bfloat16, 3)
    h, y = residual_norm(x.cuda(), weight=w.cuda(), post_weight=w.cuda(), scale=2.0)
    for i in (2, 3):
        assert bool(torch.isnan(y[i]).all())
    assert bool((h[1] == 0).all()) and bool((y[1] == 0).all())
    keep = [0, 1, 4, 5]
    _check(h[keep], y[keep], x[keep], None, w, w, None, 2.0, 1e-6, 0.0)
    h, (codes, scales) = residual_norm(x.cuda(), weight=w.cuda(), quant=True)
    assert bool(torch.isnan(scales[[2, 3]]).all()) and bool((codes[[2, 3]] == 0).all()) and bool((codes[1] == 0).all())
    assert bool(torch.isfinite(scales[keep]).all())


def test_empty_and_captured():
    from lightcompress_b200.block_ops import residual_norm
    w = _data((256,), torch.bfloat16, 3).cuda()
    e = torch.zeros(2, 0, 256, dtype=torch.bfloat16, device='cuda')
    h, y = residual_norm(e, e, weight=w, gate=torch.zeros(2, 1, 256, dtype=torch.bfloat16, device='cuda'))
    assert h.shape == y.shape == e.shape
    h, q = residual_norm(e, e, weight=w, quant=True)
    assert q[0].shape == e.shape and q[1].shape == (2, 0, 1)
    xs = [_data((30, 256), torch.bfloat16, s).cuda() for s in range(3)]
    held = xs[0].clone()
    want = [residual_norm(x, x, weight=w, post_weight=w, quant=True) for x in xs]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = residual_norm(held, held, weight=w, post_weight=w, quant=True)
    for x, (wh, (wc, ws)) in zip(xs, want):
        held.copy_(x)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], wh) and torch.equal(out[1][0], wc) and torch.equal(out[1][1], ws)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('c', [256, 1000, 4096, 8192, 11008, 16384])
def test_a_row_does_not_depend_on_the_others(dtype, c):
    from lightcompress_b200.block_ops import residual_norm
    x, res, w = _data((400, c), dtype, 1).cuda(), _data((400, c), dtype, 2).cuda(), _data((c,), dtype, 3).cuda()
    h, q = residual_norm(x, res, weight=w, post_weight=w, quant=True)
    _, y = residual_norm(x, res, weight=w, post_weight=w)
    for rows in (slice(0, 1), slice(399, 400), slice(7, 30)):
        hs, qs = residual_norm(x[rows], res[rows], weight=w, post_weight=w, quant=True)
        _, ys = residual_norm(x[rows], res[rows], weight=w, post_weight=w)
        assert torch.equal(hs, h[rows]) and torch.equal(ys, y[rows])
        assert torch.equal(qs[0], q[0][rows]) and torch.equal(qs[1], q[1][rows])


# Rows by pairs and by single values on every shape that holds them, and just beyond the widest
NARROW = [(3, 2), (9, 6), (17, 129), (200, 254), (5, 511), (4, 1022), (3, 1023), (150, 1026), (149, 2046), (3, 2047), (4, 4094),
          (150, 4095), (2, 8190), (2, 8191), (2, 16382), (2, 16385), (1, 32766), (2, 32770)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', NARROW)
def test_rows_that_begin_anywhere(dtype, shape):
    test_residual_norm(dtype, shape)
    test_quantised_form(dtype, True, shape)
    test_quantised_form(dtype, False, shape)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('first', [1, 2, 3, 4])
def test_rows_of_a_slice(dtype, first):
    """Rows of 1020 of 1030 values: every other way in which a row may lie, inputs alike and not."""
    from lightcompress_b200.block_ops import residual_norm
    wide, other = _data((5, 1030), dtype, 1), _data((5, 1030), dtype, 2)
    w, post = _data((1020,), dtype, 3), _data((1020,), dtype, 4)
    x = wide.cuda()[:, first:first + 1020]
    for start in (first, 0):
        res = other.cuda()[:, start:start + 1020]
        h, y = residual_norm(x, res, weight=w.cuda(), post_weight=post.cuda())
        _check(h, y, x.cpu(), res.cpu(), w, post, None, 1.0, 1e-6, 0.0)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', [(5, 4096), (3, 1022), (7, 129), (2, 16384), (2, 40001)])
def test_both_forms_of_the_norm_in_one_call(dtype, shape):
    """The C interface gives y and its codes together: the same bits as either alone."""
    from lightcompress_b200 import _lib as L
    from lightcompress_b200.block_ops import residual_norm
    rows, c = shape
    x, res, w = _data(shape, dtype, 1).cuda(), _data(shape, dtype, 2).cuda(), _data((c,), dtype, 3).cuda()
    for sym in (True, False):
        want_h, want_y = residual_norm(x, res, weight=w, scale=0.3)
        _, q = residual_norm(x, res, weight=w, scale=0.3, quant=True, sym=sym)
        h, y = torch.empty_like(x), torch.empty_like(x)
        ldc = (c + 15) // 16 * 16
        codes = torch.empty(rows, ldc, dtype=torch.int8, device='cuda')
        scales = torch.empty(rows, device='cuda')
        zeros = torch.empty(rows, dtype=torch.int32, device='cuda')
        L.launch(0, 'lc_residual_norm', L.RESIDUAL_NORM.pack(
            x.data_ptr(), res.data_ptr(), 0, 0, 0, w.data_ptr(), L._DTYPES[dtype], rows, c, c, c, 0.3, 1e-6, 0.0, h.data_ptr(),
            y.data_ptr(), codes.data_ptr(), ldc, scales.data_ptr(), 0 if sym else zeros.data_ptr()))
        assert torch.equal(h, want_h) and torch.equal(y, want_y)
        assert torch.equal(codes[:, :c], q[0]) and torch.equal(scales, q[1].flatten())
        if not sym:
            assert torch.equal(zeros, q[2].flatten())

"""The 8-bit integer linear against its 64-bit restatement (oracle/w8a8_ref.py).

The product is held to the bit: the sum of products is a whole number that 32 bits hold, and the three fp32
operations behind it and the rounding are named by the interface, so every tile and every split must give the same.
Codes of a plain quantisation are held to the bit as well: the definition rounds v * r once, from an exact product.
Codes of the gated activation come from an fp32 value of a few roundings; tolerances stand beside the tests."""
import pytest
import torch

from oracle import w8a8_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _acts(m, k, dtype, seed=0, shift=0.0):
    g = torch.Generator().manual_seed(seed + 131 * m + k)
    x = torch.randn(m, k, generator=g) + shift
    x[:, :: max(1, k // 3)] *= 9
    return x.to(dtype)


def _weight(n, k, seed=0):
    g = torch.Generator().manual_seed(seed + 17 * n + k)
    b = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
    room = torch.full((n, (k + 15) // 16 * 16 + 16), 77, dtype=torch.int8)      # what lies behind a row is not read
    room[:, :k] = b
    return b, room.cuda()[:, :k], (torch.rand(n, generator=g) * 0.01 + 1e-4)


# ---- quantisation -------------------------------------------------------------------------------------------

@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('sym', [True, False])
@pytest.mark.parametrize('shape', [(1, 1), (1, 7), (3, 64), (5, 129), (2, 3, 256), (70, 1399), (9, 4096), (2, 11008), (3, 40000)])
def test_codes_are_the_definition_to_the_bit(dtype, sym, shape):
    from lightcompress_b200.int8_linear import act_quant
    x = _acts(shape[0] * (shape[1] if len(shape) == 3 else 1), shape[-1], dtype, shift=0.0 if sym else 0.6).reshape(shape)
    got = act_quant(x.cuda(), sym)
    q, s, z = ref.quant_rows(x.reshape(-1, shape[-1]), sym)
    assert got[0].dtype == torch.int8 and got[0].shape == x.shape and got[1].shape == (*shape[:-1], 1)
    assert torch.equal(got[0].cpu().long().reshape(q.shape), q)
    assert torch.equal(got[1].cpu().reshape(-1), s)
    if not sym:
        assert got[2].dtype == torch.int32 and torch.equal(got[2].cpu().long().reshape(-1), z)


@pytest.mark.parametrize('sym', [True, False])
def test_rows_that_are_special(sym):
    """Rows of zeros, of one sign, of the floor of the scale, of values next to rounding borders, with NaN and
    infinities, with the type's largest values."""
    from lightcompress_b200.int8_linear import act_quant
    k = 96
    rows = [torch.zeros(k), torch.full((k,), 3.0), torch.full((k,), -2.5), torch.linspace(-1e-6, 1e-6, k),
            torch.linspace(-63.5, 63.5, k).mul(2).round().div(2), torch.linspace(0, 255, k), torch.linspace(-255, 0, k),
            torch.full((k,), 3e38), torch.linspace(-3e38, 3e38, k), torch.linspace(1, 2, k)]
    for bad in (float('nan'), float('inf'), -float('inf')):
        r = torch.linspace(-1, 1, k)
        r[k - 1] = bad
        rows.append(r)
    x = torch.stack(rows)
    got = act_quant(x.cuda(), sym)
    q, s, z = ref.quant_rows(x, sym)
    assert torch.equal(got[0].cpu().long(), q)
    assert torch.equal(torch.isnan(got[1].cpu().reshape(-1)), torch.isnan(s))
    assert torch.equal(got[1].cpu().reshape(-1).nan_to_num(), s.nan_to_num())
    if not sym:
        assert torch.equal(got[2].cpu().long().reshape(-1), z)


@pytest.mark.parametrize('dtype', TYPES)
def test_strided_rows_and_what_lies_behind_them(dtype):
    from lightcompress_b200 import _lib as L
    from lightcompress_b200.int8_linear import act_quant
    base = _acts(12, 300, dtype).cuda()
    for view in (base[:, 3:260], base[::2, :256], base[:, 8:264], base.t()[:, :9], base[:1].expand(5, 300), base[:, ::2]):
        q, s, _ = ref.quant_rows(view.cpu().contiguous())
        codes, scales = act_quant(view)
        assert torch.equal(codes.cpu().long(), q) and torch.equal(scales.cpu().reshape(-1), s)
    # bytes behind a row and rows behind the last stay as they were
    room = torch.full((8, 320), 55, dtype=torch.int8, device='cuda')
    scales = torch.full((8,), -1.0, device='cuda')
    x = base[:6, :257].contiguous()
    L.launch(0, 'lc_int8_act_quant', x.data_ptr(), L.lc_dtype(x), 6, 257, 257, room.data_ptr(), 320, scales.data_ptr(), None)
    q, s, _ = ref.quant_rows(x.cpu())
    assert torch.equal(room[:6, :257].cpu().long(), q) and torch.equal(scales[:6].cpu(), s)
    assert bool((room[:6, 257:] == 55).all()) and bool((room[6:] == 55).all()) and bool((scales[6:] == -1).all())


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('act', ['silu', 'gelu', 'gelu_tanh'])
@pytest.mark.parametrize('m,k,sym', [(1, 1, True), (5, 130, False), (33, 1399, True), (4, 11008, True), (7, 4096, False)])
def test_gated_quantisation(dtype, act, m, k, sym):
    """v = act(gate) * up has a relative error of a few fp32 roundings, and exp one that grows with its argument
    (|x| 2^-23 at |x| < 32): under 2^-17 of the largest value of the row in all, i.e. 2^-10 of a code step (at 127 or 255
    steps a row). So a code is at most half a step and that from v / s, and the scale within 2^-17."""
    from lightcompress_b200.int8_linear import gated_act_quant
    gate, up = _acts(m, k, dtype, 1), _acts(m, k, dtype, 2)
    got = gated_act_quant(gate.cuda(), up.cuda(), act, sym)
    v = ref.act(gate, act) * up.double()
    _, s, z = ref.quant_rows(v, sym)
    assert torch.allclose(got[1].cpu().reshape(-1).double(), s.double(), rtol=2.0 ** -17, atol=0)
    codes = got[0].cpu().double()
    if not sym:
        gz = got[2].cpu().double()
        assert float((gz.reshape(-1) - z).abs().max()) <= 1
        codes = codes - gz
    off = (codes - v / got[1].cpu().double()).abs()
    # with a zero point the ends of the range may be cut by the rounding of z: half a step more, at the ends only
    limit = torch.full_like(off, 0.5 + 2.0 ** -9)
    if not sym:
        limit[(got[0].cpu() == 127) | (got[0].cpu() == -128)] += 0.5
    assert bool((off <= limit).all()), float(off.max())


# ---- product ------------------------------------------------------------------------------------------------

PRODUCTS = [(1, 1, 1), (1, 16, 16), (1, 4096, 4096), (2, 130, 1399), (3, 1000, 31), (8, 257, 256), (16, 4096, 4096), (17, 96, 2048),
            (24, 11008, 512), (33, 72, 100), (64, 128, 128), (65, 520, 640), (100, 1000, 1000), (128, 256, 256), (129, 384, 384),
            (200, 64, 11008), (256, 256, 512), (257, 513, 1025), (333, 1001, 1399), (512, 1024, 144), (600, 2048, 2048),
            (1000, 1408, 2048), (2048, 4096, 1024), (2500, 520, 272), (5, 33000, 64)]


@pytest.mark.parametrize('m,n,k', PRODUCTS)
def test_product_is_exact(m, n, k):
    from lightcompress_b200.int8_linear import act_quant, int8_gemm
    b, bd, bs = _weight(n, k)
    g = torch.Generator().manual_seed(m + n + k)
    bias = torch.randn(n, generator=g)
    for sym in (True, False):
        x = _acts(m, k, torch.float32, shift=0.0 if sym else 0.5).cuda()
        q = act_quant(x, sym)
        a, a_s = q[0].cpu(), q[1].cpu()
        a_z = None if sym else q[2].cpu()
        total = (q[0].double() - (0 if sym else q[2].double())) @ bd.double().t()       # exact whole numbers
        for dtype in TYPES:
            bi = bias.to(dtype).cuda() if dtype != torch.float16 else None
            c = int8_gemm(q[0], q[1], bd, bs.cuda(), bi, None if sym else q[2],
                          None if sym else b.sum(1, dtype=torch.int32).cuda(), dtype)
            y = total.float() * q[1] * bs.cuda()
            y = (y if bi is None else y + bi.float()).to(dtype)
            assert c.shape == (m, n) and c.dtype == dtype
            assert torch.equal(c, y), (sym, dtype, float((c.float() - y.float()).abs().max()))
    # the restatement on the CPU agrees with what the loop compared with
    if m * n * k < 1 << 24:
        assert torch.equal(int8_gemm(q[0], q[1], bd, bs.cuda(), None, q[2], b.sum(1, dtype=torch.int32).cuda(),
                                     torch.float32).cpu(), ref.int8_product(a, a_s, b, bs, None, a_z))


def test_more_tokens_than_a_grid_dimension_holds():
    """More 128-token tiles than 65535, of few channels: every row of the output against the exact sums."""
    from lightcompress_b200.int8_linear import int8_gemm
    m, n, k = 128 * 65536 + 77, 8, 16
    g = torch.Generator(device='cuda').manual_seed(1)
    a = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8, device='cuda')
    b = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8, device='cuda')
    one = torch.ones(m, device='cuda')
    c = int8_gemm(a, one, b, one[:n], out_dtype=torch.float32)
    assert torch.equal(c, a.float() @ b.float().t())            # sums below 2^24: exact in fp32


@pytest.mark.parametrize('m', [1, 20, 300])
def test_largest_sums(m):
    """Sums at the ends of 32 bits: all codes -128, with and without a zero point at the other end."""
    from lightcompress_b200.int8_linear import int8_gemm
    k, n = 131071, 40
    pitch = (k + 15) // 16 * 16
    a = torch.full((m, pitch), -128, dtype=torch.int8, device='cuda')[:, :k]
    b = torch.full((n, pitch), -128, dtype=torch.int8, device='cuda')[:, :k]
    one = torch.ones(max(m, n), device='cuda')
    c = int8_gemm(a, one[:m], b, one[:n], out_dtype=torch.float32)
    assert bool((c == float(128 * 128 * k)).all())
    k = 65793
    a, b = a[:, :k], b[:, :k]
    z = torch.full((m, 1), 127, dtype=torch.int32, device='cuda')
    c = int8_gemm(a, one[:m], b, one[:n], a_z=z, b_sum=b.sum(1, dtype=torch.int32), out_dtype=torch.float32)
    assert bool((c == torch.tensor(float(255 * 128 * k), device='cuda')).all())


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('m,n,k', [(1, 1, 1), (1, 64, 64), (1, 4096, 4096), (1, 4096, 4099), (1, 300, 11008), (1, 50, 4080), (1, 50, 4100),
                                   (1, 20000, 16000), (2, 333, 11008), (3, 1000, 9000), (8, 520, 4096),
                                   (5, 11008, 4096), (7, 130, 130), (8, 40, 17), (4, 1000, 11008), (9, 130, 1399), (40, 256, 512),
                                   (300, 520, 1040)])
def test_linear_is_quantisation_and_product(dtype, m, n, k):
    from lightcompress_b200.int8_linear import act_quant, check_status, int8_dynamic_forward_func, int8_gemm
    b, bd, bs = _weight(n, k)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    w_sum = b.sum(1, dtype=torch.int32).cuda()
    for sym in (True, False):
        x = _acts(m, k, dtype, shift=0.0 if sym else 0.7).cuda()
        q = act_quant(x, sym)
        want = int8_gemm(q[0], q[1], bd, bs.cuda(), bias, None if sym else q[2], None if sym else w_sum, dtype)
        got = int8_dynamic_forward_func(x, bd, bs.cuda(), bias, None if sym else w_sum)
        assert torch.equal(got, want)
        wide = torch.zeros(m, k + 11, dtype=dtype, device='cuda')
        wide[:, 5:5 + k] = x
        assert torch.equal(int8_dynamic_forward_func(wide[:, 5:5 + k], bd, bs.cuda(), bias, None if sym else w_sum), want)
        assert torch.equal(int8_dynamic_forward_func(x.reshape(1, m, 1, k), bd, bs.cuda(), bias, None if sym else w_sum),
                           want.reshape(1, m, 1, n))
    check_status()


@pytest.mark.parametrize('m', [1, 5, 150])
def test_rows_that_are_not_finite_stay_apart(m):
    from lightcompress_b200.int8_linear import int8_dynamic_forward_func
    b, bd, bs = _weight(200, 320)
    x = _acts(m + 1, 320, torch.bfloat16).cuda()
    clean = int8_dynamic_forward_func(x, bd, bs.cuda())
    x[0, 17] = float('inf')
    y = int8_dynamic_forward_func(x, bd, bs.cuda())
    assert bool(torch.isnan(y[0]).all()) and torch.equal(y[1:], clean[1:])


def test_empty_batches():
    from lightcompress_b200 import int8_linear as il
    _, bd, bs = _weight(48, 64)
    x = torch.zeros(0, 64, dtype=torch.bfloat16, device='cuda')
    assert il.int8_dynamic_forward_func(x, bd, bs.cuda()).shape == (0, 48)
    assert il.int8_dynamic_forward_func(x.reshape(2, 0, 64), bd, bs.cuda()).shape == (2, 0, 48)
    codes, scales = il.act_quant(x)
    assert codes.shape == (0, 64) and scales.shape == (0, 1)
    assert il.int8_gemm(codes, scales, bd, bs.cuda()).shape == (0, 48)
    y = il.int8_dynamic_forward_func(torch.ones(3, 64, device='cuda'), bd[:0], bs[:0].cuda())
    assert y.shape == (3, 0)
    codes, scales = il.act_quant(torch.ones(64, device='cuda'))
    assert codes.shape == (64,) and scales.shape == (1,)
    assert il.int8_gemm(codes, scales, bd, bs.cuda()).shape == (48,)


@pytest.mark.parametrize('m', [1, 12, 70, 700])
def test_captured_and_replayed_and_on_other_streams(m):
    from lightcompress_b200.int8_linear import int8_dynamic_forward_func
    n, k = 640, 1104
    b, bd, bs = _weight(n, k)
    bs = bs.cuda()
    xs = [_acts(m, k, torch.bfloat16, seed).cuda() for seed in range(3)]
    want = [int8_dynamic_forward_func(x, bd, bs) for x in xs]
    torch.cuda.synchronize()
    held = xs[0].clone()
    graphs = []
    for _ in range(2):                                     # two graphs of the same weights and input
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = int8_dynamic_forward_func(held, bd, bs)
        graphs.append((g, y))
    for x, w in zip(xs, want):
        held.copy_(x)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, w) for _, y in graphs)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for _ in range(5):
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                outs.append(int8_dynamic_forward_func(x, bd, bs))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i % 3]) for i, o in enumerate(outs))


@pytest.mark.parametrize('m', [3, 40, 300, 2100])
def test_product_waits_for_whatever_wrote_its_operands(m):
    """Operands written right before the product by a copy, a fill, a kernel of torch, this library's quantisation and on
    another stream, eagerly and captured."""
    from lightcompress_b200.int8_linear import act_quant, int8_gemm
    n, k = 2304, 1040
    xs = [_acts(m, k, torch.bfloat16, seed).cuda() for seed in range(4)]
    ws = [_weight(n, k, seed)[1].contiguous() for seed in range(4)]
    bs = [torch.full((n,), 0.5 + i, device='cuda') for i in range(4)]
    want = [int8_gemm(*act_quant(x), w, b) for x, w, b in zip(xs, ws, bs)]
    x, w, b = xs[0].clone(), ws[0].clone(), bs[0].clone()
    side = torch.cuda.Stream()
    picked = torch.zeros(1, dtype=torch.int64, device='cuda')
    all_x, all_w = torch.stack(xs), torch.stack(ws)

    def by_copies(i):
        q = act_quant(xs[i])
        w.copy_(ws[i])
        b.copy_(bs[i])
        return int8_gemm(*q, w, b)

    def by_a_fill(i):
        q = act_quant(xs[i])
        b.fill_(0.5 + i)
        return int8_gemm(*q, ws[i], b)

    def by_a_kernel(i):
        q = act_quant(xs[i])
        return int8_gemm(*q, (all_w[i].int() + 0).to(torch.int8), bs[i])

    def on_another_stream(i):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            x.copy_(xs[i])
            q = act_quant(x)
        torch.cuda.current_stream().wait_stream(side)
        w.copy_(ws[i])
        y = int8_gemm(*q, w, bs[i])
        for t in q:
            t.record_stream(torch.cuda.current_stream())
        return y
    for way in (by_copies, by_a_fill, by_a_kernel, on_another_stream):
        for rep in range(3):
            for i in range(4):
                assert torch.equal(way(i), want[i]), (way.__name__, i)

    def picks():
        i = picked
        x.copy_(all_x.index_select(0, i)[0])
        q = act_quant(x)
        w.copy_(all_w.index_select(0, i)[0])
        b.zero_()
        b.add_(0.5).add_(i)
        return int8_gemm(*q, w, b), int8_gemm(*act_quant(x), w, b)
    picks()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ys = picks()
    for rep in range(3):
        for i in range(4):
            picked.fill_(i)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(ys[0], want[i]) and torch.equal(ys[1], want[i])


def test_module_from_a_quantised_linear():
    from lightcompress_b200 import Int8Linear, IntegerQuantizer, RTN
    torch.manual_seed(0)
    lin = torch.nn.Linear(256, 192).to(torch.bfloat16).cuda()
    wq = IntegerQuantizer(8, True, 'per_channel')
    x = torch.randn(2, 9, 256, device='cuda').to(torch.bfloat16)
    full = lin(x).detach().float()
    for aq in (None, IntegerQuantizer(8, True, 'per_token'), IntegerQuantizer(8, False, 'per_token')):
        m = Int8Linear.new(lin, RTN(wq).w_q, wq, aq)
        y = m(x)
        assert y.dtype == torch.bfloat16 and y.shape == (2, 9, 192)
        codes, s, _ = wq.real_quant_weight_dynamic(lin.weight.data)
        sym = aq is None or aq.sym
        q, a_s, a_z = ref.quant_rows(x.reshape(18, 256).cpu(), sym)
        want = ref.int8_product(q, a_s, codes.cpu(), s.float().cpu(), lin.bias.data.cpu(), None if sym else a_z, torch.bfloat16)
        assert torch.equal(y.reshape(18, 192).cpu(), want)
        # 8 bits on both sides: each element off by half a step of 1/127 of its row's largest at most, ~1 % in the norm
        assert float((y.float() - full).norm() / full.norm()) < 0.03
        again = Int8Linear(m.weight.clone(), m.weight_scale, m.bias, sym)
        again.load_state_dict(m.state_dict())
        assert torch.equal(again(x), y)
    with pytest.raises(NotImplementedError):
        asym = IntegerQuantizer(8, False, 'per_channel')
        Int8Linear.new(lin, RTN(asym).w_q, asym)
    with pytest.raises(NotImplementedError):
        Int8Linear.new(lin, RTN(wq).w_q, wq, IntegerQuantizer(4, True, 'per_token'))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', [(3, 2), (9, 6), (17, 129), (200, 254), (4, 1022), (150, 1026), (149, 2046), (3, 2047), (4, 4094),
                                   (150, 4095), (2, 8190), (2, 16382), (2, 16385), (1, 32766), (2, 32770)])
def test_codes_of_rows_that_begin_anywhere(dtype, shape):
    for sym in (True, False):
        test_codes_are_the_definition_to_the_bit(dtype, sym, shape)
    for act in ('silu', 'gelu', 'gelu_tanh'):
        test_gated_quantisation(dtype, act, *shape, True)
    test_gated_quantisation(dtype, 'silu', *shape, False)


@pytest.mark.parametrize('m,n,k', [(24, 4096, 11008), (232, 256, 9600), (51, 512, 7040), (7, 179, 1189), (2400, 1280, 128),
                                   (1837, 268, 528), (1250, 256, 4224), (139, 384, 1792), (25, 2048, 6144)])
def test_product_in_many_small_blocks_and_large_clusters(m, n, k):
    test_product_is_exact(m, n, k)

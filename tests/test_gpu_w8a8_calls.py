"""The compiled front of the W8A8 operators against the Python functions it stands before: the same values to the bit
where it serves a call, and None (the Python function's turn) where it must not."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


class Silent:
    """A front that serves nothing."""

    def __getattr__(self, name):
        return (lambda *a: None) if name != 'set_status' else (lambda *a: None)


def _both(monkeypatch, f):
    """f() through the front and without it; the front has to have served it."""
    from lightcompress_b200 import _calls, block_ops, int8_linear
    served = []

    class Watched:
        def __getattr__(self, name):
            def call(*a):
                out = getattr(_calls, name)(*a)
                if name != 'set_status':
                    served.append(out is not None)
                return out
            return call
    results = []
    for front in (Watched(), Silent()):
        with monkeypatch.context() as m:
            m.setattr(int8_linear, '_calls', front)
            m.setattr(block_ops, '_calls', front)
            results.append(f())
    assert served and all(served)
    return results


def _leaves(v):
    return [v] if v is None or isinstance(v, torch.Tensor) else [t for x in v for t in _leaves(x)]


def _same(a, b):
    a, b = _leaves(a), _leaves(b)
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert (x is None) == (y is None)
        if x is not None:
            assert x.dtype == y.dtype and x.shape == y.shape and x.device == y.device and torch.equal(x, y)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', [(1, 64), (24, 1399), (2, 3, 256), (2, 1, 4, 100), (77,), (300, 4096)])
def test_quantisation_and_products(monkeypatch, dtype, shape):
    from lightcompress_b200 import int8_linear as il
    torch.manual_seed(len(shape) + shape[-1])
    x, up = torch.randn(shape, device='cuda').to(dtype), torch.randn(shape, device='cuda').to(dtype)
    w = il.aligned_rows(torch.randint(-128, 128, (130, shape[-1]), dtype=torch.int8, device='cuda'))
    ws, bias, total = torch.rand(130, device='cuda'), torch.randn(130, device='cuda').to(dtype), w.sum(1, dtype=torch.int32)
    il.int8_dynamic_forward_func(x, w, ws)                      # the status word exists from here on
    for sym in (True, False):
        _same(*_both(monkeypatch, lambda: il.act_quant(x, sym)))
        _same(*_both(monkeypatch, lambda: il.gated_act_quant(x, up, 'gelu_tanh', sym)))
        _same(*_both(monkeypatch, lambda: il.int8_dynamic_forward_func(x, w, ws, bias, None if sym else total)))
        q = il.act_quant(x, sym)
        for out in TYPES:
            _same(*_both(monkeypatch, lambda: il.int8_gemm(q[0], q[1], w, ws[:, None], bias if out == dtype else None,
                                                           None if sym else q[2], None if sym else total, out)))
    if len(shape) == 2 and shape[0] > 1:
        wide = torch.zeros(shape[0], shape[1] + 24, dtype=dtype, device='cuda')
        wide[:, 8:8 + shape[1]] = x
        _same(*_both(monkeypatch, lambda: il.int8_dynamic_forward_func(wide[:, 8:8 + shape[1]], w, ws, bias)))
        _same(*_both(monkeypatch, lambda: il.act_quant(wide[::2, 8:8 + shape[1]])))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', [(1, 64), (24, 1399), (2, 3, 256), (2, 1, 4, 100), (300, 4096)])
def test_residual_norm(monkeypatch, dtype, shape):
    from lightcompress_b200.block_ops import residual_norm
    torch.manual_seed(shape[-1])
    t = lambda *s: torch.randn(*s, device='cuda').to(dtype)  # noqa: E731
    x, r, w, p = t(*shape), t(*shape), t(shape[-1]), t(shape[-1])
    gates = [None, t(shape[-1]), t(*shape), t(*[1] * (len(shape) - 1), shape[-1])]
    if len(shape) == 3:
        gates.append(t(shape[0], 1, shape[-1]))
    for gate in gates:
        _same(*_both(monkeypatch, lambda: residual_norm(x, r, weight=w, post_weight=p, gate=gate, scale=0.5, weight_offset=1.0)))
        for sym in (True, False):
            _same(*_both(monkeypatch, lambda: residual_norm(x, r, weight=w, gate=gate, quant=True, sym=sym)))
    _same(*_both(monkeypatch, lambda: residual_norm(x, r, post_weight=p)))
    _same(*_both(monkeypatch, lambda: residual_norm(x, r, scale=2)))
    for h, _ in _both(monkeypatch, lambda: residual_norm(x, weight=w)):
        assert h is x


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('inter', [False, True])
def test_rotary(monkeypatch, dtype, inter):
    from lightcompress_b200.block_ops import rope_frequencies, rotary_embed
    freq, _ = rope_frequencies(48)
    for b, t in ((1, 1), (3, 7), (2, 1)):
        q, k = torch.randn(b, t, 6, 64, device='cuda').to(dtype).transpose(1, 2), torch.randn(b, 2, t, 64, device='cuda').to(dtype)
        for pos in (torch.randint(0, 9999, (b, t), device='cuda'), torch.arange(t, device='cuda')[None], torch.arange(t, device='cuda')):
            for kk in (k, None):
                got = _both(monkeypatch, lambda: rotary_embed(q, kk, pos, freq, inter, 1.25))
                _same(*got)
                assert got[0][0].stride() == got[1][0].stride()


def test_what_is_left_to_python():
    """The front serves none of these, and Python says why or does it."""
    from lightcompress_b200 import _calls, block_ops, int8_linear as il
    x = torch.randn(4, 64, device='cuda')
    w, ws = torch.zeros(8, 64, dtype=torch.int8, device='cuda'), torch.ones(8, device='cuda')
    il.int8_dynamic_forward_func(x, w, ws)
    assert _calls.act_quant(x, True) is not None
    for bad in (x.cpu(), x.t(), x[:0], x.double(), x.clone().requires_grad_(), x[0, 0], None, 3):
        assert _calls.act_quant(bad, True) is None
    with torch.no_grad():
        assert _calls.act_quant(x.clone().requires_grad_(), True) is not None
    assert _calls.act_quant(x, 1) is None and _calls.act_quant(x) is None
    assert _calls.int8_linear(x, w, ws, None, None) is not None
    for args in ((x, w[:, :60], ws, None, None), (x[:, :60], w, ws, None, None), (x, w, ws[:4], None, None), (x, w, ws.double(), None, None),
                 (x, w, ws, ws.half(), None), (x, w, ws, None, ws), (x, w.float(), ws, None, None), (x, w.t(), ws, None, None),
                 (x, w, ws.cpu(), None, None), (x, w[:0], ws[:0], None, None), (x, w, ws.clone().requires_grad_(), None, None)):
        assert _calls.int8_linear(*args) is None
    q = il.act_quant(x)
    assert _calls.int8_gemm(*q, w, ws, None, None, None, torch.float16) is not None
    z = torch.zeros(4, 1, dtype=torch.int32, device='cuda')
    for args in ((*q, w, ws, None, None, None, torch.float64), (*q, w, ws, None, z, None, torch.float16), (q[0], q[1][:2], w, ws, None, None, None, torch.float16),
                 (*q, w, ws, None, None, None, 'half'), (q[0][:, 1:33], q[1], w[:, :32], ws, None, None, None, torch.float16)):
        assert _calls.int8_gemm(*args) is None
    one = torch.ones(64, device='cuda')
    assert _calls.residual_norm(x, x, one, None, None, 1.0, 1e-6, 0.0, False, True) is not None
    for args in ((x, x[:2], one, None, None, 1.0, 1e-6, 0.0, False, True), (x, x, one.half(), None, None, 1.0, 1e-6, 0.0, False, True),
                 (x, x, one[:32], None, None, 1.0, 1e-6, 0.0, False, True), (x, x, None, None, None, 1.0, 1e-6, 0.0, True, True),
                 (x, x, one, None, x[:2], 1.0, 1e-6, 0.0, False, True), (x, None, None, None, None, 1.0, 1e-6, 0.0, False, True),
                 (x, x, one, None, None, '1', 1e-6, 0.0, False, True)):
        assert _calls.residual_norm(*args) is None
    h, y = block_ops.residual_norm(x)
    assert h is x and y is None
    a = torch.randn(1, 2, 3, 8, device='cuda')
    pos, f = torch.arange(3, device='cuda'), torch.ones(4, device='cuda')
    assert _calls.rotary_embed(a, None, pos, f, False, 1.0) is not None
    for args in ((a, None, pos.int(), f, False, 1.0), (a, None, pos[:2], f, False, 1.0), (a, None, pos, torch.ones(5, device='cuda'), False, 1.0),
                 (a[0], None, pos, f, False, 1.0), (a, a[:, :, :2], pos, f, False, 1.0), (a[:, :, :0], None, pos[:0], f, False, 1.0),
                 (a.transpose(2, 3), None, pos, f, False, 1.0), (a, None, pos.cpu(), f, False, 1.0)):
        assert _calls.rotary_embed(*args) is None

"""Views with a pending negation (the imaginary part of a conjugated tensor): their memory holds the other sign.  Each operand
of each W8A8 operator, against the same values laid out plainly."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _leaves(v):
    return [] if v is None else [v] if isinstance(v, torch.Tensor) else [t for x in v for t in _leaves(x)]


def _negated(t):
    v = torch._neg_view(-t)
    assert v.is_neg() and torch.equal(v, t)
    return v


@pytest.mark.parametrize('name', ['act_quant', 'gated_act_quant', 'int8_gemm', 'int8_linear', 'residual_norm', 'rotary_embed'])
def test_negated_operands(name):
    from lightcompress_b200 import block_ops as bo, int8_linear as il
    torch.manual_seed(0)
    x, r = torch.randn(5, 64, device='cuda') + 1, torch.randn(5, 64, device='cuda')
    one, gate = torch.rand(64, device='cuda') + 0.5, torch.randn(64, device='cuda')
    w, ws = torch.randint(-127, 128, (8, 64), dtype=torch.int8, device='cuda'), torch.rand(8, device='cuda') + 0.1
    bias, total = torch.randn(8, device='cuda'), w.sum(1, dtype=torch.int32)
    codes, scales = torch.randint(-127, 128, (5, 64), dtype=torch.int8, device='cuda'), torch.rand(5, 1, device='cuda') + 0.1
    zeros = torch.randint(-9, 9, (5, 1), dtype=torch.int32, device='cuda')
    q, k = torch.randn(1, 2, 3, 8, device='cuda'), torch.randn(1, 1, 3, 8, device='cuda')
    pos, freq = torch.arange(3, device='cuda') + 1, torch.rand(4, device='cuda')
    call, args = {
        'act_quant': (lambda x: il.act_quant(x, False), [x]),
        'gated_act_quant': (lambda g, u: il.gated_act_quant(g, u, 'silu', False), [x, r]),
        'int8_gemm': (lambda a, a_s, b, b_s, bi, z, t: il.int8_gemm(a, a_s, b, b_s, bi, z, t, torch.float32),
                      [codes, scales, w, ws, bias, zeros, total]),
        'int8_linear': (il.int8_dynamic_forward_func, [x, w, ws, bias, total]),
        'residual_norm': (lambda *a: bo.residual_norm(*a, scale=0.5), [x, r, one, one * 2, gate]),
        'rotary_embed': (bo.rotary_embed, [q, k, pos, freq])}[name]
    want = _leaves(call(*args))
    for i in range(len(args)):
        got = _leaves(call(*args[:i], _negated(args[i]), *args[i + 1:]))
        assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want)), (name, i)
    z = torch.complex(x, x).conj().imag                    # as a program comes by one
    assert z.is_neg()
    assert all(torch.equal(a, b) for a, b in zip(il.act_quant(z), il.act_quant(-x)))


def test_negated_in_place():
    from lightcompress_b200.block_ops import rotary_embed
    q, pos, freq = torch.randn(1, 2, 3, 8, device='cuda'), torch.arange(3, device='cuda'), torch.rand(4, device='cuda')
    for a, b in ((_negated(q), None), (q.clone(), _negated(q))):
        with pytest.raises(ValueError, match='negation'):
            rotary_embed(a, b, pos, freq, inplace=True)

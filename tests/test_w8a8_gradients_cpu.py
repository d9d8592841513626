"""Tensors whose derivatives the W8A8 operators would drop are refused, whichever operand they are.  A call that is not
refused ends at 'no CPU path' here."""
import pytest
import torch
import torch.autograd.forward_ad as fw


def calls():
    """(name, call of one operand, that operand) for every operand of a floating-point type"""
    from lightcompress_b200 import block_ops as bo, int8_linear as il
    x, r, one = torch.ones(2, 64), torch.ones(2, 64), torch.ones(64)
    a, a_s = torch.ones(2, 64, dtype=torch.int8), torch.ones(2, 1)
    w, ws, bias = torch.ones(8, 64, dtype=torch.int8), torch.ones(8), torch.ones(8)
    q, k, pos, freq = torch.ones(1, 2, 3, 8), torch.ones(1, 1, 3, 8), torch.arange(3), torch.ones(4)
    kw = dict(out_dtype=torch.float32)
    yield 'act_quant x', lambda t: il.act_quant(t), x
    yield 'gated gate', lambda t: il.gated_act_quant(t, r), x
    yield 'gated up', lambda t: il.gated_act_quant(x, t), r
    yield 'gemm a_s', lambda t: il.int8_gemm(a, t, w, ws, bias, **kw), a_s
    yield 'gemm b_s', lambda t: il.int8_gemm(a, a_s, w, t, bias, **kw), ws
    yield 'gemm bias', lambda t: il.int8_gemm(a, a_s, w, ws, t, **kw), bias
    yield 'linear x', lambda t: il.int8_dynamic_forward_func(t, w, ws, bias), x
    yield 'linear w_scale', lambda t: il.int8_dynamic_forward_func(x, w, t, bias), ws
    yield 'linear bias', lambda t: il.int8_dynamic_forward_func(x, w, ws, t), bias
    yield 'norm x', lambda t: bo.residual_norm(t, r, weight=one), x
    yield 'norm residual', lambda t: bo.residual_norm(x, t, weight=one), r
    yield 'norm weight', lambda t: bo.residual_norm(x, r, weight=t), one
    yield 'norm post_weight', lambda t: bo.residual_norm(x, r, post_weight=t), one
    yield 'norm gate', lambda t: bo.residual_norm(x, r, gate=t), one
    yield 'rotary q', lambda t: bo.rotary_embed(t, k, pos, freq), q
    yield 'rotary k', lambda t: bo.rotary_embed(q, t, pos, freq), k
    yield 'rotary inv_freq', lambda t: bo.rotary_embed(q, k, pos, t), freq


NAMES = ['act_quant x', 'gated gate', 'gated up', 'gemm a_s', 'gemm b_s', 'gemm bias', 'linear x', 'linear w_scale', 'linear bias',
         'norm x', 'norm residual', 'norm weight', 'norm post_weight', 'norm gate', 'rotary q', 'rotary k', 'rotary inv_freq']


def test_names():
    assert [name for name, _, _ in calls()] == NAMES


@pytest.mark.parametrize('name', NAMES)
def test_derivatives_are_not_dropped(name):
    call, t = next((c, t) for n, c, t in calls() if n == name)
    with pytest.raises(RuntimeError, match='no CPU path'):
        call(t)
    with pytest.raises(RuntimeError, match='no backward'):
        call(t.clone().requires_grad_())
    with torch.no_grad(), pytest.raises(RuntimeError, match='no CPU path'):
        call(t.clone().requires_grad_())
    with fw.dual_level():
        with pytest.raises(RuntimeError, match='no CPU path'):
            call(t)
        for mode in (torch.enable_grad, torch.no_grad):          # no_grad leaves forward mode on
            with mode(), pytest.raises(RuntimeError, match='forward-mode'):
                call(fw.make_dual(t, torch.ones_like(t)))


def test_module_refuses_dual_tensors():
    from lightcompress_b200 import Int8Linear
    lin = Int8Linear(torch.ones(8, 64, dtype=torch.int8), torch.ones(8))
    with fw.dual_level(), pytest.raises(RuntimeError, match='forward-mode'):
        lin(fw.make_dual(torch.ones(2, 64), torch.ones(2, 64)))

"""What the compiled front of the W8A8 operators has to leave to Python: operands that are no tensors of the device, one
position at a time."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _calls_and_operands():
    """name -> (arguments that the front serves, positions of its tensors, positions that may be left out)"""
    x, r = torch.randn(4, 64, device='cuda'), torch.randn(4, 64, device='cuda')
    one = torch.ones(64, device='cuda')
    w, ws = torch.ones(8, 64, dtype=torch.int8, device='cuda'), torch.ones(8, device='cuda')
    bias, total = torch.zeros(8, device='cuda'), w.sum(1, dtype=torch.int32)
    codes, scales = torch.ones(4, 64, dtype=torch.int8, device='cuda'), torch.ones(4, 1, device='cuda')
    zeros = torch.zeros(4, 1, dtype=torch.int32, device='cuda')
    q, k = torch.randn(1, 2, 3, 8, device='cuda'), torch.randn(1, 1, 3, 8, device='cuda')
    pos, freq = torch.arange(3, device='cuda'), torch.ones(4, device='cuda')
    return {'act_quant': ([x, True], [0], []),
            'gated_act_quant': ([x, r, 1, True], [0, 1], []),
            'int8_gemm': ([codes, scales, w, ws, bias, zeros, total, torch.float32], range(7), [4, 5]),
            'int8_linear': ([x, w, ws, bias, total], range(5), [3, 4]),
            'residual_norm': ([x, r, one, one, one, 1.0, 1e-6, 0.0, False, True], range(5), [1, 2, 3, 4]),
            'rotary_embed': ([q, k, pos, freq, False, 1.0], range(4), [1])}


@pytest.mark.parametrize('name', ['act_quant', 'gated_act_quant', 'int8_gemm', 'int8_linear', 'residual_norm', 'rotary_embed'])
def test_operands_that_are_no_tensors_of_the_device(name):
    from lightcompress_b200 import _calls, int8_linear as il
    il.int8_dynamic_forward_func(torch.ones(1, 16, device='cuda'), torch.ones(1, 16, dtype=torch.int8, device='cuda'),
                                 torch.ones(1, device='cuda'))          # the status word exists from here on
    args, tensors, optional = _calls_and_operands()[name]
    assert getattr(_calls, name)(*args) is not None
    for i in tensors:
        for bad in (None, 3, 'x', args[i].cpu()):
            if bad is None and i in optional:
                continue
            assert getattr(_calls, name)(*args[:i], bad, *args[i + 1:]) is None, (name, i, bad)


def test_a_norm_without_its_input_is_an_error():
    """A sub-layer that returned None, in front of a residual or a weight on the device."""
    from lightcompress_b200.block_ops import residual_norm
    x, one = torch.randn(4, 64, device='cuda'), torch.ones(64, device='cuda')
    for kw in ({'residual': x}, {'weight': one}, {'residual': x, 'weight': one, 'post_weight': one}, {'gate': one}):
        with pytest.raises((AttributeError, TypeError)):
            residual_norm(None, **kw)
        with torch.no_grad(), pytest.raises((AttributeError, TypeError)):
            residual_norm(None, **kw)


@pytest.mark.parametrize('name', ['act_quant', 'gated_act_quant', 'int8_gemm', 'int8_linear', 'residual_norm', 'rotary_embed'])
def test_dual_tensors_are_left_to_python(name):
    """Forward-mode derivatives: the front may not drop a tangent; Python refuses the call."""
    import torch.autograd.forward_ad as fw
    from lightcompress_b200 import _calls, block_ops as bo, int8_linear as il
    il.int8_dynamic_forward_func(torch.ones(1, 16, device='cuda'), torch.ones(1, 16, dtype=torch.int8, device='cuda'),
                                 torch.ones(1, device='cuda'))
    args, tensors, _ = _calls_and_operands()[name]
    public = {'act_quant': il.act_quant, 'gated_act_quant': lambda g, u, kind, sym: il.gated_act_quant(g, u, 'silu', sym),
              'int8_gemm': il.int8_gemm, 'int8_linear': il.int8_dynamic_forward_func, 'residual_norm': bo.residual_norm,
              'rotary_embed': bo.rotary_embed}[name]
    with fw.dual_level():
        assert getattr(_calls, name)(*args) is not None
        for i in tensors:
            if not args[i].is_floating_point():
                continue
            dual = fw.make_dual(args[i], torch.ones_like(args[i]))
            given = (*args[:i], dual, *args[i + 1:])
            with torch.no_grad():
                assert getattr(_calls, name)(*given) is None
                with pytest.raises(RuntimeError, match='forward-mode'):
                    public(*given)

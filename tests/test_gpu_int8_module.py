"""Int8Linear moved to the GPU and cast, against the functional call on the same codes, bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _codes(k):
    g = torch.Generator().manual_seed(k)
    return (torch.randint(-128, 128, (40, k), generator=g, dtype=torch.int8), torch.rand(40, generator=g) * 0.01 + 1e-3,
            torch.randn(40, generator=g))


def _want(codes, scale, bias, x, sym):
    from lightcompress_b200 import int8_linear as il
    w = il.aligned_rows(codes.cuda())
    return il.int8_dynamic_forward_func(x, w, scale.cuda(), bias.to(x.dtype).cuda(), None if sym else w.sum(1, dtype=torch.int32))


@pytest.mark.parametrize('sym', [True, False])
@pytest.mark.parametrize('k', [30, 64, 1399])
def test_built_on_the_cpu_and_moved(k, sym):
    from lightcompress_b200 import Int8Linear
    codes, scale, bias = _codes(k)
    m = Int8Linear(codes, scale, bias, sym).cuda()
    x = torch.randn(5, k, device='cuda')
    assert torch.equal(m(x), _want(codes, scale, bias, x, sym))
    there = m.cpu().to('cuda:0')
    assert torch.equal(there(x), _want(codes, scale, bias, x, sym))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_cast_with_a_model(dtype):
    from lightcompress_b200 import Int8Linear
    for k, sym in ((30, True), (256, False)):
        codes, scale, bias = _codes(k)
        model = torch.nn.Sequential(torch.nn.Linear(k, k), Int8Linear(codes, scale, bias, sym)).to('cuda').to(dtype)
        x = torch.randn(5, k, device='cuda').to(dtype)
        assert torch.equal(model[1](x), _want(codes, scale, bias, x, sym))


def test_zero_points_beside_those_of_the_fake_quantiser():
    """The grid of IntegerQuantizer(8, False, 'per_token') for tokens of both signs: the same steps (a division apart, 2^-23) and
    values at most a step apart (zero points next to a rounding border, and codes next to one).  Tokens of one sign: the range
    is widened to hold zero, so that every value is within half a step; the quantiser cuts off what lies beyond max - min."""
    from lightcompress_b200 import IntegerQuantizer
    from lightcompress_b200.int8_linear import act_quant
    g = torch.Generator().manual_seed(4)
    both = torch.randn(64, 512, generator=g).cuda()
    one = (torch.rand(64, 512, generator=g) + 1).cuda()                     # between 1 and 2
    fake = IntegerQuantizer(8, False, 'per_token')
    for x in (both, one, -one):
        codes, scales, zeros = act_quant(x, sym=False)
        value = (codes.float() - zeros) * scales
        # the ends of a range of both signs may be cut by the zero point's rounding, half a step
        assert bool(((value - x).abs() <= scales * (1.01 if x is both else 0.5 + 2.0 ** -10)).all())
        off = (value - fake.fake_quant_act_dynamic(x)).abs()
        if x is both:
            want = (x.amax(1, keepdim=True) - x.amin(1, keepdim=True)) / 255
            assert torch.allclose(scales, want, rtol=2.0 ** -22, atol=0)
            assert bool((off <= scales * 1.01).all())
        else:
            assert float(off.max()) > 0.5                                    # the far end, not a step (2 / 255)

"""Int8Linear as a module among others: moved, cast, copied, saved and loaded.  The products read rows that begin at multiples
of 16 bytes and scales in fp32, whatever is done to the module.  The meta device stands for another device here."""
import copy
import io

import pytest
import torch


def _module(k=30, sym=True, bias=True):
    from lightcompress_b200 import Int8Linear
    g = torch.Generator().manual_seed(k)
    codes = torch.randint(-128, 128, (8, k), generator=g, dtype=torch.int8)
    return Int8Linear(codes, torch.rand(8, generator=g) + 0.1, torch.randn(8, generator=g) if bias else None, sym), codes


def _laid_out(m):
    from lightcompress_b200.int8_linear import _rows_aligned
    assert _rows_aligned(m.weight), m.weight.stride()
    with pytest.raises(RuntimeError, match='no CPU path'):          # nothing else is wrong with a call
        m(torch.zeros(2, m.in_features, dtype=torch.float32 if m.bias is None else m.bias.dtype))


@pytest.mark.parametrize('k', [30, 32, 1])
@pytest.mark.parametrize('sym', [True, False])
def test_rows_stay_laid_out(k, sym):
    m, codes = _module(k, sym)
    _laid_out(m)
    away = copy.deepcopy(m).to('meta')
    assert away.weight.device.type == 'meta' and (k % 16 == 0 or away.weight.stride()[0] % 16 == 0)
    back = away.to_empty(device='cpu')                              # as a model is built before it is loaded
    back.load_state_dict(m.state_dict())
    _laid_out(back)
    assert torch.equal(back.weight, codes)
    # a copy on the same device by force, as a move makes one
    moved = copy.deepcopy(m)._apply(lambda t: t.contiguous().clone(memory_format=torch.contiguous_format))
    _laid_out(moved)
    assert torch.equal(moved.weight, codes) and torch.equal(moved.weight_scale, m.weight_scale)
    state = {name: t.contiguous() for name, t in m.state_dict().items()}
    for assign in (False, True):
        other, _ = _module(k, sym)
        other.weight.zero_()
        other.load_state_dict(state, assign=assign)
        _laid_out(other)
        assert torch.equal(other.weight, codes)
    file = io.BytesIO()
    torch.save(m, file)
    file.seek(0)
    again = torch.load(file, weights_only=False)
    _laid_out(again)
    assert torch.equal(again.weight, codes)
    block = torch.nn.Sequential(torch.nn.Linear(k, k), copy.deepcopy(m))
    block._apply(lambda t: t.clone(memory_format=torch.contiguous_format))
    _laid_out(block[1])


@pytest.mark.parametrize('cast', ['half', 'bfloat16', 'double', 'to', 'to_both', 'type', 'to_meta'])
def test_scales_keep_their_type_and_value(cast):
    for k, sym in ((30, True), (64, False)):
        m, codes = _module(k, sym)
        want = m.weight_scale.clone()
        outer = torch.nn.Sequential(m)
        if cast == 'to':
            outer.to(torch.bfloat16)
        elif cast == 'to_both':
            outer.to(device='cpu', dtype=torch.float16)
        elif cast == 'type':
            outer.type(torch.float16)
        elif cast == 'to_meta':
            outer.to(device='meta', dtype=torch.float16)
        else:
            getattr(outer, cast)()
        assert m.weight.dtype == torch.int8 and m.weight_scale.dtype == torch.float32
        assert sym or m.weight_sum.dtype == torch.int32
        assert m.bias.dtype == {'half': torch.float16, 'bfloat16': torch.bfloat16, 'double': torch.float64, 'to': torch.bfloat16}.get(cast, torch.float16)
        if cast == 'to_meta':
            assert {t.device.type for t in m.state_dict().values()} == {'meta'}
            continue
        assert torch.equal(m.weight_scale, want) and torch.equal(m.weight, codes)
        if cast != 'double':
            _laid_out(m)
            outer.float()                                           # there and back: only the bias was rounded
            assert torch.equal(m.weight_scale, want)
            _laid_out(m)


def test_quantisers_that_it_is_no_deployment_of_are_refused():
    """Settings of the activations' quantiser that the module would otherwise pass over."""
    from lightcompress_b200 import FloatQuantizer, Int8Linear, IntegerQuantizer
    lin = torch.nn.Linear(16, 8)
    codes, scale = torch.ones(8, 16, dtype=torch.int8), torch.ones(8, 1)

    def new(aq):
        return Int8Linear.new(lin, lambda module, wq: (codes, scale, None), object(), aq)
    for aq in (None, IntegerQuantizer(8, True, 'per_token'), IntegerQuantizer(8, False, 'per_token'),
               IntegerQuantizer(8, True, 'per_token', round_zp=False)):
        assert new(aq).in_features == 16
    for aq in (IntegerQuantizer(8, True, 'per_token', calib_algo='static_minmax'), IntegerQuantizer(8, True, 'per_token', calib_algo='mse'),
               IntegerQuantizer(8, True, 'per_token', calib_algo='static_hist'), IntegerQuantizer(8, False, 'per_token', round_zp=False),
               IntegerQuantizer(8, True, 'per_tensor'), IntegerQuantizer(6, True, 'per_token'),
               FloatQuantizer('e4m3', True, 'per_token', use_qtorch=True)):
        with pytest.raises(NotImplementedError, match='Int8Linear'):
            new(aq)

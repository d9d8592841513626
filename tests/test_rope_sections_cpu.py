"""What a configuration's section says of the base is not passed over."""
import pytest
import torch


def _f(*a, **kw):
    from lightcompress_b200.block_ops import rope_frequencies
    return rope_frequencies(*a, device='cpu', **kw)


@pytest.mark.parametrize('kind,more', [('default', {}), ('linear', {'factor': 2.0}),
                                       ('yarn', {'factor': 4.0, 'original_max_position_embeddings': 64}),
                                       ('llama3', {'factor': 8.0, 'low_freq_factor': 1.0, 'high_freq_factor': 4.0,
                                                   'original_max_position_embeddings': 256}),
                                       ('dynamic', {'factor': 4.0, 'original_max_position_embeddings': 64})])
def test_the_sections_own_base(kind, more):
    section = dict(more, rope_type=kind)
    want, scale = _f(64, 500000.0, section, seq_len=300)
    other, _ = _f(64, scaling=section, seq_len=300)
    assert not torch.equal(want, other) and torch.equal(other, _f(64, 10000.0, section, seq_len=300)[0])
    given = dict(section, rope_theta=500000.0, partial_rotary_factor=0.5)
    got, same = _f(64, scaling=given, seq_len=300)
    assert torch.equal(got, want) and same == scale
    assert torch.equal(_f(64, 500000.0, given, seq_len=300)[0], want)
    with pytest.raises(ValueError, match='rope_theta'):
        _f(64, 10000.0, given, seq_len=300)


def test_sections_for_several_kinds_of_layer():
    both = {'full_attention': {'rope_type': 'linear', 'factor': 8.0, 'rope_theta': 1e6}, 'sliding_attention': {'rope_type': 'default', 'rope_theta': 1e4}}
    with pytest.raises(ValueError, match='kind'):
        _f(64, scaling=both)
    assert torch.equal(_f(64, scaling=both['full_attention'])[0], _f(64, 1e6, {'type': 'linear', 'factor': 8.0})[0])


def test_no_section_at_all():
    assert torch.equal(_f(8)[0], _f(8, 10000.0)[0]) and torch.equal(_f(8)[0], torch.tensor([1.0, 0.1, 0.01, 0.001]))

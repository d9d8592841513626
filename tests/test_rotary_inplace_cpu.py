"""What rotary_embed refuses to do in place: elements that two heads share would be read and written in any order.  The
refusals come before anything touches a GPU; tensors on the CPU that are not refused end at 'no CPU path'."""
import itertools
import random

import pytest
import torch


def _rope(q, k):
    from lightcompress_b200.block_ops import rotary_embed
    t = q.shape[2]
    return rotary_embed(q, k, torch.arange(t), torch.ones(2), inplace=True)


def test_heads_that_share_elements_are_refused():
    room = torch.zeros(4096)
    q = room[:2 * 4 * 3 * 8].view(2, 3, 4, 8).transpose(1, 2)              # (2, 4, 3, 8)
    for k in (q[:, 1:], q[:, 2:3], q[1:].expand(1, 4, 3, 8).reshape(1, 4, 3, 8).expand(2, 4, 3, 8), q[:, 1:2, :, :],
              room[4:4 + 2 * 3 * 8].view(2, 1, 3, 8), room[8 * 23:8 * 23 + 48].view(2, 3, 1, 8).transpose(1, 2)):
        with pytest.raises(ValueError, match='in place'):
            _rope(q, k)
    # heads that begin 4 elements apart, tokens that overlap
    for bad in (torch.as_strided(room, (1, 3, 2, 8), (0, 4, 64, 1)), torch.as_strided(room, (1, 2, 3, 8), (0, 16, 16, 1)),
                torch.as_strided(room, (2, 2, 2, 8), (24, 8, 16, 1)), torch.as_strided(room, (2, 3, 5, 8), (40, 16, 8, 1))):
        with pytest.raises(ValueError, match='in place'):
            _rope(bad, None)


def test_views_of_one_projection_are_not():
    b, t, h, g, d = 2, 3, 4, 2, 8
    qkv = torch.zeros(b, t, (h + 2 * g) * d + 3)
    q = qkv[..., :h * d].unflatten(-1, (h, d)).transpose(1, 2)
    k = qkv[..., h * d:(h + g) * d].unflatten(-1, (g, d)).transpose(1, 2)
    apart = torch.zeros(b, t, h, 3, d)                                      # q, k and v of a head side by side
    pairs = [(q, k), (k, q), (apart[..., 0, :].transpose(1, 2), apart[..., 1, :].transpose(1, 2)), (q, None),
             (torch.zeros(b, h, t, d), torch.zeros(b, g, t, d)), (torch.zeros(b, h, t, d)[:, :2], None)]
    one = torch.zeros(1, 1, h + g, d)                                       # strides of dimensions of one index say nothing
    pairs.append((one[:, :, :h].transpose(1, 2), one[:, :, h:].transpose(1, 2)))
    cache = torch.zeros(b, 64, g, d)                                        # a cache's rows beside a fresh q
    pairs.append((torch.zeros(b, t, h, d).transpose(1, 2), cache[:, 5:5 + t].transpose(1, 2)))
    halves = torch.zeros(b, h, t, 2 * d)
    pairs.append((halves[..., :d], halves[:, :2, :, d:]))
    for a, c in pairs:
        with pytest.raises(RuntimeError, match='no CPU path'):
            _rope(a, c)


def test_shared_elements_against_a_count_of_all_of_them():
    from lightcompress_b200.block_ops import _layouts_meet, _meets_itself
    rng, room = random.Random(3), torch.zeros(4000)

    def view():
        shape = [rng.choice([1, 1, 2, 3, 4]) for _ in range(3)] + [rng.choice([1, 2, 4])]
        stride = [rng.choice([1, 2, 4, 5, 8, 12, 16, 24, 48, 96]) for _ in range(3)] + [1]
        return torch.as_strided(room, shape, stride, rng.randint(0, 120))

    def places(x):
        return [x.storage_offset() + sum(i * s for i, s in zip(at, x.stride())) for at in itertools.product(*map(range, x.shape))]
    seen = set()
    for _ in range(4000):
        a, b = view(), view()
        pa, pb = places(a), places(b)
        assert _meets_itself(a.shape, a.stride()) == (len(set(pa)) < len(pa))
        shared = bool(set(pa) & set(pb))
        apart = b.storage_offset() - a.storage_offset()
        layouts = (a.shape, a.stride()), (b.shape, b.stride())
        assert _layouts_meet(apart, *layouts[0], *layouts[1]) == shared == _layouts_meet(-apart, *layouts[1], *layouts[0])
        seen.add(shared)
    assert seen == {True, False}


def test_autograd_learns_of_what_changed_in_place(monkeypatch):
    """A tensor that a backward pass still needs: changed in place, that pass refuses, as it does behind torch's own
    operators.  (The launch itself is left out: there is no GPU here.)"""
    from lightcompress_b200 import block_ops as bo
    monkeypatch.setattr(bo.L, 'launch', lambda *a: None)
    pos, freq = torch.arange(3), torch.ones(2)
    for which in (0, 1):
        x = torch.randn(2, 4, 3, 8, requires_grad=True)
        y = x.exp()                                    # kept for the backward pass
        other = torch.zeros(2, 4, 3, 8)
        before = other._version
        with torch.no_grad():
            bo.rotary_embed(*((y, other) if which == 0 else (other, y)), pos, freq, inplace=True)
        assert other._version > before
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            y.sum().backward()
    y = x.exp()
    with torch.no_grad():
        bo.rotary_embed(y, None, pos, freq)            # not in place: nothing changed
    y.sum().backward()
    with torch.inference_mode():
        z = torch.zeros(2, 4, 3, 8)
        assert bo.rotary_embed(z, None, pos, freq, inplace=True)[0] is z
    assert bo.rotary_embed(z, None, pos, freq, inplace=True)[0] is z

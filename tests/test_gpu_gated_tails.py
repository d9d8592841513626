"""Gated quantisation of tokens whose gates all lie in the negative tail of the activation, where nothing larger hides its
error: scale and codes follow from values that are small themselves.

Tolerance, with e = 2^-23: an exponential of argument y is off by (2 + 1.17 |y|) e relative (CUDA's bound for the fast one),
a fast quotient by 2 e, the sum under it by e / 2.
  silu       y = x                                            (5 + 1.2 |x|) e
  gelu_tanh  y = u of seven roundings: 3.5 |u| e besides      (5 + 4.7 |u|) e
  gelu       y = x^2 / 2, itself of a rounding: 0.25 x^2 e and 0.59 x^2 e; the quotient t and its sum 2.5 e, which the
             polynomial passes on at most once; its fit and its seven roundings 13 e; three products 1.5 e: in all
             (18 + 0.9 x^2) e, measured on the CPU for the fit alone: 1.5e-6 = 12.6 e
and a rounding of act * up, of the division by 127 and of the scale: 2 e.  So much of a row's largest value is its scale off;
a code, which is half a step from v / s, by 127 times that of its own value besides."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -23


def _value(x, act):
    """act(x) in fp64 without cancellation below zero, and its relative tolerance."""
    x = x.double()
    if act == 'silu':
        return x / (1 + torch.exp(-x)), (5 + 1.2 * x.abs()) * E
    if act == 'gelu_tanh':
        u = 2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
        return x / (1 + torch.exp(-u)), (5 + 4.7 * u.abs()) * E
    return x * torch.special.erfc(-x / math.sqrt(2)) / 2, (18 + 0.9 * x * x) * E


RANGES = [('silu', -8, -2), ('silu', -48, -30), ('silu', -86, -60), ('silu', -1, 0), ('gelu_tanh', -4.5, -2), ('gelu_tanh', -9, -5),
          ('gelu_tanh', -1, 0), ('gelu', -3, -2.5), ('gelu', -8, -2), ('gelu', -7.5, -6.5), ('gelu', -12, -9), ('gelu', -1, 0), ('gelu', -20, 20)]


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize('act,low,high', RANGES)
@pytest.mark.parametrize('power', [0, 14, 40, 110])
def test_tokens_in_the_tail(dtype, act, low, high, power):
    from lightcompress_b200.int8_linear import gated_act_quant
    if dtype == torch.float16 and power > 14:
        pytest.skip('beyond the type')
    g = torch.Generator().manual_seed(power + int(1000 * high))
    gate = (low + (high - low) * torch.rand(64, 96, generator=g)).to(dtype)
    up = ((0.5 + torch.rand(64, 96, generator=g)) * 2.0 ** power).to(dtype)
    a, tol = _value(gate, act)
    keep = (a * up.double()).abs().amax(-1) < 1e38
    v, tol = (a * up.double())[keep], tol[keep]
    codes, scale = gated_act_quant(gate[keep].cuda(), up[keep].cuda(), act)
    codes, scale = codes.cpu().double(), scale.cpu().double()
    tol = tol + 2 * E
    top = v.abs().amax(-1, keepdim=True)
    # every value within its own tolerance: the largest of them lies within the largest tolerance of all that come near it
    upper, lower = (v.abs() * (1 + tol)).amax(-1, keepdim=True), (v.abs() * (1 - tol)).amax(-1, keepdim=True)
    floor = torch.full_like(top, 1e-5)
    assert bool((scale * 127 <= torch.maximum(upper, floor) * (1 + 2 * E)).all())
    assert bool((scale * 127 >= torch.maximum(lower, floor) * (1 - 2 * E)).all())
    off = (codes - v / scale).abs()
    assert bool((off <= 0.5 + 127 * (tol + 2 * E)).all()), float(off.max())

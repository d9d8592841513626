"""Fused element-wise pieces of the calibration block forward.

The reference's block_forward (llmc/compression/quantization/base_blockwise_quantization.py:378-401)
runs the decoder block's stock module code.  Three chains of small tensor ops in that code -- the
RMS norms, the rotary embedding of q and k and the gated activation of the MLP -- cost more HBM
passes than all quantisation kernels together, so the staged Llama schedule swaps them for one
kernel each.  The kernels round after every op of the chain they replace (the RMS norm also
associates its sum of squares like torch's row reduction); before a swap is used it is compared
bit for bit with the stock code on random data, and the stock code is kept if they differ (another
rotary convention, activation or norm, or a torch build that reduces in another order).

The second half of the file are the operators of a deployed block that such a check cannot cover, because
they round once instead of after every op: residual_norm (the residual add with the norms on both sides of
it, a gate and a multiplier, and the 8-bit quantisation the next integer linear needs) and rotary_embed
(rotary positions from inv_freq: both pair layouts, part of a head, scaled frequencies).
"""
import contextlib
import functools
import math
import sys

import numpy as np
import torch

from . import _lib as L
from . import int8_linear
from ._lib import _calls

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_checked = {}


def rejected():
    """The self-checks that failed so far, i.e. the module kinds for which the stock tensor ops were kept
    because the fused kernel did not reproduce them bit for bit: [(kind, detail), ...].  Empty on the
    Llama block this library is built for; a benchmark or a caller that expects the fused path reads this
    instead of guessing."""
    return [(k[0], str(k[1])) for k, ok in _checked.items() if not ok]


def rope_apply_one(x, cos, sin):
    """x: (B, H, T, D) view of a (B, T, H, D) contiguous tensor; cos, sin: (B, T, D) or (1, T, D)
    contiguous.  Returns the embedded tensor with x's shape and memory layout."""
    B, H, T, D = x.shape
    mem = x.transpose(1, 2)
    out = torch.empty_like(mem)
    L.call('lc_rope_apply', L.ptr(mem), L.ptr(cos), L.ptr(sin), L.lc_dtype(x), B * T, H, D, cos.shape[0] * T,
           L.ptr(out), L.stream_of(x))
    return out.transpose(1, 2)


def _rope_fits(q, k, cos, sin, unsqueeze_dim):
    if unsqueeze_dim != 1 or not q.is_cuda or q.dtype not in _DTYPES or q.dim() != 4 or k.dim() != 4:
        return False
    if not (k.dtype == cos.dtype == sin.dtype == q.dtype):
        return False
    B, _, T, D = q.shape
    if cos.shape not in ((B, T, D), (1, T, D)) or sin.shape != cos.shape or k.shape[0] != B \
            or k.shape[2:] != (T, D):
        return False
    if D % (8 if q.dtype == torch.float32 else 16):
        return False
    return (q.transpose(1, 2).is_contiguous() and k.transpose(1, 2).is_contiguous() and cos.is_contiguous()
            and sin.is_contiguous() and all(t.data_ptr() % 16 == 0 for t in (q, k, cos, sin)))


def _make_rope(orig):
    def apply_rotary_pos_emb(q, k, cos, sin, unsqueeze_dim=1, **kw):
        if kw or not _rope_fits(q, k, cos, sin, unsqueeze_dim):
            return orig(q, k, cos, sin, unsqueeze_dim=unsqueeze_dim, **kw)
        return rope_apply_one(q, cos, sin), rope_apply_one(k, cos, sin)
    return apply_rotary_pos_emb


def _rope_matches(orig, device, dtype):
    """True if `orig` is the rotate-half convention the kernel implements (checked on random data)."""
    key = ('rope', id(orig), str(device), dtype)
    if key not in _checked:
        g = torch.Generator().manual_seed(7)
        q = torch.randn(2, 5, 3, 32, generator=g).to(dtype).to(device).transpose(1, 2)
        k = torch.randn(2, 5, 1, 32, generator=g).to(dtype).to(device).transpose(1, 2)
        cos = torch.randn(2, 5, 32, generator=g).to(dtype).to(device)
        sin = torch.randn(2, 5, 32, generator=g).to(dtype).to(device)
        try:
            rq, rk = orig(q, k, cos, sin)
            ok = torch.equal(rq, rope_apply_one(q, cos, sin)) and torch.equal(rk, rope_apply_one(k, cos, sin))
        except (TypeError, RuntimeError, ValueError):
            ok = False
        _checked[key] = ok
    return _checked[key]


@contextlib.contextmanager
def fused_rotary(attn_module, device, dtype):
    """While active, the Python module that defines `attn_module`'s class applies the rotary
    embedding through lc_rope_apply.  Yields whether the swap took place."""
    mod = sys.modules.get(type(attn_module).__module__)
    orig = getattr(mod, 'apply_rotary_pos_emb', None)
    if orig is None or dtype not in _DTYPES or not _rope_matches(orig, device, dtype):
        yield False
        return
    mod.apply_rotary_pos_emb = _make_rope(orig)
    try:
        yield True
    finally:
        mod.apply_rotary_pos_emb = orig


def silu_mul(gate, up):
    out = torch.empty_like(gate)
    L.call('lc_silu_mul', L.ptr(gate), L.ptr(up), L.lc_dtype(gate), gate.numel(), L.ptr(out), L.stream_of(gate))
    return out


def gated_act(act_fn, gate, up):
    """act_fn(gate) * up; through lc_silu_mul when act_fn is SiLU (verified once per activation type,
    device and dtype on random data) and the tensors fit the kernel, else with the stock ops."""
    fits = (gate.is_cuda and gate.dtype in _DTYPES and up.dtype == gate.dtype and gate.shape == up.shape
            and gate.is_contiguous() and up.is_contiguous() and gate.numel() % 8 == 0
            and gate.data_ptr() % 16 == 0 and up.data_ptr() % 16 == 0)
    if fits:
        key = ('act', type(act_fn), str(gate.device), gate.dtype)
        if key not in _checked:
            g = torch.Generator().manual_seed(11)
            a = (torch.randn(4096, generator=g) * 4).to(gate.dtype).to(gate.device)
            b = torch.randn(4096, generator=g).to(gate.dtype).to(gate.device)
            _checked[key] = torch.equal(act_fn(a) * b, silu_mul(a, b))
        if _checked[key]:
            return silu_mul(gate, up)
    return act_fn(gate) * up


def _rms_raw(x, weight, eps):
    x2 = x.reshape(-1, x.shape[-1])
    rows, C = x2.shape
    out = torch.empty_like(x2)
    # 1/C the way the mean it replaces forms it: fp32 rows / fp32 (rows * C)
    factor = float(np.float32(rows) / np.float32(rows * C))
    L.call('lc_rmsnorm', L.ptr(x2), L.ptr(weight), L.lc_dtype(x2), rows, C, factor, float(eps), L.ptr(out),
           L.stream_of(x2))
    return out.view(x.shape)


def rms_norm(module, x):
    """module(x) for a Llama-style RMS norm (weight, variance_epsilon) through lc_rmsnorm when the
    kernel reproduces the module bit for bit (checked once per module type, width, dtype and device
    on random rows that include the row count of `x`), else the module itself."""
    w = getattr(module, 'weight', None)
    eps = getattr(module, 'variance_epsilon', None)
    C = x.shape[-1]
    fits = (w is not None and eps is not None and x.is_cuda and x.dtype in _DTYPES and w.dtype == x.dtype
            and w.dim() == 1 and w.shape[0] == C and C % 128 == 0 and 128 <= C < 8192 and x.is_contiguous()
            and w.is_contiguous() and x.data_ptr() % 16 == 0 and w.data_ptr() % 16 == 0 and x.numel() > 0)
    if not fits:
        return module(x)
    rows = x.numel() // C
    key = ('rms', type(module), C, rows, float(eps), str(x.device), x.dtype)
    if key not in _checked:
        g = torch.Generator().manual_seed(13)
        t = torch.randn(rows, C, generator=g)
        t[: rows // 2] *= torch.rand(rows // 2, 1, generator=g) * 30     # a spread of row norms
        wt = torch.randn(C, generator=g) * 0.5 + 1
        saved = module.weight.data
        ok = True
        try:
            # in fp32 nothing hides a differently associated sum; then the dtype actually used
            for dt in (torch.float32, x.dtype):
                module.weight.data = wt.to(dt).to(x.device)
                td = t.to(dt).to(x.device).view(x.shape)
                ok = ok and torch.equal(module(td), _rms_raw(td, module.weight.data, eps))
        finally:
            module.weight.data = saved
        _checked[key] = ok
    if _checked[key]:
        return _rms_raw(x, w.data, eps)
    return module(x)


@contextlib.contextmanager
def fused_gated_mlp(mlp):
    """While active, `type(mlp).forward` is down_proj(act_fn(gate_proj(x)) * up_proj(x)) with the
    activation and the product in one kernel (gated_act).  Only swapped in if the class's own forward
    gives the same bits on random data for this module's layout; yields whether it was."""
    cls = type(mlp)
    need = all(hasattr(mlp, a) for a in ('gate_proj', 'up_proj', 'down_proj', 'act_fn'))
    w = getattr(getattr(mlp, 'gate_proj', None), 'weight', None)
    if not need or w is None or not w.is_cuda or w.dtype not in _DTYPES:
        yield False
        return
    orig = cls.forward

    def forward(self, x):
        return self.down_proj(gated_act(self.act_fn, self.gate_proj(x), self.up_proj(x)))
    key = ('mlp', cls, str(w.device), w.dtype)
    if key not in _checked:
        g = torch.Generator().manual_seed(17)
        t = torch.randn(2, 24, w.shape[1], generator=g).to(w.dtype).to(w.device)
        with torch.no_grad():
            _checked[key] = torch.equal(orig(mlp, t), forward(mlp, t))
    if not _checked[key]:
        yield False
        return
    cls.forward = forward
    try:
        yield True
    finally:
        cls.forward = orig


# ---- operators of a deployed block ---------------------------------------------------------------
def _strided_rows(x):
    """(..., C) as a 2-D view (a copy where there is none) with contiguous rows."""
    if x.stride(-1) != 1 and x.shape[-1] != 1:
        x = x.contiguous()
    return x if x.dim() == 2 else x.reshape(-1, x.shape[-1])


def _gate_rows(gate, x):
    """How many rows of gate there are, given that it broadcasts against x (..., C) over trailing tokens: one value
    per channel (C,), one row per leading index ((B, 1, C), (B, 1, 1, C)) or one per token (x's shape)."""
    lead = x.shape[:-1]
    g = tuple(gate.shape[:-1])
    if gate.shape[-1:] != x.shape[-1:] or len(g) > len(lead):
        return None
    g = (1,) * (len(lead) - len(g)) + g
    n = 0
    while n < len(lead) and g[n] == lead[n]:
        n += 1
    # after the indices it shares with x come ones; a shared 1 may stand on either side
    if any(v != 1 for v in g[n:]):
        return None
    return math.prod(g[:n])


def residual_norm(x, residual=None, weight=None, post_weight=None, gate=None, scale=1.0, eps=1e-6, weight_offset=0.0,
                  quant=False, sym=True):
    """The residual add of a decoder block and the norms on both sides of it, in one pass:

        t = x                     or  x * rsqrt(mean(x^2) + eps) * (post_weight + weight_offset)
        h = residual + scale * gate * t
        y = h * rsqrt(mean(h^2) + eps) * (weight + weight_offset)

    x, residual: (..., C) of one type (bf16, fp16, fp32), any strides; weight, post_weight: (C,); gate: (C,), one row
    per leading index such as (B, 1, C), or x's shape; all of x's type.  residual, post_weight, gate and weight may each
    be left out; weight_offset is 1 for norms that store their weight less one.  Statistics and sums are fp32; h is
    rounded once and y is formed from the rounded h.  A row's result does not depend on the other rows; the order of its
    sums, and so its last bits, follows the alignment that all rows have: 16 bytes, two values or one.

    Returns (h, y).  Without weight, y is None.  With quant, y is what int8_linear.act_quant returns for it, (codes,
    scales) or, with sym=False, (codes, scales, zeros), quantised from fp32.  Where h would equal x, it is x."""
    out = _calls.residual_norm(x, residual, weight, post_weight, gate, scale, eps, weight_offset, quant, sym)
    if out is not None:
        return out
    name = 'residual_norm'
    L.refuse_grad(name, x, residual, weight, post_weight, gate)
    x, residual, weight, post_weight, gate = L.resolved(x, residual, weight, post_weight, gate)
    dtype, shape, dev = x.dtype, x.shape, x.get_device()
    dt = L._DTYPES.get(dtype)
    if dt is None:
        raise TypeError(f'{name}: unsupported dtype {dtype}')
    C = shape[-1] if shape else 0
    if C == 0:
        raise ValueError(f'{name}: the last dimension must not be empty')
    rows, gate_rows = x.numel() // C, 0
    x2 = _strided_rows(x)
    ldx = x2.stride()[0]
    r2, ldr = residual, C
    if residual is not None:
        if residual.shape != shape or residual.dtype != dtype or residual.get_device() != dev:
            _refuse_operand(name, 'residual', residual, x, shape)
        r2 = _strided_rows(residual)
        ldr = r2.stride()[0]
    if weight is not None:
        if weight.dtype != dtype or weight.dim() != 1 or weight.numel() != C or weight.get_device() != dev:
            _refuse_operand(name, 'weight', weight, x, (C,))
        weight = weight.contiguous()
    elif quant:
        raise ValueError(f'{name}: quant needs the weight of the norm whose result it quantises')
    if post_weight is not None:
        if post_weight.dtype != dtype or post_weight.dim() != 1 or post_weight.numel() != C or post_weight.get_device() != dev:
            _refuse_operand(name, 'post_weight', post_weight, x, (C,))
        post_weight = post_weight.contiguous()
    if gate is not None:
        gate_rows = _gate_rows(gate, x)
        if gate_rows is None or gate.dtype != dtype or gate.get_device() != dev:
            _refuse_operand(name, 'gate', gate, x, None if gate_rows is None else gate.shape)
        gate = gate.contiguous()
    kept = residual is None and post_weight is None and gate is None and scale == 1.0
    if kept and weight is None:
        return x, None
    h = x if kept else x.new_empty(shape)
    y = codes = scales = zeros = None
    pitch = 0
    if quant:
        codes, pitch, scales, zeros, quantised = int8_linear._codes_like(x, shape, sym)
    elif weight is not None:
        y = x.new_empty(shape)
    if rows:
        L.launch(dev, 'lc_residual_norm', L.RESIDUAL_NORM.pack(
            x2.data_ptr(), _at(r2), _at(post_weight), _at(gate), gate_rows, _at(weight), dt, rows, C, ldx, ldr, scale, eps,
            weight_offset, 0 if kept else h.data_ptr(), _at(y), _at(codes), pitch, _at(scales), _at(zeros)))
    return h, quantised if quant else y


def _refuse_operand(name, key, t, x, shape):
    """Says what is wrong with an operand that does not go with x."""
    if t.dtype != x.dtype:
        raise TypeError(f'{name}: {key} is {t.dtype}, x is {x.dtype}')
    if shape is None:
        raise ValueError(f'{name}: gate {tuple(t.shape)} must be ({x.shape[-1]},), one row per leading index, or x\'s shape')
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f'{name}: {key} must have shape {tuple(shape)}, got {tuple(t.shape)}')
    L.refuse_devices(name, x, **{key: t})


def _at(t):
    return 0 if t is None else t.data_ptr()


def rotary_embed(q, k, positions, inv_freq, interleaved=False, attention_scale=1.0, inplace=False):
    """Rotary embedding of q (B, H, T, D) and k (B, G, T, D; may be None) from positions, one launch for both:
    with angle = positions * inv_freq[i], pair i of the first R = 2 * len(inv_freq) elements of every head becomes
    attention_scale * (x1 cos - x2 sin, x2 cos + x1 sin); pairs are (i, i + R/2) or, interleaved, (2i, 2i + 1); the
    other D - R elements are kept.  The angle is formed in 64 bits (positions under 2^31 lose nothing), the result rounded once.

    q, k: bf16, fp16 or fp32 with contiguous heads (any other strides, e.g. views of one projection's output);
    positions: int64, (B, T), (1, T) or (T,); inv_freq: (R / 2,) fp32, see rope_frequencies.  Returns (q, k) in new memory,
    (B, T, H, D) contiguous seen as (B, H, T, D) like the stock projections, or the given tensors if inplace; in place, no two
    heads may share elements."""
    out = None if inplace else _calls.rotary_embed(q, k, positions, inv_freq, interleaved, attention_scale)
    if out is not None:
        return out
    name = 'rotary_embed'
    L.refuse_grad(name, q, k, inv_freq)
    if inplace and (q.is_neg() or (k is not None and k.is_neg())):
        raise ValueError(f'{name}: cannot work in place on a view with a pending negation')
    q, k, positions, inv_freq = L.resolved(q, k, positions, inv_freq)
    dt = L._DTYPES.get(q.dtype)
    if dt is None:
        raise TypeError(f'{name}: unsupported dtype {q.dtype}')
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError(f'{name}: q and k must be (B, heads, T, D)')
    B, H, T, D = q.shape
    G = 0
    if k is not None:
        kb, G, kt, kd = k.shape
        if kb != B or kt != T or kd != D or k.dtype != q.dtype:
            raise ValueError(f'{name}: k {tuple(k.shape)} {k.dtype} does not go with q {tuple(q.shape)} {q.dtype}')
    shape = tuple(positions.shape)
    if positions.dtype != torch.int64 or shape not in ((B, T), (1, T), (T,)):
        raise ValueError(f'{name}: positions must be int64 of shape ({B}, {T}), (1, {T}) or ({T},), got {positions.dtype} '
                         f'{shape}')
    half = inv_freq.numel()
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not 0 < 2 * half <= D:
        raise ValueError(f'{name}: inv_freq must be between 1 and {D // 2} fp32 values, got {inv_freq.dtype} '
                         f'{tuple(inv_freq.shape)}')
    if D > 1024 or H + G > 1023:
        raise NotImplementedError(f'{name}: heads of at most 1024 elements and at most 1023 of them, got {D} and {H + G}')
    dev = q.get_device()
    if not (positions.get_device() == inv_freq.get_device() == dev) or (k is not None and k.get_device() != dev):
        L.refuse_devices(name, q, k=k, positions=positions, inv_freq=inv_freq)
    if inplace and k is not None and k.data_ptr() == q.data_ptr() and k.numel():
        raise ValueError(f'{name}: cannot work in place on one tensor as q and k')
    q, q_out, qb, qh, qt = _heads(name, q, B, H, T, D, inplace)
    if k is None:
        k_out, k_at, ko_at, kb, kh, kt = None, 0, 0, 0, 0, 0
    else:
        k, k_out, kb, kh, kt = _heads(name, k, B, G, T, D, inplace)
        k_at, ko_at = k.data_ptr(), k_out.data_ptr()
    if B and T:
        if inplace:
            fault = _shared_in_place(B, T, D, H, qb, qh, qt, G, kb, kh, kt, k_at - q.data_ptr() if G else 0, q.element_size())
            if fault is not None:
                raise ValueError(f'{name}: cannot work in place on {fault}')
        positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
        L.launch(dev, 'lc_rotary_embed', L.ROTARY_EMBED.pack(
            q.data_ptr(), q_out.data_ptr(), H, qb, qt, qh, k_at, ko_at, G, kb, kt, kh, positions.data_ptr(),
            T if len(shape) == 2 and shape[0] > 1 else 0, inv_freq.data_ptr(), dt, B, T, D, 2 * half, interleaved,
            attention_scale))
        if inplace:
            # what autograd keeps of them for a backward pass is no longer what it was; tensors of inference mode are never kept
            torch.autograd.graph.increment_version([t for t in (q_out, k_out) if t is not None and not t.is_inference()])
    return q_out, k_out


def _heads(name, x, B, H, T, D, inplace):
    """(x with contiguous heads, where its result goes, strides of batch, head and token)"""
    sb, sh, st, sd = x.stride()
    if sd != 1 and D != 1:
        if inplace:
            raise ValueError(f'{name}: the elements of a head must be contiguous')
        x = x.contiguous()
        sb, sh, st, sd = x.stride()
    if inplace:
        if (sb == 0 and B > 1) or (sh == 0 and H > 1) or (st == 0 and T > 1):
            raise ValueError(f'{name}: cannot work in place on an expanded tensor')
        return x, x, sb, sh, st
    return x, x.new_empty((B, T, H, D)).transpose(1, 2), sb, sh, st


def _hits(off, steps):
    """Whether off is a sum of i * stride with low <= i <= high over steps, a list of (stride > 0, low, high) by falling
    stride.  What the smaller strides reach leaves few i for each; a layout that still takes long counts as a hit."""
    reach = [(0, 0)]
    for stride, low, high in reversed(steps):
        reach.append((reach[-1][0] + low * stride, reach[-1][1] + high * stride))
    reach.reverse()
    looks = [0]

    def look(n, rest):
        if not reach[n][0] <= rest <= reach[n][1]:
            return False
        if n == len(steps):
            return True
        looks[0] += 1
        if looks[0] > 4096:
            return True
        stride, low, high = steps[n]
        least, most = reach[n + 1]
        first, last = max(low, -((most - rest) // stride)), min(high, (rest - least) // stride)
        return any(look(n + 1, rest - i * stride) for i in range(first, last + 1))
    return look(0, off)


@functools.lru_cache(maxsize=256)      # of layouts alone: a model asks for the same few at every step
def _shared_in_place(B, T, D, H, qb, qh, qt, G, kb, kh, kt, apart, size):
    """What is wrong with working in place on q (B, H, T, D) and k (B, G, T, D) `apart` bytes behind it, by their strides of batch,
    head and token; None where no element of memory belongs to two places of them."""
    q, k = ((B, H, T, D), (qb, qh, qt, 1)), ((B, G, T, D), (kb, kh, kt, 1))
    for n, layout in ((H, q), (G, k)):
        if n and _meets_itself(*layout):
            return 'a tensor whose heads overlap'
    # views that lie off one another's elements are taken as shared
    if H and G and (apart % size or _layouts_meet(apart // size, *q, *k)):
        return 'q and k that share elements'
    return None


def _layouts_meet(apart, a_shape, a_stride, b_shape, b_stride):
    """Whether two tensors, the second one `apart` elements behind the first, have an element in common."""
    # a's element at sum i * stride is b's at apart + sum j * stride; equal strides count as one step, i - j
    steps = {}
    for sign, shape, strides in ((1, a_shape, a_stride), (-1, b_shape, b_stride)):
        for n, stride in zip(shape, strides):
            if n > 1:
                low, high = steps.get(stride, (0, 0))
                steps[stride] = (low, high + n - 1) if sign > 0 else (low - n + 1, high)
    steps.pop(0, None)
    return _hits(apart, sorted(((s, *r) for s, r in steps.items()), reverse=True))


def _meets_itself(shape, strides):
    """Whether two different indices of a tensor of that layout name the same element."""
    dims = sorted(((s, n) for s, n in zip(strides, shape) if n > 1), reverse=True)
    inner = 1
    for s, n in reversed(dims):                        # the usual layouts: each stride steps over all that is inside it
        if s < inner:
            break
        inner = s * (n - 1) + inner
    else:
        return False
    # some dimension differs, by at least one step up; the others by any
    return any(_hits(0, [(t, 1 if j == i else 1 - m, m - 1) for j, (t, m) in enumerate(dims)]) for i in range(len(dims)))


def rope_frequencies(rotary_dim, base=None, scaling=None, seq_len=None, device='cuda'):
    """(inv_freq fp32 (rotary_dim / 2,), attention_scale) for rotary_embed.  `scaling` is a model configuration's
    rope_scaling / rope_parameters section: None or type 'default', 'linear' (factor), 'dynamic' (factor,
    original_max_position_embeddings; uses seq_len), 'llama3' (factor, low_freq_factor, high_freq_factor,
    original_max_position_embeddings) or 'yarn' (factor, original_max_position_embeddings, optional beta_fast, beta_slow,
    mscale, mscale_all_dim, attention_factor).  base: the model's rope_theta; where it is left out it is the section's own
    rope_theta, else 10000.  A section that holds one for each kind of layer is handed in one kind at a time."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f'rope_frequencies: rotary_dim must be even and positive, got {rotary_dim}')
    s = dict(scaling or {})
    if any(isinstance(v, dict) for v in s.values()):
        raise ValueError(f'rope_frequencies: sections for several kinds of layer ({", ".join(map(str, s))}): hand in one of them')
    theta = s.get('rope_theta')
    if base is None:
        base = 10000.0 if theta is None else theta
    elif theta is not None and theta != base:
        raise ValueError(f'rope_frequencies: base {base} and the section\'s rope_theta {theta} differ')
    kind = s.get('rope_type', s.get('type', 'default'))
    expo = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
    inv = float(base) ** -expo
    attention_scale = 1.0
    if kind == 'linear':
        inv = inv / s['factor']
    elif kind == 'dynamic':
        # the base grows with the sequence once it is longer than what the model was trained on
        trained = s['original_max_position_embeddings']
        length = max(seq_len or 0, trained)
        if rotary_dim > 2:      # a single pair turns once a position, whatever the base
            grown = base * (s['factor'] * length / trained - (s['factor'] - 1)) ** (rotary_dim / (rotary_dim - 2))
            inv = float(grown) ** -expo
    elif kind == 'llama3':
        # wave lengths beyond the trained context are stretched, short ones kept, the ones between blended
        turns = s['original_max_position_embeddings'] * inv / (2 * math.pi)     # turns within the trained context
        keep = ((turns - s['low_freq_factor']) / (s['high_freq_factor'] - s['low_freq_factor'])).clamp(0, 1)
        inv = keep * inv + (1 - keep) * inv / s['factor']
    elif kind == 'yarn':
        trained, factor = s['original_max_position_embeddings'], s['factor']

        def pair_with(turns):      # the (fractional) pair that makes so many turns within the trained context
            return rotary_dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = pair_with(s.get('beta_fast') or 32), pair_with(s.get('beta_slow') or 1)
        if s.get('truncate', True):
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, rotary_dim - 1)
        if low == high:
            high += 0.001
        ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - low) / (high - low)).clamp(0, 1)
        inv = inv / factor * ramp + inv * (1 - ramp)

        def magnitude(m):
            return 0.1 * m * math.log(factor) + 1 if factor > 1 else 1.0
        if s.get('attention_factor') is not None:
            attention_scale = float(s['attention_factor'])
        elif s.get('mscale') and s.get('mscale_all_dim'):
            attention_scale = magnitude(s['mscale']) / magnitude(s['mscale_all_dim'])
        else:
            attention_scale = magnitude(1.0)
    elif kind != 'default':
        raise NotImplementedError(f'rope_frequencies: scaling type {kind!r}')
    return inv.float().to(device), attention_scale

"""The 8-bit integer linear: what a W8A8-quantised linear is deployed as.

Counterpart of the reference's VllmQuantLinearInt8 (llmc/compression/quantization/module_utils.py:145-209), which
hands the per-token quantisation of the activations and the scaled product to third-party kernels, and the integer
sibling of fp8_linear.  Codes are int8 with an fp32 scale per token (activations) and per output channel (weights);
activations may carry a zero point per token as well.

Nothing here reads device memory on the host, and nothing synchronises but the first product on a device, which makes the word
that an expired wait is reported in; so every call can be captured into a CUDA graph (a product whose device has no such word
yet reports nothing).

Each function asks the compiled front (_calls) first, which serves the ordinary call in half of the host time and returns
None for any other; the Python below it knows every case and says what is wrong with a call.
"""
import threading

import torch
import torch.nn as nn

from . import _lib as L
from ._lib import _calls

_ACTS = {'silu': 1, 'gelu': 2, 'gelu_tanh': 3}
_status, _status_made = {}, threading.Lock()
_DTYPES = L._DTYPES


def _status_of(t, dev):
    """Address of the device's status word (a bounded wait that expired in a product), which is made on first use; 0
    where that first use is inside a capture."""
    s = _status.get(dev)
    if s is None:
        if dev < 0 or torch.cuda.is_current_stream_capturing():
            return 0
        with _status_made:                      # one word for all threads: kernels and graphs keep its address
            s = _status.get(dev)
            if s is None:
                with torch.inference_mode(False):       # check_status clears the word outside that mode as well
                    s = torch.zeros(1, dtype=torch.int32, device=t.device)
                torch.cuda.current_stream(dev).synchronize()      # other streams may use it from here on
                _status[dev] = s
                _calls.set_status(dev, s.data_ptr())
    return s.data_ptr()


def check_status(device=None):
    """Waits for the device and raises LcError if a product since the last check gave up waiting (its outputs are
    NaN where that happened)."""
    dev = torch.device('cuda' if device is None else device)
    dev = torch.cuda.current_device() if dev.index is None else dev.index
    torch.cuda.synchronize(dev)
    s = _status.get(dev)
    code = int(s.item()) if s is not None else 0
    if code:
        s.zero_()
        raise L.LcError('lc_int8_gemm', code, L.status_string(code))


def _float_rows(name, x):
    """x (..., K) as a 2-D view (or, where no view exists, a copy) whose rows are contiguous, and its type's number."""
    dt = _DTYPES.get(x.dtype)
    if dt is None:
        raise TypeError(f'{name}: unsupported dtype {x.dtype}')
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f'{name}: the last dimension must not be empty')
    if x.stride(-1) != 1 and x.shape[-1] != 1:
        x = x.contiguous()
    return (x if x.dim() == 2 else x.reshape(-1, x.shape[-1])), dt


def _codes_like(x, shape, sym):
    """Room for the codes of a tensor of `shape` (rows 16 bytes apart or a multiple of that, as the products read them),
    scales, zeros; and what the caller returns of it."""
    cols = shape[-1]
    pitch = (cols + 15) & -16
    lead = shape[:-1]
    codes = x.new_empty((*lead, pitch), dtype=torch.int8)
    scales = x.new_empty((*lead, 1), dtype=torch.float32)
    zeros = None if sym else x.new_empty((*lead, 1), dtype=torch.int32)
    seen = codes if pitch == cols else codes[..., :cols]
    return codes, pitch, scales, zeros, (seen, scales) if sym else (seen, scales, zeros)


def act_quant(x, sym=True):
    """(int8 codes of x's shape, fp32 scales (..., 1)), with sym=False also int32 zero points (..., 1): per token
    s = max(|x|) / 127 and q = rint(x / s), or, with a zero point, 255 steps over the token's range widened to
    hold zero, x ~ (q - z) s.  x: (..., K) of bf16, fp16 or fp32, any strides.  A token that holds a NaN or an
    infinity gets scale NaN.  The codes' rows lie a multiple of 16 bytes apart, which the products require."""
    out = _calls.act_quant(x, sym)
    return _act_quant(x, sym) if out is None else out


def _act_quant(x, sym):
    L.refuse_grad('act_quant', x)
    x, = L.resolved(x)
    x2, dt = _float_rows('act_quant', x)
    rows, cols = x2.shape
    codes, pitch, scales, zeros, out = _codes_like(x, x.shape, sym)
    if rows:
        L.launch(x2.get_device(), 'lc_int8_act_quant', x2.data_ptr(), dt, rows, cols, x2.stride()[0], codes.data_ptr(), pitch,
                 scales.data_ptr(), None if sym else zeros.data_ptr())
    return out


def gated_act_quant(gate, up, act='silu', sym=True):
    """act_quant(act(gate) * up) in one pass, the product formed in fp32 and not rounded in between: the input of an
    MLP's down projection.  act: 'silu', 'gelu' or 'gelu_tanh'."""
    kind = _ACTS.get(act)
    if kind is None:
        raise NotImplementedError(f'gated_act_quant: activation {act!r}; there are {sorted(_ACTS)}')
    out = _calls.gated_act_quant(gate, up, kind, sym)
    return _gated_act_quant(gate, up, kind, sym) if out is None else out


def _gated_act_quant(gate, up, kind, sym):
    shape = gate.shape
    if shape != up.shape or gate.dtype != up.dtype:
        raise ValueError(f'gated_act_quant: gate {tuple(shape)} {gate.dtype} and up {tuple(up.shape)} {up.dtype} differ')
    L.refuse_grad('gated_act_quant', gate, up)
    gate, up = L.resolved(gate, up)
    dev = gate.get_device()
    if up.get_device() != dev:
        L.refuse_devices('gated_act_quant', gate, up=up)
    g2, dt = _float_rows('gated_act_quant', gate)
    u2, _ = _float_rows('gated_act_quant', up)
    rows, cols = g2.shape
    codes, pitch, scales, zeros, out = _codes_like(gate, shape, sym)
    if rows:
        L.launch(dev, 'lc_int8_gated_act_quant', g2.data_ptr(), u2.data_ptr(), dt, rows, cols, g2.stride()[0], u2.stride()[0], kind,
                 codes.data_ptr(), pitch, scales.data_ptr(), None if sym else zeros.data_ptr())
    return out


def aligned_rows(codes):
    """codes (N, K) int8 as the products read them: rows beginning at multiples of 16 bytes.  The tensor itself where
    it is laid out so already, else a copy (made once, when a weight is loaded)."""
    if codes.dtype != torch.int8 or codes.dim() != 2:
        raise TypeError('aligned_rows: int8 codes (N, K) expected')
    if _rows_aligned(codes):
        return codes
    n, k = codes.shape
    room = torch.zeros((n, (k + 15) // 16 * 16), dtype=torch.int8, device=codes.device)
    room[:, :k] = codes
    return room[:, :k]


def _rows_aligned(t):
    rows, cols = t.shape
    pitch, step = t.stride()
    return not t.data_ptr() & 15 and (step == 1 or cols == 1) and ((not pitch & 15 and pitch >= cols) or rows <= 1)


def _pitch(t, rows, cols):
    """Row pitch of an aligned 2-D code tensor; a single row may carry any stride."""
    return t.stride()[0] if rows > 1 else (cols + 15) & -16


def _check_weight(name, b, b_s, b_sum, bias, zeros, out_dtype):
    """(N, K) of the weight; refuses what the products do not take."""
    if b.dtype != torch.int8 or b.dim() != 2:
        raise TypeError(f'{name}: the weight must be int8 codes (N, K), got {b.dtype} {tuple(b.shape)}')
    N, K = b.shape
    if not _rows_aligned(b):
        raise ValueError(f'{name}: the rows of the weight must begin at multiples of 16 bytes (int8_linear.aligned_rows '
                         'lays them out once)')
    if b_s.dtype != torch.float32 or b_s.numel() != N or not b_s.is_contiguous():
        raise ValueError(f'{name}: the weight needs one fp32 scale per output channel ({N}), contiguous')
    if zeros:
        if b_sum is None:
            raise ValueError(f'{name}: zero points need the sums of the weight\'s rows, w.sum(1, dtype=torch.int32)')
        if b_sum.dtype != torch.int32 or b_sum.numel() != N or not b_sum.is_contiguous():
            raise ValueError(f'{name}: the sums of the weight\'s rows must be {N} int32 values, contiguous')
    if bias is not None and (bias.dtype != out_dtype or bias.numel() != N or not bias.is_contiguous()):
        raise ValueError(f'{name}: bias must be {N} contiguous values of {out_dtype}')
    if K > (65793 if zeros else 131071):
        raise ValueError(f'{name}: {K} products may leave 32 bits (at most 131071, with zero points 65793)')
    return N, K


def int8_gemm(a, a_s, b, b_s, bias=None, a_z=None, b_sum=None, out_dtype=torch.bfloat16):
    """a: (..., K) int8 codes with scales a_s (..., 1) and, if given, zero points a_z (..., 1), as act_quant returns
    them; b: (N, K) int8 with b_s (N fp32 values) and, with zero points, b_sum (N int32 sums of b's rows).  Returns
    (..., N) = ((a - a_z) b^T) * a_s * b_s + bias in out_dtype; the sum of products is exact."""
    c = _calls.int8_gemm(a, a_s, b, b_s, bias, a_z, b_sum, out_dtype)
    return _int8_gemm(a, a_s, b, b_s, bias, a_z, b_sum, out_dtype) if c is None else c


def _int8_gemm(a, a_s, b, b_s, bias, a_z, b_sum, out_dtype):
    name = 'int8_gemm'
    L.refuse_grad(name, a_s, b_s, bias)
    a, a_s, b, b_s, bias, a_z, b_sum = L.resolved(a, a_s, b, b_s, bias, a_z, b_sum)
    out = _DTYPES.get(out_dtype)
    if out is None:
        raise TypeError(f'{name}: unsupported output type {out_dtype}')
    if a.dtype != torch.int8 or a.dim() == 0:
        raise TypeError(f'{name}: the activations must be int8 codes (..., K), got {a.dtype}')
    N, K = _check_weight(name, b, b_s, b_sum, bias, a_z is not None, out_dtype)
    if a.shape[-1] != K or K == 0:
        raise ValueError(f'{name}: activations of {a.shape[-1]} and a weight of {K} input channels')
    a2 = a if a.dim() == 2 else a.reshape(-1, K)
    M = a2.shape[0]
    if not _rows_aligned(a2):
        raise ValueError(f'{name}: the rows of the activations\' codes must begin at multiples of 16 bytes, as act_quant lays '
                         'them out')
    if a_s.dtype != torch.float32 or a_s.numel() != M or not a_s.is_contiguous():
        raise ValueError(f'{name}: the activations need one fp32 scale per token ({M}), contiguous')
    if a_z is not None and (a_z.dtype != torch.int32 or a_z.numel() != M or not a_z.is_contiguous()):
        raise ValueError(f'{name}: zero points must be {M} int32 values, contiguous')
    dev = a.get_device()
    if not (a_s.get_device() == b.get_device() == b_s.get_device() == dev) or (bias is not None and bias.get_device() != dev) \
            or (a_z is not None and not a_z.get_device() == b_sum.get_device() == dev):
        L.refuse_devices(name, a, a_s=a_s, a_z=a_z, b=b, b_s=b_s, b_sum=b_sum, bias=bias)
    c = a.new_empty((*a.shape[:-1], N), dtype=out_dtype)
    if M and N:
        L.launch(dev, 'lc_int8_gemm', L.INT8_GEMM.pack(
            a2.data_ptr(), _pitch(a2, M, K), a_s.data_ptr(), 0 if a_z is None else a_z.data_ptr(), b.data_ptr(), _pitch(b, N, K),
            b_s.data_ptr(), 0 if a_z is None else b_sum.data_ptr(), 0 if bias is None else bias.data_ptr(), M, N, K,
            c.data_ptr(), out, _status_of(a, dev)))
    return c


def int8_dynamic_forward_func(x, w, w_scale, bias=None, w_sum=None):
    """The W8A8 linear's forward: x (..., K) quantised per token and multiplied with w (N, K) int8, scales w_scale (N fp32
    values), in one call.  With w_sum (N int32 sums of w's rows) the activations get a zero point per token, without it
    they are quantised symmetrically.  Returns (..., N) of x's type; bias has that type too."""
    c = _calls.int8_linear(x, w, w_scale, bias, w_sum)
    return _int8_dynamic_forward(x, w, w_scale, bias, w_sum) if c is None else c


def _int8_dynamic_forward(x, w, w_scale, bias, w_sum):
    name = 'int8_dynamic_forward_func'
    L.refuse_grad(name, x, w_scale, bias)
    x, w, w_scale, bias, w_sum = L.resolved(x, w, w_scale, bias, w_sum)
    x2, dt = _float_rows(name, x)
    sym = w_sum is None
    N, K = _check_weight(name, w, w_scale, w_sum, bias, not sym, x.dtype)
    M, k = x2.shape
    if k != K:
        raise ValueError(f'{name}: activations of {k} and a weight of {K} input channels')
    dev = x.get_device()
    if not (w.get_device() == w_scale.get_device() == dev) or (bias is not None and bias.get_device() != dev) \
            or (not sym and w_sum.get_device() != dev):
        L.refuse_devices(name, x, w=w, w_scale=w_scale, bias=bias, w_sum=w_sum)
    c = x.new_empty((*x.shape[:-1], N))
    if M and N:
        room = L.lib.lc_int8_linear_scratch(M, K)
        scratch = x.new_empty(room, dtype=torch.int8) if room else None
        L.launch(dev, 'lc_int8_linear', L.INT8_LINEAR.pack(
            x2.data_ptr(), dt, x2.stride()[0], w.data_ptr(), _pitch(w, N, K), w_scale.data_ptr(), 0 if sym else w_sum.data_ptr(),
            0 if bias is None else bias.data_ptr(), M, N, K, sym, c.data_ptr(), scratch.data_ptr() if room else 0, room,
            _status_of(x, dev)))
    return c


class Int8Linear(nn.Module):
    """Replacement linear with int8 weights and dynamically quantised activations (the role of the reference's
    VllmQuantLinearInt8).  Moved and cast like any module: the bias takes the type that the activations then have, codes and
    scales keep theirs.  `new` takes what the algorithms' replacement linears take: the module and its
    w_q(module, wquantizer) -> (codes, scales, zeros)."""

    def __init__(self, codes, scale, bias=None, sym_act=True):
        super().__init__()
        if codes.dtype != torch.int8:
            raise TypeError('Int8Linear: symmetric int8 weight codes expected')
        if scale.numel() != codes.shape[0]:
            raise NotImplementedError('Int8Linear: one scale per output channel (per_channel weights) expected, got '
                                      f'{scale.numel()} for {codes.shape[0]} channels')
        self.out_features, self.in_features = codes.shape
        self.register_buffer('weight', aligned_rows(codes))
        self.register_buffer('weight_scale', scale.detach().reshape(-1).float().contiguous())
        self.register_buffer('weight_sum', None if sym_act else codes.sum(1, dtype=torch.int32))
        self.register_buffer('bias', None if bias is None else bias.detach().contiguous())

    @classmethod
    @torch.no_grad()
    def new(cls, module, w_q, wquantizer=None, aquantizer=None):
        """module: an nn.Linear; w_q: e.g. RTN(wquantizer).w_q, for 8-bit symmetric per_channel weights; aquantizer:
        the activations' quantizer (8 bits, per_token), whose symmetry is kept; None means symmetric.  With zero points the
        token's range is widened to hold zero, as act_quant says: for a token of both signs that is the quantiser's own
        grid, for a token of one sign it is not (the quantiser steps over max - min from a zero point cut to its codes, and
        so cuts off the values of the far end)."""
        if aquantizer is not None and (aquantizer.bit != 8 or aquantizer.granularity != 'per_token'):
            raise NotImplementedError('Int8Linear: activations are quantised to 8 bits per token')
        if aquantizer is not None and getattr(aquantizer, 'calib_algo', 'minmax') != 'minmax':
            raise NotImplementedError(f'Int8Linear: activations take their range from each token, not by {aquantizer.calib_algo}')
        if aquantizer is not None and not aquantizer.sym and not getattr(aquantizer, 'round_zp', True):
            raise NotImplementedError('Int8Linear: zero points are whole numbers (round_zp)')
        codes, scale, zeros = w_q(module, wquantizer) if wquantizer is not None else w_q(module)
        if zeros is not None:
            raise NotImplementedError('Int8Linear: weights with zero points are not supported')
        bias = getattr(module, 'bias', None)
        return cls(codes, scale, None if bias is None else bias.data, aquantizer is None or aquantizer.sym)

    def _lay_out(self):
        # where in_features is no multiple of 16 the weight is a view of padded rows, which torch makes contiguous when it
        # copies it to another device or takes it over from a state dict
        self.weight = aligned_rows(self.weight)

    def _apply(self, fn, recurse=True):
        kept = {name: getattr(self, name) for name in ('weight', 'weight_scale', 'weight_sum')}
        super()._apply(fn, recurse)
        for name, before in kept.items():       # .half() and the like cast the bias; codes, sums and scales keep their types
            now = getattr(self, name)
            if before is not None and now.dtype != before.dtype:
                setattr(self, name, before.to(now.device))
        self._lay_out()
        return self

    def _load_from_state_dict(self, *args, **kwargs):
        super()._load_from_state_dict(*args, **kwargs)
        self._lay_out()

    @torch.no_grad()
    def forward(self, x):
        return int8_dynamic_forward_func(x, self.weight, self.weight_scale, self.bias, self.weight_sum)

    def extra_repr(self):
        return f'in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}'

"""Refusals of the operators of a deployed W8A8 block, and the rotary frequencies: nothing here needs a GPU."""
import ctypes
import math
import os
import re

import pytest
import torch

A = 4096                           # an aligned address that no refused call may touch
P = ctypes.c_void_p(A)


def _lib():
    from lightcompress_b200 import _lib
    return _lib, _lib.lib


def test_quantisation_refusals_at_the_c_boundary():
    L, lib = _lib()
    f = lib.lc_int8_act_quant
    assert f(P, 9, 2, 64, 64, P, 64, P, None, None) == L.LC_ERR_ARG            # type
    assert f(P, 1, -1, 64, 64, P, 64, P, None, None) == L.LC_ERR_ARG           # rows
    assert f(P, 1, 2, 0, 64, P, 64, P, None, None) == L.LC_ERR_ARG             # width
    assert f(P, 1, 2, 64, 64, P, 63, P, None, None) == L.LC_ERR_ARG            # rows of codes that overlap
    assert f(None, 1, 2, 64, 64, P, 64, P, None, None) == L.LC_ERR_ARG
    assert f(None, 1, 0, 64, 64, None, 64, None, None, None) == L.LC_OK        # no rows
    g = lib.lc_int8_gated_act_quant
    assert g(P, P, 1, 2, 64, 64, 64, 0, P, 64, P, None, None) == L.LC_ERR_ARG  # activation
    assert g(P, P, 1, 2, 64, 64, 64, 4, P, 64, P, None, None) == L.LC_ERR_ARG
    assert g(P, None, 1, 2, 64, 64, 64, 1, P, 64, P, None, None) == L.LC_ERR_ARG


def test_product_refusals_at_the_c_boundary():
    L, lib = _lib()

    def gemm(a=A, lda=64, a_s=A, a_z=0, b=A, ldb=64, b_s=A, b_sum=0, M=4, N=4, K=64, c=A, out=1):
        return lib.lc_int8_gemm(L.INT8_GEMM.pack(a, lda, a_s, a_z, b, ldb, b_s, b_sum, 0, M, N, K, c, out, 0), None)
    assert gemm(out=3) == L.LC_ERR_ARG
    assert gemm(K=0) == L.LC_ERR_ARG
    assert gemm(lda=72) == L.LC_ERR_ALIGN and gemm(ldb=72) == L.LC_ERR_ALIGN
    assert gemm(a=4100) == L.LC_ERR_ALIGN and gemm(b=4100) == L.LC_ERR_ALIGN
    assert gemm(lda=48) == L.LC_ERR_ARG and gemm(ldb=48) == L.LC_ERR_ARG
    assert gemm(a_z=A) == L.LC_ERR_ARG                                         # zero points without b_sum
    assert gemm(K=131072, lda=131072, ldb=131072) == L.LC_ERR_SHAPE
    assert gemm(K=65794, lda=65808, ldb=65808, a_z=A, b_sum=A) == L.LC_ERR_SHAPE
    assert gemm(M=0, a=0, c=0) == L.LC_OK and gemm(N=0, b=0, c=0) == L.LC_OK

    def linear(M=40, K=64, ldb=64, sym=1, scratch=A, room=1 << 20, dtype=1, b_sum=0, x=A):
        return lib.lc_int8_linear(L.INT8_LINEAR.pack(x, dtype, 64, A, ldb, A, b_sum, 0, M, 4, K, sym, A, scratch, room, 0), None)
    assert lib.lc_int8_linear_scratch(40, 65) == 40 * 80 + 320 and lib.lc_int8_linear_scratch(1, 4097) == 4112 + 8
    assert lib.lc_int8_linear_scratch(1, 4096) == 0 and lib.lc_int8_linear_scratch(0, 65) == 0
    assert linear(room=40 * 64 + 319) == L.LC_ERR_WORKSPACE
    assert linear(scratch=0) == L.LC_ERR_ARG and linear(x=0) == L.LC_ERR_ARG
    assert linear(scratch=4104) == L.LC_ERR_ALIGN
    assert linear(sym=0) == L.LC_ERR_ARG and linear(dtype=5) == L.LC_ERR_ARG
    assert linear(M=0, scratch=0, room=0) == L.LC_OK


def test_norm_and_rotary_refusals_at_the_c_boundary():
    L, lib = _lib()

    def norm(x=A, res=0, post=0, gate=0, gate_rows=0, w=A, dtype=1, rows=4, cols=64, scale=1.0, h=0, y=A,
             codes=0, ldc=64, scales=0):
        return lib.lc_residual_norm(L.RESIDUAL_NORM.pack(x, res, post, gate, gate_rows, w, dtype, rows, cols, 64, 64, scale, 1e-6,
                                                         0.0, h, y, codes, ldc, scales, 0), None)
    assert norm(dtype=7) == L.LC_ERR_ARG and norm(cols=0) == L.LC_ERR_ARG
    assert norm(gate=A, gate_rows=3, h=A) == L.LC_ERR_SHAPE and norm(gate=A, gate_rows=0, h=A) == L.LC_ERR_SHAPE
    assert norm(res=A) == L.LC_ERR_ARG and norm(scale=0.5) == L.LC_ERR_ARG      # a changed stream without room for it
    assert norm(w=0, y=0) == L.LC_ERR_ARG and norm(w=0) == L.LC_ERR_ARG and norm(y=0) == L.LC_ERR_ARG
    assert norm(codes=A) == L.LC_ERR_ARG and norm(codes=A, scales=A, ldc=63) == L.LC_ERR_ARG
    assert norm(rows=0, x=0) == L.LC_OK

    def rope(q=A, qh=2, k=A, kh=1, pos=A, freq=A, dtype=1, B=1, T=1, D=64, R=64):
        return lib.lc_rotary_embed(L.ROTARY_EMBED.pack(q, q, qh, 0, 0, 64, k, k, kh, 0, 0, 64, pos, 0, freq, dtype, B, T, D, R, 0,
                                                       1.0), None)
    assert rope(dtype=3) == L.LC_ERR_ARG and rope(R=0) == L.LC_ERR_ARG
    assert rope(R=63) == L.LC_ERR_SHAPE and rope(R=66) == L.LC_ERR_SHAPE and rope(D=1026, R=64) == L.LC_ERR_SHAPE
    assert rope(q=0) == L.LC_ERR_ARG and rope(k=0) == L.LC_ERR_ARG and rope(pos=0) == L.LC_ERR_ARG
    assert rope(T=0, q=0) == L.LC_OK and rope(qh=0, kh=0, q=0, k=0) == L.LC_OK
    assert rope(qh=1000, kh=24) == L.LC_ERR_SHAPE
    for f in (lib.lc_int8_gemm, lib.lc_int8_linear, lib.lc_residual_norm, lib.lc_rotary_embed):
        assert f(None, None) == L.LC_ERR_ARG


def test_packed_structs_match_the_header():
    """Every member is 8 bytes wide, and the packed formats name the header's members one by one."""
    L, _ = _lib()
    text = open(os.path.join(os.path.dirname(L.__file__), '..', 'include', 'lc_b200.h')).read()
    for fmt, name in ((L.INT8_GEMM, 'int8_gemm'), (L.INT8_LINEAR, 'int8_linear'), (L.RESIDUAL_NORM, 'residual_norm'),
                      (L.ROTARY_EMBED, 'rotary_embed')):
        body = re.search(r'typedef struct \{([^}]*)\} lc_%s_args;' % name, text).group(1)
        want = '@'
        for line in filter(None, (v.strip() for v in body.split(';'))):
            kind = 'P' if '*' in line else 'd' if line.startswith('double') else 'q'
            assert kind == 'P' or line.startswith(('int64_t ', 'double '))
            want += kind * (line.count(',') + 1)
        assert fmt.format == want and fmt.size == 8 * (len(want) - 1)


def test_int8_linear_refusals():
    from lightcompress_b200 import int8_linear as il
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    w, ws = torch.zeros(8, 64, dtype=torch.int8), torch.ones(8)
    with pytest.raises(RuntimeError, match='no CPU path'):
        il.act_quant(x)
    with pytest.raises(RuntimeError, match='no CPU path'):
        il.int8_dynamic_forward_func(x, w, ws)
    with pytest.raises(TypeError, match='dtype'):
        il.act_quant(x.double())
    with pytest.raises(ValueError, match='empty'):
        il.act_quant(torch.zeros(3, 0))
    with pytest.raises(RuntimeError, match='no backward'):
        il.act_quant(torch.zeros(2, 8, requires_grad=True))
    with pytest.raises(NotImplementedError, match='relu'):
        il.gated_act_quant(x, x, 'relu')
    with pytest.raises(ValueError, match='differ'):
        il.gated_act_quant(x, x[:1])
    with pytest.raises(ValueError, match='16 bytes'):
        il.int8_dynamic_forward_func(torch.zeros(2, 60), torch.zeros(8, 60, dtype=torch.int8), ws)
    with pytest.raises(ValueError, match='16 bytes'):
        il.int8_dynamic_forward_func(x, torch.zeros(64, 8, dtype=torch.int8).t(), ws)
    with pytest.raises(ValueError, match='input channels'):
        il.int8_dynamic_forward_func(x[:, :32], w, ws)
    with pytest.raises(ValueError, match='scale per output channel'):
        il.int8_dynamic_forward_func(x, w, ws.double())
    with pytest.raises(ValueError, match='scale per output channel'):
        il.int8_dynamic_forward_func(x, w, ws[:4])
    with pytest.raises(ValueError, match='bias'):
        il.int8_dynamic_forward_func(x, w, ws, torch.zeros(8))
    with pytest.raises(TypeError, match='int8 codes'):
        il.int8_dynamic_forward_func(x, w.to(torch.uint8), ws)
    with pytest.raises(ValueError, match='leave 32 bits'):
        il.int8_dynamic_forward_func(torch.zeros(1, 131072), torch.zeros(1, 131072, dtype=torch.int8), torch.ones(1))
    with pytest.raises(ValueError, match='int32'):
        il.int8_dynamic_forward_func(x, w, ws, w_sum=torch.zeros(8))
    a, a_s = torch.zeros(2, 64, dtype=torch.int8), torch.ones(2, 1)
    with pytest.raises(RuntimeError, match='no CPU path'):
        il.int8_gemm(a, a_s, w, ws)
    with pytest.raises(ValueError, match='per token'):
        il.int8_gemm(a, a_s[:1], w, ws)
    with pytest.raises(ValueError, match='sums of the weight'):
        il.int8_gemm(a, a_s, w, ws, a_z=torch.zeros(2, 1, dtype=torch.int32))
    with pytest.raises(ValueError, match='zero points'):
        il.int8_gemm(a, a_s, w, ws, a_z=torch.zeros(2, 1), b_sum=torch.zeros(8, dtype=torch.int32))
    with pytest.raises(TypeError, match='output type'):
        il.int8_gemm(a, a_s, w, ws, out_dtype=torch.float64)
    with pytest.raises(TypeError, match='int8 codes'):
        il.int8_gemm(a.float(), a_s, w, ws)
    with pytest.raises(NotImplementedError, match='per output channel'):
        il.Int8Linear(w, torch.ones(8, 2))
    with pytest.raises(TypeError, match='int8'):
        il.Int8Linear(w.to(torch.uint8), ws)


def test_aligned_rows():
    from lightcompress_b200.int8_linear import aligned_rows
    w = torch.randint(-128, 128, (5, 30), dtype=torch.int8)
    p = aligned_rows(w)
    assert torch.equal(p, w) and p.stride() == (32, 1) and p.data_ptr() % 16 == 0
    assert aligned_rows(p) is p
    t = torch.randint(-128, 128, (32, 5), dtype=torch.int8).t()
    assert torch.equal(aligned_rows(t), t) and aligned_rows(t).stride(1) == 1


def test_block_operator_refusals():
    from lightcompress_b200 import block_ops as bo
    x, w = torch.zeros(2, 3, 64), torch.ones(64)
    with pytest.raises(RuntimeError, match='no CPU path'):
        bo.residual_norm(x, x, weight=w)
    with pytest.raises(RuntimeError, match='no backward'):
        bo.residual_norm(x, x, weight=torch.nn.Parameter(w))
    with pytest.raises(ValueError, match='residual'):
        bo.residual_norm(x, x[:1], weight=w)
    with pytest.raises(TypeError, match='weight'):
        bo.residual_norm(x, x, weight=w.half())
    with pytest.raises(ValueError, match='shape'):
        bo.residual_norm(x, x, weight=w[:32])
    with pytest.raises(ValueError, match='quant'):
        bo.residual_norm(x, x, quant=True)
    for bad in ((3, 64), (2, 2, 64), (1, 3, 64), (2, 3, 1), (1, 2, 3, 64)):
        with pytest.raises(ValueError, match='gate'):
            bo.residual_norm(x, x, weight=w, gate=torch.ones(bad))
    q, k, pos, freq = torch.zeros(2, 4, 3, 64), torch.zeros(2, 1, 3, 64), torch.zeros(2, 3, dtype=torch.int64), torch.ones(32)
    with pytest.raises(RuntimeError, match='no CPU path'):
        bo.rotary_embed(q, k, pos, freq)
    with pytest.raises(ValueError, match='positions'):
        bo.rotary_embed(q, k, pos.int(), freq)
    with pytest.raises(ValueError, match='positions'):
        bo.rotary_embed(q, k, pos[:, :2], freq)
    with pytest.raises(ValueError, match='inv_freq'):
        bo.rotary_embed(q, k, pos, torch.ones(33))
    with pytest.raises(ValueError, match='inv_freq'):
        bo.rotary_embed(q, k, pos, freq.double())
    with pytest.raises(ValueError, match='does not go'):
        bo.rotary_embed(q, k[:, :, :2], pos, freq)
    with pytest.raises(ValueError, match='heads, T, D'):
        bo.rotary_embed(q[0], k, pos, freq)
    with pytest.raises(NotImplementedError, match='1024'):
        bo.rotary_embed(torch.zeros(1, 1, 1, 1026), None, pos[:1, :1], freq)
    with pytest.raises(RuntimeError, match='no backward'):
        bo.rotary_embed(q.requires_grad_(), k, pos, freq)
    with pytest.raises(NotImplementedError, match='scaling type'):
        bo.rope_frequencies(64, scaling={'rope_type': 'other'}, device='cpu')
    with pytest.raises(ValueError, match='rotary_dim'):
        bo.rope_frequencies(63, device='cpu')


def test_gate_rows():
    from lightcompress_b200.block_ops import _gate_rows
    x = torch.zeros(2, 3, 8)
    assert _gate_rows(torch.zeros(8), x) == 1 and _gate_rows(torch.zeros(1, 1, 8), x) == 1
    assert _gate_rows(torch.zeros(2, 1, 8), x) == 2 and _gate_rows(torch.zeros(2, 3, 8), x) == 6
    assert _gate_rows(torch.zeros(3, 8), x[:1]) == 3 and _gate_rows(torch.zeros(1, 8), torch.zeros(5, 8)) == 1


_CONFIGS = [
    ('default', None), ('linear', {'factor': 4.0}),
    ('dynamic', {'factor': 4.0, 'original_max_position_embeddings': 64}),
    ('llama3', {'factor': 8.0, 'low_freq_factor': 1.0, 'high_freq_factor': 4.0, 'original_max_position_embeddings': 256}),
    ('yarn', {'factor': 8.0, 'original_max_position_embeddings': 256}),
    ('yarn', {'factor': 8.0, 'original_max_position_embeddings': 256, 'mscale': 0.7, 'mscale_all_dim': 1.0,
              'beta_fast': 16, 'beta_slow': 2}),
]


@pytest.mark.parametrize('kind,section', _CONFIGS)
def test_rope_frequencies_against_transformers(kind, section):
    """The frequencies of a model configuration's scaling section, as transformers computes them for it.  Both are fp32
    values of the same real number, computed in fp64 here and in fp32 there: a power with relative error 2^-24 per
    rounding and its exponent's error times ln(base): under 1e-5 relative."""
    tr = pytest.importorskip('transformers')
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    from lightcompress_b200.block_ops import rope_frequencies
    base, dim = 10000.0, 64
    params = dict(section or {}, rope_type=kind)
    seq = 300 if kind == 'dynamic' else None
    if kind == 'default':
        want, want_scale = 1.0 / base ** (torch.arange(0, dim, 2).float() / dim), 1.0
    else:
        trained = params.get('original_max_position_embeddings', 64)
        try:
            cfg = tr.LlamaConfig(hidden_size=128, num_attention_heads=2, head_dim=dim, max_position_embeddings=trained,
                                 rope_theta=base, rope_scaling=dict(params, rope_theta=base))
            want, want_scale = ROPE_INIT_FUNCTIONS[kind](cfg, torch.device('cpu'), seq_len=seq)
        except (TypeError, KeyError, AttributeError) as e:
            pytest.skip(f'this transformers has another interface: {e}')
    got, scale = rope_frequencies(dim, base, params, seq_len=seq, device='cpu')
    assert got.dtype == torch.float32 and got.shape == (dim // 2,)
    assert math.isclose(scale, want_scale, rel_tol=1e-6)
    assert torch.allclose(got, want.float(), rtol=1e-5, atol=0)


def test_rope_frequencies_of_a_single_pair():
    from lightcompress_b200.block_ops import rope_frequencies
    for kind in ('default', 'dynamic'):
        inv, _ = rope_frequencies(2, scaling={'rope_type': kind, 'factor': 2.0, 'original_max_position_embeddings': 8}, seq_len=20,
                                  device='cpu')
        assert inv.tolist() == [1.0]


def test_launches_on_the_tensors_device_and_leaves_the_current_one(monkeypatch):
    """The device and stream that a call is given, against fakes of the library and of torch's device functions."""
    import contextlib
    from lightcompress_b200 import _lib as L
    seen, current = [], [0]

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], d
        try:
            yield
        finally:
            current[0] = before

    class Lib:
        code = 0

        def lc_set_device(self, d):
            seen.append(('device', d))
            return 0

        def lc_thing(self, *args):
            seen.append(('call', current[0], args))
            return self.code

        def lc_status_string(self, code):
            return b'fake'
    lib = Lib()
    monkeypatch.setattr(L, 'lib', lib)
    monkeypatch.setattr(L, '_current_device', lambda: current[0])
    monkeypatch.setattr(torch.cuda, 'device', device)
    monkeypatch.setattr(L, '_raw_stream', lambda d: 100 + d)
    L.launch(0, 'lc_thing', b'x')
    assert seen == [('device', 0), ('call', 0, (b'x', 100))]
    seen.clear()
    L.launch(3, 'lc_thing', b'x')
    assert seen == [('device', 3), ('call', 3, (b'x', 103)), ('device', 0)] and current == [0]
    seen.clear()
    lib.code = L.LC_ERR_SHAPE
    with pytest.raises(L.LcError, match='lc_thing failed'):
        L.launch(3, 'lc_thing')
    assert seen[-1] == ('device', 0) and current == [0]
    with pytest.raises(RuntimeError, match='no CPU path'):
        L.launch(-1, 'lc_thing')


def test_an_expired_wait_is_reported_once(monkeypatch):
    """check_status on a status word that a kernel would have written."""
    from lightcompress_b200 import _lib as L
    from lightcompress_b200 import int8_linear as il
    word = torch.zeros(1, dtype=torch.int32)
    monkeypatch.setattr(torch.cuda, 'synchronize', lambda d=None: None)
    monkeypatch.setattr(il, '_status', {0: word})
    il.check_status('cuda:0')
    word.fill_(L.LC_ERR_TIMEOUT)
    with pytest.raises(L.LcError, match='timed out'):
        il.check_status(0)
    il.check_status(0)
    il.check_status(1)          # a device that has run no product

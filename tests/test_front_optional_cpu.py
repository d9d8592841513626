"""The package without its compiled front, or with one that does not load: everything but the host time of the W8A8 operators is
as it was."""
import os
import subprocess
import sys

import pytest

PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'lightcompress_b200')

CHECK = '''
import sys, warnings
sys.path.insert(0, sys.argv[1])
with warnings.catch_warnings(record=True) as seen:
    warnings.simplefilter('always')
    import lightcompress_b200 as lc
    from lightcompress_b200 import block_ops, int8_linear, _lib
assert lc.__file__.startswith(sys.argv[1]), lc.__file__
assert sum('_calls.so' in str(w.message) and w.category is RuntimeWarning for w in seen) == 1, [str(w.message) for w in seen]
assert isinstance(_lib._calls, _lib.NoFront)
import torch
lc.IntegerQuantizer(4, False, 'per_group', group_size=128), lc.GPTQ, lc.Awq
x, w, s, one = torch.ones(2, 64), torch.ones(8, 64, dtype=torch.int8), torch.ones(8), torch.ones(64)
q = torch.ones(1, 2, 3, 8)
launched = []
_lib.launch = lambda dev, name, *args: launched.append(name)
int8_linear.act_quant(x)
int8_linear.gated_act_quant(x, x)
int8_linear.int8_gemm(x.to(torch.int8), x[:, :1].contiguous(), w, s)
int8_linear.int8_dynamic_forward_func(x, w, s)
block_ops.residual_norm(x, x, weight=one)
block_ops.rotary_embed(q, None, torch.arange(3), torch.ones(4))
assert launched == ['lc_int8_act_quant', 'lc_int8_gated_act_quant', 'lc_int8_gemm', 'lc_int8_linear', 'lc_residual_norm',
                    'lc_rotary_embed'], launched
print('fine')
'''


@pytest.mark.parametrize('front', ['missing', 'not a library'])
def test_the_package_without_its_front(tmp_path, front):
    there = tmp_path / 'lightcompress_b200'
    there.mkdir()
    for f in os.listdir(PACKAGE):
        if f.endswith('.py') or f == 'liblc_b200.so':
            os.symlink(os.path.join(PACKAGE, f), there / f)
    if front != 'missing':
        (there / '_calls.so').write_text('nothing that loads')
    r = subprocess.run([sys.executable, '-c', CHECK, str(tmp_path)], capture_output=True, text=True, cwd=tmp_path, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == 'fine', r.stdout + r.stderr

"""The compiled front is for one torch and one interpreter: another one neither runs it nor takes it for up to date."""
import importlib.util
import os
import sys
import sysconfig

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _build_module():
    spec = importlib.util.spec_from_file_location('front_build', os.path.join(ROOT, 'lightcompress_b200', 'build.py'))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_what_it_is_built_for():
    from lightcompress_b200 import _calls, _lib
    here = f'torch {torch.__version__}, {sysconfig.get_config_var("SOABI")}'
    assert _build_module().front_for(os.path.dirname(torch.__file__)) == here
    assert _calls.built_for == here and _lib._calls is _calls


def test_another_torch_makes_it_stale(tmp_path, monkeypatch):
    b = _build_module()
    (tmp_path / 'version.py').write_text("__version__ = '9.9.9+other'\ngit_version = 'x'\n")
    other, here = b.front_for(str(tmp_path)), b.front_for(os.path.dirname(torch.__file__))
    assert other.startswith('torch 9.9.9+other, ')
    calls, note = tmp_path / '_calls.so', tmp_path / 'note'
    monkeypatch.setattr(b, 'CALLS', str(calls))
    monkeypatch.setattr(b, 'CALLS_NOTE', str(note))
    assert b._front_is_stale(here)                          # there is none
    calls.write_text('')
    assert b._front_is_stale(here)                          # nobody knows what for
    note.write_text(here + '\n')
    assert not b._front_is_stale(here) and b._front_is_stale(other)
    os.utime(calls, (1, 1))
    assert b._front_is_stale(here)                          # older than its source


def test_one_built_for_another_torch_is_not_called(monkeypatch):
    import warnings
    from lightcompress_b200 import _lib
    import lightcompress_b200

    class Other:
        built_for = 'torch 9.9.9+other, ' + str(sysconfig.get_config_var('SOABI'))

    class Unnamed:
        pass
    for front in (Other(), Unnamed()):
        monkeypatch.setattr(lightcompress_b200, '_calls', front)
        monkeypatch.setitem(sys.modules, 'lightcompress_b200._calls', front)
        with warnings.catch_warnings(record=True) as seen:
            warnings.simplefilter('always')
            assert isinstance(_lib._load_front(), _lib.NoFront)
        assert len(seen) == 1 and 'does not fit' in str(seen[0].message)

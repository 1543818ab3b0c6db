"""When the host module of tensor lists is built again, and that one of another torch or Python is refused (no GPU needed)."""
import re
import sys

import pytest
import torch

from nerf_amd import _lib, build


def test_the_host_module_goes_stale_with_torch_and_python(monkeypatch, tmp_path):
    module, record = tmp_path / 'lists.so', tmp_path / 'lists.txt'
    monkeypatch.setattr(build, 'LISTS', str(module))
    monkeypatch.setattr(build, 'LISTS_RECORD', str(record))
    assert build.lists_stale()                      # nothing there
    module.write_bytes(b'')
    assert build.lists_stale()                      # nobody knows what it was built with
    record.write_text(build.lists_record())
    assert not build.lists_stale()
    for owner, name, other in ((torch, '__version__', '9.9.9'), (sys, 'version', '9.9 (other)'),
                               (torch, '__file__', '/elsewhere/torch/__init__.py')):
        with monkeypatch.context() as m:
            m.setattr(owner, name, other)
            assert build.lists_stale(), name
    assert not build.lists_stale()


@pytest.mark.parametrize('name', ['torch', 'python'])
def test_a_host_module_of_another_version_is_refused(monkeypatch, name):
    good = _lib.lists()
    assert good.built_for == (re.match(r'[\d.]*\d', torch.__version__).group(), '%d.%d' % sys.version_info[:2])
    monkeypatch.setattr(_lib, '_lists', None)
    if name == 'torch':
        monkeypatch.setattr(torch, '__version__', '9.9.9+other')
    else:
        monkeypatch.setattr(sys, 'version_info', (9, 9, 0, 'final', 0))
    with pytest.raises(ImportError, match='nerf_amd.build'):
        _lib.lists()
    assert _lib._lists is None

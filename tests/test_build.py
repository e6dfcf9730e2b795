"""kernelfoundry_b200.build: what is built, where and when (CPU; nothing here needs a compiler run that is not cached)."""
from __future__ import annotations

import os
import subprocess
import sys

import pytest

from conftest import REPO


def _python(code, **env):
    res = subprocess.run([sys.executable, "-c", code], cwd=REPO, env={**os.environ, **env}, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr
    return res.stdout.strip()


@pytest.mark.parametrize("error", [RuntimeError("g++ failed (1): Python.h"), FileNotFoundError("g++")])
def test_library_is_built_without_pythons_headers(kf_lib, monkeypatch, capsys, error):
    """The C ABI's library does not wait for the Python module; what the module could not be built for is reported."""
    from kernelfoundry_b200 import build

    def fail(force=False):
        raise error

    monkeypatch.setattr(build, "build_host", fail)
    assert build.build() == build.LIB_PATH and os.path.exists(build.LIB_PATH)
    assert str(error) in capsys.readouterr().err


def test_a_library_elsewhere_has_its_module_beside_it(kf_lib, tmp_path):
    """With KF_LIB_PATH nothing is built into the package's own lib/; a library without a module uses the package's."""
    from kernelfoundry_b200 import build

    lib = tmp_path / "libkf_attn.so"
    lib.symlink_to(os.path.abspath(build.LIB_PATH))
    where = "from kernelfoundry_b200 import build; print(build.HOST_PATH)"
    assert os.path.dirname(_python(where, KF_LIB_PATH=str(lib))) == str(tmp_path)
    assert os.path.dirname(_python(where, KF_LIB_PATH="")) == build.LIB_DIR
    assert _python("from kernelfoundry_b200._lib import host; print(host().form())", KF_LIB_PATH=str(lib)) == "b''"
    assert os.listdir(tmp_path) == ["libkf_attn.so"]


def test_module_belongs_to_one_torch(kf_lib):
    """Another torch or Python means another file: it is built anew there, and one built for another is never loaded."""
    import sysconfig

    import torch

    from kernelfoundry_b200 import build

    name = os.path.basename(build.HOST_PATH)
    assert torch.__version__ in name and name.endswith(sysconfig.get_config_var("EXT_SUFFIX"))
    code = ("import torch; torch.__version__ = '0.0.1'; from kernelfoundry_b200 import _lib, build\n"
            "assert build.HOST_PATH != %r\ntry: _lib.host()\nexcept ImportError as e: print(e)" % build.HOST_PATH)
    assert "0.0.1" in _python(code)


def test_a_failed_build_leaves_no_outdated_module(monkeypatch, tmp_path):
    """A module older than its source goes even if the new one cannot be built; an up-to-date one stays."""
    from kernelfoundry_b200 import build

    source, module = tmp_path / "kf_host.cpp", tmp_path / "_kf_host.so"
    source.write_text("not C++")
    module.write_text("")
    monkeypatch.setattr(build, "HOST_SOURCE", str(source))
    monkeypatch.setattr(build, "HOST_PATH", str(module))
    os.utime(module, (os.path.getmtime(source) + 5,) * 2)
    assert build.build_host() == str(module)
    os.utime(module, (os.path.getmtime(source) - 5,) * 2)
    with pytest.raises(RuntimeError, match="g"):
        build.build_host()
    assert not module.exists()

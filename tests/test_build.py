"""kernelfoundry_b200.build: what is built, where and when (CPU; nothing here needs a compiler run that is not cached)."""
from __future__ import annotations

import os

import pytest


@pytest.mark.parametrize("error", [RuntimeError("g++ failed (1): Python.h"), FileNotFoundError("g++")])
def test_library_is_built_without_pythons_headers(kf_lib, monkeypatch, capsys, error):
    """The C ABI's library does not wait for the Python module; what the module could not be built for is reported."""
    from kernelfoundry_b200 import build

    def fail(force=False):
        raise error

    monkeypatch.setattr(build, "build_host", fail)
    assert build.build() == build.LIB_PATH and os.path.exists(build.LIB_PATH)
    assert str(error) in capsys.readouterr().err

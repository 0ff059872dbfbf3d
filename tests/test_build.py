"""The build notices what its outputs depend on (ltx-2_b200/build.py)."""
from __future__ import annotations

import importlib.util
import os

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ltx-2_b200")


@pytest.fixture
def build(tmp_path, monkeypatch):
    """build.py with its outputs in tmp_path and a compiler that only counts its calls."""
    spec = importlib.util.spec_from_file_location("ltx_build_under_test", os.path.join(PKG, "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    monkeypatch.setattr(mod, "LIB_DIR", str(tmp_path))
    monkeypatch.setattr(mod, "BINDING_PATH", str(tmp_path / "_ltxfp8_torch.so"))
    mod.calls = []

    class Compiler:
        @staticmethod
        def check_call(cmd):
            mod.calls.append(cmd)
            with open(cmd[cmd.index("-o") + 1], "wb") as f:
                f.write(b"built")

        @staticmethod
        def check_output(cmd):
            return b" (NEEDED) Shared library: [libstdc++.so.6]"

    monkeypatch.setattr(mod, "subprocess", Compiler)
    return mod


def test_binding_is_rebuilt_for_another_torch(build, monkeypatch):
    import torch
    build.build_binding()
    build.build_binding()
    assert len(build.calls) == 1  # up to date
    monkeypatch.setattr(torch, "__version__", torch.__version__ + ".other")
    build.build_binding()
    assert len(build.calls) == 2 and os.path.getsize(build.BINDING_PATH) == 5
    build.build_binding()
    assert len(build.calls) == 2


def test_binding_without_a_record_is_rebuilt(build):
    """A library from before the record, or from an interrupted build."""
    with open(build.BINDING_PATH, "wb") as f:
        f.write(b"old")
    build.build_binding()
    assert len(build.calls) == 1


def test_binding_of_another_torch_is_not_used():
    """The loader compares the torch it was compiled for with the one that runs."""
    import torch
    from ltx_kernels import _lib
    assert _lib.binding().torch_version == torch.__version__

    class Other:
        torch_version = "0.0"

    with pytest.raises(ImportError, match="built for torch 0.0"):
        _lib.check_binding(Other)

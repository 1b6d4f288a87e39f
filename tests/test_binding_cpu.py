"""CPU: how the torch binding is built: for one torch and interpreter, on the C++ runtime that they have loaded."""
import sys

import pytest
import torch


def test_another_torch_means_another_build(monkeypatch):
    from omlx_exl3_b200 import _lib, build
    assert _lib.torch_calls().__doc__ == f"built for torch {torch.__version__}, {sys.implementation.cache_tag}"
    assert build.binding_up_to_date()
    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", torch.__version__ + "0")
        assert not build.binding_up_to_date()
    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", "1.0")
        assert not build.binding_up_to_date()
    assert build.binding_up_to_date()


@pytest.mark.parametrize("compiler", [None, "g++"])
def test_the_binding_has_no_cxx_runtime_of_its_own(monkeypatch, tmp_path, compiler):
    """Whichever compiler the environment names: the shared library is needed, and none of it is inside."""
    from omlx_exl3_b200 import _lib, build
    _lib.torch_calls()
    path = build.BINDING
    if compiler:
        path = tmp_path / "_exl3_torch.so"
        monkeypatch.setenv("CXX", compiler)
        monkeypatch.setattr(build, "BINDING", path)
        build.build_binding(force=True)
    held = path.read_bytes()
    assert b"libstdc++.so.6\0" in held and b"std::locale::_Impl" not in held and b"_ZNSt6locale5_ImplC1Em\0" not in held

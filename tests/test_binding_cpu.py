"""CPU: how the torch binding is built: on the C++ runtime that torch has loaded."""
import pytest


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

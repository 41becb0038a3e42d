"""The operations' module is bound to one PyTorch, Python and C++ ABI: the build notices others, and the loader refuses them."""

import importlib.util
import json
import os

import pytest

from conftest import REPO, wf


@pytest.fixture
def build():
    path = os.path.join(REPO, "comfyui-weightferry_b200", "csrc", "build.py")
    spec = importlib.util.spec_from_file_location("wf_build_under_test", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("key,other", [("torch", "2.0.0"), ("python", ".cpython-39-x86_64-linux-gnu.so"), ("cxx11_abi", -1)])
def test_another_abi_is_stale(build, tmp_path, key, other):
    path = tmp_path / "abi"
    assert build._other_abi(str(path))  # nothing written down
    path.write_text("{")
    assert build._other_abi(str(path))
    path.write_text(json.dumps(build._ops_abi()))
    assert not build._other_abi(str(path))
    path.write_text(json.dumps({**build._ops_abi(), key: other}))
    assert build._other_abi(str(path))


def test_built_module_is_written_down(build):
    assert not build._other_abi(os.path.join(build.LIB_DIR, build.ABI_NAME))


@pytest.mark.parametrize("abi", [False, True])
def test_flag_is_pytorchs(build, monkeypatch, abi):
    import torch
    monkeypatch.setattr(torch, "compiled_with_cxx11_abi", lambda: abi)
    assert f"-D_GLIBCXX_USE_CXX11_ABI={int(abi)}" in build._cxx_cmd("/usr/local/cuda/bin/nvcc", "a.cpp", "a.o")


@pytest.mark.parametrize("built", [{"torch": "2.0.0"}, {"python": ".cpython-39-x86_64-linux-gnu.so"}])
def test_loader_refuses_another_abi(build, monkeypatch, tmp_path, built):
    ext = wf("_ext")
    ext.ops()
    path = tmp_path / "abi"
    monkeypatch.setattr(ext, "ABI_PATH", str(path))
    monkeypatch.setattr(ext, "_ops", None)
    path.write_text(json.dumps({**build._ops_abi(), **built}))
    with pytest.raises(ext.ExtensionMissing, match="were built for"):
        ext.ops()

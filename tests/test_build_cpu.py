"""The build (flash_eq/_build.py) of one small source, into a folder of its own."""
import ctypes
import importlib.util
import os

import pytest

from flash_eq import _build


@pytest.fixture
def small(tmp_path, monkeypatch):
    if not os.path.exists(_build.HIPCC):
        pytest.skip("no hipcc")
    (tmp_path / "csrc").mkdir()
    (tmp_path / "csrc" / "one.hip").write_text('extern "C" int feq_one() { return 1; }\n')
    real = _build.CSRC
    for name, path in (("CSRC", "csrc"), ("BUILD_DIR", "build"), ("LIB_DIR", "lib"), ("LIB_PATH", "lib/libflasheq.so"),
                       ("NODES_PATH", "lib/flasheq_torch.so")):
        monkeypatch.setattr(_build, name, str(tmp_path / path))
    (tmp_path / "csrc" / "torch_nodes.cpp").symlink_to(os.path.join(real, "torch_nodes.cpp"))
    (tmp_path / "lib").mkdir()
    (tmp_path / "lib" / "flasheq_torch.so").write_text("of an earlier build")
    return monkeypatch


def test_the_library_is_built_where_the_pytorch_module_is_not(small):
    small.setenv("CXX", "false")                 # a compiler that fails
    with pytest.raises(RuntimeError, match="torch_nodes.cpp"):
        _build.build()
    assert ctypes.CDLL(_build.LIB_PATH).feq_one() == 1
    assert not os.path.exists(_build.NODES_PATH)


def test_the_library_is_built_without_pytorch(small):
    find = importlib.util.find_spec
    small.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    assert _build.build() == _build.LIB_PATH
    assert ctypes.CDLL(_build.LIB_PATH).feq_one() == 1
    assert not os.path.exists(_build.NODES_PATH)

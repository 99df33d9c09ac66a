"""The extension module of the native host side is a way to the kernels, not a condition of them: what happens where it
cannot be built or loaded, or was built for another torch."""
import os

import pytest
import torch


@pytest.fixture
def elsewhere(tmp_path, monkeypatch):
    """The extension's place, empty; the library stays."""
    from embodied_efficiency_b200 import _lib, build
    build.build()
    monkeypatch.setattr(build, "TORCH_LIB", str(tmp_path / "ee_torch.so"))
    monkeypatch.setattr(_lib, "_native", None)
    return tmp_path


def _through_python():
    """A call that the Python function refuses: it was asked."""
    from embodied_efficiency_b200 import quantize_tokens
    with pytest.raises(RuntimeError, match="no CPU path"):
        quantize_tokens(torch.zeros(2, 64, dtype=torch.bfloat16))


@pytest.mark.parametrize("error", [ImportError("No module named 'torch'"), FileNotFoundError("g++"),
                                   RuntimeError("g++ failed")])
def test_library_is_built_without_the_extension(elsewhere, monkeypatch, error):
    from embodied_efficiency_b200 import build

    def fail():
        raise error

    monkeypatch.setattr(build, "_build_torch", fail)
    with pytest.warns(RuntimeWarning, match="was not built"):
        assert build.build() == build.LIB
    assert build.up_to_date() and not build.torch_up_to_date()


def test_missing_extension(elsewhere):
    with pytest.warns(RuntimeWarning, match="is not used"):
        _through_python()
    _through_python()  # said once


def test_file_that_is_no_extension(elsewhere):
    (elsewhere / "ee_torch.so").write_bytes(b"nothing of the kind")
    with pytest.warns(RuntimeWarning, match="is not used"):
        _through_python()


def test_another_torch(monkeypatch):
    from embodied_efficiency_b200 import _lib, build
    build.build()
    assert build.torch_up_to_date() and torch.__version__ in build.torch_version()
    monkeypatch.setattr(build, "torch_version", lambda: "0.1 cpython-312")
    assert build.up_to_date() and not build.torch_up_to_date()
    monkeypatch.setattr(_lib, "_native", None)
    with pytest.warns(RuntimeWarning, match="built for"):
        _through_python()


def test_extension_is_loaded():
    from embodied_efficiency_b200 import _lib, build
    build.build()
    assert _lib.native().torch_version == build.torch_version() and os.path.exists(build.TORCH_LIB)

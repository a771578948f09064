"""Which library an operator call takes: B2DIT_SO is looked at in every call."""
import shutil

import pytest
import torch


def test_operator_calls_follow_the_variable(pkg, monkeypatch, tmp_path):
    lib = pkg._lib
    monkeypatch.delenv("B2DIT_SO", raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)      # what a CPU tensor's get_device() says
    calls = pkg.ops.launch_count

    def call():                                             # no rows: returns before anything is launched
        pkg.ops._call("b2_dequantize_int8_rowwise", torch.zeros(1), None, None, None, 0, 4, None)

    sizes = (1, 2, 2, 1, 65536, -1, 0, 0)
    first = lib.load()
    call()
    need = pkg.ops._window_workspace(*sizes)
    assert need > 0 and lib.current() is first
    try:
        monkeypatch.setenv("B2DIT_SO", str(tmp_path / "missing.so"))
        for refused in (call, lambda: pkg.ops._window_workspace(*sizes)):
            with pytest.raises(RuntimeError, match="Cannot load"):
                refused()
        other = tmp_path / "other.so"
        shutil.copy(lib.DEFAULT_SO, other)
        monkeypatch.setenv("B2DIT_SO", str(other))
        call()
        assert lib._lib_path == other and lib.current() is lib.load() is not first
        assert pkg.ops._window_workspace(*sizes) == need
    finally:
        monkeypatch.delenv("B2DIT_SO")
        lib.load()
    call()
    assert lib._lib_path == lib.DEFAULT_SO and pkg.ops.launch_count == calls + 3

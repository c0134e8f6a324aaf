"""CPU tests: the CPython module of the row operators' calls is optional.  One that
does not load, or is not there, leaves the ctypes path."""
import os
import subprocess
import warnings

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash1017-engine_b200")


@pytest.fixture
def fresh(ffn, monkeypatch):
    """The binding as before its first row operator."""
    for name in ("_T", "_dts", "_dev_now", "_raw_stream", "_calls"):
        monkeypatch.setattr(ffn, name, None)
    return ffn


def refuses_as_ever(ffn):
    import torch
    x = torch.zeros(4, 64)
    for call in (lambda: ffn.BlockNorm().forward(x), lambda: ffn.moe_combine(x, torch.zeros(4, 2, dtype=torch.int32))):
        with pytest.raises(ffn.FfnError):
            call()


def test_a_module_that_does_not_load(fresh, tmp_path, monkeypatch):
    bad = tmp_path / "ffn_b200_torch.so"
    bad.write_bytes(b"not a shared object")
    monkeypatch.setattr(fresh, "_calls_path", lambda: str(bad), raising=False)
    with pytest.warns(RuntimeWarning, match="ctypes"):
        refuses_as_ever(fresh)
    assert fresh._calls is None and fresh._T is not None
    with warnings.catch_warnings():  # once
        warnings.simplefilter("error")
        refuses_as_ever(fresh)


def test_no_module(fresh, tmp_path, monkeypatch):
    monkeypatch.setattr(fresh, "_calls_path", lambda: str(tmp_path / "none.so"))
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        refuses_as_ever(fresh)
    assert fresh._calls is None


def make(**variables):
    return subprocess.run(["make", "-n", "-C", PKG, *(f"{k}={v}" for k, v in variables.items())], check=True,
                          capture_output=True, text=True).stdout


def test_the_module_is_built_for_one_python_and_one_torch(ffn, tmp_path):
    """The name that is built is the one that is loaded, and another torch's is another."""
    import sys
    out = str(tmp_path / "out")
    assert os.path.basename(ffn._calls_path()) in make(PYTHON=sys.executable, OUT=out)
    other = tmp_path / "torch"
    for part in ("include/ATen", "lib"):
        (other / part).mkdir(parents=True)
    (other / "version.py").write_text("__version__ = '9.9.9+cu128'\n")
    (other / "include" / "ATen" / "ATen.h").write_text("")
    # without CUDA's half of torch there is nothing to link against
    assert "ffn_b200_torch" not in make(PYTHON=sys.executable, OUT=out, TORCH=str(other))
    (other / "lib" / "libc10_cuda.so").write_text("")
    plan = make(PYTHON=sys.executable, OUT=out, TORCH=str(other))
    assert "torch-9.9.9+cu128.so" in plan and os.path.basename(ffn._calls_path()) not in plan


def test_a_module_that_does_not_compile_is_left_out(ffn, tmp_path):
    """make goes on without it and says so."""
    import sys
    lib, module = tmp_path / "libffn_b200.so", tmp_path / os.path.basename(ffn._calls_path())
    lib.write_bytes(b""), module.write_bytes(b"of an older source")
    os.utime(module, (1, 1))
    r = subprocess.run(["make", "-C", PKG, f"PYTHON={sys.executable}", f"OUT={tmp_path}", "CXX=false", "-o", str(lib),
                        str(module)], capture_output=True, text=True)
    assert r.returncode == 0 and "ctypes" in r.stderr, r.stderr
    assert not module.exists()

"""The int8 layer's calls on torch tensors have a compiled form (_calls-*.so) and Python forms:
where the first cannot be built or loaded, the others do its work."""
import os
import subprocess
import warnings

import pytest

torch = pytest.importorskip("torch")

import mini_llama_b200 as mlb  # noqa: E402
from mini_llama_b200 import build  # noqa: E402


def no_compiler(*args, **kw):
    raise FileNotFoundError("g++")


def no_headers(cmd, *args, **kw):
    raise subprocess.CalledProcessError(1, cmd)


def broken(tmp_path):
    path = tmp_path / "_calls-broken.so"
    path.write_bytes(b"not a library")
    return str(path)


def unloadable(monkeypatch, tmp_path, how):
    """Leaves mlb without the compiled form, in one of the ways it can be missing."""
    monkeypatch.setattr(mlb, "_fast", None)
    if how == "broken":
        monkeypatch.setattr(build, "calls_path", lambda: broken(tmp_path))
    else:
        monkeypatch.setattr(build, "calls_path", lambda: str(tmp_path / "_calls-none.so"))
        monkeypatch.setattr(build.subprocess, "run",
                            no_compiler if how == "no compiler" else no_headers)


HOW = ["no compiler", "no headers", "broken"]


@pytest.mark.parametrize("how", HOW)
def test_the_python_forms_are_reached(monkeypatch, tmp_path, how):
    unloadable(monkeypatch, tmp_path, how)
    x = torch.zeros(2, 32)
    with pytest.warns(RuntimeWarning, match="Python forms"):
        with pytest.raises(mlb.MlbError, match="must be on a CUDA device"):
            mlb.CudaInt8QuantizeDeviceInput(x)
    with warnings.catch_warnings():  # said once
        warnings.simplefilter("error")
        with pytest.raises(mlb.MlbError, match="must be on a CUDA device"):
            mlb.CudaRmsNormInt8DeviceWeight(x, x[0], 1e-5)
    assert os.listdir(tmp_path) in ([], ["_calls-broken.so"])


def test_a_warning_made_an_error_ends_one_call_alone(monkeypatch, tmp_path):
    unloadable(monkeypatch, tmp_path, "no compiler")
    x = torch.zeros(2, 32)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        with pytest.raises(RuntimeWarning):
            mlb.CudaInt8QuantizeDeviceInput(x)
        with pytest.raises(mlb.MlbError, match="must be on a CUDA device"):
            mlb.CudaInt8QuantizeDeviceInput(x)


def test_a_file_for_another_torch_or_source_is_not_taken(monkeypatch, tmp_path):
    here = build.calls_path()
    assert here == build.calls_path()
    monkeypatch.setattr(build, "_torch_version", lambda torch: "0.0.1")
    other = build.calls_path()
    assert other != here and os.path.dirname(other) == os.path.dirname(here)
    monkeypatch.undo()
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    (csrc / "torch_calls.cc").write_text("// another source\n")
    monkeypatch.setattr(build, "CSRC", str(csrc))
    assert build.calls_path() not in (here, other)


def test_two_processes_that_build_at_once_stay_apart(monkeypatch, tmp_path):
    """Each writes a file of its own and puts it in place whole."""
    at = str(tmp_path / "_calls-x.so")
    monkeypatch.setattr(build, "calls_path", lambda: at)
    written = []

    def compile_one(cmd, check):
        made = cmd[cmd.index("-o") + 1]
        written.append(made)
        with open(made, "w") as f:
            f.write("whole")
        assert not os.path.exists(at)

    monkeypatch.setattr(build.subprocess, "run", compile_one)
    assert build.build_calls() == at and os.listdir(tmp_path) == ["_calls-x.so"]
    assert build.build_calls() == at and len(written) == 1  # there already
    os.remove(at)
    monkeypatch.setattr(build.os, "getpid", lambda: 1)
    build.build_calls()
    assert len(set(written)) == 2


@pytest.mark.parametrize("there", [True, False])
def test_a_build_without_headers_leaves_out_the_calls(monkeypatch, there):
    made = []
    for name in ("build_synth", "build_cuda", "build_calls"):
        monkeypatch.setattr(build, name, lambda *a, name=name: made.append(name))
    monkeypatch.setattr(build, "_torch_dir", lambda: "/torch")
    real = os.path.exists
    monkeypatch.setattr(build.os.path, "exists", lambda p: there or real(p))
    build.build()
    assert made == ["build_synth", "build_cuda"] + ["build_calls"] * there


@pytest.mark.gpu
@pytest.mark.parametrize("how", HOW)
def test_the_same_bits_without_it(cuda, monkeypatch, tmp_path, how):
    x = torch.randn(5, 96, device="cuda")
    w = torch.rand(96, device="cuda")
    q, pos = x.view(5, 3, 32), torch.arange(5, device="cuda", dtype=torch.int32)
    table = mlb.RopeTable(32)

    def calls():
        c, s, h = mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5, residual=x)
        return [c, s, h, *mlb.CudaInt8QuantizeDeviceInput(x), *mlb.CudaSiluMulInt8DeviceInput(x, h),
                mlb.CudaInt8DequantizeDeviceInput(c, s), mlb.CudaInt8LinearDeviceInput(c, s, c, s),
                *mlb.CudaRopeRowsDeviceInput(q, q, pos, table)]

    want = calls()
    unloadable(monkeypatch, tmp_path, how)
    with pytest.warns(RuntimeWarning, match="Python forms"):
        got = calls()
    for a, b in zip(got, want):
        assert torch.equal(a, b)

"""What the native build makes, in which order, and with what missing; commands are recorded, not run."""
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

from nccl_plugin_gpudirecttcpx_b200 import _build

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture
def made(tmp_path, monkeypatch):
    """Names of the files that build commands would have made."""
    names = []

    def run(cmd):
        out = Path(cmd[cmd.index("-o") + 1])
        out.parent.mkdir(parents=True, exist_ok=True)
        out.touch()
        names.append(out.name)

    monkeypatch.setattr(_build, "_run", run)
    monkeypatch.setattr(_build, "OUT", tmp_path)
    monkeypatch.setattr(_build, "OBJ", tmp_path / "obj")
    return names


def test_the_plugin_needs_no_torch(made, monkeypatch):
    monkeypatch.setitem(sys.modules, "torch", None)  # an import of it fails
    outs = [p.name for p in _build.build_cuda()]
    assert {"libtcpxb_kernels.so", "libtcpxb_train.so", "libnccl-net.so", "tcpxb_rxdm_gpu"} <= set(made) & set(outs)
    assert not any("torch" in name for name in made + outs)


def test_the_torch_module_comes_last(made, monkeypatch):
    """Headers that do not compile cost nothing else."""
    run = _build._run

    def fail(cmd):
        if "torch" in Path(cmd[cmd.index("-o") + 1]).name:
            raise RuntimeError("native build failed")
        run(cmd)

    monkeypatch.setattr(_build, "_run", fail)
    with pytest.raises(RuntimeError):
        _build.build_cuda()
    assert {"libtcpxb_train.so", "libnccl-net.so", "tcpxb_rxdm_gpu"} <= set(made)
    monkeypatch.setattr(_build, "_run", run)
    made.clear()
    assert "tcpxb_train_torch.so" in [p.name for p in _build.build_cuda()] and "tcpxb_train_torch.so" in made and "libnccl-net.so" not in made


def test_another_torch_rebuilds_its_module_alone(made, monkeypatch):
    import torch
    _build.build_cuda()
    assert "tcpxb_train_torch.so" in made
    made.clear()
    _build.build_cuda()
    assert not made
    monkeypatch.setattr(torch, "__version__", torch.__version__ + ".other")
    _build.build_cuda()
    assert sorted(made) == ["tcpxb_train_torch.so", "torch_bind_train_torch.o"]
    made.clear()
    _build.build_cuda()
    assert not made


@pytest.mark.skipif(not shutil.which("cmake") or not _build._nvcc(), reason="needs cmake and nvcc")
def test_cmake_configures_without_python_headers(tmp_path):
    cmd = ["cmake", "-S", str(ROOT), "-B", str(tmp_path), f"-DCMAKE_CUDA_COMPILER={_build._nvcc()}"]
    r = subprocess.run([*cmd, "-DCMAKE_DISABLE_FIND_PACKAGE_Python3=TRUE"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    targets = subprocess.run(["cmake", "--build", str(tmp_path), "--target", "help"], capture_output=True, text=True, timeout=60).stdout
    assert "nccl-net" in targets and "tcpxb_train" in targets and "tcpxb_train_torch" not in targets

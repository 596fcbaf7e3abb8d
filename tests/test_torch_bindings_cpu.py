"""The torch bindings (libctu_torch.so) are bound to one torch build: without a library for the installed torch the
ops that it registers refuse, saying why, and every other op of the package works as before."""

import importlib.util
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1] / "comfyui-turing-utils_b200"
PACKAGE = ROOT / "comfyui_turing_utils_kernel"
TORCH_LIB = PACKAGE / "libctu_torch.so"

PROGRAM = """
import torch
import comfyui_turing_utils_kernel as k
from comfyui_turing_utils_kernel import _lib

x = torch.empty((3, 512), dtype=torch.bfloat16, device="meta")
codes, scale = k.turing_bf16_int8_convrot_quantize(x, 256)
assert codes.shape == (3, 512) and codes.dtype == torch.int8 and scale.shape == (3, 1)
k.turing_layer_norm_adaln(x.view(1, 3, 512), torch.empty((1, 1, 512), dtype=torch.bfloat16, device="meta"),
                          torch.empty((1, 1, 512), dtype=torch.bfloat16, device="meta"))
tiles = k.turing_fp4_block_scale_tiles(torch.zeros((4, 8), dtype=torch.uint8).view(torch.float8_e4m3fn))
assert tiles.shape == (1, 2, 32, 16)
calls = [lambda: k.turing_fp4_quantize(x), lambda: k.turing_fp4_dequantize(x, x, x), lambda: k.turing_layer_norm(x),
         lambda: k.turing_fp4_linear(x, x, x, x, x, x), lambda: k.turing_fp4_linear_grad_input(x, x, x, x),
         lambda: k.turing_convrot_fp4_linear(x, x, x, x)]
for call in calls:
    try:
        call()
    except _lib.KernelUnavailable as exc:
        print(exc)
    else:
        raise AssertionError("not refused")
"""


def run(folder):
    return subprocess.run([sys.executable, "-c", PROGRAM], cwd=folder, capture_output=True, text=True, timeout=300)


@pytest.fixture
def package(tmp_path):
    copy = tmp_path / PACKAGE.name
    copy.mkdir()
    for source in PACKAGE.glob("*.py"):
        shutil.copy(source, copy)
    (copy / "libctu_b200.so").symlink_to(PACKAGE / "libctu_b200.so")
    return copy


def other_torch():
    """The library's bytes with another torch version in its mark."""
    import torch
    from comfyui_turing_utils_kernel import _lib

    version = torch.__version__.encode()
    data = TORCH_LIB.read_bytes()
    assert _lib.torch_bindings_version(TORCH_LIB) == torch.__version__
    return data.replace(b"ctu-built-for-torch=" + version, b"ctu-built-for-torch=0" + version[1:])


def test_missing_library_refuses_its_own_ops_alone(package):
    res = run(package.parent)
    assert res.returncode == 0, res.stderr
    assert res.stdout.count("is not built") == 6


def test_library_of_another_torch_is_not_loaded(package):
    import torch

    (package / TORCH_LIB.name).write_bytes(other_torch())
    res = run(package.parent)
    assert res.returncode == 0, res.stderr
    assert res.stdout.count("built for torch 0" + torch.__version__[1:]) == 6


def test_library_that_does_not_load(package):
    import torch

    (package / TORCH_LIB.name).write_bytes(b"not a library ctu-built-for-torch=" + torch.__version__.encode() + b"\0")
    res = run(package.parent)
    assert res.returncode == 0, res.stderr
    assert len(res.stdout.splitlines()) >= 6 and res.stdout.count(TORCH_LIB.name) >= 6


def test_library_that_cannot_be_read(package):
    (package / TORCH_LIB.name).mkdir()
    res = run(package.parent)
    assert res.returncode == 0, res.stderr
    assert res.stdout.count(TORCH_LIB.name) >= 6


def test_library_of_another_torch_is_stale(tmp_path):
    spec = importlib.util.spec_from_file_location("ctu_build", ROOT / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    assert not build._torch_stale(TORCH_LIB)
    other = tmp_path / TORCH_LIB.name
    other.write_bytes(other_torch())
    assert build._torch_stale(other) and build._torch_stale(tmp_path / "none.so")

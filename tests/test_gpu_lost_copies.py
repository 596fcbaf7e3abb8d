"""Failure path of the 4-bit and layer norm kernels, without a GPU fault: one copy of the first CTA is not issued, the
wait for it runs out after a short limit, and the kernel stops, raises its flag in the device error word and leaves
no finite result that hangs on that copy.  The next call is whole again."""

import contextlib

import pytest
import torch

from test_gpu_fp4 import random_operand

pytestmark = pytest.mark.gpu

UNTOUCHED = 7.0


@pytest.fixture(scope="module")
def k():
    import comfyui_turing_utils_kernel as kernel

    return kernel


@pytest.fixture(scope="module")
def lib():
    from comfyui_turing_utils_kernel import _lib

    return _lib.load()


@contextlib.contextmanager
def lost_copy(which):
    """The copy is lost in here; on the way out the error word must tell of it, and is cleared."""
    from comfyui_turing_utils_kernel import _lib

    device = torch.cuda.current_device()
    assert _lib.device_error(device) == 0
    _lib.check(_lib.load().ctu_debug_lose_copy(which, 30_000_000))
    try:
        yield
        torch.cuda.synchronize()
    finally:
        _lib.load().ctu_debug_lose_copy(-1, 0)
    assert _lib.device_error(device) & 7  # a tile's, a stage's or an accumulator's wait
    assert _lib.device_error(device) == 0


def stream():
    return torch.cuda.current_stream().cuda_stream


def check(rc):
    from comfyui_turing_utils_kernel import _lib

    _lib.check(rc)


# ---------------------------------------------------------------------------- product of few rows
@pytest.mark.parametrize("fmt", ("nvfp4", "mxfp4"))
# K split over a cluster of eight, three and four, one CTA a strip, and a copy that waits for a free stage.
@pytest.mark.parametrize("m,n,width,which", [(1, 500, 5120, 0), (1, 5120, 5120, 3), (9, 4096, 2048, 1), (17, 13824, 512, 1),
                                             (100, 1000, 13824, 5), (40, 13800, 5120, 12)])
def test_few_rows(k, lib, fmt, m, n, width, which):
    (a, a_s, a_r), _ = random_operand(k, m, width, fmt, 1)
    (w, w_s, w_r), _ = random_operand(k, n, width, fmt, 2)

    def call():
        out = torch.full((m, n), UNTOUCHED, dtype=torch.bfloat16, device="cuda")
        check(lib.ctu_fp4_linear(a.data_ptr(), w.data_ptr(), a_s.data_ptr(), w_s.data_ptr(), a_r.data_ptr(), w_r.data_ptr(),
                                 n, None, out.data_ptr(), m, n, width, 0 if fmt == "nvfp4" else 1, stream()))
        return out

    before = lib.ctu_debug_set_fp4_kernel(2)
    try:
        whole = call()
        with lost_copy(which):
            cut = call()
        # The first cluster has the first strip of 128 weight rows, for the first tokens; nothing else is lost.
        strip = (cut == UNTOUCHED)[:, :128]
        assert strip.all()
        assert torch.equal(cut[:, 128:], whole[:, 128:])
        assert torch.equal(call(), whole)
    finally:
        lib.ctu_debug_set_fp4_kernel(before)

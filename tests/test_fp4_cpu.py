"""4-bit floating point and layer norm entry points without a GPU: formats, refusals, fake shapes."""

import ctypes

import numpy as np
import pytest
import torch

import fp4_oracle as oracle

FAKE = ctypes.c_void_p(0x10000)  # aligned, never dereferenced: the checked argument fails first
NULL = ctypes.c_void_p(0)


@pytest.fixture(scope="module")
def lib():
    from comfyui_turing_utils_kernel import _lib

    return _lib.load()


def refused(lib, rc, text):
    from comfyui_turing_utils_kernel import _lib

    message = lib.ctu_last_error().decode()
    return rc in (_lib.CTU_ERR_INVALID_ARGUMENT, _lib.CTU_ERR_UNSUPPORTED) and text in message


def test_oracle_rotation_is_the_orthogonal_one():
    x = np.random.default_rng(0).standard_normal((6, 512)).astype(np.float32)
    r = oracle.rotation_matrix()
    np.testing.assert_allclose(r @ r, np.eye(256), atol=1e-15)  # its own inverse
    exact = (x.astype(np.float64).reshape(-1, 256) @ r).reshape(x.shape)
    # Four stages of three additions on values bounded by the rotated magnitudes.
    bound = 12 * 2.0**-24 * (np.abs(x).astype(np.float64).reshape(-1, 256) @ np.abs(r)).reshape(x.shape)
    assert (np.abs(oracle.rotate(x) - exact) <= bound).all()


@pytest.mark.parametrize("fmt", ("nvfp4", "mxfp4"))
@pytest.mark.parametrize("rotation", (0, 256))
def test_oracle_values_are_nearest(fmt, rotation):
    """A code's value is within half a grid step of what it stands for, unless it saturates."""
    x = (np.random.default_rng(1).standard_normal((40, 512)) * 8).astype(np.float32)
    codes, scales, row = oracle.quantize(x, fmt, rotation)
    v = oracle.rotate(x) if rotation else x
    got = oracle.values(codes, scales, fmt) * row[:, None]
    step = np.repeat(oracle.scale_values(fmt)[scales], oracle.BLOCK[fmt], axis=1) * row[:, None]
    far = np.abs(got - v) / step
    size = np.abs(v) / step
    allowed = np.where(size <= 2, 0.25, np.where(size <= 4, 0.5, 1.0)) * (1 + 1e-6)
    assert ((far <= allowed) | (np.abs(got) == 6 * step)).all()
    assert (np.frexp(row)[0] == 0.5).all()


def test_tiles_round_trip():
    import comfyui_turing_utils_kernel as k

    for rows, blocks in ((1, 1), (3, 5), (127, 4), (128, 8), (300, 98)):
        plain = np.random.default_rng(rows).integers(0, 127, (rows, blocks)).astype(np.uint8)
        want = oracle.tiles(plain)
        got = k.turing_fp4_block_scale_tiles(torch.from_numpy(plain).view(torch.float8_e4m3fn))
        np.testing.assert_array_equal(got.view(torch.uint8).numpy(), want)
        np.testing.assert_array_equal(oracle.untile(want, rows, blocks), plain)
    with pytest.raises(RuntimeError):
        k.turing_fp4_block_scale_tiles(torch.zeros(4, 4))


def test_sizes(lib):
    assert lib.ctu_fp4_block_scale_bytes(1, 32, 0) == 512 and lib.ctu_fp4_block_scale_bytes(129, 1568, 0) == 2 * 25 * 512
    assert lib.ctu_fp4_block_scale_bytes(129, 1568, 1) == 2 * 13 * 512 and lib.ctu_fp4_block_scale_bytes(0, 32, 0) == 0
    assert lib.ctu_fp4_grad_workspace_bytes(4096, 5120, 5120) >= 2 * 5120 * 5120
    assert lib.ctu_fp4_grad_workspace_bytes(0, 5120, 5120) == 0
    assert lib.ctu_layer_norm_backward_workspace_bytes(10, 64) == 2 * 10 * 64 * 4
    assert lib.ctu_layer_norm_backward_workspace_bytes(1 << 20, 64) == 2 * 148 * 64 * 4


def test_quantizer_refusals(lib):
    def call(x=FAKE, rows=4, k=256, dtype=0, fmt=0, rotation=0, codes=FAKE):
        return lib.ctu_fp4_quantize(x, rows, k, dtype, fmt, rotation, codes, FAKE, FAKE, NULL)

    assert refused(lib, call(k=48), "K%32=0") and refused(lib, call(k=0), "K%32=0") and refused(lib, call(rows=-1), "K%32=0")
    assert refused(lib, call(fmt=2), "nvfp4 or mxfp4") and refused(lib, call(dtype=2), "float16 or bfloat16")
    assert refused(lib, call(rotation=128), "0 or 256") and refused(lib, call(k=96, rotation=256), "divisible by the rotation")
    assert refused(lib, call(k=49152 + 256), "at most") and refused(lib, call(x=NULL), "null")
    assert refused(lib, call(codes=ctypes.c_void_p(0x10008)), "aligned") and refused(lib, call(rows=1 << 40), "range")
    assert call(rows=0, x=NULL) == 0


def test_dequantizer_refusals(lib):
    def call(count=4, rows=4, k=256, fmt=0, dtype=0, out=FAKE):
        return lib.ctu_fp4_dequantize(FAKE, FAKE, FAKE, count, rows, k, fmt, dtype, out, NULL)

    assert refused(lib, call(k=16), "K%32=0") and refused(lib, call(fmt=-1), "nvfp4") and refused(lib, call(dtype=3), "output")
    assert refused(lib, call(count=3), "one row scale") and refused(lib, call(out=NULL), "null")
    assert call(rows=0, count=0) == 0


def test_linear_refusals(lib):
    def call(m=4, n=8, k=256, count=8, fmt=0, out=FAKE):
        return lib.ctu_fp4_linear(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, count, NULL, out, m, n, k, fmt, NULL)

    assert refused(lib, call(k=33), "K%32=0") and refused(lib, call(n=-8), "K%32=0") and refused(lib, call(fmt=7), "nvfp4")
    assert refused(lib, call(count=7), "scalar") and refused(lib, call(out=NULL), "null")
    assert refused(lib, call(out=ctypes.c_void_p(0x10002)), "aligned")
    assert refused(lib, call(m=1 << 30, n=1 << 30, count=1), "range")
    assert call(m=0) == 0 and call(n=0, count=0) == 0
    assert refused(lib, lib.ctu_debug_set_fp4_kernel(3), "unknown")


def test_gradient_refusals(lib):
    def call(m=4, n=8, k=256, count=8, fmt=0, rotation=0, ws=FAKE):
        return lib.ctu_fp4_linear_grad_input(FAKE, FAKE, FAKE, FAKE, count, rotation, ws, FAKE, m, n, k, fmt, NULL)

    assert refused(lib, call(n=9), "N%8=0") and refused(lib, call(k=40), "K%32=0") and refused(lib, call(rotation=1), "0 or 256")
    assert refused(lib, call(k=288, rotation=256), "divisible") and refused(lib, call(count=3), "scalar")
    assert refused(lib, call(ws=NULL), "null") and call(m=0) == 0


def test_layer_norm_refusals(lib):
    def forward(x=FAKE, rows=4, hidden=64, eps=1e-5, dtype=0, wdtype=0):
        return lib.ctu_layer_norm(x, NULL, NULL, FAKE, FAKE, FAKE, rows, hidden, eps, dtype, wdtype, NULL)

    assert refused(lib, forward(dtype=3), "float16") and refused(lib, forward(wdtype=1), "type or float32")
    assert refused(lib, forward(hidden=0), "positive") and refused(lib, forward(eps=0.0), "epsilon")
    assert refused(lib, forward(eps=float("inf")), "epsilon") and refused(lib, forward(x=NULL), "null")
    assert forward(rows=0) == 0

    def backward(grad=FAKE, dx=FAKE, dw=FAKE, ws=FAKE, rows=4, dtype=0):
        return lib.ctu_layer_norm_backward(grad, FAKE, NULL, FAKE, FAKE, dx, dw, NULL, ws, rows, 64, dtype, dtype, NULL)

    assert refused(lib, backward(grad=NULL), "null") and refused(lib, backward(ws=NULL), "workspace")
    assert refused(lib, backward(dtype=-1), "float16")
    assert backward(dx=NULL, dw=NULL) == 0 and backward(rows=0, dw=NULL) == 0


def test_fake_shapes_and_gradients():
    import comfyui_turing_utils_kernel as k

    x = torch.empty((3, 512), dtype=torch.bfloat16, device="meta")
    for fmt, blocks, dtype in (("nvfp4", 32, torch.float8_e4m3fn), ("mxfp4", 16, torch.float8_e8m0fnu)):
        codes, scale, row = k.turing_fp4_quantize(x, fmt, 256)
        assert codes.shape == (3, 256) and codes.dtype == torch.uint8 and row.shape == (3, 1)
        assert scale.shape == (1, blocks // 4, 32, 16) and scale.dtype == dtype
        assert k.turing_fp4_dequantize(codes, scale, row, torch.float32).shape == (3, 512)
        w, ws, wr = (t.new_empty(s) for t, s in ((codes, (24, 256)), (scale, scale.shape), (row, (24, 1))))
        y = k.turing_fp4_linear(codes, w, scale, ws, row, wr)
        assert y.shape == (3, 24) and y.dtype == torch.bfloat16
        assert k.turing_fp4_linear_grad_input(y, w, ws, wr, 256).shape == (3, 512)
        leaf = torch.empty((3, 512), dtype=torch.bfloat16, device="meta", requires_grad=True)
        k.turing_convrot_fp4_linear(leaf, w, ws, wr).sum().backward()
        assert leaf.grad.shape == (3, 512)
    leaf = torch.empty((2, 3, 64), device="meta", requires_grad=True)
    weight = torch.empty(64, device="meta", requires_grad=True)
    y = k.turing_layer_norm(leaf, weight)
    y.sum().backward()
    assert y.shape == leaf.grad.shape == (2, 3, 64) and weight.grad.shape == (64,)


def test_cpu_tensors_are_refused():
    import comfyui_turing_utils_kernel as k

    x = torch.zeros((2, 256), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        k.turing_fp4_quantize(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        k.turing_layer_norm(x)
    codes, scale = torch.zeros((2, 128), dtype=torch.uint8), torch.zeros((1, 4, 32, 16), dtype=torch.float8_e4m3fn)
    with pytest.raises(RuntimeError, match="CUDA"):
        k.turing_fp4_linear(codes, codes, scale, scale, torch.ones(2), torch.ones(2))
    with pytest.raises(RuntimeError, match="CUDA"):
        k.turing_fp4_dequantize(codes, scale, torch.ones(2))
    with pytest.raises(RuntimeError, match="CUDA"):
        k.turing_fp4_linear_grad_input(x, codes, scale, torch.ones(2))


def test_wrapper_refusals():
    from comfyui_turing_utils_b200 import dispatch, fusions

    x = torch.zeros((2, 256), dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError):
        dispatch.convrot_fp4_linear(x, x, x, x, convrot_groupsize=128)
    with pytest.raises(RuntimeError, match="does not fit"):
        fusions.affine_layer_norm(torch.nn.LayerNorm([2, 256]), x)


def differentiable_calls():
    """(call, differentiable leaves) of the differentiable ops on meta tensors."""
    import comfyui_turing_utils_kernel as k

    x = torch.empty((3, 512), dtype=torch.bfloat16, device="meta")
    codes, scale, row = k.turing_fp4_quantize(torch.empty((24, 512), dtype=torch.bfloat16, device="meta"), "nvfp4", 256)
    norm = torch.empty((2, 3, 64), device="meta"), torch.empty(64, device="meta"), torch.empty(64, device="meta")
    return [(lambda x: k.turing_convrot_fp4_linear(x, codes, scale, row), (x,)), (k.turing_layer_norm, norm)]


@pytest.mark.parametrize("requires_grad", (False, True))
@pytest.mark.parametrize("no_grad", (False, True))
def test_forward_mode_is_refused(requires_grad, no_grad):
    """There is no forward-mode derivative: a tangent raises, it does not come out as zero."""
    import torch.autograd.forward_ad as fwd

    for call, leaves in differentiable_calls():
        for i in range(len(leaves)):
            args = [t.clone().requires_grad_(requires_grad) for t in leaves]
            with fwd.dual_level(), torch.set_grad_enabled(not no_grad):
                args[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*args)
                primals = [fwd.unpack_dual(t).primal for t in args]
                assert call(*primals).shape == call(*leaves).shape  # without a tangent it runs inside the level too


def test_functional_forward_mode_is_refused():
    for call, leaves in differentiable_calls():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(call, leaves, tuple(torch.ones_like(t) for t in leaves))


def test_tangent_of_a_gradient_is_refused():
    """Forward mode over the backward pass: the gradient that comes in carries the tangent."""
    import torch.autograd.forward_ad as fwd

    for call, leaves in differentiable_calls():
        args = [t.clone().requires_grad_(True) for t in leaves]
        y = call(*args)
        with fwd.dual_level():
            grad = fwd.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(y, args, grad, retain_graph=True)
        assert torch.autograd.grad(y, args, torch.ones_like(y))[0].shape == leaves[0].shape


def test_timeout_hook_refusals(lib):
    for limit in (0, 5_000_000_001):
        assert refused(lib, lib.ctu_debug_inject_timeout(0, limit), "limit")
    assert lib.ctu_debug_inject_timeout(3, 1000) == 0 and lib.ctu_debug_inject_timeout(-1, 0) == 0

"""``turing_utils::*`` torch custom ops over the B200 kernels.

Op names, signatures, defaults, device/capability errors and fake (meta) kernels
follow the reference's kernel/comfyui_turing_utils_kernel/ops.py, so graph capture,
torch.compile tracing and shape propagation see the same contract.  Each op calls
the matching function of ``_C`` (the C-ABI shim); there is no CPU path.
"""

from __future__ import annotations

import functools

import torch

from . import _C, _lib


def _require_cuda(t: torch.Tensor, what: str) -> None:
    if t.device.type != "cuda":
        raise RuntimeError(f"{what} requires CUDA tensors")
    if torch.cuda.get_device_capability(t.device) < (7, 5):
        raise RuntimeError(f"{what} requires sm75 or newer")


# ops.py:8-35
@torch.library.custom_op("turing_utils::w4a8_linear", mutates_args=())
def turing_w4a8_linear(
    activation: torch.Tensor,
    weight: torch.Tensor,
    activation_scale: torch.Tensor,
    weight_scale: torch.Tensor,
    bias: torch.Tensor | None = None,
) -> torch.Tensor:
    """Signed packed-int4 W4A8 linear (int4 sign-extended in shared memory, tcgen05 MMA)."""
    _require_cuda(activation, "Turing W4A8")
    return _C.turing_w4a8_linear(
        activation.contiguous(),
        weight.contiguous(),
        activation_scale.contiguous(),
        weight_scale.contiguous(),
        None if bias is None else bias.contiguous(),
    )


@turing_w4a8_linear.register_fake
def _turing_w4a8_linear_fake(activation, weight, activation_scale, weight_scale, bias=None):
    return torch.empty((activation.size(0), weight.size(0)), dtype=torch.bfloat16, device=activation.device)


# ops.py:38-93
@torch.library.custom_op("turing_utils::codebook_w4a8_linear", mutates_args=())
def turing_codebook_w4a8_linear(
    activation: torch.Tensor,
    weight: torch.Tensor,
    activation_scale: torch.Tensor,
    group_scale: torch.Tensor,
    channel_scale: torch.Tensor,
    codebook: torch.Tensor,
    bias: torch.Tensor | None = None,
    group_size: int = 16,
    chunk_rows: int = 0,
) -> torch.Tensor:
    """Grouped-codebook W4A8: codes decoded to int8 ahead of the tcgen05 GEMM.

    ``chunk_rows=0`` selects the production policy, ``-1`` forces the long-sequence
    policy (group_size 16, M > 8192), and a positive multiple of eight forces that many
    output channels per decoded chunk.
    """
    _require_cuda(activation, "Turing codebook W4A8")
    if group_scale.dtype == torch.float8_e4m3fn:
        group_scale = group_scale.view(torch.uint8)
    if group_scale.dtype != torch.uint8:
        raise TypeError("group_scale must be float8_e4m3fn or its raw uint8 view")
    return _C.turing_codebook_w4a8_linear(
        activation.contiguous(), weight.contiguous(), activation_scale.contiguous(), group_scale.contiguous(),
        channel_scale.contiguous(), codebook.contiguous(), None if bias is None else bias.contiguous(),
        group_size, chunk_rows)


@turing_codebook_w4a8_linear.register_fake
def _turing_codebook_w4a8_linear_fake(activation, weight, activation_scale, group_scale, channel_scale, codebook,
                                      bias=None, group_size=16, chunk_rows=0):
    return torch.empty((activation.size(0), weight.size(0)), dtype=torch.bfloat16, device=activation.device)


@torch.library.custom_op("turing_utils::int8_linear", mutates_args=())
def turing_int8_linear(
    activation: torch.Tensor,
    weight: torch.Tensor,
    activation_scale: torch.Tensor,
    weight_scale: torch.Tensor,
    bias: torch.Tensor | None = None,
) -> torch.Tensor:
    """W8A8 contraction with the fused dequant + bias epilogue (tcgen05 kind::i8)."""
    _require_cuda(activation, "Turing INT8 linear")
    return _C.turing_int8_linear(
        activation.contiguous(),
        weight.contiguous(),
        activation_scale.contiguous(),
        weight_scale.contiguous(),
        None if bias is None else bias.contiguous(),
    )


@turing_int8_linear.register_fake
def _turing_int8_linear_fake(activation, weight, activation_scale, weight_scale, bias=None):
    return torch.empty((activation.size(0), weight.size(0)), dtype=torch.bfloat16, device=activation.device)


@torch.library.custom_op("turing_utils::bf16_int8_convrot_quantize_b128", mutates_args=())
def turing_bf16_int8_convrot_quantize_b128(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """ConvRot int8 quantize with rotation block 128 (no reference op: the reference's
    quantizers take block 256 only; the block-128 rotation is defined in ctu_b200.h)."""
    _require_cuda(x, "block-128 ConvRot")
    return _C.bf16_int8_convrot_quantize_b128(x.contiguous())


@turing_bf16_int8_convrot_quantize_b128.register_fake
def _turing_bf16_int8_convrot_quantize_b128_fake(x):
    return (torch.empty_like(x, dtype=torch.int8),
            torch.empty((x.size(0), 1), dtype=torch.float32, device=x.device))


@torch.library.custom_op("turing_utils::convrot_int8_linear", mutates_args=())
def turing_convrot_int8_linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    weight_scale: torch.Tensor,
    bias: torch.Tensor | None = None,
    group_size: int = 256,
) -> torch.Tensor:
    """ConvRot W8A8 linear from bf16 rows (quantize + int8_linear in one call; no
    reference op: the plugin composes the two in dispatch.int8_linear, dispatch.py:748-800)."""
    _require_cuda(x, "ConvRot INT8 linear")
    return _C.convrot_int8_linear(x, weight, weight_scale, bias, group_size)


@turing_convrot_int8_linear.register_fake
def _turing_convrot_int8_linear_fake(x, weight, weight_scale, bias=None, group_size=256):
    return torch.empty((x.size(0), weight.size(0)), dtype=torch.bfloat16, device=x.device)


# ops.py:129-160
@torch.library.custom_op("turing_utils::dequantize_int8_bf16", mutates_args=())
def turing_dequantize_int8_bf16(
    accumulator: torch.Tensor,
    activation_scale: torch.Tensor,
    weight_scale: torch.Tensor,
    output_columns: int = -1,
) -> torch.Tensor:
    """Dequantize an INT32 GEMM workspace directly into bf16."""
    _require_cuda(accumulator, "Turing BF16 epilogue")
    if accumulator.dtype != torch.int32 or accumulator.ndim != 2:
        raise TypeError("accumulator must be a 2D int32 tensor")
    return _C.turing_dequantize_int8_bf16(
        accumulator.contiguous(), activation_scale.contiguous(), weight_scale.contiguous(), output_columns
    )


@turing_dequantize_int8_bf16.register_fake
def _turing_dequantize_int8_bf16_fake(accumulator, activation_scale, weight_scale, output_columns=-1):
    columns = accumulator.size(1) if output_columns < 0 else output_columns
    return torch.empty((accumulator.size(0), columns), dtype=torch.bfloat16, device=accumulator.device)


def _check_bf16_2d(x: torch.Tensor, what: str) -> None:
    if x.dtype != torch.bfloat16:
        raise TypeError(f"{what} input must be bfloat16")
    if x.ndim != 2:
        raise ValueError(f"{what} input must be 2D")


# ops.py:290-315
@torch.library.custom_op("turing_utils::bf16_int8_convrot_quantize", mutates_args=())
def turing_bf16_int8_convrot_quantize(
    x: torch.Tensor,
    group_size: int = 256,
    *,
    swiglu: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Fused ConvRot rotation + per-token int8 quantization of a bf16 row block."""
    _require_cuda(x, "BF16 row-buffer ConvRot")
    _check_bf16_2d(x, "BF16 row-buffer ConvRot")
    return _C.turing_bf16_int8_convrot_quantize(x.contiguous(), group_size, swiglu)


@turing_bf16_int8_convrot_quantize.register_fake
def _turing_bf16_int8_convrot_quantize_fake(x, group_size=256, *, swiglu=False):
    hidden = x.size(1) // 2 if swiglu else x.size(1)
    return (
        torch.empty((x.size(0), hidden), dtype=torch.int8, device=x.device),
        torch.empty((x.size(0), 1), dtype=torch.float32, device=x.device),
    )


# ops.py:318-343
@torch.library.custom_op("turing_utils::bf16_int4_convrot_quantize", mutates_args=())
def turing_bf16_int4_convrot_quantize(
    x: torch.Tensor,
    group_size: int = 256,
    *,
    swiglu: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Fused ConvRot rotation + per-token packed-int4 quantization."""
    _require_cuda(x, "BF16 row-buffer INT4 ConvRot")
    _check_bf16_2d(x, "BF16 row-buffer INT4 ConvRot")
    return _C.turing_bf16_int4_convrot_quantize(x.contiguous(), group_size, swiglu)


@turing_bf16_int4_convrot_quantize.register_fake
def _turing_bf16_int4_convrot_quantize_fake(x, group_size=256, *, swiglu=False):
    hidden = x.size(1) // 2 if swiglu else x.size(1)
    return (
        torch.empty((x.size(0), hidden // 2), dtype=torch.int8, device=x.device),
        torch.empty((x.size(0), 1), dtype=torch.float32, device=x.device),
    )


# ops.py:346-365
@torch.library.custom_op("turing_utils::bf16_gelu_int8_convrot_quantize", mutates_args=())
def turing_bf16_gelu_int8_convrot_quantize(
    x: torch.Tensor,
    group_size: int = 256,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Fused tanh-GELU + ConvRot + per-token int8 quantization."""
    _require_cuda(x, "BF16 GELU ConvRot")
    _check_bf16_2d(x, "BF16 GELU ConvRot")
    return _C.turing_bf16_gelu_int8_convrot_quantize(x.contiguous(), group_size)


@turing_bf16_gelu_int8_convrot_quantize.register_fake
def _turing_bf16_gelu_int8_convrot_quantize_fake(x, group_size=256):
    return (
        torch.empty(x.shape, dtype=torch.int8, device=x.device),
        torch.empty((x.size(0), 1), dtype=torch.float32, device=x.device),
    )


# ops.py:368-385
@torch.library.custom_op("turing_utils::bf16_gelu_int4_convrot_quantize", mutates_args=())
def turing_bf16_gelu_int4_convrot_quantize(
    x: torch.Tensor,
    group_size: int = 256,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Fused tanh-GELU + ConvRot + per-token packed-int4 quantization."""
    _require_cuda(x, "BF16 GELU INT4 ConvRot")
    _check_bf16_2d(x, "BF16 GELU INT4 ConvRot")
    return _C.turing_bf16_gelu_int4_convrot_quantize(x.contiguous(), group_size)


@turing_bf16_gelu_int4_convrot_quantize.register_fake
def _turing_bf16_gelu_int4_convrot_quantize_fake(x, group_size=256):
    return (
        torch.empty((x.size(0), x.size(1) // 2), dtype=torch.int8, device=x.device),
        torch.empty((x.size(0), 1), dtype=torch.float32, device=x.device),
    )


# ops.py:163-186, 222-287: the staged entries share the fused kernel (bf16 input).
@torch.library.custom_op("turing_utils::swiglu_int8_convrot_quantize", mutates_args=())
def turing_swiglu_int8_convrot_quantize(x: torch.Tensor, group_size: int = 256) -> tuple[torch.Tensor, torch.Tensor]:
    """SwiGLU + ConvRot int8 quantization of a [M, 2K] (gate | up) block."""
    _require_cuda(x, "Turing SwiGLU ConvRot")
    if x.ndim != 2:
        raise ValueError("SwiGLU ConvRot input must be 2D [M, 2K]")
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("SwiGLU ConvRot input must be float16 or bfloat16")
    return _C.turing_swiglu_int8_convrot_quantize(x.contiguous(), group_size)


@turing_swiglu_int8_convrot_quantize.register_fake
def _turing_swiglu_int8_convrot_quantize_fake(x, group_size=256):
    hidden = x.size(1) // 2
    return (
        torch.empty((x.size(0), hidden), dtype=torch.int8, device=x.device),
        torch.empty((x.size(0), 1), dtype=torch.float32, device=x.device),
    )


# ops.py:189-219: one channel shard quantized with precomputed whole-row scales.
@torch.library.custom_op("turing_utils::swiglu_int8_convrot_quantize_scaled", mutates_args=())
def turing_swiglu_int8_convrot_quantize_scaled(
    x: torch.Tensor,
    scales: torch.Tensor,
    group_size: int = 256,
) -> torch.Tensor:
    """Quantize a SwiGLU+ConvRot shard with precomputed whole-row scales."""
    _require_cuda(x, "scaled Turing SwiGLU ConvRot")
    if x.dtype not in (torch.float16, torch.bfloat16) or x.ndim != 2:
        raise TypeError("scaled SwiGLU ConvRot input must be 2D float16 or bfloat16")
    if scales.dtype != torch.float32 or scales.numel() != x.shape[0]:
        raise TypeError("scaled SwiGLU ConvRot requires one FP32 scale per row")
    return _C.turing_swiglu_int8_convrot_quantize_scaled(x.contiguous(), scales.contiguous(), group_size)


@turing_swiglu_int8_convrot_quantize_scaled.register_fake
def _turing_swiglu_int8_convrot_quantize_scaled_fake(x, scales, group_size=256):
    return torch.empty((x.size(0), x.size(1) // 2), dtype=torch.int8, device=x.device)


@torch.library.custom_op("turing_utils::swiglu_int4_convrot_quantize", mutates_args=())
def turing_swiglu_int4_convrot_quantize(x: torch.Tensor, group_size: int = 256) -> tuple[torch.Tensor, torch.Tensor]:
    """SwiGLU + ConvRot packed-int4 quantization of a [M, 2K] block."""
    _require_cuda(x, "Turing SwiGLU INT4 ConvRot")
    if x.ndim != 2:
        raise ValueError("SwiGLU INT4 ConvRot input must be 2D [M, 2K]")
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("SwiGLU INT4 ConvRot input must be float16 or bfloat16")
    return _C.turing_swiglu_int4_convrot_quantize(x.contiguous(), group_size)


@turing_swiglu_int4_convrot_quantize.register_fake
def _turing_swiglu_int4_convrot_quantize_fake(x, group_size=256):
    hidden = x.size(1) // 2
    return (
        torch.empty((x.size(0), hidden // 2), dtype=torch.int8, device=x.device),
        torch.empty((x.size(0), 1), dtype=torch.float32, device=x.device),
    )


@torch.library.custom_op("turing_utils::gelu_int8_convrot_quantize", mutates_args=())
def turing_gelu_int8_convrot_quantize(x: torch.Tensor, group_size: int = 256) -> tuple[torch.Tensor, torch.Tensor]:
    """tanh-GELU + ConvRot int8 quantization."""
    _require_cuda(x, "Turing GELU ConvRot")
    if x.dtype not in (torch.float16, torch.bfloat16) or x.ndim != 2:
        raise TypeError("GELU ConvRot input must be 2D float16 or bfloat16")
    return _C.turing_gelu_int8_convrot_quantize(x.contiguous(), group_size)


@turing_gelu_int8_convrot_quantize.register_fake
def _turing_gelu_int8_convrot_quantize_fake(x, group_size=256):
    return (
        torch.empty(x.shape, dtype=torch.int8, device=x.device),
        torch.empty((x.size(0), 1), dtype=torch.float32, device=x.device),
    )


@torch.library.custom_op("turing_utils::gelu_int4_convrot_quantize", mutates_args=())
def turing_gelu_int4_convrot_quantize(x: torch.Tensor, group_size: int = 256) -> tuple[torch.Tensor, torch.Tensor]:
    """tanh-GELU + ConvRot packed-int4 quantization."""
    _require_cuda(x, "Turing GELU INT4 ConvRot")
    if x.dtype not in (torch.float16, torch.bfloat16) or x.ndim != 2:
        raise TypeError("GELU INT4 ConvRot input must be 2D float16 or bfloat16")
    return _C.turing_gelu_int4_convrot_quantize(x.contiguous(), group_size)


@turing_gelu_int4_convrot_quantize.register_fake
def _turing_gelu_int4_convrot_quantize_fake(x, group_size=256):
    return (
        torch.empty((x.size(0), x.size(1) // 2), dtype=torch.int8, device=x.device),
        torch.empty((x.size(0), 1), dtype=torch.float32, device=x.device),
    )


# ops.py:388-425
@torch.library.custom_op("turing_utils::segmented_rms_adaln", mutates_args=())
def turing_segmented_rms_adaln(
    x: torch.Tensor,
    weight: torch.Tensor,
    scale: torch.Tensor,
    shift: torch.Tensor,
    segments: torch.Tensor,
    epsilon: float = 1.0e-5,
) -> torch.Tensor:
    """Fused affine RMSNorm and segmented AdaLN modulation."""
    if x.device.type != "cuda":
        raise RuntimeError("Segmented RMSNorm+AdaLN requires CUDA tensors")
    if torch.cuda.get_device_capability(x.device) < (7, 5):
        raise RuntimeError("Segmented RMSNorm+AdaLN requires sm75 or newer")
    if x.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise TypeError("segmented RMSNorm+AdaLN input must be float16, bfloat16, or float32")
    if x.ndim != 2:
        raise ValueError("segmented RMSNorm+AdaLN input must be 2D [M, K]")
    if weight.device != x.device or scale.device != x.device or shift.device != x.device:
        raise ValueError("weight, scale, and shift must be on the input device")
    weight = weight.to(dtype=x.dtype).contiguous()
    scale = scale.to(dtype=x.dtype)
    shift = shift.to(dtype=x.dtype)
    if scale.stride(-1) != 1:
        scale = scale.contiguous()
    if shift.stride(-1) != 1:
        shift = shift.contiguous()
    if segments.device != x.device or segments.dtype != torch.int32:
        raise ValueError("segments must be an int32 tensor on the input device")
    return _C.turing_segmented_rms_adaln(x.contiguous(), weight, scale, shift, segments.contiguous(), epsilon)


@turing_segmented_rms_adaln.register_fake
def _turing_segmented_rms_adaln_fake(x, weight, scale, shift, segments, epsilon=1.0e-5):
    return torch.empty_like(x)


# ops.py:432-447
@torch.library.custom_op("turing_utils::layer_norm_adaln", mutates_args=())
def turing_layer_norm_adaln(
    x: torch.Tensor,
    scale: torch.Tensor,
    shift: torch.Tensor,
    epsilon: float = 1.0e-5,
) -> torch.Tensor:
    """Fused FP32-reduction LayerNorm and Wan AdaLN modulation."""
    if x.device.type != "cuda" or torch.cuda.get_device_capability(x.device) < (7, 5):
        raise RuntimeError("LayerNorm+AdaLN requires an sm75-or-newer CUDA tensor")
    if x.dtype not in (torch.float16, torch.bfloat16, torch.float32) or x.ndim != 3:
        raise TypeError("LayerNorm+AdaLN input must be 3D float16, bfloat16, or float32")
    scale = scale.to(device=x.device, dtype=x.dtype).contiguous()
    shift = shift.to(device=x.device, dtype=x.dtype).contiguous()
    return _C.turing_layer_norm_adaln(x.contiguous(), scale, shift, epsilon)


@turing_layer_norm_adaln.register_fake
def _turing_layer_norm_adaln_fake(x, scale, shift, epsilon=1.0e-5):
    return torch.empty_like(x)


# Per-group (128 along K) formats.  No reference op carries them (the reference's W4A4
# path calls comfy-kitchen's int4_linear with 64-column weight groups, dispatch.py:876-936,
# and it has no per-group asymmetric W4A8 format); the names follow the turing_utils::
# convention and the arithmetic is documented in ctu_b200.h.
@torch.library.custom_op("turing_utils::bf16_int4_g128_convrot_quantize", mutates_args=())
def turing_bf16_int4_g128_convrot_quantize(x: torch.Tensor, group_size: int = 256) -> tuple[torch.Tensor, torch.Tensor]:
    """ConvRot rotation + int4 codes with one scale per token per 128 columns."""
    _require_cuda(x, "per-group INT4 ConvRot")
    _check_bf16_2d(x, "per-group INT4 ConvRot")
    return _C.bf16_int4_g128_convrot_quantize(x.contiguous(), group_size)


@turing_bf16_int4_g128_convrot_quantize.register_fake
def _turing_bf16_int4_g128_convrot_quantize_fake(x, group_size=256):
    return (
        torch.empty((x.size(0), x.size(1) // 2), dtype=torch.int8, device=x.device),
        torch.empty((x.size(0), x.size(1) // 128), dtype=torch.float32, device=x.device),
    )


@torch.library.custom_op("turing_utils::asym_w4a8_g128_linear", mutates_args=())
def turing_asym_w4a8_g128_linear(
    activation: torch.Tensor,
    weight: torch.Tensor,
    activation_scale: torch.Tensor,
    weight_scale: torch.Tensor,
    weight_zero: torch.Tensor,
    bias: torch.Tensor | None = None,
) -> torch.Tensor:
    """Asymmetric uint4 W4A8: fp16 scale and uint4 zero point per 128 columns of K."""
    _require_cuda(activation, "asymmetric W4A8")
    return _C.asym_w4a8_g128_linear(activation, weight, activation_scale, weight_scale, weight_zero, bias)


@turing_asym_w4a8_g128_linear.register_fake
def _turing_asym_w4a8_g128_linear_fake(activation, weight, activation_scale, weight_scale, weight_zero, bias=None):
    return torch.empty((activation.size(0), weight.size(0)), dtype=torch.bfloat16, device=activation.device)


@torch.library.custom_op("turing_utils::w4a4_g128_linear", mutates_args=())
def turing_w4a4_g128_linear(
    activation: torch.Tensor,
    weight: torch.Tensor,
    activation_scale: torch.Tensor,
    weight_scale: torch.Tensor,
    bias: torch.Tensor | None = None,
) -> torch.Tensor:
    """W4A4 with per-token-per-group-128 activation scales and fp16 per-group weight scales."""
    _require_cuda(activation, "per-group W4A4")
    return _C.w4a4_g128_linear(activation, weight, activation_scale, weight_scale, bias)


@turing_w4a4_g128_linear.register_fake
def _turing_w4a4_g128_linear_fake(activation, weight, activation_scale, weight_scale, bias=None):
    return torch.empty((activation.size(0), weight.size(0)), dtype=torch.bfloat16, device=activation.device)


# 4-bit floating point linear and affine layer norm (no reference ops; arithmetic and layouts in
# ctu_b200.h).  A single token's call is bound by host time, so these ops, their checks and their
# gradients are registered from C++ (csrc/torch_ops.cpp): 1 x 5120 x 5120 costs 17 us of host time as a
# Python op over ctypes.  Their fake kernels are here.  Where the library of bindings does not fit the installed
# torch, these ops refuse and the others, which need no such library, work.
try:
    _lib.load_torch_ops()
    _torch_ops_error = None
except _lib.KernelUnavailable as exc:
    _torch_ops_error = str(exc)


def _register_fake(name: str):
    return torch.library.register_fake(name) if _torch_ops_error is None else lambda fn: fn


def _torch_op(fn):
    """``fn``, or a refusal in its place where the bindings are not loaded."""
    if _torch_ops_error is None:
        return fn

    @functools.wraps(fn)
    def refuse(*args, **kwargs):
        raise _lib.KernelUnavailable(_torch_ops_error)

    return refuse


_FP4_FORMATS = {"nvfp4": (16, torch.float8_e4m3fn), "mxfp4": (32, torch.float8_e8m0fnu)}


@_register_fake("turing_utils::fp4_quantize")
def _fp4_quantize_fake(x, format="nvfp4", rotation=0):
    block, dtype = _FP4_FORMATS[format]
    rows, k = x.shape
    return (x.new_empty((rows, k // 2), dtype=torch.uint8),
            x.new_empty(((rows + 127) // 128, (k // block + 3) // 4, 32, 16), dtype=dtype),
            x.new_empty((rows, 1), dtype=torch.float32))


@_torch_op
def turing_fp4_quantize(x: torch.Tensor, format: str = "nvfp4", rotation: int = 0):
    """bf16/fp16 rows to 4-bit floating point: (packed codes, block scale tiles, row scales).

    ``format`` is ``"nvfp4"`` (e4m3 scale per 16 values, power-of-two row scale) or ``"mxfp4"`` (e8m0
    scale per 32 values); ``rotation=256`` applies the ConvRot rotation first."""
    return torch.ops.turing_utils.fp4_quantize.default(x, format, rotation)


@_register_fake("turing_utils::fp4_dequantize")
def _fp4_dequantize_fake(codes, block_scale, scale, out_dtype=torch.bfloat16):
    return codes.new_empty((codes.size(0), codes.size(1) * 2), dtype=out_dtype)


@_torch_op
def turing_fp4_dequantize(codes: torch.Tensor, block_scale: torch.Tensor, scale: torch.Tensor,
                          out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that FP4 codes and scales stand for (rotated values stay rotated); ``scale`` is one
    fp32 value or one per row."""
    return torch.ops.turing_utils.fp4_dequantize.default(codes, block_scale, scale, out_dtype)


@_register_fake("turing_utils::fp4_linear")
def _fp4_linear_fake(activation, weight, activation_block_scale, weight_block_scale, activation_scale, weight_scale,
                     bias=None):
    return activation.new_empty((activation.size(0), weight.size(0)), dtype=torch.bfloat16)


@_torch_op
def turing_fp4_linear(activation: torch.Tensor, weight: torch.Tensor, activation_block_scale: torch.Tensor,
                      weight_block_scale: torch.Tensor, activation_scale: torch.Tensor, weight_scale: torch.Tensor,
                      bias: torch.Tensor | None = None) -> torch.Tensor:
    """W4A4 product of two FP4 operands of one format (tcgen05 block-scaled MMA), bf16 [m, n]."""
    return torch.ops.turing_utils.fp4_linear.default(activation, weight, activation_block_scale, weight_block_scale,
                                                     activation_scale, weight_scale, bias)


@_register_fake("turing_utils::fp4_linear_grad_input")
def _fp4_linear_grad_input_fake(grad_output, weight, weight_block_scale, weight_scale, rotation=0):
    return grad_output.new_empty((grad_output.size(0), weight.size(1) * 2))


@_torch_op
def turing_fp4_linear_grad_input(grad_output: torch.Tensor, weight: torch.Tensor, weight_block_scale: torch.Tensor,
                                 weight_scale: torch.Tensor, rotation: int = 0) -> torch.Tensor:
    """Gradient with respect to the input of a linear with frozen FP4 weights: bf16 [m, k]."""
    return torch.ops.turing_utils.fp4_linear_grad_input.default(grad_output, weight, weight_block_scale, weight_scale,
                                                                rotation)


@_register_fake("turing_utils::convrot_fp4_linear")
def _convrot_fp4_linear_fake(x, weight, weight_block_scale, weight_scale, bias=None, rotation=256):
    return x.new_empty((x.size(0), weight.size(0)), dtype=torch.bfloat16)


@_torch_op
def turing_convrot_fp4_linear(x: torch.Tensor, weight: torch.Tensor, weight_block_scale: torch.Tensor,
                              weight_scale: torch.Tensor, bias: torch.Tensor | None = None,
                              rotation: int = 256) -> torch.Tensor:
    """Linear of bf16/fp16 rows with FP4 weights: the rows are rotated and quantized to the weights'
    format, then multiplied.  Differentiable in ``x`` (bf16): the quantization passes the gradient
    straight through, the weights are frozen."""
    return torch.ops.turing_utils.convrot_fp4_linear.default(x, weight, weight_block_scale, weight_scale, bias, rotation)


@_register_fake("turing_utils::layer_norm")
def _layer_norm_fake(x, weight=None, bias=None, epsilon=1.0e-5):
    rows = x.numel() // x.size(-1)
    return (torch.empty_like(x, memory_format=torch.contiguous_format), x.new_empty(rows, dtype=torch.float32),
            x.new_empty(rows, dtype=torch.float32))


@_register_fake("turing_utils::layer_norm_backward")
def _layer_norm_backward_fake(grad, x, mean, rstd, weight=None, bias=None, needs=7):
    none = x.new_empty(0)
    return (torch.empty_like(x, memory_format=torch.contiguous_format) if needs & 1 else none,
            torch.empty_like(weight) if needs & 2 and weight is not None else none,
            torch.empty_like(bias) if needs & 4 and bias is not None else none)


@_torch_op
def turing_layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                      epsilon: float = 1.0e-5) -> torch.Tensor:
    """Affine layer norm over the last dimension, differentiable in x, weight and bias.

    x is bf16, fp16 or fp32; weight and bias have its type or are fp32."""
    return torch.ops.turing_utils.layer_norm.default(x, weight, bias, epsilon)[0]


def turing_fp4_block_scale_tiles(block_scale: torch.Tensor) -> torch.Tensor:
    """Plain block scales [rows, k / block] (float8_e4m3fn or float8_e8m0fnu), as checkpoints store them,
    in the tiles that the FP4 ops read: once, when a layer is loaded."""
    if block_scale.dim() != 2 or block_scale.dtype not in (torch.float8_e4m3fn, torch.float8_e8m0fnu):
        raise RuntimeError("block scales must be 2D float8_e4m3fn or float8_e8m0fnu")
    rows, blocks = block_scale.shape
    mt, kt = (rows + 127) // 128, (blocks + 3) // 4
    full = torch.zeros((mt * 128, kt * 4), dtype=torch.uint8, device=block_scale.device)
    full[:rows, :blocks] = block_scale.view(torch.uint8)
    tiles = full.view(mt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).reshape(mt, kt, 32, 16)
    return tiles.contiguous().view(block_scale.dtype)

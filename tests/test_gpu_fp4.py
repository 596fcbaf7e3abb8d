"""4-bit floating point quantizer, dequantizer, linear and its input gradient against 64-bit definitions."""

import contextlib

import numpy as np
import pytest
import torch

import fp4_oracle as oracle

pytestmark = pytest.mark.gpu

FORMATS = ("nvfp4", "mxfp4")
HALF_BF16 = 2.0**-8  # a bf16 rounding, relative


@pytest.fixture(scope="module")
def k():
    import comfyui_turing_utils_kernel as kernel

    yield kernel
    from comfyui_turing_utils_kernel import _lib

    assert _lib.device_error(torch.cuda.current_device()) == 0


def rows_like(rows, width, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))
    x[:, :: max(1, width // 5)] *= 16
    return x.to(dtype)


def quantized(rows, width, fmt, seed, rotation=0):
    """Codes, tiles and row scales on the GPU from the oracle, and the float64 values they stand for."""
    x = rows_like(rows, width, seed)
    codes, scales, row = oracle.quantize(x.float().numpy(), fmt, rotation)
    dtype = torch.float8_e4m3fn if fmt == "nvfp4" else torch.float8_e8m0fnu
    t = torch.from_numpy(oracle.tiles(scales)).cuda().view(dtype)
    return (torch.from_numpy(codes).cuda(), t, torch.from_numpy(row).view(-1, 1).cuda()), oracle.values(codes, scales, fmt), row


def check_quantized(k, x, fmt, rotation):
    codes, tiles, row = k.turing_fp4_quantize(x.cuda() if not x.is_cuda else x, fmt, rotation)
    want_codes, want_scales, want_row = oracle.quantize(x.float().cpu().numpy(), fmt, rotation)
    np.testing.assert_array_equal(row.view(-1).cpu().numpy(), want_row)
    np.testing.assert_array_equal(tiles.view(torch.uint8).cpu().numpy(), oracle.tiles(want_scales))
    np.testing.assert_array_equal(codes.cpu().numpy(), want_codes)


# ---------------------------------------------------------------------------- quantizer
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("rows,width,rotation", [
    (1, 32, 0), (1, 256, 256), (3, 64, 0), (127, 96, 0), (129, 1568, 0), (5, 512, 256), (130, 5120, 256),
    (2, 5120, 0), (33, 13824, 256), (7, 13824, 0), (1, 16384, 256), (2, 49152, 256), (1, 49152, 0), (300, 768, 256)])
def test_quantizer_bits(k, fmt, dtype, rows, width, rotation):
    check_quantized(k, rows_like(rows, width, rows + width, dtype), fmt, rotation)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rotation", (0, 256))
def test_quantizer_edge_rows(k, fmt, rotation):
    width = 512
    x = rows_like(40, width, 7)
    x[0] = 0
    x[1] = -0.0
    x[2] = float("nan")
    x[3, 5] = float("inf")
    x[4, 300] = float("-inf")
    x[5, 17] = float("nan")
    x[6] = 1e-40  # bf16 subnormals
    x[7] = torch.finfo(torch.bfloat16).tiny
    x[8] = 3e38
    x[9, :] = 0
    x[9, 100] = 3.0e38
    x[10] = 2688.0  # the row scale's own border
    x[11] = 2704.0
    x[12] = 1e-30
    x[12, 0] = 1.0  # blocks far below the row's largest
    x[13, :256] = 0
    x[14] = 6.0
    # Every tie of the code grid, at several block scales.
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    for i in range(16):
        scale = (8 + i % 8) / 8.0 * 2.0 ** (i - 8)
        x[15 + i] = (ties * scale).repeat(width // 8).bfloat16()
        x[15 + i, 1::2] *= -1
    check_quantized(k, x, fmt, rotation)


def test_quantizer_block_scale_ties(k):
    # block amax = 6 * (a midpoint of two e4m3 values): bf16 holds it, the division must keep the tie.
    x = torch.zeros(8, 512, dtype=torch.bfloat16)
    for i in range(8):
        for b in range(32):
            x[i, 16 * b] = 6.0 * (2 * ((8 + (b % 8))) + 1) / 16.0 * 2.0 ** (i - 3)
        x[i, 511] = 2688.0
    check_quantized(k, x, "nvfp4", 0)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantizer_takes_strided_rows(k, fmt):
    x = rows_like(20, 1024, 3).cuda()
    check_quantized(k, x[::2, 256:768], fmt, 256)
    check_quantized(k, rows_like(512, 64, 4).cuda().t()[:, :256], fmt, 0)
    flat = rows_like(1, 3 * 512 + 8, 5).cuda().view(-1)
    check_quantized(k, flat[3 : 3 + 1024].view(2, 512), fmt, 256)  # rows start off a 16-byte boundary


@pytest.mark.parametrize("fmt", FORMATS)
def test_empty_rows(k, fmt):
    codes, tiles, row = k.turing_fp4_quantize(torch.empty(0, 256, dtype=torch.bfloat16, device="cuda"), fmt, 256)
    assert codes.shape == (0, 128) and row.shape == (0, 1) and tiles.shape[0] == 0
    assert k.turing_fp4_dequantize(codes, tiles, row).shape == (0, 256)
    (w, ws, wr), _, _ = quantized(24, 256, fmt, 1)
    assert k.turing_fp4_linear(codes, w, tiles, ws, row, wr).shape == (0, 24)
    assert k.turing_fp4_linear_grad_input(torch.empty(0, 24, dtype=torch.bfloat16, device="cuda"), w, ws, wr).shape == (0, 256)


# ---------------------------------------------------------------------------- dequantizer
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16, torch.float32))
@pytest.mark.parametrize("rows,width", [(1, 32), (3, 96), (129, 1568), (130, 512), (2, 13824)])
def test_dequantizer(k, fmt, dtype, rows, width):
    (codes, tiles, row), values, row_np = quantized(rows, width, fmt, rows)
    out = k.turing_fp4_dequantize(codes, tiles, row, dtype)
    want = torch.from_numpy(values * row_np[:, None].astype(np.float64)).to(dtype)  # one rounding, or none
    torch.testing.assert_close(out.cpu(), want, rtol=0, atol=0)
    scalar = k.turing_fp4_dequantize(codes, tiles, torch.full((1,), 0.25, device="cuda"), dtype)
    torch.testing.assert_close(scalar.cpu(), torch.from_numpy(values * 0.25).to(dtype), rtol=0, atol=0)


def test_every_code_and_scale_byte(k):
    for fmt, block in oracle.BLOCK.items():
        rows = 256
        width = 2 * block
        codes = np.tile(np.arange(256, dtype=np.uint8), (rows, 1))[:, :block]
        for r in range(rows):
            codes[r] = (np.arange(block) * 17 + r) % 256
        scales = np.stack([np.arange(256), np.arange(255, -1, -1)], 1).astype(np.uint8)
        dtype = torch.float8_e4m3fn if fmt == "nvfp4" else torch.float8_e8m0fnu
        t = torch.from_numpy(oracle.tiles(scales)).cuda().view(dtype)
        out = k.turing_fp4_dequantize(torch.from_numpy(codes).cuda(), t, torch.ones(1, device="cuda"), torch.float32)
        np.testing.assert_array_equal(out.cpu().numpy(), oracle.values(codes, scales, fmt).astype(np.float32))
        assert out.shape == (rows, width)


# ---------------------------------------------------------------------------- linear
@contextlib.contextmanager
def forced_kernel(which):
    from comfyui_turing_utils_kernel import _lib

    before = _lib.load().ctu_debug_set_fp4_kernel(which)
    try:
        yield
    finally:
        _lib.load().ctu_debug_set_fp4_kernel(before)


def linear_bound(av, ar, wv, wr, exact):
    """Half a bf16 step of the result, and the accumulation: at most one truncation (2^-23 of the sum of
    magnitudes) for each K = 64 instruction and each of the sums inside it, taken as eight levels,
    doubled for the products with the two fp32 scales."""
    mags = np.abs(av) @ np.abs(wv).T * np.abs(ar)[:, None] * np.abs(wr)[None, :]
    steps = -(-av.shape[1] // 64) + 8
    return HALF_BF16 * np.abs(exact) + 2 * steps * 2.0**-23 * mags + 1e-37


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,width", [
    (1, 1, 32), (1, 8, 64), (1, 5120, 5120), (2, 193, 96), (3, 64, 256), (7, 191, 288), (8, 192, 512), (9, 333, 1568),
    (16, 384, 1024), (17, 1537, 2048), (31, 129, 13824), (32, 200, 768), (33, 64, 320), (64, 500, 512), (65, 72, 416),
    (100, 1000, 1056), (127, 385, 544), (128, 128, 256), (129, 257, 512), (255, 40, 96), (256, 192, 256),
    (257, 576, 2080), (300, 1153, 800), (513, 384, 5120), (1025, 1537, 1568)])
def test_linear(k, fmt, m, n, width):
    (a, a_s, a_r), av, ar = quantized(m, width, fmt, m + n)
    (w, w_s, w_r), wv, wr = quantized(n, width, fmt, n + width)
    bias = torch.linspace(-3, 3, n, device="cuda")
    ar, wr = ar.astype(np.float64), wr.astype(np.float64)
    plain = (av @ wv.T) * ar[:, None] * wr[None, :]
    for b, which in ((None, 0), (bias, 0), (bias, 1), (None, 2), (bias, 2)):  # by size, CTA pair, few rows
        with forced_kernel(which):
            out = k.turing_fp4_linear(a, w, a_s, w_s, a_r, w_r, b)
        exact = plain if b is None else plain + b.double().cpu().numpy()[None, :]
        assert out.shape == (m, n) and out.dtype == torch.bfloat16
        off = np.abs(out.double().cpu().numpy() - exact)
        bound = linear_bound(av, ar, wv, wr, exact)
        assert (off <= bound).all(), (off / bound).max()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", (1, 40, 300))
def test_linear_scalar_weight_scale_and_nan_rows(k, fmt, m):
    (a, a_s, a_r), av, ar = quantized(m, 512, fmt, 1)
    (w, w_s, _), wv, _ = quantized(200, 512, fmt, 2)
    a_r = a_r.clone()
    a_r[m // 2] = float("nan")
    out = k.turing_fp4_linear(a, w, a_s, w_s, a_r, torch.full((1,), 0.37, device="cuda")).double().cpu().numpy()
    assert np.isnan(out[m // 2]).all()
    keep = np.arange(m) != m // 2
    scale = np.full(200, np.float32(0.37), np.float64)
    exact = (av @ wv.T) * ar[:, None].astype(np.float64) * scale[None, :]
    bound = linear_bound(av, ar.astype(np.float64), wv, scale, exact) + 2.0**-23 * np.abs(exact)
    assert (np.abs(out - exact) <= bound)[keep].all()


@pytest.mark.parametrize("m", (1, 5, 300))
def test_linear_nan_block_scales(k, m):
    # An e8m0 scale byte of 255 is NaN: its row's (or column's) outputs are, and no others.
    (a, a_s, a_r), _, _ = quantized(m, 256, "mxfp4", 1)
    (w, w_s, w_r), _, _ = quantized(200, 256, "mxfp4", 2)
    clean = k.turing_fp4_linear(a, w, a_s, w_s, a_r, w_r)
    w_s = w_s.clone()
    w_s.view(torch.uint8)[0, 1, 7, 4 * 1 + 2] = 255  # row 39, block 6
    out = k.turing_fp4_linear(a, w, a_s, w_s, a_r, w_r)
    bad = torch.isnan(out)
    assert bad[:, 39].all() and bad.sum() == m
    assert torch.equal(out[:, :39], clean[:, :39]) and torch.equal(out[:, 40:], clean[:, 40:])


@pytest.mark.parametrize("fmt", FORMATS)
def test_linear_repeats_bits_and_leaves_neighbours(k, fmt):
    for m, n, width in ((1, 300, 2048), (20, 1000, 5120), (400, 777, 512)):
        (a, a_s, a_r), _, _ = quantized(m, width, fmt, 5)
        (w, w_s, w_r), _, _ = quantized(n, width, fmt, 6)
        first = k.turing_fp4_linear(a, w, a_s, w_s, a_r, w_r)
        for _ in range(3):
            assert torch.equal(first, k.turing_fp4_linear(a, w, a_s, w_s, a_r, w_r))
        # The C entry into a buffer with a margin on both sides.
        from comfyui_turing_utils_kernel import _lib

        buf = torch.full((m * n + 64,), 7.0, dtype=torch.bfloat16, device="cuda")
        _lib.check(_lib.load().ctu_fp4_linear(
            a.data_ptr(), w.data_ptr(), a_s.data_ptr(), w_s.data_ptr(), a_r.data_ptr(), w_r.data_ptr(), n, None,
            buf.data_ptr() + 64, m, n, width, 0 if fmt == "nvfp4" else 1, torch.cuda.current_stream().cuda_stream))
        assert torch.equal(buf[32 : 32 + m * n].view(m, n), first)
        assert (buf[:32] == 7).all() and (buf[32 + m * n :] == 7).all()


# ---------------------------------------------------------------------------- input gradient
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,width,rotation", [
    (1, 8, 32, 0), (1, 64, 256, 256), (3, 200, 96, 0), (17, 1544, 512, 256), (128, 72, 288, 0), (129, 520, 768, 256),
    (257, 256, 1024, 256), (300, 1000, 1568, 0), (40, 5120, 5120, 256), (5, 13824, 512, 0)])
def test_grad_input(k, fmt, m, n, width, rotation):
    (w, w_s, w_r), wv, wr = quantized(n, width, fmt, n + width, rotation)
    g = torch.randn(m, n, generator=torch.Generator().manual_seed(m)).bfloat16()
    dx = k.turing_fp4_linear_grad_input(g.cuda(), w, w_s, w_r, rotation)
    gd, wd = g.double().numpy(), wv * wr[:, None].astype(np.float64)
    exact = gd @ wd
    # Sums: one truncation per K = 16 instruction and four levels inside; rotation: four stages of three
    # fp32 additions, of values bounded by the rotated magnitudes; up to 16 parts added; then half a bf16 step.
    mags = np.abs(gd) @ np.abs(wd)
    off = (-(-n // 16) + 4) * 2.0**-23 * mags + 16 * 2.0**-24 * mags
    if rotation:
        r = oracle.rotation_matrix()
        exact = (exact.reshape(-1, 256) @ r).reshape(m, width)
        mixed = (mags.reshape(-1, 256) @ np.abs(r)).reshape(m, width)
        off = (off.reshape(-1, 256) @ np.abs(r)).reshape(m, width) + (12 + 16) * 2.0**-24 * mixed
    assert dx.dtype == torch.bfloat16 and dx.shape == (m, width)
    got = dx.double().cpu().numpy()
    bound = HALF_BF16 * (np.abs(exact) + off) + off + 1e-37
    assert (np.abs(got - exact) <= bound).all(), (np.abs(got - exact) / bound).max()


def test_grad_input_arbitrary_channel_scales(k):
    (w, w_s, _), wv, _ = quantized(64, 256, "nvfp4", 3)
    scale = torch.rand(64, device="cuda") + 0.1
    g = torch.randn(20, 64, generator=torch.Generator().manual_seed(1)).bfloat16()
    for s in (scale, scale[:1]):
        dx = k.turing_fp4_linear_grad_input(g.cuda(), w, w_s, s).double().cpu().numpy()
        wd = wv * np.broadcast_to(s.double().cpu().numpy(), 64)[:, None]
        gd = g.double().numpy()
        exact, mags = gd @ wd, np.abs(gd) @ np.abs(wd)
        off = (HALF_BF16 + 10 * 2.0**-23) * mags  # each decoded weight rounds once
        assert (np.abs(dx - exact) <= HALF_BF16 * (np.abs(exact) + off) + off).all()


def test_gradient_is_the_adjoint_of_the_layer(k):
    """<grad, layer(d)> = <dx, d>: the layer is linear in what it multiplies, so its differences are exact."""
    m, n, width = 24, 136, 512
    (w, w_s, w_r), wv, wr = quantized(n, width, "nvfp4", 9, 256)
    g = torch.randn(m, n, generator=torch.Generator().manual_seed(2)).bfloat16()
    dx = k.turing_fp4_linear_grad_input(g.cuda(), w, w_s, w_r, 256).double().cpu().numpy()
    wd = wv * wr[:, None].astype(np.float64)
    r = oracle.rotation_matrix()
    rng = np.random.default_rng(0)
    for _ in range(8):
        d = rng.standard_normal((m, width))
        moved = (d.reshape(-1, 256) @ r).reshape(m, width) @ wd.T
        left, right = (g.double().numpy() * moved).sum(), (dx * d).sum()
        # dx carries one bf16 rounding per value.
        assert abs(left - right) <= 1.01 * HALF_BF16 * (np.abs(dx) * np.abs(d)).sum()


def test_autograd_of_the_layer(k):
    m, n, width = 37, 200, 768
    (w, w_s, w_r), _, _ = quantized(n, width, "mxfp4", 4, 256)
    x = rows_like(m, width, 1).cuda().requires_grad_(True)
    bias = torch.randn(n, device="cuda")
    y = k.turing_convrot_fp4_linear(x, w, w_s, w_r, bias, 256)
    codes, scale, row = k.turing_fp4_quantize(x.detach(), "mxfp4", 256)
    assert torch.equal(y, k.turing_fp4_linear(codes, w, scale, w_s, row, w_r, bias))
    g = torch.randn(n, m, device="cuda").bfloat16().t()  # a gradient that is not contiguous
    (dx,) = torch.autograd.grad(y, x, g)
    assert torch.equal(dx, k.turing_fp4_linear_grad_input(g.contiguous(), w, w_s, w_r, 256))
    (dx1,) = torch.autograd.grad(k.turing_convrot_fp4_linear(x, w, w_s, w_r, bias, 256).sum(), x)  # expanded gradient
    assert torch.equal(dx1, k.turing_fp4_linear_grad_input(torch.ones_like(g).contiguous(), w, w_s, w_r, 256))
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(k.turing_convrot_fp4_linear(x, w, w_s, w_r, None, 256).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="frozen"):
        k.turing_convrot_fp4_linear(x, w, w_s, w_r, bias.requires_grad_(True), 256)


# ---------------------------------------------------------------------------- streams, graphs, refusals
@pytest.mark.parametrize("m", (1, 48, 300))
def test_other_stream_and_graph(k, m):
    width, n = 1024, 520
    x = rows_like(m, width, 2).cuda()
    (w, w_s, w_r), _, _ = quantized(n, width, "nvfp4", 8, 256)
    want = k.turing_convrot_fp4_linear(x, w, w_s, w_r, None, 256)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = k.turing_convrot_fp4_linear(x, w, w_s, w_r, None, 256)
    stream.synchronize()
    assert torch.equal(got, want)
    graphs = []
    static = [x.clone(), x.clone()]
    for s in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = k.turing_convrot_fp4_linear(s, w, w_s, w_r, None, 256)
            back = k.turing_fp4_linear_grad_input(y, w, w_s, w_r, 256)
        graphs.append((graph, y, back))
    other = rows_like(m, width, 3).cuda()
    static[1].copy_(other)
    for graph, _, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    wants = [want, k.turing_convrot_fp4_linear(other, w, w_s, w_r, None, 256)]
    for (_, y, back), y0 in zip(graphs, wants):
        assert torch.equal(y, y0)
        assert torch.equal(back, k.turing_fp4_linear_grad_input(y0, w, w_s, w_r, 256))


def test_two_streams_at_once(k):
    width, n = 2048, 1000
    (w, w_s, w_r), _, _ = quantized(n, width, "nvfp4", 8)
    inputs = [quantized(m, width, "nvfp4", m)[0] for m in (1, 9, 60, 500)]
    want = [k.turing_fp4_linear(a, w, s, w_s, r, w_r) for a, s, r in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    got = [[] for _ in inputs]
    for _ in range(10):
        for i, (st, (a, s, r)) in enumerate(zip(streams, inputs)):
            with torch.cuda.stream(st):
                got[i].append(k.turing_fp4_linear(a, w, s, w_s, r, w_r))
    torch.cuda.synchronize()
    for y, ys in zip(want, got):
        assert all(torch.equal(y, z) for z in ys)


def test_refusals_on_the_gpu(k):
    (a, a_s, a_r), _, _ = quantized(4, 256, "nvfp4", 1)
    (w, w_s, w_r), _, _ = quantized(9, 256, "nvfp4", 2)
    (v, v_s, v_r), _, _ = quantized(9, 256, "mxfp4", 2)
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device="cuda")
    for call in (
        lambda: k.turing_fp4_quantize(x.float()), lambda: k.turing_fp4_quantize(x[0]),
        lambda: k.turing_fp4_quantize(x[:, :48].contiguous()), lambda: k.turing_fp4_quantize(x[:, :96], "nvfp4", 256),
        lambda: k.turing_fp4_quantize(x, "fp4"), lambda: k.turing_fp4_quantize(x, "nvfp4", 128),
        lambda: k.turing_fp4_quantize(torch.zeros(1, 49408, dtype=torch.bfloat16, device="cuda")),
        lambda: k.turing_fp4_linear(a, v, a_s, v_s, a_r, v_r),
        lambda: k.turing_fp4_linear(a, w, a_s[:, :2], w_s, a_r, w_r),
        lambda: k.turing_fp4_linear(a, w[:, :64], a_s, w_s, a_r, w_r),
        lambda: k.turing_fp4_linear(a, w, a_s, w_s, a_r[:2], w_r),
        lambda: k.turing_fp4_linear(a, w, a_s, w_s, a_r, w_r.double()),
        lambda: k.turing_fp4_linear(a, w, a_s, w_s, a_r, w_r, torch.zeros(8, device="cuda")),
        lambda: k.turing_fp4_linear(a, w, a_s, w_s, a_r, w_r.requires_grad_(True)),
        lambda: k.turing_fp4_linear_grad_input(torch.zeros(4, 9, dtype=torch.bfloat16, device="cuda"), w, w_s, v_r),
        lambda: k.turing_fp4_linear_grad_input(torch.zeros(4, 8, dtype=torch.bfloat16, device="cuda"), w, w_s, v_r),
        lambda: k.turing_fp4_dequantize(a, a_s, a_r, torch.float64),
        lambda: k.turing_fp4_dequantize(a.view(torch.int8), a_s, a_r),
        lambda: k.turing_fp4_dequantize(a, a_s.view(torch.uint8), a_r),
    ):
        with pytest.raises(RuntimeError):
            call()


# ---------------------------------------------------------------------------- together
@pytest.mark.parametrize("m", (1, 70, 300))
def test_norm_linear_and_their_gradients_together(k, m):
    """An adapter-tuning step through frozen weights: affine norm, rotated 4-bit linear, gradients of the
    norm's input and parameters, against the formulas in 64 bits from the values that the layers hold."""
    from comfyui_turing_utils_b200 import dispatch, fusions

    width, n = 768, 200
    norm = torch.nn.LayerNorm(width).cuda()  # fp32 master parameters
    with torch.no_grad():
        norm.weight.add_(0.1 * torch.randn(width, device="cuda", generator=torch.Generator("cuda").manual_seed(1)))
        norm.bias.add_(0.1 * torch.randn(width, device="cuda", generator=torch.Generator("cuda").manual_seed(2)))
    x = rows_like(m, width, 3).cuda().view(1, m, width).requires_grad_(True)
    (w, w_s, w_r), wv, wr = quantized(n, width, "nvfp4", 4, 256)
    h = fusions.affine_layer_norm(norm, x)
    h.retain_grad()
    y = dispatch.convrot_fp4_linear(h, w, w_s, w_r)
    g = torch.randn(1, m, n, device="cuda", generator=torch.Generator("cuda").manual_seed(5)).bfloat16()
    y.backward(g)
    # The product of what the quantizer holds of h.
    codes, scales, row = oracle.quantize(h.detach().view(m, width).float().cpu().numpy(), "nvfp4", 256)
    av, ar, wr = oracle.values(codes, scales, "nvfp4"), row.astype(np.float64), wr.astype(np.float64)
    exact = (av @ wv.T) * ar[:, None] * wr[None, :]
    off = np.abs(y.detach().view(m, n).double().cpu().numpy() - exact)
    assert (off <= linear_bound(av, ar, wv, wr, exact)).all()
    # Its input gradient, then the norm's backward pass from the bf16 gradient that reaches it.
    gd, wd, r = g.view(m, n).double().cpu().numpy(), wv * wr[:, None], oracle.rotation_matrix()
    mags = (np.abs(gd) @ np.abs(wd)).reshape(-1, 256) @ np.abs(r)
    dh = ((gd @ wd).reshape(-1, 256) @ r).reshape(m, width)
    got = h.grad.view(m, width).double().cpu().numpy()
    slack = (-(-n // 16) + 32) * 2.0**-23 * mags.reshape(m, width)
    assert (np.abs(got - dh) <= HALF_BF16 * (np.abs(dh) + slack) + slack).all()
    xd = x.detach().view(m, width).double().cpu().numpy()
    mean, var = xd.mean(1, keepdims=True), xd.var(1, keepdims=True)
    rstd = 1 / np.sqrt(var + norm.eps)
    n_ = (xd - mean) * rstd
    gw = got * norm.weight.detach().double().cpu().numpy()
    dx = rstd * (gw - gw.mean(1, keepdims=True) - n_ * (gw * n_).mean(1, keepdims=True))
    # fp32 statistics: under 2^-18 of the terms' magnitudes (768 terms, sums at most 40 deep), and a bf16 step.
    terms = rstd * (np.abs(gw) + np.abs(gw).mean(1, keepdims=True) + np.abs(n_) * (np.abs(gw * n_)).mean(1, keepdims=True))
    assert (np.abs(x.grad.view(m, width).double().cpu().numpy() - dx) <= HALF_BF16 * np.abs(dx) + 2.0**-16 * terms).all()
    for grad, want, size in ((norm.weight.grad, (got * n_).sum(0), np.abs(got * n_).sum(0)), (norm.bias.grad, got.sum(0), np.abs(got).sum(0))):
        assert (np.abs(grad.double().cpu().numpy() - want) <= 2.0**-16 * size + 1e-30).all()


def test_captured_training_step(k):
    """Forward and backward captured together, replayed on other data."""
    m, n, width = 64, 256, 512
    (w, w_s, w_r), _, _ = quantized(n, width, "mxfp4", 6, 256)
    weight, bias = (torch.randn(width, device="cuda").requires_grad_(True) for _ in range(2))
    g = torch.randn(m, n, device="cuda").bfloat16()

    def step(x):
        h = k.turing_layer_norm(x, weight, bias)
        y = k.turing_convrot_fp4_linear(h, w, w_s, w_r, None, 256)
        return (y.detach(), *torch.autograd.grad(y, (x, weight, bias), g))

    first, second = (rows_like(m, width, s).cuda() for s in (1, 2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(first.clone().requires_grad_(True))
    torch.cuda.current_stream().wait_stream(side)
    static = first.clone().requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for data in (second, first):
        with torch.no_grad():
            static.copy_(data)
        graph.replay()
        torch.cuda.synchronize()
        want = step(data.clone().requires_grad_(True))
        assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_long_offsets(k):
    """Rows whose elements lie beyond 2^31: the last ones come out as they do alone."""
    width, rows = 13824, 156000  # 2.16e9 values
    x = torch.zeros((rows, width), dtype=torch.bfloat16, device="cuda")
    tail = rows_like(200, width, 1).cuda()
    x[-200:] = tail
    codes, tiles, row = k.turing_fp4_quantize(x, "nvfp4", 256)
    some, _, some_row = k.turing_fp4_quantize(tail, "nvfp4", 256)
    assert torch.equal(codes[-200:], some) and torch.equal(row[-200:], some_row)
    (w, w_s, w_r), _, _ = quantized(40, width, "nvfp4", 2, 256)
    y = k.turing_convrot_fp4_linear(x, w, w_s, w_r)
    # The reference takes the same product kernel, over enough rows of it.
    assert torch.equal(y[-200:], k.turing_convrot_fp4_linear(x[-1000:], w, w_s, w_r)[-200:])
    back = k.turing_fp4_dequantize(codes, tiles, row)
    del x, codes, tiles
    last = k.turing_fp4_quantize(tail, "nvfp4", 256)
    assert torch.equal(back[-200:], k.turing_fp4_dequantize(*last))
    del back
    z = torch.zeros((rows, width), dtype=torch.bfloat16, device="cuda")
    z[-200:] = tail
    assert torch.equal(k.turing_layer_norm(z)[-200:], k.turing_layer_norm(tail))


def test_calls_from_a_fresh_thread(k):
    """A thread that has made no CUDA call yet, its outputs served from the allocator's cache."""
    import threading

    (a, a_s, a_r), _, _ = quantized(300, 512, "nvfp4", 1)
    (w, w_s, w_r), _, _ = quantized(256, 512, "nvfp4", 2)
    x = rows_like(300, 512, 3).cuda()
    g = torch.randn(300, 256, device="cuda").bfloat16()
    calls = [lambda: k.turing_fp4_linear(a, w, a_s, w_s, a_r, w_r), lambda: k.turing_fp4_linear(a[:3], w, a_s[:1], w_s, a_r[:3], w_r),
             lambda: k.turing_fp4_quantize(x, "mxfp4", 256)[0], lambda: k.turing_fp4_linear_grad_input(g, w, w_s, w_r, 256)]
    want = [f() for f in calls]
    for f in calls:
        f()  # leaves blocks of the sizes in the cache
    torch.cuda.synchronize()
    for f, y in zip(calls, want):
        got = []
        t = threading.Thread(target=lambda: got.append(f()))  # noqa: B023
        t.start()
        t.join()
        assert len(got) == 1 and torch.equal(got[0], y)


def test_ops_trace_and_compile(k):
    """Fake kernels, autograd registration and traced gradients agree with the ops; a compiled layer gives
    the eager one's bits."""
    from torch.library import opcheck

    ops = torch.ops.turing_utils
    (w, w_s, w_r), _, _ = quantized(64, 512, "nvfp4", 1, 256)
    x = rows_like(40, 512, 2).cuda()
    codes, scale, row = k.turing_fp4_quantize(x, "nvfp4", 256)
    leaf = x.clone().requires_grad_(True)
    weight, bias = (torch.randn(512, device="cuda").requires_grad_(True) for _ in range(2))
    stats = torch.zeros(40, device="cuda"), torch.ones(40, device="cuda")
    checks = ("test_autograd_registration", "test_faketensor", "test_aot_dispatch_dynamic")
    for op, args in ((ops.fp4_quantize, (x, "nvfp4", 256)), (ops.fp4_dequantize, (codes, scale, row)),
                     (ops.fp4_linear, (codes, w, scale, w_s, row, w_r)),
                     (ops.fp4_linear_grad_input, (torch.randn(40, 64, device="cuda").bfloat16(), w, w_s, w_r, 256)),
                     (ops.convrot_fp4_linear, (leaf, w, w_s, w_r)), (ops.layer_norm, (leaf, weight, bias)),
                     (ops.layer_norm, (leaf, None, bias)),
                     (ops.layer_norm_backward, (x, x, *stats, weight.detach(), bias.detach(), 7))):
        opcheck(op.default, args, test_utils=checks)

    def layer(x, weight, bias):
        return k.turing_convrot_fp4_linear(k.turing_layer_norm(x, weight, bias), w, w_s, w_r).float().square().sum()

    leaves = (leaf, weight, bias)
    eager = torch.autograd.grad(layer(*leaves), leaves)
    compiled = torch.autograd.grad(torch.compile(layer, backend="aot_eager", fullgraph=True)(*leaves), leaves)
    assert all(torch.equal(p, q) for p, q in zip(eager, compiled))


@pytest.mark.parametrize("m,n,width,rotation", [(16, 2048, 512, 256), (333, 4096, 768, 0), (1300, 1024, 4096, 256)])
def test_gradient_repeats_bits(k, m, n, width, rotation):
    """Split sums are joined in a fixed order; rows beyond the gradient's stay as they were."""
    from comfyui_turing_utils_kernel import _lib

    (w, w_s, w_r), _, _ = quantized(n, width, "mxfp4", 3, rotation)
    g = torch.randn(m, n, device="cuda").bfloat16()
    first = k.turing_fp4_linear_grad_input(g, w, w_s, w_r, rotation)
    for _ in range(3):
        assert torch.equal(first, k.turing_fp4_linear_grad_input(g, w, w_s, w_r, rotation))
    lib = _lib.load()
    buf = torch.full((m + 2, width), 7.0, dtype=torch.bfloat16, device="cuda")
    room = lib.ctu_fp4_grad_workspace_bytes(m, n, width)
    work = torch.full((room + 256,), 9, dtype=torch.uint8, device="cuda")
    _lib.check(lib.ctu_fp4_linear_grad_input(
        g.data_ptr(), w.data_ptr(), w_s.data_ptr(), w_r.data_ptr(), n, rotation, work.data_ptr(), buf[1:].data_ptr(), m, n,
        width, 1, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(buf[1 : 1 + m], first) and (buf[0] == 7).all() and (buf[-1] == 7).all()
    assert (work[room:] == 9).all()


# ---------------------------------------------------------------------------- more tiles than pairs
def random_operand(k, rows, width, fmt, seed):
    """Codes, tiles and row scales drawn as bytes on the GPU, and the values that they stand for (float64,
    there too): sizes for which the oracle on the host takes too long."""
    g = torch.Generator("cuda").manual_seed(seed)
    low, high, dtype = (48, 73, torch.float8_e4m3fn) if fmt == "nvfp4" else (124, 130, torch.float8_e8m0fnu)
    codes = torch.randint(0, 256, (rows, width // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.randint(low, high, (rows, width // oracle.BLOCK[fmt]), generator=g, device="cuda", dtype=torch.uint8)
    row = torch.exp2(torch.randint(-6, -3, (rows, 1), generator=g, device="cuda").float())
    grid = torch.from_numpy(np.concatenate((oracle.GRID, -oracle.GRID))).cuda()
    v = grid[torch.stack((codes & 15, codes >> 4), 2).view(rows, width).int()]
    v = v * torch.from_numpy(oracle.scale_values(fmt)).cuda()[scales.int()].repeat_interleave(oracle.BLOCK[fmt], 1)
    return (codes, k.turing_fp4_block_scale_tiles(scales.view(dtype)), row), v * row.double()


def rotate64(v):
    r = torch.from_numpy(oracle.rotation_matrix()).to(v.device)
    return (v.view(-1, 256) @ r).view(v.shape), r.abs()


# A B200 runs 74 CTA pairs: each takes three to four tiles here, so both accumulators, the tensor-memory columns that they
# share and the ring's phase go from tile to tile.  By size: output rows on 16 bytes (tile stores) or not, K from
# 4096 on (four epilogue warps, on 16 bytes) or below (eight), one stage a tile, last tiles that end inside.
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,width", [(3850, 3976, 4128), (3850, 3975, 4128), (3850, 3976, 544), (3850, 3973, 544),
                                       (4096, 4096, 256), (57100, 248, 4096), (200, 75000, 1056)])
def test_linear_of_several_tiles_a_pair(k, fmt, m, n, width):
    (a, a_s, a_r), av = random_operand(k, m, width, fmt, m + n)
    (w, w_s, w_r), wv = random_operand(k, n, width, fmt, n + width)
    bias = torch.linspace(-30, 30, n, device="cuda")
    out = k.turing_fp4_linear(a, w, a_s, w_s, a_r, w_r, bias)
    exact = av @ wv.t() + bias.double()
    # linear_bound's, over the whole output.
    steps = -(-width // 64) + 8
    bound = HALF_BF16 * exact.abs() + 2 * steps * 2.0**-23 * (av.abs() @ wv.t().abs()) + 1e-37
    worst = ((out.double() - exact).abs() / bound).max().item()
    assert worst <= 1, worst
    assert torch.equal(out, k.turing_fp4_linear(a, w, a_s, w_s, a_r, w_r, bias))


# More work items than pairs: tiles of several rounds without a split, and whole tiles beside the parts of the last
# round's, whose sums a second kernel joins; rows, columns and sums that end inside a tile.
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,width,rotation,mixed", [(4700, 1000, 4352, 256, False), (4790, 520, 4000, 0, False),
                                                      (2450, 5000, 2080, 0, True), (2300, 4104, 2304, 256, True),
                                                      (4096, 5120, 5120, 256, True)])
def test_gradient_of_several_items_a_pair(k, fmt, m, n, width, rotation, mixed):
    from comfyui_turing_utils_kernel import _lib

    tiles = -(-m // 256) * -(-width // 256)
    parts = (_lib.load().ctu_fp4_grad_workspace_bytes(m, n, width) - 2 * n * width) // (256 * 256 * 4)
    assert tiles > 74 and (parts > tiles % 74 if mixed else parts == 0)
    (w, w_s, w_r), wd = random_operand(k, n, width, fmt, n + width)
    g = torch.randn(m, n, device="cuda", generator=torch.Generator("cuda").manual_seed(m)).bfloat16()
    dx = k.turing_fp4_linear_grad_input(g, w, w_s, w_r, rotation)
    exact, mags = g.double() @ wd, g.double().abs() @ wd.abs()
    # As in test_grad_input.
    off = (-(-n // 16) + 4) * 2.0**-23 * mags + 16 * 2.0**-24 * mags
    if rotation:
        exact, r = rotate64(exact)
        off = (off.view(-1, 256) @ r).view(off.shape) + (12 + 16) * 2.0**-24 * (mags.view(-1, 256) @ r).view(off.shape)
    bound = HALF_BF16 * (exact.abs() + off) + off + 1e-37
    worst = ((dx.double() - exact).abs() / bound).max().item()
    assert worst <= 1, worst
    assert torch.equal(dx, k.turing_fp4_linear_grad_input(g, w, w_s, w_r, rotation))


# ---------------------------------------------------------------------------- every block scale's division
def test_quantizer_every_block_scale(k):
    """All 126 positive e4m3 scales as divisors: of bf16 values on and beside every border of the code grid, and of
    rotated, so fp32, values."""
    values = oracle.e4m3_values()[1:127]
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    x = torch.zeros(127, 64, dtype=torch.bfloat16)
    for i, s in enumerate(values):
        on = (borders * float(s)).bfloat16()  # four bits of scale, three of border: exact
        off = torch.where(torch.arange(7) % 2 == i % 2, 1, -1).to(torch.int16)
        beside = (on.view(torch.int16) + off).view(torch.bfloat16)
        x[i, :16] = torch.cat((torch.tensor([6.0 * s]).bfloat16(), on, beside, -on[:1]))
        x[i, 63] = 2688.0  # row scale 1
    _, scales, row = oracle.quantize(x[:126].float().numpy(), "nvfp4", 0)
    assert (scales[:, 0] == np.arange(1, 127)).all() and (row == 1).all()
    check_quantized(k, x, "nvfp4", 0)
    # Groups of 256 columns below the row's largest by up to 2^18, so that their scales are all of them.
    g = torch.Generator().manual_seed(11)
    y = torch.randn(400, 20, 256, generator=g) * torch.exp2(-18 * torch.rand(400, 20, 1, generator=g))
    y = y.view(400, -1).bfloat16()
    _, scales, _ = oracle.quantize(y.float().numpy(), "nvfp4", 256)
    assert set(range(1, 127)) <= set(np.unique(scales).tolist())
    check_quantized(k, y, "nvfp4", 256)

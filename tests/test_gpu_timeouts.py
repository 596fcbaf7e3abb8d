"""Failure path of the 4-bit and layer norm kernels, without a GPU fault: one wait of the first CTA for a copy is on a
barrier that nothing arrives on and runs out after a short limit.  The kernel stops, raises its flag in the device
error word and leaves no finite result that hangs on that copy; the next call is whole again."""

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
def timeout(which):
    """The wait runs out in here; on the way out the error word must tell of it, and is cleared."""
    from comfyui_turing_utils_kernel import _lib

    device = torch.cuda.current_device()
    assert _lib.device_error(device) == 0
    _lib.check(_lib.load().ctu_debug_inject_timeout(which, 30_000_000))
    try:
        yield
        torch.cuda.synchronize()
    finally:
        _lib.load().ctu_debug_inject_timeout(-1, 0)
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
        with timeout(which):
            cut = call()
        # The first cluster has the first strip of 128 weight rows, for the first tokens; nothing else is lost.
        assert torch.isnan(cut[:, :128]).all()
        assert torch.equal(cut[:, 128:], whole[:, 128:])
        assert torch.equal(call(), whole)
    finally:
        lib.ctu_debug_set_fp4_kernel(before)


# ---------------------------------------------------------------------------- rotating quantizer
@pytest.mark.parametrize("fmt", ("nvfp4", "mxfp4"))
# Several rows a warp, a row a warp, two rows a CTA of several warps, a row a CTA; the first wait and a later one.
@pytest.mark.parametrize("rows,width,which", [(70000, 256, 1), (20000, 1280, 2), (9, 2048, 0), (3000, 5120, 1), (1000, 13824, 1),
                                              (5, 49152, 0)])
def test_rotating_quantizer(k, lib, fmt, rows, width, which):
    x = torch.randn(rows, width, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).bfloat16()
    room = lib.ctu_fp4_block_scale_bytes(rows, width, 0 if fmt == "nvfp4" else 1)

    def call():
        codes = torch.full((rows, width // 2), 171, dtype=torch.uint8, device="cuda")
        scales = torch.full((room,), 171, dtype=torch.uint8, device="cuda")
        row = torch.full((rows,), UNTOUCHED, device="cuda")
        check(lib.ctu_fp4_quantize(x.data_ptr(), rows, width, 0, 0 if fmt == "nvfp4" else 1, 256, codes.data_ptr(),
                                   scales.data_ptr(), row.data_ptr(), stream()))
        # A row's block scales, [rows, blocks], out of the tiles.
        blocks = width // (16 if fmt == "nvfp4" else 32)
        plain = scales.view(-(-rows // 128), -1, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-(-rows // 128) * 128, -1)
        return codes, plain[:rows, :blocks], row

    whole = call()
    with timeout(which):
        cut = call()
    # Each row is as it should be, or comes out as a row with a NaN does: those of the first CTA's rows that the warp has a
    # part of, from that wait on.
    same = torch.stack([(p == q).view(rows, -1).all(1) for p, q in zip(whole, cut)])
    lost = torch.stack([(cut[0] == 0).all(1), (cut[1] == 0).all(1), torch.isnan(cut[2])])
    done, lost = same.all(0), lost.all(0)
    assert (done ^ lost).all() and lost.any() and 100 * lost.sum() <= max(rows, 2500)
    assert bool(lost[0]) == (which == 0)
    assert all(torch.equal(p, q) for p, q in zip(call(), whole))


# ---------------------------------------------------------------------------- layer norm, backward pass
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
# Sixteen teams a CTA, four or two, one; on and off 16 bytes; rows two deep, and (the last, fp32) one deep.
@pytest.mark.parametrize("rows,hidden,which", [(9000, 320, 1), (5000, 641, 2), (3000, 2560, 0), (2000, 5121, 1), (700, 10240, 2),
                                               (450, 10244, 1)])
def test_layer_norm_backward(k, lib, dtype, rows, hidden, which):
    from test_gpu_layer_norm import formulas, make

    x, w, b, dy = make(rows, hidden, dtype, torch.float32, rows)
    f = formulas(x, w, b, dy)
    mean, rstd = f["mean"].float().view(-1), f["rstd"].float().view(-1)
    room = lib.ctu_layer_norm_backward_workspace_bytes(rows, hidden)

    def call():
        dx = torch.full_like(x, UNTOUCHED)
        dw, db = torch.full_like(w, UNTOUCHED), torch.full_like(b, UNTOUCHED)
        work = torch.full((room // 4,), UNTOUCHED, device="cuda")
        kind = {torch.bfloat16: 0, torch.float32: 2}[dtype]
        check(lib.ctu_layer_norm_backward(dy.data_ptr(), x.data_ptr(), w.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                                          dx.data_ptr(), dw.data_ptr(), db.data_ptr(), work.data_ptr(), rows, hidden, kind, 2,
                                          stream()))
        return dx, dw, db

    whole = call()
    with timeout(which):
        dx, dw, db = call()
    # The first team's rows from that wait on, and every column's sums.
    done, lost = (dx == whole[0]).all(1), torch.isnan(dx).all(1)
    assert (done ^ lost).all() and lost.any() and 20 * lost.sum() <= rows
    assert bool(lost[0]) == (which == 0)
    assert torch.isnan(dw).all() and torch.isnan(db).all()
    assert all(torch.equal(p, q) for p, q in zip(call(), whole))


# ---------------------------------------------------------------------------- CTA pairs: product and gradient
def lost_tiles(whole, cut, along_rows):
    """Numbers of the 256 x 256 tiles that are NaN, counted along rows or down columns; the others have their bits."""
    (m, n), found = whole.shape, []
    rows, cols = -(-m // 256), -(-n // 256)
    for i in range(rows):
        for j in range(cols):
            at = (slice(256 * i, 256 * i + 256), slice(256 * j, 256 * j + 256))
            if torch.isnan(cut[at]).all():
                found.append(i * cols + j if along_rows else j * rows + i)
            else:
                assert torch.equal(cut[at], whole[at])
    return sorted(found)


@pytest.mark.parametrize("fmt", ("nvfp4", "mxfp4"))
# One tile a pair; several, lost in the second one, with eight epilogue warps, with own stores, and with four warps.
@pytest.mark.parametrize("m,n,width,which", [(300, 1153, 800, 0), (3850, 3976, 544, 4), (3850, 3973, 544, 3),
                                             (3850, 3976, 4128, 20)])
def test_pair_product(k, lib, fmt, m, n, width, which):
    (a, a_s, a_r), _ = random_operand(k, m, width, fmt, 1)
    (w, w_s, w_r), _ = random_operand(k, n, width, fmt, 2)

    def call():
        return k.turing_fp4_linear(a, w, a_s, w_s, a_r, w_r)

    whole = call()
    with timeout(which):
        cut = call()
    lost = lost_tiles(whole, cut, True)
    if which < -(-width // 256):
        assert lost == [0]
    else:  # the first pair's tiles from the second on
        assert lost and lost[0] >= 60 and lost == [lost[0] * (i + 1) for i in range(len(lost))]
    assert torch.equal(call(), whole)


@pytest.mark.parametrize("fmt", ("nvfp4", "mxfp4"))
# Every tile split; several whole tiles a pair, lost in the second one; a whole tile and a part of a split one.
@pytest.mark.parametrize("m,n,width,rotation,which,lost", [(40, 5120, 5120, 256, 2, [0]), (4700, 1000, 4352, 256, 20, [74, 148, 222, 296]),
                                                           (2450, 5000, 2080, 0, 3, [0, 74])])
def test_pair_gradient(k, lib, fmt, m, n, width, rotation, which, lost):
    (w, w_s, w_r), _ = random_operand(k, n, width, fmt, 2)
    g = torch.randn(m, n, device="cuda", generator=torch.Generator("cuda").manual_seed(m)).bfloat16()

    def call():
        return k.turing_fp4_linear_grad_input(g, w, w_s, w_r, rotation)

    whole = call()
    with timeout(which):
        cut = call()
    assert lost_tiles(whole, cut, False) == lost
    assert torch.equal(call(), whole)

"""Affine layer norm, forward and backward, against 64-bit formulas and differences."""

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 1.0e-5
U = 2.0**-24


@pytest.fixture(scope="module")
def k():
    import comfyui_turing_utils_kernel as kernel

    return kernel


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(rows, hidden, dtype, wdtype, seed=0, shift=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, hidden, generator=g) * torch.exp(torch.randn(rows, 1, generator=g)) + shift).to(dtype)
    w = (1 + 0.2 * torch.randn(hidden, generator=g)).to(wdtype)
    b = (0.3 * torch.randn(hidden, generator=g)).to(wdtype)
    dy = torch.randn(rows, hidden, generator=g).to(dtype)
    return [t.cuda() for t in (x, w, b, dy)]


def formulas(x, w, b, dy):
    x, dy = x.double(), dy.double()
    w = torch.ones(x.size(1), dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + EPS)
    xhat = (x - mean) * rstd
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return dict(y=xhat * w + b, dx=dx, dw=(dy * xhat).sum(0), db=dy.sum(0), mean=mean, rstd=rstd, xhat=xhat, g=g, w=w, b=b)


def check(out, grads, x, w, b, dy):
    """Bounds: sums of h terms run at most h / 128 + 32 deep, so they are off by that many 2^-24 of the
    sum of magnitudes; the rest is a handful of roundings, and one to the storage type."""
    f = formulas(x, w, b, dy)
    rows, h = x.shape
    c = (h / 128 + 32) * U
    xd = x.double()
    far = xd.abs().mean(1, keepdim=True) + xd.abs()  # what the mean's and the difference's errors are relative to
    xhat_off = c * (far * f["rstd"] + 2 * f["xhat"].abs())
    y_off = xhat_off * f["w"].abs() + 4 * U * (f["xhat"] * f["w"]).abs() + U * f["b"].abs()
    limit = y_off + half_step(out.dtype) * (f["y"].abs() + y_off) + 1e-30
    assert ((out.double() - f["y"]).abs() <= limit).all()
    if grads is None:
        return
    dx, dw, db = grads
    if dx is not None:
        g, n = f["g"].abs(), f["xhat"].abs()
        s2 = (g * n).mean(1, keepdim=True)
        s2_off = c * s2 + (g * xhat_off).mean(1, keepdim=True)
        off = f["rstd"] * (8 * U * g + 2 * c * g.mean(1, keepdim=True) + n * s2_off + (xhat_off + 4 * U * n) * s2)
        off = off + (c + 4 * U) * f["dx"].abs() + f["dx"].abs() * c * (far * f["rstd"]).mean(1, keepdim=True)
        limit = off + half_step(dx.dtype) * (f["dx"].abs() + off) + 1e-30
        assert ((dx.double() - f["dx"]).abs() <= limit).all(), ((dx.double() - f["dx"]).abs() / limit).max()
    depth = (rows / 64 + 64 + 32) * U
    dyd = dy.double().abs()
    if dw is not None:
        off = depth * (dyd * f["xhat"].abs()).sum(0) + (dyd * (xhat_off + 2 * U * f["xhat"].abs())).sum(0)
        assert ((dw.double() - f["dw"]).abs() <= off + half_step(dw.dtype) * (f["dw"].abs() + off) + 1e-30).all()
    if db is not None:
        off = depth * dyd.sum(0)
        assert ((db.double() - f["db"]).abs() <= off + half_step(db.dtype) * (f["db"].abs() + off) + 1e-30).all()


SHAPES = [(1, 1), (1, 7), (3, 2), (5, 8), (2, 33), (64, 64), (33, 255), (7, 256), (130, 257), (9, 1000), (200, 1536),
          (31, 1537), (65, 5120), (300, 5120), (4, 5376), (17, 8192), (3, 8200), (5, 13824), (2, 13825), (2, 40000), (1000, 96)]
TYPES = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
         (torch.float16, torch.float32), (torch.float32, torch.float32)]


@pytest.mark.parametrize("dtype,wdtype", TYPES)
@pytest.mark.parametrize("rows,hidden", SHAPES)
def test_forward_and_backward(k, rows, hidden, dtype, wdtype):
    x, w, b, dy = make(rows, hidden, dtype, wdtype, rows + hidden)
    for t in (x, w, b):
        t.requires_grad_(True)
    y = k.turing_layer_norm(x, w, b, EPS)
    grads = torch.autograd.grad(y, (x, w, b), dy)
    assert y.dtype == dtype and grads[0].dtype == dtype and grads[1].dtype == wdtype and grads[2].dtype == wdtype
    check(y.detach(), grads, x.detach(), w.detach(), b.detach(), dy)


@pytest.mark.parametrize("hidden", (48, 1537, 5120))
def test_optional_parameters_and_needs(k, hidden):
    x, w, b, dy = make(70, hidden, torch.bfloat16, torch.float32, 1)
    for weight, bias in ((None, None), (w, None), (None, b)):
        leaves = [t for t in (x, weight, bias) if t is not None]
        for t in leaves:
            t.requires_grad_(True)
        y = k.turing_layer_norm(x, weight, bias, EPS)
        got = iter(torch.autograd.grad(y, leaves, dy))
        full = [next(got), next(got) if weight is not None else None, next(got) if bias is not None else None]
        check(y.detach(), full, *(None if t is None else t.detach() for t in (x, weight, bias)), dy)
    # Any one gradient alone has the bits that it has among the others.
    y = k.turing_layer_norm(x, w, b, EPS)
    all_of = torch.autograd.grad(y, (x, w, b), dy, retain_graph=True)
    for i, leaf in enumerate((x, w, b)):
        others = [t.detach() for t in (x, w, b)]
        others[i] = leaf
        alone = torch.autograd.grad(k.turing_layer_norm(*others, EPS), leaf, dy)[0]
        assert torch.equal(alone, all_of[i])


def test_values_that_cancel_and_extremes(k):
    x, w, b, dy = make(40, 1024, torch.float32, torch.float32, 3, shift=100.0)
    x[0] = 5.0  # no variance
    x[1] = 0.0
    x[2] *= 1e-20
    x[3] *= 1e15
    x[4, 7] = 1e6
    for t in (x, w, b):
        t.requires_grad_(True)
    y = k.turing_layer_norm(x, w, b, EPS)
    check(y.detach(), torch.autograd.grad(y, (x, w, b), dy), x.detach(), w.detach(), b.detach(), dy)


def test_not_finite_rows_stay_alone(k):
    x, w, b, dy = make(12, 640, torch.bfloat16, torch.bfloat16, 4)
    clean = k.turing_layer_norm(x, w, b, EPS)
    x[3, 5], x[7, 600] = float("nan"), float("inf")
    y = k.turing_layer_norm(x, w, b, EPS)
    bad = torch.isnan(y).all(1)
    assert bad.tolist() == [i in (3, 7) for i in range(12)]
    keep = [i for i in range(12) if i not in (3, 7)]
    assert torch.equal(y[keep], clean[keep])


def test_differences(k):
    """Central differences of the fp32 kernel's own forward pass along random directions."""
    x, w, b, dy = make(6, 96, torch.float32, torch.float32, 5)
    for t in (x, w, b):
        t.requires_grad_(True)
    grads = torch.autograd.grad(k.turing_layer_norm(x, w, b, EPS), (x, w, b), dy)
    g = torch.Generator(device="cuda").manual_seed(1)
    loss = lambda *p: (k.turing_layer_norm(*p, EPS).double() * dy.double()).sum()  # noqa: E731
    with torch.no_grad():
        scale = (1.0 / formulas(x, w, b, dy)["rstd"]).float()
        for i, leaf in enumerate((x, w, b)):
            for _ in range(4):
                d = torch.randn(leaf.shape, generator=g, device="cuda")
                if i == 0:
                    d = d * scale
                h = 2.0**-8
                at = lambda s: [t + s * h * d if j == i else t for j, t in enumerate((x, w, b))]  # noqa: E731,B023
                numeric = (loss(*at(1)) - loss(*at(-1))) / (2 * h)
                analytic = (grads[i].double() * d.double()).sum()
                # The forward's errors (2^-19 of each output's magnitude, at random signs taken as their
                # sum) over 2 h, and the cubic term: h^2 times third derivatives of order ten.
                size = (k.turing_layer_norm(x, w, b, EPS).double().abs() * dy.double().abs()).sum()
                assert (numeric - analytic).abs() <= 2.0**-19 * size / h + 10 * h * h * size


def test_layouts(k):
    x, w, b, dy = make(60, 512, torch.bfloat16, torch.bfloat16, 6)
    y = k.turing_layer_norm(x, w, b, EPS)
    assert torch.equal(k.turing_layer_norm(x.view(3, 20, 512), w, b, EPS), y.view(3, 20, 512))
    wide = torch.zeros(60, 1024, dtype=torch.bfloat16, device="cuda")
    wide[:, 256:768] = x
    assert torch.equal(k.turing_layer_norm(wide[:, 256:768], w, b, EPS), y)
    flat = torch.empty(60 * 512 + 1, dtype=torch.bfloat16, device="cuda")
    flat[1:] = x.reshape(-1)
    assert torch.equal(k.turing_layer_norm(flat[1:].view(60, 512), w, b, EPS), y)  # 2 bytes off alignment
    assert torch.equal(k.turing_layer_norm(x.t().contiguous().t(), w, b, EPS), y)
    # Gradients of misaligned rows and of an expanded gradient.
    leaf = flat[1:].view(60, 512).detach().requires_grad_(True)
    aligned = x.clone().requires_grad_(True)
    for grad in (dy, dy[:, :1].expand(60, 512), dy[:1].expand(60, 512)):
        one = torch.autograd.grad(k.turing_layer_norm(leaf, w, b, EPS), leaf, grad)[0]
        two = torch.autograd.grad(k.turing_layer_norm(aligned, w, b, EPS), aligned, grad)[0]
        assert torch.equal(one, two)


def test_empty(k):
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    b = torch.ones(64, device="cuda", requires_grad=True)
    y = k.turing_layer_norm(x, w, b, EPS)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()


def test_same_bits_again(k):
    x, w, b, dy = make(3000, 1536, torch.bfloat16, torch.float32, 7)
    for t in (x, w, b):
        t.requires_grad_(True)
    first = torch.autograd.grad(k.turing_layer_norm(x, w, b, EPS), (x, w, b), dy)
    for _ in range(3):
        again = torch.autograd.grad(k.turing_layer_norm(x, w, b, EPS), (x, w, b), dy)
        assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_graph_and_stream(k):
    x, w, b, dy = make(100, 768, torch.bfloat16, torch.float32, 8)

    def step(x):
        y, mean, rstd = torch.ops.turing_utils.layer_norm(x, w, b, EPS)
        return (y, *torch.ops.turing_utils.layer_norm_backward(dy, x, mean, rstd, w, b, 7))

    want = step(x)
    static = torch.zeros_like(x)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(static)
        graphs.append((graph, out))
    static.copy_(x)
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(p, q) for p, q in zip(out, want))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = step(x)
    stream.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_refusals(k):
    x, w, b, dy = make(4, 64, torch.bfloat16, torch.bfloat16)
    for call in (lambda: k.turing_layer_norm(x.double()), lambda: k.turing_layer_norm(x, w[:32]),
                 lambda: k.turing_layer_norm(x, w.half()), lambda: k.turing_layer_norm(x, w, b.float()),
                 lambda: k.turing_layer_norm(x, w, b, 0.0), lambda: k.turing_layer_norm(x, w, b, float("nan")),
                 lambda: k.turing_layer_norm(x[:, :0]), lambda: k.turing_layer_norm(x, w.cpu())):
        with pytest.raises(RuntimeError):
            call()
    x.requires_grad_(True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(k.turing_layer_norm(x, w, b).sum(), x, create_graph=True)


# Rows of a C caller that start anywhere within 16 bytes: x, dy and the results at one offset, or the results
# at another than x; results in the middle of a larger buffer, whose other values stay.
@pytest.mark.parametrize("dtype,offset,result_offset", [(torch.bfloat16, 0, 0), (torch.bfloat16, 3, 3), (torch.float16, 7, 7),
                                                        (torch.float32, 1, 1), (torch.float32, 2, 2), (torch.bfloat16, 5, 0),
                                                        (torch.float32, 0, 3)])
@pytest.mark.parametrize("rows,hidden", [(1, 32), (7, 33), (8, 47), (9, 256), (41, 1281), (700, 2562), (30, 5119),
                                         (1300, 5124), (3, 10247)])
def test_rows_anywhere_within_16_bytes(k, rows, hidden, dtype, offset, result_offset):
    from comfyui_turing_utils_kernel import _lib

    lib = _lib.load()
    x, w, b, dy = make(rows, hidden, dtype, torch.float32, rows + hidden + offset)
    kind = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}[dtype]
    guard = 24

    def placed(t, at):
        buf = torch.full((t.numel() + 2 * guard,), -77.0, dtype=dtype, device="cuda")
        view = buf[guard + at:guard + at + t.numel()]
        view.copy_(t.reshape(-1))
        return buf, view.view(rows, hidden)

    def outside(buf, at):
        return torch.cat((buf[:guard + at], buf[guard + at + rows * hidden:]))

    _, x = placed(x, offset)
    _, dy = placed(dy, offset)
    w = torch.cat((w[:1], w))[1:]  # 4 bytes off 16
    y_buf, y = placed(torch.zeros_like(x), result_offset)
    dx_buf, dx = placed(torch.zeros_like(x), result_offset)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    dw, db = torch.empty(hidden, device="cuda"), torch.empty(hidden, device="cuda")
    room = lib.ctu_layer_norm_backward_workspace_bytes(rows, hidden) // 4
    work = torch.full((room + 64,), -77.0, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    _lib.check(lib.ctu_layer_norm(x.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                                  rows, hidden, EPS, kind, 2, stream))
    _lib.check(lib.ctu_layer_norm_backward(dy.data_ptr(), x.data_ptr(), w.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                                           dx.data_ptr(), dw.data_ptr(), db.data_ptr(), work.data_ptr(), rows, hidden,
                                           kind, 2, stream))
    check(y, (dx, dw, db), x, w, b, dy)
    assert (outside(y_buf, result_offset) == -77).all() and (outside(dx_buf, result_offset) == -77).all()
    assert (work[room:] == -77).all()


# fp32 rows that take more than five pieces a thread, more rows than CTAs.
@pytest.mark.parametrize("rows,hidden", [(450, 10244), (310, 12289), (150, 14336), (149, 14335), (20, 14345)])
def test_widest_fp32_rows(k, rows, hidden):
    x, w, b, dy = make(rows, hidden, torch.float32, torch.float32, hidden)
    for t in (x, w, b):
        t.requires_grad_(True)
    y = k.turing_layer_norm(x, w, b, EPS)
    grads = torch.autograd.grad(y, (x, w, b), dy)
    check(y.detach(), grads, x.detach(), w.detach(), b.detach(), dy)
    # The weights' gradients alone: the rows' own are not asked for.
    y = k.turing_layer_norm(x.detach(), w, b, EPS)
    dw, db = torch.autograd.grad(y, (w, b), dy)
    assert torch.equal(dw, grads[1]) and torch.equal(db, grads[2])


# Rows that share 16 bytes with their neighbours.
@pytest.mark.parametrize("dtype,hidden", [(torch.bfloat16, 641), (torch.float16, 5121), (torch.float32, 1027)])
def test_rows_off_16_bytes_stay_alone(k, dtype, hidden):
    x, w, b, dy = make(40, hidden, dtype, torch.float32, 8)
    leaf = x.clone().requires_grad_(True)
    clean = k.turing_layer_norm(leaf, w, b, EPS)
    clean_dx = torch.autograd.grad(clean, leaf, dy)[0]
    bad = x.clone()
    bad[3, 0], bad[7, -1], bad[20, hidden // 2] = float("nan"), float("inf"), float("-inf")
    bad.requires_grad_(True)
    y = k.turing_layer_norm(bad, w, b, EPS)
    dx = torch.autograd.grad(y, bad, dy)[0]
    rows = [i in (3, 7, 20) for i in range(40)]
    assert torch.isnan(y).all(1).tolist() == rows and torch.isnan(dx).any(1).tolist() == rows
    keep = [i for i in range(40) if not rows[i]]
    assert torch.equal(y[keep], clean[keep]) and torch.equal(dx[keep], clean_dx[keep])


@pytest.mark.parametrize("dtype,hidden", [(torch.bfloat16, 1537), (torch.float32, 10245)])
def test_off_16_bytes_captured_and_again(k, dtype, hidden):
    x, w, b, dy = make(900, hidden, dtype, torch.float32, 9)

    def step():
        y, mean, rstd = torch.ops.turing_utils.layer_norm(x, w, b, EPS)
        return (y, *torch.ops.turing_utils.layer_norm_backward(dy, x, mean, rstd, w, b, 7))

    first = [t.clone() for t in step()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(2):
        for t in held:
            t.zero_()
        graph.replay()
        assert all(torch.equal(a, c) for a, c in zip(first, held))
    x.mul_(0.5)
    graph.replay()
    assert all(torch.equal(a, c) for a, c in zip(step(), held))


# Rows on 16 bytes, several to each of the backward pass's teams (one to sixteen a CTA), whose buffers are loaded again and
# again; the last round of rows leaves some teams without one.
@pytest.mark.parametrize("dtype,wdtype", TYPES)
@pytest.mark.parametrize("rows,hidden", [(9001, 640), (5003, 1536), (3001, 5120), (1201, 10240), (701, 13824)])
def test_several_rows_a_team(k, rows, hidden, dtype, wdtype):
    x, w, b, dy = make(rows, hidden, dtype, wdtype, rows + hidden)
    for t in (x, w, b):
        t.requires_grad_(True)
    y = k.turing_layer_norm(x, w, b, EPS)
    check(y.detach(), torch.autograd.grad(y, (x, w, b), dy), x.detach(), w.detach(), b.detach(), dy)


def test_widest_row_accepted(k):
    """One row of 2^30 values: twice the width, which the join of the sums counts to, is beyond 31 bits."""
    from comfyui_turing_utils_kernel import _lib

    lib, hidden = _lib.load(), 1 << 30
    x = torch.full((hidden,), 0.5, dtype=torch.bfloat16, device="cuda")
    x[::2] = -0.5  # mean 0; xhat of one size
    dy = torch.ones_like(x)
    dy[-1], dy[0] = 3.0, -2.0
    mean, rstd = torch.zeros(1, device="cuda"), torch.full((1,), 2.0, device="cuda")
    dw, db = torch.full_like(x, -77), torch.full_like(x, -77)
    work = torch.empty(lib.ctu_layer_norm_backward_workspace_bytes(1, hidden), dtype=torch.uint8, device="cuda")
    _lib.check(lib.ctu_layer_norm_backward(dy.data_ptr(), x.data_ptr(), None, mean.data_ptr(), rstd.data_ptr(), None,
                                           dw.data_ptr(), db.data_ptr(), work.data_ptr(), 1, hidden, 0, 0,
                                           torch.cuda.current_stream().cuda_stream))
    assert torch.equal(db, dy)  # one row: its gradient, exact in every step
    assert torch.equal(dw, dy * (2 * x))

"""Layer norm: values and gradients against the definition in 64 bits.

Tolerances come from the arithmetic, not from a run. u = 2^-24 is half an
fp32 step. A sum over a row adds at most S = max(32, cols/512) + 12 terms in
sequence (a thread's own, then a tree), so it is off by at most S u times the
sum of magnitudes; results are rounded once to their type, half a step.
"""
import itertools

import pytest
import torch
import torch.autograd.forward_ad as fw

from torched_impala_amd.ops.layernorm import layer_norm

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _ref(x, w, b, eps, dy):
    """y, dx, dw, db in 64 bits, each with its error bound."""
    x, dy = x.double(), dy.double()
    n = x.shape[-1]
    one = torch.ones(n, dtype=torch.float64, device=x.device)
    wd = one if w is None else w.double()
    bd = 0 * one if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    rstd = (var + eps) ** -0.5
    xh = (x - mean) * rstd
    y = xh * wd + bd
    h = dy * wd
    m1, m2 = h.mean(-1, keepdim=True), (h * xh).mean(-1, keepdim=True)
    dx = rstd * (h - m1 - xh * m2)
    S = max(32, n / 512) + 12
    # xhat: the mean's error, the difference's and rstd's
    e = U * (S * rstd * x.abs().mean(-1, keepdim=True)
             + (S + 8) * xh.abs())
    ty = e * wd.abs() + 4 * U * (y.abs() + bd.abs())
    ah = h.abs().mean(-1, keepdim=True)
    ahx = (h * xh).abs().mean(-1, keepdim=True)
    tdx = rstd * ((S + 8) * U * (h.abs() + ah + 2 * xh.abs() * ahx)
                  + m2.abs() * e
                  + xh.abs() * (h.abs() * e).mean(-1, keepdim=True)) \
        + (S + 8) * U * dx.abs()
    rows = x.numel() // n
    xh2, dy2, e2 = (t.reshape(-1, n) for t in (xh, dy, e.expand_as(x)))
    R = rows / 512 + 96
    dw, db = (dy2 * xh2).sum(0), dy2.sum(0)
    tdw = R * U * (dy2 * xh2).abs().sum(0) + (dy2.abs() * e2).sum(0)
    tdb = R * U * dy2.abs().sum(0)
    return (y, ty), (dx, tdx), (dw, tdw), (db, tdb)


def _close(got, ref, what):
    val, tol = ref
    assert got.shape == val.shape, what
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).tiny
    err = (got.double() - val).abs()
    ok = err <= tol * (1 + half) + half * val.abs() + tiny
    assert bool(ok.all()), (what, float((err - tol).max()),
                            int((~ok).sum()))


def _case(shape, dtype, pdtype, affine, device, offset=1.0, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    n = shape[-1]
    x = (torch.randn(*shape, generator=g, device=device) * 1.5
         + offset * torch.randn(*shape[:-1], 1, generator=g, device=device)
         ).to(dtype)
    dy = torch.randn(*shape, generator=g, device=device).to(dtype)
    w = b = None
    if "w" in affine:
        w = (1 + 0.3 * torch.randn(n, generator=g, device=device)).to(pdtype)
    if "b" in affine:
        b = (0.3 * torch.randn(n, generator=g, device=device)).to(pdtype)
    return x, w, b, dy


def _run(x, w, b, dy, eps=1e-5):
    ins = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    it = iter(ins)
    xr = next(it)
    wr = next(it) if w is not None else None
    br = next(it) if b is not None else None
    y = layer_norm(xr, wr, br, eps)
    return y, torch.autograd.grad(y, ins, dy)


def _check(x, w, b, dy, eps=1e-5):
    y, grads = _run(x, w, b, dy, eps)
    ry, rdx, rdw, rdb = _ref(x, w, b, eps, dy)
    assert y.dtype is x.dtype and y.is_contiguous()
    _close(y, ry, "y")
    _close(grads[0], rdx, "dx")
    k = 1
    if w is not None:
        assert grads[k].dtype is w.dtype
        _close(grads[k], rdw, "dw")
        k += 1
    if b is not None:
        _close(grads[k], rdb, "db")
    return y, grads


# --------------------------------------------------------------- CPU
def test_forward_mode_on_cpu():
    """torch's ops carry a tangent on."""
    x, w, b, t = _case((3, 5), torch.float32, torch.float32, "wb", "cpu")
    with fw.dual_level():
        y = layer_norm(fw.make_dual(x, t), w, b)
        assert fw.unpack_dual(y).tangent is not None


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(grad):
    """The kernels have no forward-mode derivative: never a result without
    one."""
    x, w, b, t = _case((3, 5), torch.float32, torch.float32, "wb", "cuda")
    for i in range(3):
        a = [x, w, b]
        with fw.dual_level():
            a[i] = fw.make_dual(a[i], torch.ones_like(a[i]))
            if grad:
                a[0] = a[0].requires_grad_()
            with pytest.raises(RuntimeError, match="forward-mode"):
                layer_norm(*a)
            y = layer_norm(*a, force_eager=True)
            assert fw.unpack_dual(y).tangent is not None


@pytest.mark.parametrize("dtype", DTYPES)
def test_cpu_path(dtype):
    _check(*_case((3, 5, 19), dtype, torch.float32, "wb", "cpu"))


def test_refusals():
    x = torch.randn(4, 8)
    with pytest.raises(TypeError):
        layer_norm(x.double())
    with pytest.raises(TypeError):
        layer_norm(x.long())
    with pytest.raises(ValueError):
        layer_norm(torch.tensor(1.0))
    with pytest.raises(ValueError):
        layer_norm(torch.empty(3, 0))
    with pytest.raises(ValueError):
        layer_norm(x, torch.ones(7))
    with pytest.raises(ValueError):
        layer_norm(x, torch.ones(8), torch.zeros(8, 1))
    with pytest.raises(TypeError):
        layer_norm(x, torch.ones(8).bfloat16())
    with pytest.raises(TypeError):
        layer_norm(x.bfloat16(), torch.ones(8), torch.zeros(8).bfloat16())
    for eps in (-1e-5, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            layer_norm(x, eps=eps)
    with pytest.raises(ValueError):
        layer_norm(x, torch.ones(8, device="meta"))


# --------------------------------------------------------------- GPU
# one column; part of a wave; a wave; a block of 256 and of 512 threads; the
# looped kernels; rows that are multiples of 16 bytes and rows that are not
COLS = [1, 2, 3, 7, 8, 31, 64, 65, 256, 263, 1000, 1025, 2048, 2056, 4096,
        4097, 8192, 8193, 10240, 16384, 16392]


@pytest.mark.gpu
@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_row_lengths(cols, dtype):
    for rows in (1, 13):
        _check(*_case((rows, cols), dtype, dtype, "wb", "cuda", seed=cols))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 5, 672, 4099, 20001])
@pytest.mark.parametrize("cols", [8, 64, 263])
def test_row_counts(rows, cols):
    _check(*_case((rows, cols), torch.float32, torch.float32, "wb", "cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,pdtype,affine", [
    (d, p, a) for d, p, a in itertools.product(
        DTYPES, [torch.float32, "same"], ["", "w", "b", "wb"])])
def test_types_and_parameters(dtype, pdtype, affine):
    pdtype = dtype if pdtype == "same" else pdtype
    for cols in (136, 77, 20000):
        _check(*_case((9, cols), dtype, pdtype, affine, "cuda"))


@pytest.mark.gpu
def test_strides_and_alignment():
    dev = "cuda"
    base = torch.randn(7, 6, 3 * 64, device=dev)
    for x in (base[..., 64:128],                 # rows with a common stride
              base[..., 1:65],                   # off 16-byte alignment
              base.transpose(0, 1)[..., :64],    # rows without one
              base[..., ::3],                    # columns apart
              base[:, :1, :64].expand(7, 6, 64),  # broadcast rows
              base[0, 0, :64]):                  # one row
        dy = torch.randn(x.shape, device=dev)
        w, b = torch.randn(x.shape[-1], device=dev), None
        _check(x, w, b, dy)
    # weight off alignment, gradient of the output not contiguous
    x = torch.randn(40, 64, device=dev)
    w = torch.randn(65, device=dev)[1:]
    dy = torch.randn(64, 40, device=dev).t()
    _check(x, w, None, dy)
    _check(x, w, None, torch.randn(1, 1, device=dev).expand(40, 64))


@pytest.mark.gpu
def test_more_columns_than_a_launch_has_threads():
    """Of the column sums, 32 threads a column: 2^26 columns and some."""
    _check(*_case((2, 2 ** 26 + 40), torch.float16, torch.float16, "wb",
                  "cuda"))


@pytest.mark.gpu
def test_no_rows():
    x = torch.randn(0, 33, device="cuda", requires_grad=True)
    w = torch.ones(33, device="cuda", requires_grad=True)
    b = torch.zeros(33, device="cuda", requires_grad=True)
    y = layer_norm(x, w, b)
    assert y.shape == (0, 33)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.randn(0, 33).cuda())
    assert dx.shape == (0, 33)
    assert not dw.any() and not db.any()


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [64, 263, 4096, 20000])
def test_large_offset_and_constant_rows(cols):
    # an offset of 1000 spreads: the variance is taken around the mean
    x, w, b, dy = _case((11, cols), torch.float32, torch.float32, "wb",
                        "cuda", offset=1000.0)
    _check(x, w, b, dy)
    x = torch.full((3, cols), 7.0, device="cuda")
    y = layer_norm(x)
    assert torch.equal(y, torch.zeros_like(y))


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [40, 1024, 5000, 20000])
def test_non_finite_rows_stay_alone(cols):
    x = torch.randn(9, cols, device="cuda")
    clean = layer_norm(x)
    bad = x.clone()
    bad[2, 3] = float("nan")
    bad[5, cols - 1] = float("inf")
    y = layer_norm(bad)
    keep = [i for i in range(9) if i not in (2, 5)]
    assert torch.equal(y[keep], clean[keep])
    assert not y[2].isfinite().any() and not y[5].isfinite().all()


@pytest.mark.gpu
def test_partial_gradients():
    """Each gradient alone equals the one computed with the others."""
    x, w, b, dy = _case((301, 72), torch.bfloat16, torch.float32, "wb",
                        "cuda")
    _, full = _run(x, w, b, dy)
    for k in range(3):
        ts = [t.detach().clone() for t in (x, w, b)]
        ts[k].requires_grad_()
        g, = torch.autograd.grad(layer_norm(*ts), ts[k], dy)
        assert torch.equal(g, full[k])


@pytest.mark.gpu
def test_gradient_against_differences():
    x, w, b, dy = _case((4, 24), torch.float32, torch.float32, "wb", "cuda")
    _, (dx, dw, db) = _run(x, w, b, dy)

    def loss(x, w, b):
        xd = x.double()
        xh = torch.nn.functional.layer_norm(xd, (24,))
        del xh
        return (layer_norm(x, w, b).double() * dy.double()).sum()

    # a central difference of step h over fp32 values: truncation h^2 times
    # a third derivative of order one, rounding 2^-24 * sum|dy y| / h
    h = 2.0 ** -7
    for t, g, args in ((x, dx, 0), (w, dw, 1), (b, db, 2)):
        v = torch.randn_like(t)
        v /= v.norm()
        hi = [x, w, b]
        lo = [x, w, b]
        hi[args] = t + h * v
        lo[args] = t - h * v
        num = (loss(*hi) - loss(*lo)) / (2 * h)
        ana = (g.double() * v.double()).sum()
        tol = 100 * h * h + 96 * 64 * U / h
        assert abs(float(num - ana)) < tol


@pytest.mark.gpu
def test_repeatable_and_on_another_stream():
    x, w, b, dy = _case((5000, 264), torch.bfloat16, torch.bfloat16, "wb",
                        "cuda")
    y0, g0 = _run(x, w, b, dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y1, g1 = _run(x, w, b, dy)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y0, y1)
    for a, c in zip(g0, g1):
        assert torch.equal(a, c)


@pytest.mark.gpu
def test_captured():
    x, w, b, dy = _case((672, 256), torch.float32, torch.float32, "wb",
                        "cuda")
    sx, sdy = x.clone(), dy.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _run(sx, w, b, sdy)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, grads = _run(sx, w, b, sdy)
    for seed in range(3):
        x2, _, _, dy2 = _case((672, 256), torch.float32, torch.float32, "wb",
                              "cuda", seed=seed + 5)
        sx.copy_(x2)
        sdy.copy_(dy2)
        graph.replay()
        torch.cuda.synchronize()
        ry, rg = _run(x2, w, b, dy2)
        assert torch.equal(y, ry)
        for a, c in zip(grads, rg):
            assert torch.equal(a, c)


@pytest.mark.gpu
def test_saved_input_changed_in_place():
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    z = x * 1.0
    y = layer_norm(z)
    z.add_(1.0)
    with pytest.raises(RuntimeError):
        y.sum().backward()


@pytest.mark.gpu
def test_differentiable_once():
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(layer_norm(x, w).square().sum(), x,
                             create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()

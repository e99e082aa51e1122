"""Newton-Schulz orthogonalisation against its definition in 64 bits.

Tolerances come from the arithmetic, not from a run. A product of a round is
computed from operands of 22 bits with fp32 sums: with u = 2^-22 its relative
error, in the Frobenius norm of the product's magnitudes, stays under 4 u
(operands, dropped low product, sums). An error of X in one round is carried
on by the later ones: the derivative of p(s) = a s + b s^3 + c s^5 on [0,
1.21] is at most a = 3.4445 in magnitude, and so is that of the matrix map
between two singular directions up to a factor of 2. So an error e_k of round
k's X (its norm times 4 u for each of three products, the middle one weighted
by |b| + 2 |c| < 10) gives at most 2 a^(steps - k) e_k in the result:

    |error|_F <= sum_k 2 a^(steps-k) * 48 u * |X_k|_F,   |X_k|_F <= a^k, sqrt(m) * 1.21
"""
import math

import pytest
import torch
import torch.autograd.forward_ad as fw

from torched_impala_amd.ops.orthogonal import COEFFICIENTS, orthogonalize

A, B, C = COEFFICIENTS
U22 = 2.0 ** -22


def _ref(g, steps=5, eps=1e-7):
    x = g.detach().double().cpu()
    x = x / (torch.linalg.vector_norm(x) + eps)
    if x.shape[0] <= x.shape[1]:
        for _ in range(steps):
            m = x @ x.T
            x = A * x + B * (m @ x) + C * (m @ (m @ x))
    else:
        for _ in range(steps):
            m = x.T @ x
            x = A * x + B * (x @ m) + C * ((x @ m) @ m)
    return x


def _tol(g, steps, rho=1.0):
    m = min(g.shape)
    return sum(2 * A ** (steps - k) * 48 * U22
               * min(rho * A ** k, 1.21 * math.sqrt(m))
               for k in range(steps + 1))


def _check(mats, steps=5, eps=1e-7, out=None):
    got = orthogonalize(mats, steps=steps, eps=eps, out=out)
    for g, o in zip(mats, got):
        r = _ref(g, steps, eps)
        assert o.shape == g.shape and o.dtype is g.dtype
        norm = float(torch.linalg.vector_norm(g.detach().double()))
        rho = norm / (norm + eps) if norm + eps else 0.0
        half = torch.finfo(o.dtype).eps / 2
        err = float(torch.linalg.vector_norm(o.double().cpu() - r))
        # sizes under the type's smallest normal round by its step there
        tiny = torch.finfo(o.dtype).tiny * half * 2 * math.sqrt(r.numel())
        lim = _tol(g, steps, rho) + half * float(
            torch.linalg.vector_norm(r)) + tiny
        assert err <= lim, (tuple(g.shape), err, lim)
    return got


def _rand(m, n, dtype=torch.float32, device="cuda", seed=0, scale=1e-3):
    gen = torch.Generator().manual_seed(seed * 1000 + m * 7 + n)
    return (scale * torch.randn(m, n, generator=gen)).to(dtype).to(device)


# --------------------------------------------------------------- CPU
def test_cpu_path():
    _check([_rand(7, 19, device="cpu"), _rand(19, 7, device="cpu"),
            _rand(8, 8, torch.bfloat16, device="cpu")])
    assert orthogonalize([]) == []
    buf = [_rand(5, 6, device="cpu")]
    ref = orthogonalize(buf)
    assert orthogonalize(buf, out=buf)[0] is buf[0]
    assert torch.equal(buf[0], ref[0])


def test_singular_values_near_one():
    g = _rand(24, 60, device="cpu", scale=1.0)
    s = torch.linalg.svdvals(orthogonalize([g])[0])
    assert float(s.max()) <= 1.21 and float(s.min()) >= 0.6


# What the bound of the test below lets through, and what it does not: the
# rounds with sums in 64 bits and operands in one or two fp16 parts, as the
# kernels keep them, with mistakes that kernels could make.

def _parts(x):
    """x in two fp16 parts, its largest entry at 2^13 to 2^14."""
    s = 2.0 ** (13 - math.floor(math.log2(float(x.abs().max()))))
    hi = (x * s).half().double()
    return hi / s, (x * s - hi).half().double() / s


def _in_parts(g, mistake=None, steps=5):
    x = g.double() / (torch.linalg.vector_norm(g.double()) + 1e-7)
    old = torch.zeros_like(x)
    for _ in range(steps):
        h, l = _parts(x)
        if mistake == "one part":
            l = torch.zeros_like(l)
        elif mistake == "stale low part":
            l, old = old, l
        left = h if mistake == "left low part dropped" else h + l
        m = left @ (h + l).T
        if mistake == "low parts swapped":
            m = h @ h.T + l @ l.T
        m = sum(_parts(m)[:1 if mistake == "one part of A" else 2])
        b = A * torch.eye(len(m), dtype=m.dtype) + B * m + C * (m @ m)
        x = sum(_parts(b)[:1 if mistake == "one part of B" else 2]) @ (h + l)
    return x


MISTAKES = ["one part", "stale low part", "left low part dropped",
            "low parts swapped", "one part of A", "one part of B"]


@pytest.mark.parametrize("shape", [(128, 512), (256, 1568), (640, 640)])
def test_twice_fp32_tells_parts_from_mistakes(shape):
    """Two parts pass the bound of test_as_exact_as_fp32 and every mistake
    fails it."""
    gen = torch.Generator().manual_seed(shape[1])
    mats = [torch.randn(shape, generator=gen) for _ in range(2)]
    want = [_ref(g) for g in mats]
    lim = _mean_error([_plain_fp32(g) for g in mats], mats, want) + math.log(2)
    assert _mean_error([_in_parts(g) for g in mats], mats, want) <= lim
    for mistake in MISTAKES:
        got = [_in_parts(g, mistake) for g in mats]
        assert _mean_error(got, mats, want) > lim, mistake


def _refuse(device):
    g = _rand(6, 8, device=device)
    for exc, args, kw in [
            (TypeError, [g.double()], {}),
            (TypeError, [g.long()], {}),
            (ValueError, [g[0]], {}),
            (ValueError, [g[None]], {}),
            (ValueError, [g], dict(steps=0)),
            (ValueError, [g], dict(steps=2.5)),
            (ValueError, [g], dict(eps=-1.0)),
            (ValueError, [g], dict(eps=float("inf"))),
            (ValueError, [g, g.to("meta")], {}),
            (ValueError, [torch.empty(1 << 20, 1, device="meta")], {}),
            (ValueError, [torch.empty(32769, 32769, device="meta")], {}),
            (RuntimeError, [g.clone().requires_grad_()], {}),
            (ValueError, [g], dict(out=[])),
            (TypeError, [g], dict(out=[g.double()])),
            (ValueError, [g], dict(out=[g[:5]])),
            (ValueError, [g], dict(out=[torch.empty(6, 16, device=device)
                                        [:, ::2]])),
            (ValueError, [g], dict(out=[g[:1].expand(6, 8)])),
            (RuntimeError, [g], dict(out=[torch.empty_like(
                g, requires_grad=True)]))]:
        with pytest.raises(exc):
            orthogonalize(args, **kw)
    pool = torch.randn(200, device=device)
    a, b = pool[:48].view(6, 8), pool[40:88].view(6, 8)
    with pytest.raises(ValueError):      # two results on one memory
        orthogonalize([g, g], out=[a, b])
    with pytest.raises(ValueError):      # a result on another's matrix
        orthogonalize([a, g], out=[torch.empty_like(a), b])


def test_refusals_cpu():
    _refuse("cpu")


def _refuse_forward_mode(device):
    g = _rand(6, 8, device=device)
    with fw.dual_level():
        dual = fw.make_dual(g, g.clone())
        with pytest.raises(RuntimeError, match="forward-mode"):
            orthogonalize([g, dual])
        with pytest.raises(RuntimeError, match="forward-mode"):
            orthogonalize([g], out=[dual])


def test_forward_mode_is_refused_cpu():
    _refuse_forward_mode("cpu")


@pytest.mark.gpu
def test_forward_mode_is_refused_gpu():
    _refuse_forward_mode("cuda")


# --------------------------------------------------------------- GPU
@pytest.mark.gpu
def test_refusals_gpu():
    _refuse("cuda")


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 300), (16, 256), (63, 65), (64, 64),
          (65, 63), (128, 128), (129, 127), (200, 333), (256, 1568),
          (1024, 263), (1024, 256), (32, 288), (300, 4), (5, 5000),
          (640, 640)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16,
                                   torch.float16])
def test_shapes(shape, dtype):
    _check([_rand(*shape, dtype)])


@pytest.mark.gpu
def test_list_of_many():
    """More matrices than one launch takes, all types, empty ones among."""
    types = [torch.float32, torch.bfloat16, torch.float16]
    mats = [_rand(3 + 5 * i, 200 - 3 * i, types[i % 3]) for i in range(60)]
    mats[4] = mats[4][:0]
    mats[31] = mats[31][:, :0]
    got = _check(mats)
    for i in (0, 7, 59):   # and each equals its own call
        assert torch.allclose(got[i].float(),
                              orthogonalize([mats[i]])[0].float(),
                              atol=2 ** -8)


@pytest.mark.gpu
def test_wide_tiles():
    _check([_rand(1024, 1024), _rand(2000, 1030), _rand(1030, 2000,
                                                        torch.bfloat16),
            _rand(33, 70)])


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 2, 3, 8])
def test_steps(steps):
    _check([_rand(70, 200), _rand(200, 70)], steps=steps)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-36, 1e-20, 1e-12, 1e-8, 1e-6, 1.0, 1e6,
                                   1e18, 1e36])
def test_scales(scale):
    """Any gradient's scale: norms that overflow 32 bits when squared, and
    norms that eps outweighs, where the result stays as small as it is."""
    _check([_rand(48, 130, scale=scale)])
    _check([_rand(48, 130, scale=scale)], eps=0.0)


@pytest.mark.gpu
def test_low_rank_and_zero():
    u, v = _rand(90, 3, scale=1.0), _rand(3, 150, scale=1.0)
    _check([u @ v, torch.zeros(40, 70, device="cuda")])
    assert not orthogonalize([torch.zeros(9, 9, device="cuda")])[0].any()
    assert orthogonalize([torch.zeros(3, 3, device="cuda")],
                         eps=0.0)[0].isnan().all()


@pytest.mark.gpu
def test_non_finite_stays_in_its_matrix():
    a, b = _rand(70, 70), _rand(70, 90)
    clean = orthogonalize([a, b])
    for value in (float("nan"), float("inf")):
        bad = a.clone()
        bad[3, 4] = value
        got = orthogonalize([bad, b])
        assert not got[0].isfinite().any()
        assert torch.equal(got[1], clean[1])


@pytest.mark.gpu
def test_strides():
    base = torch.randn(70, 400, device="cuda")
    mats = [base[:, :130], base[:, 1:300:3], base.t()[5:90], base[::2, 7:],
            base[:1].expand(20, 400)]
    got = _check(mats)
    assert all(o.is_contiguous() for o in got)
    # results in a larger buffer: what lies around them stays
    pool = torch.randn(1000, device="cuda")
    before = pool.clone()
    out = [pool[100:100 + 210].view(14, 15), pool[400:400 + 210].view(15, 14)
           .t()]
    mats = [_rand(14, 15), _rand(14, 15, seed=1)]
    orthogonalize(mats, out=out)
    ref = orthogonalize(mats)
    assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])
    assert torch.equal(pool[:100], before[:100])
    assert torch.equal(pool[310:400], before[310:400])
    assert torch.equal(pool[610:], before[610:])


@pytest.mark.gpu
def test_in_place():
    mats = [_rand(70, 200), _rand(300, 40)]
    ref = orthogonalize(mats)
    got = orthogonalize(mats, out=mats)
    assert got[0] is mats[0]
    for a, b in zip(got, ref):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_repeatable_streams_and_two_at_once():
    one = [_rand(256, 1568), _rand(1024, 256)]
    two = [_rand(256, 1568, seed=2), _rand(1024, 256, seed=2)]
    r1, r2 = orthogonalize(one), orthogonalize(two)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(s1):
            g1 = orthogonalize(one)
        with torch.cuda.stream(s2):
            g2 = orthogonalize(two)
        torch.cuda.synchronize()
        for a, b in zip(r1 + r2, g1 + g2):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_captured():
    mats = [_rand(256, 1568), _rand(1024, 263), _rand(16, 256)]
    buf = [m.clone() for m in mats]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        orthogonalize(buf)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = orthogonalize(buf)
    for seed in (4, 5, 6):
        new = [_rand(*m.shape, seed=seed) for m in mats]
        for b, n in zip(buf, new):
            b.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(res, orthogonalize(new)):
            assert torch.equal(a, b)


def _plain_fp32(g, steps=5, eps=1e-7):
    x = g / (torch.linalg.vector_norm(g) + eps)
    for _ in range(steps):
        m = x @ x.T
        x = A * x + (B * m + C * (m @ m)) @ x
    return x


def _mean_error(got, mats, want):
    """Mean of the logarithm of the relative errors."""
    return sum(math.log(torch.linalg.vector_norm(y.double().cpu() - w)
                        / torch.linalg.vector_norm(w))
               for y, w in zip(got, want)) / len(mats)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(4, 2000), (7, 599), (12, 635), (16, 16),
                                   (16, 256), (32, 288), (64, 500)])
@pytest.mark.parametrize("tall", [False, True])
def test_few_rows_beside_a_large_matrix(shape, tall):
    """Few rows are as exact as in fp32 beside a matrix that takes the large
    tiles too. The bound is that of the test of few rows by themselves."""
    gen = torch.Generator().manual_seed(shape[0] * 3001 + shape[1])
    mats = [torch.randn(shape, generator=gen) for _ in range(64)]
    want = [_ref(g) for g in mats]
    big = _rand(2048, 2048)
    turn = (lambda t: t.t().contiguous()) if tall else (lambda t: t)
    got = []
    for i in range(0, 64, 8):
        res = orthogonalize([turn(g).cuda() for g in mats[i:i + 4]] + [big]
                            + [turn(g).cuda() for g in mats[i + 4:i + 8]])
        got += [turn(x) for x in res[:4] + res[5:]]
    own = _mean_error(got, mats, want)
    plain = _mean_error([_plain_fp32(g.cuda()) for g in mats], mats, want)
    assert own <= plain + math.log(1.25), (math.exp(own), math.exp(plain))


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", [
    [(640, 640)], [(256, 1568), (1024, 263), (1024, 256)],   # tiles of 64
    [(1024, 1024)], [(1024, 1024)] * 4,      # of 64 and of 128, k split
    [(2048, 2048), (65, 400), (100, 1000), (128, 2000), (263, 1024),
     (1030, 2000), (2000, 1030)]])           # of 128
def test_as_exact_as_fp32(shapes):
    """fp32 matrices of more rows, in both sizes of tiles, with and without a
    split k, against the same products in fp32. An operand of 22 bits is off by
    2^-23 of each value, independently, and so is a product of K terms by
    2^-23 sqrt(2 / K) of its magnitudes' sum; the sums, of 32 terms at a time,
    are off by 2^-24 sqrt(K / 32) of their own size or less. fp32 products sum
    the K terms with errors of the same kind, so neither is far below the
    other: twice fp32's error is allowed for the mean over four matrices. One
    part in place of two gives 2^-12, a thousand times as much."""
    gen = torch.Generator().manual_seed(len(shapes) * 100 + shapes[0][0])
    lists = [[torch.randn(s, generator=gen).cuda() for s in shapes]
             for _ in range(4)]
    got = [orthogonalize(mats) for mats in lists]

    def wide(t):
        return t if t.shape[0] <= t.shape[1] else t.t()

    for i, shape in enumerate(shapes):
        mats = [wide(m[i]) for m in lists]
        want = [_plain_fp32(g.double()).cpu() for g in mats]
        own = _mean_error([wide(x[i]) for x in got], mats, want)
        plain = _mean_error([_plain_fp32(g) for g in mats], mats, want)
        assert own <= plain + math.log(2), (shape, math.exp(own),
                                            math.exp(plain))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(4, 2000), (7, 599), (12, 635), (16, 16),
                                   (64, 500)])
def test_few_rows_as_exact_as_fp32(shape):
    """Singular values that are nearly the same make errors of one sign add
    up instead of averaging out. The mean error over 64 matrices is held
    against that of the same products in fp32, whose roundings are random. One
    matrix's two errors are apart by a factor of about e^0.35 either way, so
    their mean by e^0.044: a quarter is five times that."""
    gen = torch.Generator().manual_seed(shape[0] * 3001 + shape[1])
    mats = [torch.randn(shape, generator=gen) for _ in range(64)]
    own, plain = 0.0, 0.0
    for g, x in zip(mats, orthogonalize([g.cuda() for g in mats])):
        want = _ref(g)
        for y in (x, _plain_fp32(g.cuda())):
            err = math.log(torch.linalg.vector_norm(y.double().cpu() - want)
                           / torch.linalg.vector_norm(want))
            if y is x:
                own += err / len(mats)
            else:
                plain += err / len(mats)
    assert own <= plain + math.log(1.25), (math.exp(own), math.exp(plain))

"""Linear attention against its recurrence in 64 bits.

Tolerances come from the arithmetic, not from a run. Every result is a sum
of products of the inputs; running the same sum over the inputs' magnitudes
gives A, and a computation in 32 bits is off by at most K u A, where u is
half an fp32 step and K counts roundings in sequence: dk for a score, 64 for
a chunk's sum, another 64 for the state's, and 6 a chunk for the decays and
sums that carry the state on, plus 32 for weights and scales. With bf16
operands the scores and the state enter a product in two bf16 parts, each
off by 2^-18 of its value: 2^-17 A more for both. Then half a step of the
result's type.
"""
import itertools
import math

import pytest
import torch
import torch.autograd.forward_ad as fw

from torched_impala_amd.ops.linear_attention import (
    linear_attention, linear_attention_step)

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _ref(q, k, v, g, done, state, scale, d_out=None, d_final=None):
    """out, final and the gradients by the recurrence, in 64 bits on the CPU
    (gradients written out, not by autograd)."""
    T, B, H, dk = q.shape
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    lam = g.double().cpu().exp().view(1, H, 1, 1)
    live = (torch.ones(T, B) if done is None else (~done).double().cpu())
    f = lam * live.double().view(T, B, 1, 1, 1)
    s = (torch.zeros(B, H, dk, v.shape[-1]) if state is None
         else state.detach().cpu()).double()
    out = torch.zeros_like(v)
    hist = []
    for t in range(T):
        s = torch.where(f[t] == 0, torch.zeros_like(s), s * f[t]) \
            + k[t][..., :, None] * v[t][..., None, :]
        hist.append(s)
        out[t] = scale * (q[t][..., :, None] * s).sum(-2)
    res = [out, s]
    if d_out is None:
        return res
    do = d_out.double().cpu()
    r = torch.zeros_like(s) if d_final is None else d_final.double().cpu()
    dq, dkk, dvv = (torch.zeros_like(t) for t in (q, k, v))
    for t in reversed(range(T)):
        dq[t] = scale * (hist[t] * do[t][..., None, :]).sum(-1)
        r = r + scale * q[t][..., :, None] * do[t][..., None, :]
        dkk[t] = (r * v[t][..., None, :]).sum(-1)
        dvv[t] = (r * k[t][..., :, None]).sum(-2)
        r = torch.where(f[t] == 0, torch.zeros_like(r), r * f[t])
    return res + [dq, dkk, dvv, r]


def _bounds(dtype, T, dk, dv):
    K = max(dk, dv) + 128 + 6 * math.ceil(max(T, 1) / 64) + 32
    rel = K * U
    full = rel + (2.0 ** -17 if dtype is torch.bfloat16 else 0.0)
    return full, rel


def _close(got, ref, mag, rel, what):
    assert got.shape == ref.shape, what
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).tiny
    tol = rel * mag * (1 + half) + half * ref.abs() + tiny
    x = got.detach().double().cpu()
    ok = (x - ref).abs() <= tol
    # beyond the type's largest value plus half its step a result is infinite,
    # where the error may reach across that place it may be
    top = torch.finfo(got.dtype).max * (1 + half / 2)
    ok &= ref.abs() - tol <= top
    ok |= (x == ref.sign() * math.inf) & (ref.abs() + tol >= top)
    bad = ~ok
    assert not bool(bad.any()), (
        what, int(bad.sum()),
        float(((got.detach().double().cpu() - ref).abs() - tol).max()))


def _inputs(T, B, H, dk, dv, dtype, done=0.05, state=True, device="cuda",
            seed=0):
    gen = torch.Generator().manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, generator=gen)

    q, k = rn(T, B, H, dk).to(dtype), rn(T, B, H, dk).to(dtype)
    v, do = rn(T, B, H, dv).to(dtype), rn(T, B, H, dv).to(dtype)
    g = torch.log1p(-torch.exp2(-1.0 - 7.0 * torch.rand(H, generator=gen)))
    d = torch.rand(T, B, generator=gen) < done if done else None
    s = rn(B, H, dk, dv) if state else None
    df = rn(B, H, dk, dv) if state else None
    return [None if t is None else t.to(device)
            for t in (q, k, v, g, d, s, do, df)]


def _run(q, k, v, g, d, s, do, df, scale=None):
    ins = [t.detach().requires_grad_() for t in (q, k, v)]
    st = None if s is None else s.detach().requires_grad_()
    out, fin = linear_attention(*ins, g, done=d, state=st, scale=scale)
    outs, grads = [out], [do]
    if df is not None:
        outs.append(fin)
        grads.append(df)
    gr = torch.autograd.grad(outs, ins + ([] if st is None else [st]), grads)
    return [out, fin] + list(gr)


NAMES = ("out", "final", "dq", "dk", "dv", "dstate")


def _check(q, k, v, g, d, s, do, df, scale=None):
    T, B, H, dk = q.shape
    dv = v.shape[-1]
    sc = dk ** -0.5 if scale is None else scale
    got = _run(q, k, v, g, d, s, do, df, scale)
    ref = _ref(q, k, v, g, d, s, sc, do, df)
    mag = _ref(q.abs(), k.abs(), v.abs(), g, d,
               None if s is None else s.abs(), abs(sc), do.abs(),
               None if df is None else df.abs())
    full, rel = _bounds(q.dtype, T, dk, dv)
    for n, a, r, m in zip(NAMES, got, ref, mag):
        _close(a, r, m, rel if n in ("final", "dstate") else full, n)
        if n in ("final", "dstate"):
            assert a.dtype is torch.float32
        else:
            assert a.dtype is q.dtype
    return got


# --------------------------------------------------------------- CPU
@pytest.mark.parametrize("dtype", DTYPES)
def test_cpu_path(dtype):
    _check(*_inputs(9, 3, 2, 5, 7, dtype, 0.2, device="cpu"))
    _check(*_inputs(9, 3, 2, 5, 7, dtype, 0, False, device="cpu"))


def test_cpu_step_is_one_step():
    q, k, v, g, d, s, _, _ = _inputs(3, 4, 2, 8, 6, torch.float32, 0.3,
                                     device="cpu")
    out, fin = linear_attention(q, k, v, g, done=d, state=s)
    st = s
    for t in range(3):
        o, st = linear_attention_step(q[t], k[t], v[t], g, st, done=d[t])
        torch.testing.assert_close(o, out[t], rtol=0, atol=0)
    assert torch.equal(st, fin)
    buf = s.clone()
    o, r = linear_attention_step(q[0], k[0], v[0], g, buf, done=d[0],
                                 out_state=buf)
    assert r is buf and not torch.equal(buf, s)


def _refuse_forward_mode_of_a_step(device):
    q, k, v, g, d, s, _, _ = _inputs(1, 2, 2, 4, 5, torch.float32,
                                     device=device)
    for i in range(6):
        a = [q[0], k[0], v[0], g, s.clone(), torch.empty_like(s)]
        with fw.dual_level():
            a[i] = fw.make_dual(a[i], torch.ones_like(a[i]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                linear_attention_step(*a[:5], done=d[0], out_state=a[5])


def test_forward_mode_on_cpu():
    """torch's ops carry a tangent on; a step has no derivatives at all."""
    q, k, v, g, d, s, _, _ = _inputs(3, 2, 2, 4, 5, torch.float32,
                                     device="cpu")
    with fw.dual_level():
        out, fin = linear_attention(q, k, fw.make_dual(v, v), g, done=d,
                                    state=s)
        assert fw.unpack_dual(out).tangent is not None
        assert fw.unpack_dual(fin).tangent is not None
    _refuse_forward_mode_of_a_step("cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(grad):
    """The kernels have no forward-mode derivative: never a result without
    one."""
    q, k, v, g, d, s, _, _ = _inputs(3, 2, 2, 4, 5, torch.float32)
    for i in range(5):
        a = [q, k, v, g, s]
        with fw.dual_level():
            a[i] = fw.make_dual(a[i], torch.ones_like(a[i]))
            if grad:
                a[0] = a[0].clone().requires_grad_()
            with pytest.raises(RuntimeError, match="forward-mode"):
                linear_attention(*a[:4], done=d, state=a[4])
            out, _ = linear_attention(*a[:4], done=d, state=a[4],
                                      force_eager=True)
            assert fw.unpack_dual(out).tangent is not None
    _refuse_forward_mode_of_a_step("cuda")


def test_cpu_nothing_to_do():
    for T, B, H in ((0, 2, 3), (4, 0, 3), (4, 2, 0)):
        q, k, v, g, d, s, _, _ = _inputs(T, B, H, 4, 5, torch.float32,
                                         device="cpu")
        out, fin = linear_attention(q, k, v, g, done=d, state=s)
        assert out.shape == (T, B, H, 5)
        assert torch.equal(fin, s)


def _bad_calls(device):
    """(exception, keyword changes) for a good call of T=3 B=2 H=2 4x5."""
    def t(*s, dtype=torch.float32):
        return torch.zeros(*s, dtype=dtype, device=device)

    return [
        (TypeError, dict(q=t(3, 2, 2, 4, dtype=torch.float64))),
        (TypeError, dict(k=t(3, 2, 2, 4, dtype=torch.bfloat16))),
        (ValueError, dict(k=t(3, 2, 1, 4))),
        (ValueError, dict(v=t(3, 1, 2, 5))),
        (ValueError, dict(q=t(2, 2, 4))),
        (ValueError, dict(v=t(3, 2, 2, 129))),
        (ValueError, dict(v=t(3, 2, 2, 0))),
        (ValueError, dict(q=t(3, 2, 2, 129), k=t(3, 2, 2, 129))),
        (ValueError, dict(log_decay=t(3))),
        (TypeError, dict(log_decay=t(2, dtype=torch.float64))),
        (ValueError, dict(log_decay=t(2).requires_grad_())),
        (TypeError, dict(done=t(3, 2))),
        (ValueError, dict(done=t(2, 3, dtype=torch.bool))),
        (TypeError, dict(state=t(2, 2, 4, 5, dtype=torch.bfloat16))),
        (ValueError, dict(state=t(2, 2, 5, 4))),
        (ValueError, dict(scale=float("nan"))),
        (ValueError, dict(v=torch.zeros(3, 2, 2, 5, device="meta"))),
    ]


def _good(device):
    q, k, v, g, d, s, _, _ = _inputs(3, 2, 2, 4, 5, torch.float32,
                                     device=device)
    return dict(q=q, k=k, v=v, log_decay=g, done=d, state=s, scale=None)


def _refuse(device):
    for exc, change in _bad_calls(device):
        kw = dict(_good(device), **change)
        with pytest.raises(exc):
            linear_attention(kw.pop("q"), kw.pop("k"), kw.pop("v"),
                             kw.pop("log_decay"), **kw)
    q, k, v, g, d, s, _, _ = _inputs(1, 2, 2, 4, 5, torch.float32,
                                     device=device)
    q, k, v, d = q[0], k[0], v[0], d[0]
    with pytest.raises(RuntimeError):
        linear_attention_step(q.clone().requires_grad_(), k, v, g, s)
    for bad in (s[:1], s.transpose(2, 3).contiguous()):
        with pytest.raises(ValueError):
            linear_attention_step(q, k, v, g, s, out_state=bad)
    with pytest.raises(TypeError):
        linear_attention_step(q, k, v, g, s, out_state=s.double())
    with pytest.raises(ValueError):   # environments on one memory
        linear_attention_step(q, k, v, g, s,
                              out_state=torch.zeros_like(s[:1]).expand(
                                  s.shape))
    pool = torch.zeros(3, 2, 4, 5, device=device)
    with pytest.raises(ValueError):   # overlap that is not the same place
        linear_attention_step(q, k, v, g, pool[:2], out_state=pool[1:])
    with pytest.raises(ValueError):
        linear_attention_step(q, k, v, g, s, done=d[:1])


def test_refusals_cpu():
    _refuse("cpu")


def _states_side_by_side(device):
    """Old and new states of a pool that holds both for every environment."""
    B, H, dk, dv = 3, 2, 4, 5
    n = H * dk * dv
    q, k, v, g, d, s, _, _ = _inputs(1, B, H, dk, dv, torch.float32,
                                     device=device)
    ref, new = linear_attention_step(q[0], k[0], v[0], g, s, done=d[0])
    pool = torch.randn(B, 2 * n + 3, device=device)
    part = [pool[:, i:i + n].unflatten(1, (H, dk, dv))
            for i in (0, 1, n - 1, n, n + 3)]
    before = pool.clone()
    for i, o in ((0, 3), (0, 4), (4, 0), (3, 0)):
        pool.copy_(before)
        part[i].copy_(s)
        kept = pool.clone()
        out, r = linear_attention_step(q[0], k[0], v[0], g, part[i],
                                       done=d[0], out_state=part[o])
        assert torch.equal(out, ref) and torch.equal(r, new)
        part[o].copy_(kept[:, (0, 0, 0, n, n + 3)[o]:][:, :n]
                      .unflatten(1, (H, dk, dv)))
        assert torch.equal(pool, kept)   # and nothing else was written
    for i, o in ((0, 1), (1, 0), (0, 2), (2, 0), (2, 3), (4, 1)):
        # the last one: an environment's new state reaches into the next's
        if (i, o) == (4, 1):
            b = pool.view(-1)[n + 3:].as_strided(s.shape, s.stride())
            a = pool.view(-1).as_strided(s.shape, (n + 1, dk * dv, dv, 1))
        else:
            a, b = part[i], part[o]
        with pytest.raises(ValueError, match="without being it"):
            linear_attention_step(q[0], k[0], v[0], g, a, out_state=b)


def _refuse_results_on_inputs(device):
    """The new state over memory that the step still reads."""
    q, k, v, g, d, s, _, _ = _inputs(1, 2, 2, 4, 5, torch.float32,
                                     device=device)
    ref, want = linear_attention_step(q[0], k[0], v[0], g, s, done=d[0])
    assert s.numel() == 80
    for i in range(5):
        a = [q[0], k[0], v[0], g, d[0]]
        pool = torch.zeros(200, device=device)
        where = pool[40:] if i != 4 else pool[40:].view(torch.bool)
        n = a[i].numel()
        where[:n] = a[i].reshape(-1)
        a[i] = where[:n].view(a[i].shape)
        with pytest.raises(ValueError, match="overlaps an input"):
            linear_attention_step(*a[:4], s, done=a[4],
                                  out_state=pool[:80].view(s.shape))
        out, new = linear_attention_step(*a[:4], s, done=a[4],
                                         out_state=pool[80:160].view(s.shape))
        assert torch.equal(out, ref) and torch.equal(new, want)
    # an environment's state and query in one record
    pool = torch.zeros(2, 48, device=device)
    qr, sr = pool[:, :8].unflatten(1, (2, 4)), pool[:, 8:].view(s.shape)
    qr.copy_(q[0])
    sr.copy_(s)
    out, new = linear_attention_step(qr, k[0], v[0], g, sr, done=d[0],
                                     out_state=sr)
    assert torch.equal(out, ref) and torch.equal(new, want)
    assert torch.equal(qr, q[0])


def test_results_on_inputs_are_refused_cpu():
    _refuse_results_on_inputs("cpu")


@pytest.mark.gpu
def test_results_on_inputs_are_refused_gpu():
    _refuse_results_on_inputs("cuda")


def test_states_side_by_side_cpu():
    _states_side_by_side("cpu")


@pytest.mark.gpu
def test_states_side_by_side_gpu():
    _states_side_by_side("cuda")


def _refuse_heads(device):
    """More heads than a launch has threads for."""
    from torched_impala_amd.ops.linear_attention import MAX_HEADS
    x = torch.zeros(1, 1, 1, 1, device=device)
    g = torch.zeros(3, device=device)
    x = x.expand(1, MAX_HEADS // 3 + 1, 3, 1)
    with pytest.raises(ValueError):
        linear_attention(x, x, x, g)
    with pytest.raises(ValueError):
        linear_attention_step(x[0], x[0], x[0], g,
                              x[0].unsqueeze(-1))


def test_too_many_heads_cpu():
    _refuse_heads("cpu")


# --------------------------------------------------------------- GPU
@pytest.mark.gpu
def test_refusals_gpu():
    _refuse("cuda")


@pytest.mark.gpu
def test_too_many_heads_gpu():
    _refuse_heads("cuda")


LENGTHS = [1, 2, 15, 16, 17, 21, 33, 48, 63, 64, 65, 101, 128, 129, 200]


@pytest.mark.gpu
@pytest.mark.parametrize("T", LENGTHS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_lengths(T, dtype):
    _check(*_inputs(T, 3, 2, 64, 64, dtype, seed=T))


@pytest.mark.gpu
@pytest.mark.parametrize("eq,ek,ev,eo", [(-18, 0, 0, 0), (0, -18, 0, 0),
                                         (0, 0, -18, 0), (0, 0, 0, -18),
                                         (-18, -18, -18, -18),
                                         (12, 12, 12, 12), (12, -18, 12, -18),
                                         (-18, 12, -18, 12)])
@pytest.mark.parametrize("D", [64, 128])
def test_fp16_range(eq, ek, ev, eo, D):
    """Operands among fp16's subnormals and its largest values: products and
    states are far beyond fp16's range on both sides, and exact operands
    stay exact. The scale brings the output back into fp16."""
    q, k, v, g, d, s, do, df = _inputs(150, 2, 2, D, D, torch.float32, 0.02,
                                       seed=D + eq + 2 * ek + 3 * ev + 5 * eo)
    q, k, v, do = (((t * 2.0 ** e).clamp(-60000, 60000)).half()
                   for t, e in ((q, eq), (k, ek), (v, ev), (do, eo)))
    s, df = s * 2.0 ** (ek + ev), df * 2.0 ** (eq + eo)
    # the largest of the four results' exponents at 2^0
    top = max(eq + ek + ev, eo + ev + ek, eo + ev + eq, eo + ek + eq)
    _check(q, k, v, g, d, s, do, df, scale=2.0 ** (-5 - top))


@pytest.mark.gpu
@pytest.mark.parametrize("dk,dv", [(1, 1), (1, 128), (3, 5), (8, 16),
                                   (16, 8), (31, 33), (32, 64), (48, 80),
                                   (63, 65), (64, 32), (65, 63), (96, 40),
                                   (100, 128), (128, 1), (127, 128),
                                   (128, 128)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_head_sizes(dk, dv, dtype):
    _check(*_inputs(77, 2, 3, dk, dv, dtype, seed=dk + dv))


@pytest.mark.gpu
@pytest.mark.parametrize("T,B,H", [(512, 2, 2), (700, 1, 3), (1000, 3, 1),
                                   (2100, 1, 2), (1111, 40, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_cut_into_segments(T, B, H, dtype):
    _check(*_inputs(T, B, H, 24, 16, dtype, 0.002, seed=T))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_cut_wide_heads(dtype):
    _check(*_inputs(900, 1, 2, 128, 96, dtype, 0.002))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [40, 130, 640])
def test_no_state_and_no_done(T):
    for done, state in itertools.product([0, 0.05], [False, True]):
        _check(*_inputs(T, 2, 2, 32, 32, torch.float32, done, state))


def _with_done(rows, T=150, dtype=torch.float32):
    a = _inputs(T, 2, 2, 16, 24, dtype)
    d = torch.zeros(T, 2, dtype=torch.bool)
    for t in rows:
        d[t] = True
    a[4] = d.cuda()
    return a


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [[0], [63], [64], [65], [149], [0, 149],
                                  [62, 63, 64], list(range(150)),
                                  list(range(0, 150, 2)), [127, 128]])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_done_places(rows, dtype):
    _check(*_with_done(rows, dtype=dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [70, 600])
def test_done_equals_fresh_start(T):
    """Steps behind a done are those of an unroll that starts there."""
    q, k, v, g, _, s, _, _ = _inputs(T, 2, 2, 32, 32, torch.float32)
    cut = T - 23
    d = torch.zeros(T, 2, dtype=torch.bool, device="cuda")
    d[cut] = True
    out, fin = linear_attention(q, k, v, g, done=d, state=s)
    tail, fin2 = linear_attention(q[cut:], k[cut:], v[cut:], g)
    torch.testing.assert_close(out[cut:], tail, rtol=1e-5, atol=1e-4)
    torch.testing.assert_close(fin, fin2, rtol=1e-5, atol=1e-4)


@pytest.mark.gpu
@pytest.mark.parametrize("g", [0.0, -1e-7, -30.0, -200.0, float("-inf")])
@pytest.mark.parametrize("T", [20, 200, 600])
def test_extreme_decays(g, T):
    a = _inputs(T, 1, 2, 16, 16, torch.float32)
    a[3] = torch.tensor([g, -0.1], device="cuda")
    _check(*a)


HALF = torch.float16


@pytest.mark.gpu
@pytest.mark.parametrize("T,B,H,dk,dv", [(512, 2, 2, 24, 16),
                                         (1111, 40, 2, 24, 16),
                                         (900, 1, 2, 128, 96),
                                         (700, 1, 3, 64, 64)])
def test_fp16_cut_into_segments(T, B, H, dk, dv):
    _check(*_inputs(T, B, H, dk, dv, HALF, 0.002, seed=T))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [[0], [63], [64], [149], [62, 63, 64],
                                  list(range(150)), [127, 128]])
def test_fp16_done_places(rows):
    _check(*_with_done(rows, dtype=HALF))


@pytest.mark.gpu
@pytest.mark.parametrize("g", [0.0, -1e-7, -1.0, -30.0, -200.0,
                               float("-inf")])
@pytest.mark.parametrize("T", [20, 200, 600])
@pytest.mark.parametrize("D", [16, 128])
def test_fp16_extreme_decays(g, T, D):
    a = _inputs(T, 1, 2, D, D, HALF)
    a[3] = torch.tensor([g, -0.1], device="cuda")
    _check(*a)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [48, 128])
def test_padded_rows(dtype, D):
    """Rows of zeros at the end, or everywhere: what is left of the rows in
    front has decayed far below one and is still exact."""
    for rows in (30, 90, 150):
        a = _inputs(150, 2, 2, D, D, dtype, 0, seed=rows)
        for t in (a[0], a[1], a[2], a[6]):
            t[150 - rows:] = 0
        a[3] = torch.tensor([-1.0, -0.2], device="cuda")
        _check(*a)
        a[5] = a[7] = None
        _check(*a)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("e,scale", [(100, 2.0 ** -104), (-100, 1.0),
                                     (-140, 1.0), (40, 2.0 ** -44)])
@pytest.mark.parametrize("D", [32, 128])
def test_states_beyond_the_operands_range(dtype, e, scale, D):
    """States and their gradients are fp32: their values may be far outside
    fp16's range."""
    q, k, v, g, d, s, do, df = _inputs(140, 2, 2, D, D, dtype, 0.02, seed=D)
    df = df * 2.0 ** min(e, 0)
    _check(q, k, v, g, d, s * 2.0 ** e, do, df, scale=scale)
    z = torch.zeros_like
    _check(q, z(k), v, g, d, s * 2.0 ** e, do, df, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3])
def test_scale(scale):
    _check(*_inputs(90, 2, 2, 16, 16, torch.bfloat16), scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    T, B, H, d = 75, 3, 2, 32
    _, _, _, g, dn, s, do, df = _inputs(T, B, H, d, d, dtype)
    # parts of one projection
    x = torch.randn(T, B, 3 * H * d, device="cuda").to(dtype)
    q, k, v = (t.unflatten(-1, (H, d)) for t in x.chunk(3, -1))
    _check(q, k, v, g, dn, s, do, df)
    # off 16-byte alignment
    x = torch.randn(T, B, 3 * H * d + 1, device="cuda").to(dtype)[..., 1:]
    q, k, v = (t.unflatten(-1, (H, d)) for t in x.chunk(3, -1))
    _check(q, k, v, g, dn, s, do, df)
    # environment first, heads before steps
    q, k, v = (torch.randn(B, H, T, d, device="cuda").to(dtype)
               .permute(2, 0, 1, 3) for _ in range(3))
    _check(q, k, v, g, dn, s, do.transpose(0, 1).contiguous()
           .transpose(0, 1), df)
    # features apart, flags apart, a turned state
    q = torch.randn(T, B, H, 2 * d, device="cuda").to(dtype)[..., ::2]
    dn2 = torch.stack([dn, ~dn], -1)[..., 0]
    st = s.transpose(2, 3).contiguous().transpose(2, 3)
    _check(q, k, v, g, dn2, st, do, df)


@pytest.mark.gpu
def test_broadcast_inputs_and_gradients():
    """One key and value head for all query heads, as a broadcast view."""
    T, B, H, d = 70, 2, 4, 32
    q, k, v, g, dn, s, do, df = _inputs(T, B, H, d, d, torch.float32)
    k1, v1 = k[:, :, :1].contiguous(), v[:, :, :1].contiguous()
    ins = [t.detach().requires_grad_() for t in (q, k1, v1)]
    out, _ = linear_attention(ins[0], ins[1].expand(T, B, H, d),
                              ins[2].expand(T, B, H, d), g, done=dn, state=s)
    got = torch.autograd.grad(out, ins, do)
    kx, vx = (t.expand(T, B, H, d) for t in (k1, v1))
    full = _run(q, kx, vx, g, dn, s, do, None)
    assert torch.equal(out, full[0])
    assert torch.equal(got[0], full[2])
    torch.testing.assert_close(got[1], full[3].sum(2, keepdim=True),
                               rtol=1e-5, atol=1e-4)
    torch.testing.assert_close(got[2], full[4].sum(2, keepdim=True),
                               rtol=1e-5, atol=1e-4)


@pytest.mark.gpu
def test_far_apart_steps():
    """Offsets beyond 32 bits of elements."""
    far = 2 ** 31 + 8
    base = torch.zeros(far + 64, dtype=torch.bfloat16, device="cuda")
    q = base.as_strided((2, 1, 1, 64), (far, 64, 64, 1))
    q.copy_(torch.randn(2, 1, 1, 64))
    _, k, v, g, dn, s, do, df = _inputs(2, 1, 1, 64, 64, torch.bfloat16)
    ref = linear_attention(q.contiguous(), k, v, g, done=dn, state=s)
    got = linear_attention(q, k, v, g, done=dn, state=s)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [60, 130, 600])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_non_finite_stays_where_it_belongs(dtype, T, value):
    """Earlier steps, later episodes and other heads do not see it."""
    q, k, v, g, _, s, _, _ = _inputs(T, 2, 2, 32, 32, dtype)
    d = torch.zeros(T, 2, dtype=torch.bool, device="cuda")
    bad, cut = T // 3, T // 3 + 9
    d[cut] = True
    clean, fin = linear_attention(q, k, v, g, done=d, state=s)
    for name in "qkv":
        t = dict(q=q, k=k, v=v)
        t[name] = t[name].clone()
        t[name][bad, 0, 1, 5] = value
        out, f = linear_attention(t["q"], t["k"], t["v"], g, done=d, state=s)
        assert not out[bad, 0, 1].isfinite().all()
        o, c = out.clone(), clean.clone()
        o[bad:cut, 0, 1] = 0
        c[bad:cut, 0, 1] = 0
        assert o.isfinite().all() and f.isfinite().all()
        half = torch.finfo(dtype).eps
        torch.testing.assert_close(o, c, rtol=4 * half, atol=1e-3)
        torch.testing.assert_close(f, fin, rtol=1e-4, atol=1e-3)
        # and it reaches exactly the steps that the recurrence carries it to
        ref = _ref(t["q"], t["k"], t["v"], g, d, s, 32 ** -0.5)[0]
        assert torch.equal(out.isfinite().cpu(), ref.isfinite())


@pytest.mark.gpu
@pytest.mark.parametrize("T", [60, 600])
@pytest.mark.parametrize("dtype", [torch.bfloat16, HALF])
def test_non_finite_gradients_stay(T, dtype):
    q, k, v, g, _, s, do, df = _inputs(T, 2, 2, 32, 32, dtype)
    d = torch.zeros(T, 2, dtype=torch.bool, device="cuda")
    cut = T // 2
    d[cut] = True
    clean = _run(q, k, v, g, d, s, do, df)
    do2 = do.clone()
    do2[cut + 3, 0, 1, 5] = float("nan")
    got = _run(q, k, v, g, d, s, do2, df)
    for n, a, c in zip(NAMES[2:5], got[2:5], clean[2:5]):
        assert a[:cut].isfinite().all(), n
        assert a[cut + 4:].isfinite().all(), n
        assert not a[cut + 3, 0, 1].isfinite().all(), n
        torch.testing.assert_close(a[:cut], c[:cut], rtol=0.02, atol=1e-2)
    assert got[5].isfinite().all()


def _same_where_finite(got, ref, mag, rel, what):
    """Finite at the same places, and close there."""
    ok = ref.isfinite()
    assert torch.equal(got.isfinite().cpu(), ok), what
    z = torch.zeros_like(ref)
    _close(torch.where(ok.to(got.device), got, torch.zeros_like(got)),
           torch.where(ok, ref, z), torch.where(ok, mag, z), rel, what)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ["q", "k", "v", "s", "do", "df"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_non_finite_crosses_segments(dtype, name, value):
    """A decay that underflows over a segment is no done: what is not finite
    stays so over all later segments, up to the next done."""
    T, D = 600, 16
    q, k, v, g, _, s, do, df = _inputs(T, 1, 2, D, D, dtype, 0)
    g = torch.tensor([-3.0, -0.01], device="cuda")
    d = torch.zeros(T, 1, dtype=torch.bool, device="cuda")
    a = dict(q=q, k=k, v=v, s=s, do=do, df=df)
    mag = _ref(q.abs(), k.abs(), v.abs(), g, d, s.abs(), 0.25, do.abs(),
               df.abs())
    full, rel = _bounds(dtype, T, D, D)
    a[name] = a[name].clone()
    if name in ("s", "df"):
        a[name][0, 0, 5, 3] = value
    else:
        a[name][T - 70 if name == "do" else 70, 0, 0, 5] = value
    for cut in (None, 130, T - 130):
        if cut is not None:
            d[cut] = True
        got = _run(a["q"], a["k"], a["v"], g, d, a["s"], a["do"], a["df"])
        ref = _ref(a["q"], a["k"], a["v"], g, d, a["s"], 0.25, a["do"],
                   a["df"])
        for n, x, r, m in zip(NAMES, got, ref, mag):
            _same_where_finite(x, r, m,
                               rel if n in ("final", "dstate") else full, n)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [40, 150, 600])
@pytest.mark.parametrize("D", [16, 48, 128])
@pytest.mark.parametrize("e", [40, 60])
def test_fp16_zero_columns_under_a_large_scale(T, D, e):
    """Columns of zeros have no size to be scaled by: a scale far beyond
    fp16's range leaves them zero.

    q and do lie among fp16's subnormals, whose products the matrix
    instruction adds at the place of 2^-14: a subnormal's exponent field is
    that of 2^-14, and nothing moves its leading zeros out. The sums' roundings
    are then those of magnitudes of 2^-14 or more (measured over 32 products
    of operands of 2^-20: 2^-19.5 of their magnitudes' sum, 2^-23.6 of normal
    ones), so the bound's magnitudes are taken so."""
    q, k, v, g, d, s, do, df = _inputs(T, 1, 2, D, D, torch.float32, 0.01)
    q, k, v, do = ((t * 2.0 ** x).half()
                   for t, x in ((q, -20), (k, -10), (v, 20 - e // 2 - 10),
                                (do, -20)))
    do[..., ::2] = 0
    k[..., 1::2] = 0
    v[..., 1::3] = 0
    s[..., 1::3] = 0
    df[..., ::2] = 0
    got = _run(q, k, v, g, d, s, do, df, scale=2.0 ** e)
    ref = _ref(q, k, v, g, d, s, 2.0 ** e, do, df)
    mag = _ref(*(torch.where(t == 0, 0, t.abs().clamp_min(2.0 ** -14))
                 for t in (q, k, v)), g, d, s.abs(), 2.0 ** e,
               torch.where(do == 0, 0, do.abs().clamp_min(2.0 ** -14)),
               df.abs())
    full, rel = _bounds(q.dtype, T, D, D)
    for n, x, r, m in zip(NAMES, got, ref, mag):
        _close(x, r, m, rel if n in ("final", "dstate") else full, n)
        assert not x[(m == 0).to(x.device)].any(), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 128])
@pytest.mark.parametrize("g", [1.0, 1.395, 3.0, 80.0])
@pytest.mark.parametrize("T", [64, 600])
def test_growing_zeros(dtype, D, g, T):
    """Decays above zero, whose powers overflow: zeros stay zeros."""
    q, k, v, _, d, s, do, df = (
        torch.zeros_like(t) for t in _inputs(T, 1, 2, D, D, dtype))
    g = torch.tensor([g, -0.1], device="cuda")
    for n, x in zip(NAMES, _run(q, k, v, g, d, s, do, df)):
        assert not x.any(), n
    for n, x in zip(NAMES, _run(q, k, v, g, None, None, do, None)):
        assert not x.any(), n


@pytest.mark.gpu
@pytest.mark.parametrize("g,T", [(0.02, 1500), (0.5, 150), (1.395, 63),
                                 (1.395, 64), (3.0, 28)])
@pytest.mark.parametrize("D", [16, 128])
@pytest.mark.parametrize("state", [False, True])
def test_growing_states(g, T, D, state):
    """Results within 32 bits where a decay's powers are not. Step by step a
    contribution is rounded twice a step and scaled by a decay that is off by
    two more, which 4 T more roundings cover."""
    a = _inputs(T, 1, 2, D, D, torch.float32, 0.02, state)
    for i in (0, 1, 5, 7):   # q, k and the states
        if a[i] is not None:
            a[i] = a[i] * 2.0 ** -20
    a[3] = torch.tensor([g, -0.1], device="cuda")
    q, k, v, g, d, s, do, df = a
    got = _run(*a, scale=0.25)
    ref = _ref(q, k, v, g, d, s, 0.25, do, df)
    mag = _ref(q.abs(), k.abs(), v.abs(), g, d,
               None if s is None else s.abs(), 0.25, do.abs(),
               None if df is None else df.abs())
    rel = _bounds(q.dtype, T, D, D)[1] + 4 * T * U
    for n, x, r, m in zip(NAMES, got, ref, mag):
        _close(x, r, m, rel, n)


@pytest.mark.gpu
def test_nothing_to_do():
    for T, B, H in ((0, 2, 3), (4, 0, 3), (4, 2, 0)):
        q, k, v, g, d, s, do, df = _inputs(T, B, H, 4, 5, torch.float32)
        got = _run(q, k, v, g, d, s, do, df)
        assert got[0].shape == (T, B, H, 5)
        if T == 0:
            assert torch.equal(got[1], s) and torch.equal(got[5], df)
    q, k, v, g, d, _, _, _ = _inputs(0, 2, 3, 4, 5, torch.float32)
    assert not linear_attention(q, k, v, g)[1].any()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [50, 600])
def test_gradients_through_one_result_only(T):
    q, k, v, g, d, s, do, df = _inputs(T, 2, 2, 16, 16, torch.float32)
    ref = _ref(q, k, v, g, d, s, 0.25, do, None)
    mag = _ref(q.abs(), k.abs(), v.abs(), g, d, s.abs(), 0.25, do.abs())
    full, rel = _bounds(q.dtype, T, 16, 16)
    ins = [t.detach().requires_grad_() for t in (q, k, v, s)]
    out, fin = linear_attention(*ins[:3], g, done=d, state=ins[3])
    for n, a, r, m in zip(NAMES[2:], torch.autograd.grad(out, ins, do),
                          ref[2:], mag[2:]):
        _close(a, r, m, full, n)
    z = torch.zeros_like(do)
    ref = _ref(q, k, v, g, d, s, 0.25, z, df)
    mag = _ref(q.abs(), k.abs(), v.abs(), g, d, s.abs(), 0.25, z, df.abs())
    out, fin = linear_attention(*ins[:3], g, done=d, state=ins[3])
    for n, a, r, m in zip(NAMES[2:], torch.autograd.grad(fin, ins, df),
                          ref[2:], mag[2:]):
        _close(a, r, m, full, n)


@pytest.mark.gpu
def test_gradient_against_differences():
    q, k, v, g, d, s, do, df = _inputs(70, 1, 1, 4, 4, torch.float32)
    got = _run(q, k, v, g, d, s, do, df)[2:]

    def loss(q, k, v, s):
        out, fin = linear_attention(q, k, v, g, done=d, state=s)
        return ((out.double() * do.double()).sum()
                + (fin.double() * df.double()).sum())

    # linear in each input alone: no truncation, only roundings, which a
    # step of 1/2 keeps at 2^-24 times the magnitudes' sum
    args = [q, k, v, s]
    mag = _ref(q.abs(), k.abs(), v.abs(), g, d, s.abs(), 0.5, do.abs(),
               df.abs())
    size = float((mag[0] * do.abs().double().cpu()).sum()
                 + (mag[1] * df.abs().double().cpu()).sum())
    for i, a in enumerate(args):
        e = torch.randn_like(a)
        hi, lo = list(args), list(args)
        hi[i], lo[i] = a + 0.5 * e, a - 0.5 * e
        num = float(loss(*hi) - loss(*lo))
        ana = float((got[i].double() * e.double()).sum())
        assert abs(num - ana) <= 300 * U * 8 * size


@pytest.mark.gpu
def test_repeatable_on_streams_and_two_at_once():
    a = _inputs(600, 2, 2, 32, 32, torch.bfloat16)
    b = _inputs(600, 2, 2, 32, 32, torch.bfloat16, seed=9)
    ra, rb = _run(*a), _run(*b)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s1):
        ga = _run(*a)
    with torch.cuda.stream(s2):
        gb = _run(*b)
    torch.cuda.synchronize()
    for x, y in zip(ra + rb, ga + gb):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [21, 600])
def test_captured(T):
    a = _inputs(T, 4, 2, 32, 32, torch.float32)
    buf = [t.clone() for t in a]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _run(*buf)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = _run(*buf)
    for seed in (3, 4, 5):
        new = _inputs(T, 4, 2, 32, 32, torch.float32, seed=seed)
        for x, y in zip(buf, new):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        for n, x, y in zip(NAMES, res, _run(*new)):
            assert torch.equal(x, y), n


@pytest.mark.gpu
def test_saved_input_changed_in_place():
    q, k, v, g, d, s, do, df = _inputs(9, 1, 1, 8, 8, torch.float32)
    q.requires_grad_()
    z = k * 1.0
    out, _ = linear_attention(q, z, v, g)
    z.add_(1.0)
    with pytest.raises(RuntimeError):
        out.sum().backward()


@pytest.mark.gpu
def test_differentiable_once():
    q, k, v, g, d, s, do, df = _inputs(9, 1, 1, 8, 8, torch.float32)
    q.requires_grad_()
    out, _ = linear_attention(q, k, v, g, done=d, state=s)
    gq, = torch.autograd.grad(out.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        gq.sum().backward()


@pytest.mark.gpu
def test_one_tensor_in_all_places():
    _, _, _, g, d, s, do, df = _inputs(70, 2, 2, 16, 16, torch.float32)
    x = torch.randn(70, 2, 2, 16, device="cuda")
    a = x.clone().requires_grad_()
    out, _ = linear_attention(a, a, a, g, done=d, state=s)
    got, = torch.autograd.grad(out, a, do)
    full = _run(x, x, x, g, d, s, do, None)
    torch.testing.assert_close(got, full[2] + full[3] + full[4],
                               rtol=1e-5, atol=1e-4)


@pytest.mark.gpu
def test_gradient_of_a_sum():
    """The output's gradient comes as a broadcast view of one number."""
    a = _inputs(70, 2, 2, 16, 16, torch.float32)
    q, k, v, g, d, s, do, df = a
    ins = [t.clone().requires_grad_() for t in (q, k, v)]
    out, _ = linear_attention(*ins, g, done=d, state=s)
    got = torch.autograd.grad(out.sum(), ins)
    ref = _run(q, k, v, g, d, s, torch.ones_like(do), None)
    for x, y in zip(got, ref[2:5]):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_flags_far_apart():
    """Flags whose steps lie more than 2^25 bytes apart."""
    T, far = 70, 2 ** 25 + 3
    q, k, v, g, d, s, _, _ = _inputs(T, 1, 1, 8, 8, torch.float32)
    base = torch.zeros(far * T, dtype=torch.bool, device="cuda")
    d2 = base.as_strided((T, 1), (far, 1))
    d2.copy_(d)
    ref = linear_attention(q, k, v, g, done=d, state=s)
    got = linear_attention(q, k, v, g, done=d2, state=s)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


# --------------------------------------------------------------- one step
@pytest.mark.gpu
@pytest.mark.parametrize("dk,dv", [(1, 1), (5, 3), (8, 4), (64, 64),
                                   (48, 80), (128, 128), (128, 127),
                                   (7, 128)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_step(dk, dv, dtype):
    q, k, v, g, d, s, _, _ = _inputs(1, 5, 3, dk, dv, dtype, 0.4)
    sc = dk ** -0.5
    ref = _ref(q, k, v, g, d, s, sc)
    mag = _ref(q.abs(), k.abs(), v.abs(), g, d, s.abs(), sc)
    out, new = linear_attention_step(q[0], k[0], v[0], g, s, done=d[0])
    _close(out, ref[0][0], mag[0][0], (dk + 16) * U, "out")
    _close(new, ref[1], mag[1], 16 * U, "state")
    buf = s.clone()
    out2, r = linear_attention_step(q[0], k[0], v[0], g, buf, done=d[0],
                                    out_state=buf)
    assert r is buf and torch.equal(buf, new) and torch.equal(out2, out)


@pytest.mark.gpu
def test_step_in_a_pool():
    """Environments of a larger pool: the rows around stay as they were."""
    q, k, v, g, d, s, _, _ = _inputs(1, 4, 2, 16, 20, torch.float32, 0.3)
    pool = torch.randn(4, 3, 2, 16, 20, device="cuda")
    pool[:, 1] = s
    before = pool.clone()
    out, _ = linear_attention_step(q[0], k[0], v[0], g, pool[:, 1],
                                   done=d[0], out_state=pool[:, 1])
    ref, new = linear_attention_step(q[0], k[0], v[0], g, s, done=d[0])
    assert torch.equal(out, ref) and torch.equal(pool[:, 1], new)
    assert torch.equal(pool[:, 0], before[:, 0])
    assert torch.equal(pool[:, 2], before[:, 2])
    # one state for all environments, read as a broadcast view
    one = s[:1].expand(4, 2, 16, 20)
    o1, n1 = linear_attention_step(q[0], k[0], v[0], g, one, done=d[0])
    o2, n2 = linear_attention_step(q[0], k[0], v[0], g, one.contiguous(),
                                   done=d[0])
    assert torch.equal(o1, o2) and torch.equal(n1, n2)


@pytest.mark.gpu
def test_steps_follow_the_unroll():
    """An unroll's results are those of its steps one by one."""
    T = 90
    q, k, v, g, d, s, _, _ = _inputs(T, 3, 2, 32, 32, torch.float32)
    out, fin = linear_attention(q, k, v, g, done=d, state=s)
    st = s.clone()
    mag = _ref(q.abs(), k.abs(), v.abs(), g, d, s.abs(), 32 ** -0.5)
    full, rel = _bounds(q.dtype, T, 32, 32)
    for t in range(T):
        o, st = linear_attention_step(q[t], k[t], v[t], g, st, done=d[t],
                                      out_state=st)
        _close(o, out[t].double().cpu(), mag[0][t], 2 * full + T * U, "out")
    _close(st, fin.double().cpu(), mag[1], 2 * rel + T * U, "final")


@pytest.mark.gpu
def test_step_done_drops_a_poisoned_state():
    q, k, v, g, _, s, _, _ = _inputs(1, 2, 2, 16, 16, torch.float32)
    s[0] = float("nan")
    d = torch.tensor([True, False], device="cuda")
    out, new = linear_attention_step(q[0], k[0], v[0], g, s, done=d)
    assert out.isfinite().all() and new.isfinite().all()


@pytest.mark.gpu
def test_step_empty_and_captured():
    g = torch.zeros(2, device="cuda")
    e = torch.zeros(0, 2, 4, device="cuda")
    out, new = linear_attention_step(e, e, e, g,
                                     torch.zeros(0, 2, 4, 4, device="cuda"))
    assert out.shape == (0, 2, 4) and new.shape == (0, 2, 4, 4)
    q, k, v, g, d, s, _, _ = _inputs(1, 4, 2, 32, 32, torch.float32)
    st = s.clone()
    st0 = torch.cuda.Stream()
    st0.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st0):
        linear_attention_step(q[0], k[0], v[0], g, s, done=d[0])
    torch.cuda.current_stream().wait_stream(st0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = linear_attention_step(q[0], k[0], v[0], g, st, done=d[0],
                                       out_state=st)
    st.copy_(s)
    ref = s
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        o, ref = linear_attention_step(q[0], k[0], v[0], g, ref, done=d[0])
        assert torch.equal(out, o) and torch.equal(st, ref)

"""FlatMuon: orthogonalised momentum for matrices, RMSProp for the rest.

The reference computes a step in 64 bits from the same gradients. A step's
own roundings in 32 bits are 2^-24 of what they round; five Newton-Schulz
rounds enlarge an error of their input, 485 times at most, and add the
products' own (tests/test_orthogonal.py bounds both by 1e-4 of the update's
norm times the number of rounds' products at these sizes). The update enters
the weights times the rate.
"""
import math
import os
import queue

import pytest
import torch

from torched_impala_amd.models import MLPPolicy, ShallowNet
from torched_impala_amd.ops.optim import (FlatMuon, FlatRMSprop,
                                          muon_matrices)
from torched_impala_amd.ops.orthogonal import COEFFICIENTS

LR, MUON_LR, MU, ALPHA, EPS = 0.01, 0.02, 0.9, 0.99, 0.01


def _ns(g, steps=5):
    a, b, c = COEFFICIENTS
    x = g / (torch.linalg.vector_norm(g) + 1e-7)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    for _ in range(steps):
        m = x @ x.T
        x = a * x + (b * m + c * m @ m) @ x
    return x.T if tall else x


class _Ref:
    def __init__(self, model, max_norm, world=1):
        self.mats = {id(p) for p in muon_matrices(model)}
        self.params = list(model.parameters())
        self.w = [p.detach().double().cpu().clone() for p in self.params]
        self.s = [torch.zeros_like(w) for w in self.w]
        self.max_norm, self.world = max_norm, world

    def step(self, grads):
        g = [x.detach().double().cpu() / self.world for x in grads]
        norm = math.sqrt(sum(float((x * x).sum()) for x in g))
        c = min(1.0, self.max_norm / (norm + 1e-6))
        for i, p in enumerate(self.params):
            x = g[i] * c
            if id(p) in self.mats:
                self.s[i] = MU * self.s[i] + x
                u = (x + MU * self.s[i]).reshape(x.shape[0], -1)
                r = max(1.0, u.shape[0] / u.shape[1]) ** 0.5
                self.w[i] -= MUON_LR * r * _ns(u).reshape(x.shape)
            else:
                self.s[i] = ALPHA * self.s[i] + (1 - ALPHA) * x * x
                self.w[i] -= LR * x / (self.s[i].sqrt() + EPS)


def _make(net, max_norm, world=1):
    return FlatMuon(net.parameters(), muon_matrices(net), lr=LR, alpha=ALPHA,
                    eps=EPS, max_grad_norm=max_norm, world_size=world,
                    muon_lr=MUON_LR, muon_momentum=MU)


def _steps(net, max_norm, world=1, n=3):
    opt, ref = _make(net, max_norm, world), _Ref(net, max_norm, world)
    for k in range(n):
        gen = torch.Generator().manual_seed(k)
        opt.zero_grad()
        grads = []
        for p in net.parameters():
            x = torch.randn(p.shape, generator=gen)
            p.grad.copy_(x)
            grads.append(x)
        opt.step()
        ref.step(grads)
        for (name, p), w in zip(net.named_parameters(), ref.w):
            err = float(torch.linalg.vector_norm(p.double().cpu() - w))
            size = float(torch.linalg.vector_norm(w))
            rows = min(p.shape[0], p[0].numel()) if p.dim() > 1 else 1
            lim = (k + 1) * (2.0 ** -22 * size + 1e-4 * MUON_LR * math.sqrt(
                rows) * 16 + 1e-6 * math.sqrt(p.numel()) * LR * 64)
            assert err <= lim, (name, k, err, lim)
    return opt


def test_against_64_bits_cpu():
    torch.manual_seed(0)
    _steps(MLPPolicy((4,), 2, use_lstm=True), 40.0)
    _steps(MLPPolicy((4,), 2, use_linear_attention=True), 0.5, world=4)


def test_which_parameters():
    net = ShallowNet((4, 84, 84), 6, use_linear_attention=True)
    names = {id(p): n for n, p in net.named_parameters()}
    got = {names[id(p)] for p in muon_matrices(net)}
    assert got == {"conv1.weight", "conv2.weight", "conv3.weight",
                   "fc.weight", "core.proj_in.weight", "core.qkv.weight",
                   "core.proj_out.weight"}
    opt = _make(net, 40.0)
    n = sum(p.numel() for p in net.parameters())
    assert opt.flat_param.numel() == n
    covered = sorted(opt.slices.values())
    assert covered[0][0] == 0 and all(
        a + k == b for (a, k), (b, _) in zip(covered, covered[1:]))
    assert covered[-1][0] + covered[-1][1] == n
    with pytest.raises(AssertionError):
        FlatMuon(net.parameters(), [])
    with pytest.raises(AssertionError):
        FlatMuon(net.parameters(), [net.fc.bias])
    with pytest.raises(AssertionError):
        FlatMuon([net.fc.bias], [net.fc.weight])


def test_non_finite_step_is_skipped_cpu():
    _skip("cpu")


def _skip(device):
    torch.manual_seed(0)
    net = MLPPolicy((4,), 2, use_lstm=True).to(device)
    opt = _steps(net, 40.0, n=1) if device == "cpu" else _make(net, 40.0)
    opt.zero_grad()
    for p in net.parameters():
        p.grad.normal_()
    opt.step()
    before = [t.clone() for t in opt.state_arenas()]
    next(net.parameters()).grad.view(-1)[0] = float("nan")
    opt.step()
    for a, b in zip(before, opt.state_arenas()):
        assert torch.equal(a, b)
    assert float(opt.skip_t) == 1.0


def test_state_dict_roundtrip():
    torch.manual_seed(0)
    a = MLPPolicy((4,), 2, use_lstm=True)
    oa = _steps(a, 40.0, n=2)
    sd = oa.state_dict()
    b = MLPPolicy((4,), 2, use_lstm=True)
    b.load_state_dict(a.state_dict())
    ob = _make(b, 40.0)
    ob.load_state_dict(sd)
    for net, opt in ((a, oa), (b, ob)):
        opt.zero_grad()
        gen = torch.Generator().manual_seed(9)
        for p in net.parameters():
            p.grad.copy_(torch.randn(p.shape, generator=gen))
        opt.step()
    for x, y in zip(a.parameters(), b.parameters()):
        assert torch.equal(x, y)
    with pytest.raises(ValueError):
        ob.load_state_dict(FlatRMSprop(MLPPolicy((4,), 2).parameters())
                           .state_dict())


def _state_of(opt):
    return ([t.clone() for t in opt.state_arenas()], opt._steps,
            [{k: v for k, v in g.items() if k != "params"}
             for g in opt.param_groups])


@pytest.mark.parametrize("make", [
    lambda net: FlatRMSprop(net.parameters(), lr=0.5),
    lambda net: _make(net, 40.0)])
def test_a_state_that_does_not_fit_changes_nothing(make):
    """States of the other optimizer, of another net and damaged ones are
    refused by name before the first average is overwritten."""
    torch.manual_seed(0)
    net = MLPPolicy((4,), 2, use_lstm=True)
    opt = make(net)
    opt.flat_sqavg.normal_()
    muon = isinstance(opt, FlatMuon)
    other = MLPPolicy((5,), 2, use_lstm=True)
    states = [make(other).state_dict(),
              FlatRMSprop(net.parameters()).state_dict() if muon
              else _make(net, 40.0).state_dict()]
    opt = make(net)   # the arenas are the last optimizer's that was made
    opt.flat_sqavg.normal_()
    damaged = opt.state_dict()
    last = damaged["state"][len(damaged["state"]) - 1]
    last.pop("momentum_buffer" if muon else "square_avg")
    for sd in states + [damaged]:
        before = _state_of(opt)
        with pytest.raises(ValueError):
            opt.load_state_dict(sd)
        after = _state_of(opt)
        assert all(torch.equal(a, b) for a, b in zip(before[0], after[0]))
        assert before[1:] == after[1:]


def _train_rank(rank, world, port, q):
    """Three steps of a linear-attention policy on this rank's half of the
    batch (world 2) or on all of it (world 1)."""
    from torched_impala_amd.parallel import FlatGradReducer
    if world > 1:
        os.environ["MASTER_ADDR"] = "127.0.0.1"
        os.environ["MASTER_PORT"] = str(port)
        torch.distributed.init_process_group("gloo", rank=rank,
                                             world_size=world)
    try:
        torch.manual_seed(0)
        net = MLPPolicy((4,), 2, use_linear_attention=True)
        opt = FlatMuon(net.parameters(), muon_matrices(net), lr=0.01,
                       max_grad_norm=1e6, world_size=world, muon_lr=0.02)
        red = FlatGradReducer(net, opt, bucket_bytes=1 << 14)
        for it in range(3):
            torch.manual_seed(50 + it)
            x, done = torch.randn(5, 4, 4), torch.rand(5, 4) < 0.2
            mine = slice(2 * rank, 2 * rank + 2) if world > 1 else slice(0, 4)
            n = mine.stop - mine.start
            inputs = dict(frame=x[:, mine], reward=torch.zeros(5, n),
                          done=done[:, mine],
                          last_action=torch.zeros(5, n, dtype=torch.long))
            opt.zero_grad()
            red.prepare()
            out, _ = net(inputs, net.initial_state(n))
            ((out["policy_logits"].pow(2).sum()
              + out["baseline"].pow(2).sum()) * (world / 2)).backward()
            red.finalize()
            opt.step()
        q.put((rank, opt.flat_param.detach().numpy().copy()))
    finally:
        if world > 1:
            torch.distributed.destroy_process_group()


@pytest.mark.timeout(180)
def test_two_ranks_as_one():
    """Data parallel over two ranks: the ranks end with the same bits, and
    with what one process gets from the whole batch (its loss halved, as the
    ranks' mean is). The sums differ in order only: 20 rows through 8 layers
    are 2^-19 of a gradient's norm at most. A step's products enlarge that 485
    times, at a rate of 0.02; RMSProp moves by at most the error over eps =
    0.01 at a rate of 0.01, with norms up to 10. Over three steps together
    under 1.2e-4; a rank left out would move weights by 0.02."""
    ctx = torch.multiprocessing.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_train_rank, args=(r, 2, 29643, q))
             for r in range(2)]
    for p in procs:
        p.start()
    got = dict(q.get(timeout=120) for _ in range(2))
    for p in procs:
        p.join(timeout=30)
    assert (got[0] == got[1]).all()
    alone = queue.Queue()
    _train_rank(0, 1, 0, alone)
    torch.testing.assert_close(
        torch.from_numpy(got[0]), torch.from_numpy(alone.get()[1]),
        rtol=0, atol=1.2e-4)


@pytest.mark.gpu
def test_against_64_bits_gpu():
    torch.manual_seed(0)
    _steps(MLPPolicy((4,), 2, use_lstm=True).cuda(), 40.0)
    _steps(MLPPolicy((4,), 2, use_linear_attention=True).cuda(), 0.5,
           world=4)
    _steps(ShallowNet((4, 84, 84), 6, use_lstm=True).cuda(), 40.0)


@pytest.mark.gpu
def test_non_finite_step_is_skipped_gpu():
    _skip("cuda")


@pytest.mark.gpu
def test_equal_gradients_give_equal_weights():
    """Ranks hold the same gradients and each computes its own update: the
    weights must not drift apart by the order in which a norm is added."""
    torch.manual_seed(0)
    net = ShallowNet((4, 84, 84), 6, use_lstm=True).cuda()
    opt = _make(net, 0.5)
    opt.zero_grad()
    opt.flat_grad.normal_()
    opt.sync_lr()
    start = [t.clone() for t in opt.state_arenas()]
    first = None
    for _ in range(40):
        for t, was in zip(opt.state_arenas(), start):
            t.copy_(was)
        opt.step_device()
        got = [opt.norm_sq] + opt.state_arenas()
        if first is None:
            first = [t.clone() for t in got]
            want = float(opt.flat_grad.double().square().sum())
            assert abs(float(opt.norm_sq) / want - 1) < 1e-5
        assert all(torch.equal(a, b) for a, b in zip(got, first))


@pytest.mark.gpu
def test_captured_step():
    torch.manual_seed(0)
    nets = [MLPPolicy((4,), 2, use_lstm=True).cuda() for _ in range(2)]
    nets[1].load_state_dict(nets[0].state_dict())
    opts = [_make(n, 40.0) for n in nets]
    s = torch.cuda.Stream()
    for o in opts:
        o.zero_grad()
    snap = [t.clone() for t in opts[0].state_arenas()]
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        opts[0].step_device()
    torch.cuda.current_stream().wait_stream(s)
    for t, was in zip(opts[0].state_arenas(), snap):
        t.copy_(was)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opts[0].step_device()
    for t, was in zip(opts[0].state_arenas(), snap):
        t.copy_(was)
    for k in range(3):
        g = torch.randn_like(opts[0].flat_grad)
        for o in opts:
            o.flat_grad.copy_(g)
            for group in o.param_groups:   # the rates move between steps
                group["lr"] *= 0.9
        opts[0].sync_lr()
        graph.replay()
        torch.cuda.synchronize()
        opts[1].step()
        # the global norm is added by atomics, so its last bit may differ
        # between two runs: 2^-22 of the clipped gradients, enlarged 485
        # times at most, times the rate and the entries' size of one
        torch.testing.assert_close(opts[0].flat_param, opts[1].flat_param,
                                   rtol=1e-5, atol=485 * 2.0 ** -22 * 0.02)

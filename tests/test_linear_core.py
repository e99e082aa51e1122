"""The linear-attention core in the policy nets, and its operators in a run:
projection, norm, attention, norm per head, and the updates of the matrices.

Where two computations in 32 bits are compared, the tolerance counts their
roundings in sequence: a projection over up to 263 features, a norm over 256,
a projection over 256, an attention of up to 64 + 64 + 64 + 6 a chunk, a norm
over 64 and a projection over 256, about 1300 half steps of 2^-24 on either
side; the two norms divide by a spread and so enlarge what lies in front of
them, by 8 together at these inputs: 2 * 8 * 1300 * 2^-24 = 1.3e-3 of the
result's size at worst.
"""
import pytest
import torch

from torched_impala_amd import learner as L
from torched_impala_amd.actor import Rollout
from torched_impala_amd.config import Flags, flags_from_args
from torched_impala_amd.models import (DeepResNet, MLPPolicy, ShallowNet,
                                       build_model)
from torched_impala_amd.models.core import LinearAttentionCore
from torched_impala_amd.ops.optim import FlatMuon
from torched_impala_amd.transport import TrajectoryBuffers

REL = 1.3e-3


def _near(a, b, rel=REL):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    assert a.shape == b.shape
    err = float(torch.linalg.vector_norm(a - b))
    assert err <= rel * float(torch.linalg.vector_norm(b)) + 1e-12, err


def _inputs(T, B, obs, A, device="cpu", seed=0, dtype=None):
    g = torch.Generator().manual_seed(seed)
    frame = (torch.randn(T, B, *obs, generator=g) if len(obs) == 1 else
             torch.randint(0, 256, (T, B, *obs), dtype=torch.uint8,
                           generator=g))
    inp = dict(frame=frame, reward=torch.randn(T, B, generator=g),
               done=torch.rand(T, B, generator=g) < 0.1,
               last_action=torch.randint(0, A, (T, B), generator=g))
    return {k: v.to(device) for k, v in inp.items()}


def _ref_core(core, x, done, state):
    """The core's formulas in 64 bits."""
    p = {k: v.detach().double().cpu().requires_grad_()
         for k, v in core.named_parameters()}
    T, B = x.shape[:2]
    H, D = core.heads, core.head_size

    def norm(t, w, b, eps):
        d = t - t.mean(-1, keepdim=True)
        return d / torch.sqrt((d * d).mean(-1, keepdim=True) + eps) * w + b

    x = x.detach().double().cpu().requires_grad_()
    z = x @ p["proj_in.weight"].T + p["proj_in.bias"]
    y = norm(z, p["norm.weight"], p["norm.bias"], core.norm.eps)
    q, k, v = (y @ p["qkv.weight"].T).view(T, B, 3, H, D).unbind(2)
    lam = core.log_decay.double().cpu().exp().view(1, H, 1, 1)
    live = (~done).double().cpu()
    s = state.detach().double().cpu().view(B, H, D, D)
    outs = []
    for t in range(T):
        s = lam * live[t].view(B, 1, 1, 1) * s \
            + k[t][..., :, None] * v[t][..., None, :]
        outs.append((q[t][..., :, None] * s).sum(-2) * D ** -0.5)
    o = norm(torch.stack(outs), p["head_norm.weight"], p["head_norm.bias"],
             core.head_norm.eps)
    out = z + o.flatten(-2) @ p["proj_out.weight"].T + p["proj_out.bias"]
    return out.reshape(T * B, -1), s.reshape(B, -1), x, p


def _core_against_ref(device, T, B):
    torch.manual_seed(T)
    core = LinearAttentionCore(263)
    with torch.no_grad():
        for n in (core.norm, core.head_norm):
            n.weight.add_(0.2 * torch.randn_like(n.weight))
            n.bias.add_(0.2 * torch.randn_like(n.bias))
    core = core.to(device)
    x = torch.randn(T, B, 263).to(device).requires_grad_()
    done = (torch.rand(T, B) < 0.05).to(device)
    state = torch.randn(B, core.state_size).to(device)
    out, (s,) = core(x, done, (state,))
    ro, rs, rx, rp = _ref_core(core, x, done, state)
    _near(out, ro)
    _near(s, rs)
    d = torch.randn(T * B, 256)
    names = [n for n, _ in core.named_parameters()]
    got = torch.autograd.grad(out, [x] + list(core.parameters()),
                              d.to(device))
    ref = torch.autograd.grad(ro, [rx] + [rp[n] for n in names], d.double())
    for a, b in zip(got, ref):
        _near(a, b, 4 * REL)   # backward walks the chain a second time


def test_core_cpu():
    _core_against_ref("cpu", 21, 3)


@pytest.mark.parametrize("make,obs", [(MLPPolicy, (4,)),
                                      (ShallowNet, (4, 84, 84)),
                                      (DeepResNet, (3, 72, 96))])
def test_nets_shapes(make, obs):
    T, B, A = 4, 2, 6
    net = make(obs, A, use_linear_attention=True)
    out, core = net(_inputs(T, B, obs, A), net.initial_state(B))
    assert out["policy_logits"].shape == (T, B, A)
    assert out["baseline"].shape == (T, B)
    assert len(core) == 1 and core[0].shape == (B, 4 * 64 * 64)
    assert core[0].dtype is torch.float32


def test_parameter_names():
    names = set(ShallowNet((4, 84, 84), 6, use_linear_attention=True)
                .state_dict())
    for n in ("core.proj_in.weight", "core.norm.weight", "core.qkv.weight",
              "core.head_norm.bias", "core.proj_out.bias", "policy.weight"):
        assert n in names
    assert not any("log_decay" in n for n in names)


def test_one_core_only():
    with pytest.raises(ValueError):
        MLPPolicy((4,), 2, use_lstm=True, use_linear_attention=True)
    with pytest.raises(ValueError):
        LinearAttentionCore(8, hidden_size=30, heads=4)


def test_flags():
    f = flags_from_args(["--use-linear-attention", "--optimizer", "muon",
                         "--muon-learning-rate", "0.01"])
    assert f.use_linear_attention and f.optimizer == "muon"
    net = build_model(f, (4,), 2)
    opt, sched = L.build_optimizer(f, net)
    assert isinstance(opt, FlatMuon)
    assert opt.param_groups[1]["lr"] == 0.01
    with pytest.raises(ValueError):
        L.build_optimizer(Flags(optimizer="muon", momentum=0.5), net)
    with pytest.raises(ValueError):
        L.build_optimizer(Flags(optimizer="sgd"), net)


def test_done_resets_state():
    torch.manual_seed(0)
    T, B, A = 6, 2, 4
    net = MLPPolicy((4,), A, use_linear_attention=True).eval()
    inp = _inputs(T, B, (4,), A)
    inp["done"].zero_()
    inp["done"][3] = True
    with torch.no_grad():
        out, _ = net(inp, net.initial_state(B))
        tail, _ = net({k: v[3:] for k, v in inp.items()},
                      net.initial_state(B))
    torch.testing.assert_close(out["policy_logits"][3:],
                               tail["policy_logits"], rtol=1e-5, atol=1e-6)


def test_initial_state_replay():
    """The slot's stored state replays the actor's own rows."""
    torch.manual_seed(3)
    flags = Flags(env="synthetic-atari", envs_per_actor=2, seed=3,
                  use_linear_attention=True, actor_jit="native")
    model = build_model(flags, (4, 84, 84), 6).eval()
    roll = Rollout(flags, 0, model)
    assert roll.fast is None
    T = 5
    bufs = TrajectoryBuffers(T, (4, 84, 84), torch.uint8, 6, 2,
                             envs_per_slot=2, core_state=(1, 4 * 64 * 64))
    for m in (0, 1):
        roll.fill_slot(bufs.slot(m), T)
    s = bufs.slot(1)
    core = tuple(t.clone() for t in s["initial_core_state"].unbind(0))
    assert core[0].any()
    with torch.inference_mode():
        out, _ = model({k: s[k] for k in ("frame", "reward", "done",
                                          "last_action")}, core)
    torch.testing.assert_close(out["policy_logits"], s["behavior_logits"],
                               rtol=1e-5, atol=1e-6)


@pytest.mark.timeout(300)
@pytest.mark.parametrize("optimizer", ["rmsprop", "muon"])
def test_trains_from_actors(tmp_path, optimizer):
    flags = Flags(env="cartpole", num_actors=1, batch_size=2,
                  unroll_length=5, total_steps=1000, device="cpu",
                  use_linear_attention=True, optimizer=optimizer,
                  xpid="a", savedir=str(tmp_path), seed=7)
    stats = L.train(flags, max_learner_steps=3)
    assert stats["learner_steps"] == 3
    assert stats["total_loss"] == stats["total_loss"]
    stats = L.train(flags, max_learner_steps=1)       # resumes
    assert stats["step_frames"] == 4 * 10


def test_eval_entry():
    flags = Flags(env="cartpole", device="cpu", use_linear_attention=True)
    assert len(L.test(flags, num_episodes=1)["returns"]) == 1


# --------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("T,B", [(1, 5), (21, 32), (101, 4), (700, 1)])
def test_core_gpu(T, B):
    _core_against_ref("cuda", T, B)


@pytest.mark.gpu
def test_core_bf16_under_autocast():
    torch.manual_seed(0)
    core = LinearAttentionCore(263).cuda()
    x = torch.randn(50, 4, 263, device="cuda")
    done = torch.rand(50, 4, device="cuda") < 0.05
    state = core.initial_state(4)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out, (s,) = core(x, done, state)
        out.float().square().sum().backward()
    assert out.dtype is torch.bfloat16 and s.dtype is torch.float32
    ro, rs, _, _ = _ref_core(core, x, done, state[0])
    # the same chain with half a bf16 step a stage, six stages, times 8
    _near(out, ro, 8 * 6 * 2.0 ** -8)
    assert all(p.grad.isfinite().all() for p in core.parameters())


@pytest.mark.gpu
def test_acting_follows_the_unroll():
    """Single steps without gradients (the step kernel) against the unroll."""
    torch.manual_seed(1)
    T, B, A = 30, 6, 5
    net = MLPPolicy((4,), A, use_linear_attention=True).cuda()
    inp = _inputs(T, B, (4,), A, "cuda")
    out, (s,) = net(inp, net.initial_state(B))
    core = net.initial_state(B)
    rows = []
    with torch.no_grad():
        for t in range(T):
            o, core = net({k: v[t:t + 1] for k, v in inp.items()}, core)
            rows.append(o["policy_logits"])
    _near(torch.cat(rows), out["policy_logits"])
    _near(core[0], s)


@pytest.mark.gpu
def test_kernels_against_eager():
    torch.manual_seed(2)
    T, B, A = 21, 8, 6
    net = MLPPolicy((4,), A, use_linear_attention=True).cuda()
    inp = _inputs(T, B, (4,), A, "cuda")
    grads = []
    for eager in (False, True):
        net.force_eager_core = eager
        out, _ = net(inp, net.initial_state(B))
        loss = out["policy_logits"].square().sum() + out["baseline"].sum()
        grads.append((out["policy_logits"], torch.autograd.grad(
            loss, list(net.parameters()))))
    _near(grads[0][0], grads[1][0])
    for a, b in zip(grads[0][1], grads[1][1]):
        _near(a, b, 4 * REL)


class _StubBatcher:
    """Quacks like Batcher for GraphedStep: staging dict + _to_time_major."""

    def __init__(self, flags, staging):
        self.flags = flags
        self.k = flags.batch_size // flags.envs_per_actor
        self.staging = staging

    _to_time_major = L.Batcher._to_time_major


def _staging(flags, obs, A, seed):
    g = torch.Generator().manual_seed(seed)
    T, k, n = flags.unroll_length, flags.batch_size, 1
    st = dict(
        frame=torch.randn(k, T + 1, n, *obs, generator=g),
        reward=torch.randn(k, T + 1, n, generator=g),
        done=torch.rand(k, T + 1, n, generator=g) < 0.05,
        action=torch.randint(0, A, (k, T + 1, n), generator=g),
        last_action=torch.randint(0, A, (k, T + 1, n), generator=g),
        behavior_logits=torch.randn(k, T + 1, n, A, generator=g),
        episode_return=torch.zeros(k, T + 1, n),
        episode_step=torch.zeros(k, T + 1, n, dtype=torch.int32),
        initial_core_state=torch.randn(k, 1, n, 4 * 64 * 64, generator=g))
    return {a: b.cuda() for a, b in st.items()}


@pytest.mark.gpu
@pytest.mark.timeout(600)
@pytest.mark.parametrize("optimizer", ["rmsprop", "muon"])
def test_captured_learn_step(optimizer):
    """The whole step in a graph, two staging buffers in turns with work of
    the host between replays, against eager steps on the same batches."""
    obs, A = (4,), 6
    flags = Flags(env="cartpole", batch_size=8, unroll_length=20,
                  use_linear_attention=True, optimizer=optimizer,
                  total_steps=1 << 50)
    staging = {i: _staging(flags, obs, A, i) for i in (0, 1)}
    stub = _StubBatcher(flags, staging)

    def make():
        torch.manual_seed(42)
        model = build_model(flags, obs, A).cuda()
        return (model, *L.build_optimizer(flags, model))

    model_g, opt_g, sched_g = make()
    model_e, opt_e, sched_e = make()
    graphed = L.GraphedStep(flags, model_g, opt_g, stub)
    # the graph replays the eager kernels: what may differ is the order in
    # which library products add, 2^-24 times some hundred terms, which five
    # Newton-Schulz rounds enlarge up to 485 times in an update of norm
    # sqrt(rows) times the rate 0.02, step after step
    for n, i in enumerate((0, 1, 0, 1)):
        got = graphed.step(i, sched_g)
        torch.cuda.synchronize()
        ref = L.learn_step(flags, model_e, stub._to_time_major(staging[i]),
                           opt_e, sched_e, None)
        torch.cuda.synchronize()
        torch.testing.assert_close(got["total_loss"], ref["total_loss"],
                                   rtol=1e-3, atol=1e-2)
        for a, b in zip(opt_g.state_arenas(), opt_e.state_arenas()):
            _near(a, b, (n + 1) * 500 * 485 * 2.0 ** -24 * 0.02 * 16)
    assert float(opt_g.skip_t) == 0.0
    graphed.destroy()


@pytest.mark.gpu
@pytest.mark.timeout(600)
def test_learner_runs_on_gpu():
    flags = Flags(env="synthetic-atari", num_actors=2, batch_size=4,
                  unroll_length=6, total_steps=1 << 40, device="cuda",
                  use_linear_attention=True, optimizer="muon",
                  disable_checkpoint=True, seed=5)
    stats = L.train(flags, max_learner_steps=4)
    assert stats["learner_steps"] == 4
    assert stats["total_loss"] == stats["total_loss"]
    assert stats["graph_path_active"] and stats["grad_skip_count"] == 0.0

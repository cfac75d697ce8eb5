"""The list AdamW (PPO/optim.py) inside learn() and beside the update engine: what is clipped by which
norm, each step's values against the float64 restatement (optim_ref.py, with its per-value bounds),
and optimizer state that changes hands between the engine, the per-step paths and load_state_dict()."""
import copy

import pytest
import torch

import optim_ref as R
from test_optim_gpu import _before, _check_step

pytestmark = pytest.mark.gpu


def _adamw():
    from PPO.optim import AdamW
    return AdamW


def _ppo(make_optimizer, n=2037, k_epochs=3, mb=256, use_fused=False, use_graphs=False, **kw):
    """A discrete 4-observation PPO (seeded), and n transitions to learn from."""
    from PPO import PPO
    torch.manual_seed(0)
    ppo = PPO(False, 4, 2, lr=1e-3, k_epochs=k_epochs, batch_size=64, mini_batch_size=mb)
    ppo.show_progress, ppo.use_fused, ppo.use_graphs = False, use_fused, use_graphs
    for k, v in kw.items():
        setattr(ppo, k, v)
    if make_optimizer is not None:
        ppo.optimizer = make_optimizer(list(ppo.policy.parameters()))
    gen = torch.Generator(device="cuda").manual_seed(2)
    data = (torch.randn(n, 4, generator=gen, device="cuda"), torch.randint(0, 2, (n,), generator=gen, device="cuda").float(),
            torch.randn(n, generator=gen, device="cuda"), (torch.rand(n, generator=gen, device="cuda") < 0.01).float())
    return ppo, data


def _learn(ppo, data):
    ppo.memory.push_device(*data)
    ppo.learn()
    torch.cuda.synchronize()
    return ppo


# ---------------------------------------------------------------------------------- the clipping norm
def test_clip_and_step_clips_by_the_norm_of_the_given_parameters():
    """An optimizer of some of the parameters, and one of more than these: the norm is the parameters', theirs
    are the gradients clipped, value by value.  torch's norm is a float32 sum of n squares: off by at
    most (n + 2) / 2 roundings, its coefficient by 3 more."""
    from PPO.optim import clip_and_step
    gen = torch.Generator().manual_seed(0)
    hyper = (1e-2, (0.9, 0.999), 1e-8, 0.1)
    for of in ((0, 1), (0, 1, 2, 3), (2, 1, 0)):
        params = [torch.nn.Parameter(torch.randn(n, generator=gen).cuda()) for n in (40, 300, 90, 70)]
        raw = [(torch.randn(p.numel(), generator=gen) * s).cuda() for p, s in zip(params, (1.0, 3.0, 40.0, 9.0))]
        for p, g in zip(params, raw):
            p.grad = g.clone()
        opt = _adamw()([params[i] for i in of], lr=hyper[0], betas=hyper[1], eps=hyper[2], weight_decay=hyper[3])
        old = [p.detach().clone() for p in params]
        clipped = params[:3]
        norm = R.norm64(raw[:3])
        c = R.clip64(norm, 2.0)
        assert c < 0.01
        n = sum(p.numel() for p in clipped)
        clip_and_step(opt, clipped, 2.0)
        for i, (p, g, w) in enumerate(zip(params, raw, old)):
            if i not in of:
                assert torch.equal(p.detach(), w) and not opt.state.get(p)
                continue
            ci = c if i < 3 else 1.0
            w1, m1, v1, ew, em, ev = R.step64(w.cpu().double(), g.cpu().double(), torch.zeros(p.numel()).double(),
                                              torch.zeros(p.numel()).double(), 1, *hyper, ci)
            rel = ((n + 2) / 2 + 3) * R.U32
            st = opt.state[p]
            assert bool(((st["exp_avg"].cpu().double() - m1).abs() <= em + rel * m1.abs()).all()), (of, i)
            assert bool(((st["exp_avg_sq"].cpu().double() - v1).abs() <= ev + 2 * rel * v1).all()), (of, i)
            # m and sqrt(v) change by the same factor: the quotient by the eps beside it at most
            part = hyper[0] * m1.abs() / (1 - 0.9) / ((v1 / (1 - 0.999)).sqrt() + hyper[2])
            assert bool(((p.detach().cpu().double() - w1).abs() <= ew + rel * part).all()), (of, i)


def test_learn_with_an_optimizer_of_some_parameters_is_torchs():
    """One step of learn() with an AdamW of the first four tensors, the gradients large enough to be clipped:
    the gradients left behind are those of the same run with torch's AdamW bit for bit, the parameters both
    float32 evaluations of one step from them."""
    runs = []
    for cls in (_adamw(), torch.optim.AdamW):
        ppo, data = _ppo(lambda ps: cls(ps[:4], lr=1e-3), n=200, k_epochs=1, value_coef=300.0)
        start = [p.detach().clone() for p in ppo.policy.parameters()]
        runs.append((_learn(ppo, data), start))
    (a, start), (b, again) = runs
    assert all(torch.equal(x, y) for x, y in zip(start, again))
    ours, theirs = list(a.policy.parameters()), list(b.policy.parameters())
    total = R.norm64([p.grad for p in theirs])
    assert abs(total - 2.0) < 1e-3                   # clipped
    assert R.norm64([p.grad for p in theirs[:4]]) < 0.999 * total     # by more than the four's norm
    for i, (p, q, w) in enumerate(zip(ours, theirs, start)):
        assert torch.equal(p.grad, q.grad), i
        if i >= 4:
            assert torch.equal(p, w) and torch.equal(q, w)
            continue
        zero = torch.zeros(p.numel(), dtype=torch.float64)
        w1, _, _, ew, _, _ = R.step64(w.reshape(-1).cpu().double(), p.grad.reshape(-1).cpu().double(), zero, zero, 1, 1e-3,
                                      (0.9, 0.999), 1e-8, 1e-2, 1.0)
        for x in (p, q):
            assert bool(((x.detach().reshape(-1).cpu().double() - w1).abs() <= ew).all()), i


# ---------------------------------------------------------------------------------- the engine and the optimizer's state
def _same(a, b, steps):
    for p, q in zip(a.policy.parameters(), b.policy.parameters()):
        assert torch.equal(p, q)
        for k in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(a.optimizer.state[p][k], b.optimizer.state[q][k]), k
        assert float(a.optimizer.state[p]["step"]) == float(b.optimizer.state[q]["step"]) == steps


@pytest.mark.parametrize("torchs", [False, True])
def test_engine_goes_on_from_steps_taken_outside_it(torchs):
    """Engine -> per-step path -> engine, for this AdamW and torch's: the engine goes on as one that is
    built from the optimizer's state there."""
    make = None if torchs else lambda ps: _adamw()(ps, lr=1e-3)
    runs = []
    for fresh in (False, True):
        ppo, data = _ppo(make, use_fused=True, use_graphs=True)
        for k, path in enumerate(("fused", "graph", "fused")):
            ppo.use_fused = path == "fused"
            if fresh and k == 2:
                ppo._engine = None
            _learn(ppo, data)
            assert ppo.last_update_path == path
        runs.append(ppo)
    _same(*runs, 72.0)


@pytest.mark.parametrize("torchs", [False, True])
def test_engine_takes_loaded_state(torchs):
    """load_state_dict() on an optimizer whose state the engine holds: the next learn() starts from what was
    loaded, as an engine built after the load does; an emptied state starts from nothing."""
    make = None if torchs else lambda ps: _adamw()(ps, lr=1e-3)
    runs = []
    for fresh in (False, True):
        ppo, data = _ppo(make, use_fused=True)
        _learn(ppo, data)
        saved = copy.deepcopy(ppo.optimizer.state_dict())
        _learn(ppo, data)
        ppo.optimizer.load_state_dict(saved)
        if fresh:
            ppo._engine = None
        _learn(ppo, data)
        assert ppo.last_update_path == "fused"
        runs.append(ppo)
    _same(*runs, 48.0)
    for ppo, fresh in zip(runs, (False, True)):
        ppo.optimizer.state.clear()
        if fresh:
            ppo._engine = None
        _learn(ppo, data)
    _same(*runs, 24.0)


@pytest.mark.parametrize("held,bits", [(8, 32), (32, 8)])
def test_learn_refuses_state_of_the_other_form(held, bits):
    """State of 8-bit moments loaded into an optimizer of 32-bit ones, or the other way round: learn() refuses
    it by the state's name as step() does, and leaves parameters and state as they were."""
    ppo, data = _ppo(lambda ps: _adamw()(ps, lr=1e-3, state_bits=held), use_fused=True)
    _learn(ppo, data)
    other = _adamw()(ppo.policy.parameters(), lr=1e-3, state_bits=bits)
    other.load_state_dict(copy.deepcopy(ppo.optimizer.state_dict()))
    ppo.optimizer = other
    params = [p.detach().clone() for p in ppo.policy.parameters()]
    state = {p: {k: (t, t.clone()) for k, t in other.state[p].items()} for p in ppo.policy.parameters()}
    for ppo.use_graphs in (True, False):
        ppo.memory.push_device(*data)
        with pytest.raises(ValueError, match="exp_"):
            ppo.learn()
        torch.cuda.synchronize()
        for p, old in zip(ppo.policy.parameters(), params):
            assert torch.equal(p.detach(), old) and other.state[p].keys() == state[p].keys()
            for k, (t, was) in state[p].items():
                assert other.state[p][k] is t and torch.equal(t.float(), was.float()), k


# ---------------------------------------------------------------------------------- every step's values
def _pin(opt, bits, hyper):
    """Checks every eager step of `opt` value by value against one float64 step from what it found; returns
    the list of the steps' clip coefficients."""
    params, seen, found = [p for g in opt.param_groups for p in g["params"]], [], []

    def pre(o, args, kwargs):
        max_norm = kwargs.get("max_norm")
        c = R.clip64(R.norm64([p.grad for p in params]), max_norm)
        found.append((c, _before(o, params, bits, not o.state.get(params[0]))))

    def post(o, args, kwargs):
        c, before = found.pop()
        seen.append(c)
        _check_step(o, params, before, c, len(seen), hyper, bits)
    opt.register_step_pre_hook(pre)
    opt.register_step_post_hook(post)
    return seen


HYPER = (1e-3, (0.9, 0.999), 1e-8, 1e-2)


@pytest.mark.parametrize("bits", [32, 8])
def test_each_step_of_learn_is_the_definitions(bits):
    """The eager per-step path, some steps clipped: 24 steps of 13 tensors in the one-launch form."""
    ppo, data = _ppo(lambda ps: _adamw()(ps, lr=1e-3, state_bits=bits), value_coef=5.0)
    seen = _pin(ppo.optimizer, bits, HYPER)
    _learn(ppo, data)
    assert ppo.last_update_path == "eager" and len(seen) == 24 and min(seen) < 1.0


@pytest.mark.parametrize("bits", [32, 8])
def test_each_step_of_the_wide_policy_and_rnd_is_the_definitions(bits):
    """348 observations, 17 actions through the native gradient step (clipped by 2), and the RND predictor's
    update (not clipped)."""
    from PPO import PPO
    torch.manual_seed(0)
    ppo = PPO(True, 348, 17, action_scaling=1.0, k_epochs=2, batch_size=64, mini_batch_size=512, use_RND=True)
    ppo.show_progress = False
    ppo.optimizer = _adamw()(ppo.policy.parameters(), lr=1e-3, state_bits=bits)
    ppo.rnd.optimizer = _adamw()(ppo.rnd.pred_net.parameters(), lr=1e-3, state_bits=bits)
    policy, rnd = _pin(ppo.optimizer, bits, HYPER), _pin(ppo.rnd.optimizer, bits, HYPER)
    gen = torch.Generator(device="cuda").manual_seed(2)
    n = 1100
    _learn(ppo, (torch.randn(n, 348, generator=gen, device="cuda"), torch.randn(n, 17, generator=gen, device="cuda") * 0.1,
                 torch.randn(n, generator=gen, device="cuda"), (torch.rand(n, generator=gen, device="cuda") < 0.01).float()))
    assert ppo.last_update_path == "graph" and ppo._last_graphed.wide is not None
    assert len(policy) == 6 and rnd == [1.0] * 3


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_of_some_parameters_is_the_eager_one(bits):
    """learn() with an optimizer of the first four tensors, clipped by all parameters' norm, twice over: the
    replayed graph leaves the eager path's bits."""
    runs = []
    for graphs in (False, True):
        ppo, data = _ppo(lambda ps: _adamw()(ps[:4], lr=1e-3, state_bits=bits), use_graphs=graphs, value_coef=300.0)
        for _ in range(2):
            _learn(ppo, data)
        assert ppo.last_update_path == ("graph" if graphs else "eager") and (ppo.last_graph_replays > 0) == graphs
        runs.append(ppo)
    for i, (p, q) in enumerate(zip(*(r.policy.parameters() for r in runs))):
        assert torch.equal(p, q), i
        if i < 4:
            a, b = (r.optimizer.state[x] for r, x in zip(runs, (p, q)))
            assert float(a["step"]) == 48.0 and all(torch.equal(a[k].float(), b[k].float()) for k in a), i

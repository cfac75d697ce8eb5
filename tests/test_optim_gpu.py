"""The optimizer operators over lists of tensors (csrc/prl_optim.hip, PPO/optim.py) against their
float64 restatement (optim_ref.py).  Tolerances: float32 evaluations are held to the roundings that
optim_ref.step64 counts, per value; a 16-bit parameter to half a step of its type more; 8-bit codes are
equal to the restatement's unless the value before rounding lies within its own float32 error of a
border, and then one that a value within that error rounds to."""
import math

import pytest
import torch

import optim_ref as R

pytestmark = pytest.mark.gpu
SIZES = [1, 3, 4, 5, 255, 256, 257, 1023, 4096, 4097, 20001, 0, 17411]


def _optim():
    import PPO.optim
    return PPO.optim


def _make(sizes, dtype, seed, packed=True, lead=1):
    """Parameters and gradients as views of flat buffers (`lead` values before the first: odd
    offsets)."""
    gen = torch.Generator().manual_seed(seed)
    out, grads = [], []
    if packed:
        flat = torch.zeros(lead + sum(sizes), dtype=dtype, device="cuda")
        gflat = torch.zeros_like(flat)
    at = lead
    for n in sizes:
        w = (torch.randn(n, generator=gen) * 0.05 + 0.01).to(dtype).cuda()
        g = (torch.randn(n, generator=gen) * 10.0 ** (torch.rand(1, generator=gen) * 3 - 3)).to(dtype).cuda()
        if packed:
            flat[at:at + n], gflat[at:at + n] = w, g
            w, g = flat[at:at + n], gflat[at:at + n]
            at += n
        p = torch.nn.Parameter(w)
        p.grad = g
        out.append(p)
        grads.append(g)
    return out, grads


def _moments(st, bits, n):
    """The moments of a state in float64 on the CPU: (m, rms squared)."""
    if bits == 32:
        return st["exp_avg"].reshape(-1).cpu().double(), st["exp_avg_sq"].reshape(-1).cpu().double()

    def read(k):
        q = st[k].reshape(-1).cpu().double()
        return q * st[k + "_scale"].cpu().double().repeat_interleave(256)[:n] / 256
    return read("exp_avg"), read("exp_rms").square()


def _check_step(opt, params, before, c, t, hyper, bits):
    """Every parameter and state against one float64 step from `before`."""
    for p, (w, g, m, v) in zip(params, before):
        n = p.numel()
        w1, m1, v1, ew, em, ev = R.step64(w, g, m, v, t, *hyper, c)
        st = opt.state[p]
        assert float(st["step"]) == t
        got = st["master"] if "master" in st else p.detach()
        extra = 0.0 if got.dtype == torch.float32 else R.HALF_STEP[p.dtype] * (w1.abs() + ew) + 2.0 ** -25
        err = (got.reshape(-1).cpu().double() - w1).abs()
        assert bool((err <= ew + extra).all()), (n, float((err - ew - extra).max()))
        if "master" in st:   # the parameter is its master's rounding
            assert torch.equal(p.detach(), st["master"].to(p.dtype))
        if bits == 32:
            gm, gv = _moments(st, 32, n)
            assert bool(((gm - m1).abs() <= em).all()) and bool(((gv - v1).abs() <= ev).all()), n
            continue
        dm, dr = R.draws(n, t)
        r1 = v1.sqrt()
        er = torch.where(r1 > 0, ev / (2 * r1.clamp(min=1e-70)), torch.zeros_like(r1)) + 2 * R.U32 * r1
        for k, x, d, least, e in (("exp_avg", m1, dm, 0.0, em), ("exp_rms", r1, dr, 2.0 ** -9, er)):
            A, q, low, high = R.quantise(x, d, least, e)
            ga, gq = st[k + "_scale"].cpu().double(), st[k].reshape(-1).cpu().double()
            ea = torch.nn.functional.pad(e, (0, -n % 256)).view(-1, 256).amax(1)
            assert bool(((ga - A).abs() <= ea).all()), (n, k)
            off = gq != q
            assert bool(((gq.abs() >= low) & (gq.abs() <= high) & (gq * x >= 0)).all()), (n, k, int(off.sum()))
            # few lie so near a border, except where v is below float32's normal values: its steps
            # there are 2^-149 whatever v is, all of it may be lost (v < 2^-150 is 0 in float32)
            assert int(off.sum()) <= 0.02 * n + int((v1 < 2.0 ** -126).sum()), (n, k)


def _before(opt, params, bits, fresh):
    out = []
    for p in params:
        n, st = p.numel(), opt.state.get(p)
        w = (st["master"] if st and "master" in st else p.detach()).reshape(-1).cpu().double()
        m, v = (torch.zeros(n, dtype=torch.float64),) * 2 if fresh else _moments(st, bits, n)
        out.append((w, p.grad.reshape(-1).cpu().double(), m, v))
    return out


# ---------------------------------------------------------------------------------- norm
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_grad_norm(dtype):
    """sqrt of the float64 sum of squares: off by one float32 rounding."""
    for sizes in ([1], [3], SIZES, [7] * 300, [200_003]):
        _, grads = _make(sizes, dtype, len(sizes))
        got, want = float(_optim().grad_norm(grads)), R.norm64(grads)
        assert abs(got - want) <= 1.01 * R.U32 * want, sizes


def test_grad_norm_edges():
    f = _optim().grad_norm
    x = torch.randn(64, 48, device="cuda")
    assert abs(float(f([x.t()])) - R.norm64([x])) <= 1.01 * R.U32 * R.norm64([x])    # strided
    assert float(f(x.new_empty(0))) == 0.0 and float(f([x.new_empty(0), x.new_zeros(5)])) == 0.0
    big = torch.full((1000,), 1e30, device="cuda")         # squares past float32
    assert abs(float(f([big])) / (1e30 * math.sqrt(1000)) - 1) < 1e-6
    mixed = [x, x.bfloat16(), x.half()]
    assert abs(float(f(mixed)) - R.norm64(mixed)) <= 1.01 * R.U32 * R.norm64(mixed)
    assert math.isnan(float(f([x, x.new_full((3,), float("nan"))])))
    assert math.isinf(float(f([x.new_full((3,), float("inf")), x])))
    a = f([x])
    b = f([x])
    assert torch.equal(a, b) and a.shape == ()


# ---------------------------------------------------------------------------------- the step
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,master", [(torch.float32, False), (torch.bfloat16, False),
                                          (torch.bfloat16, True), (torch.float16, False),
                                          (torch.float16, True)])
@pytest.mark.parametrize("max_norm", [None, 0.5])
def test_adamw_steps(bits, dtype, master, max_norm):
    """Three steps (the first from empty state) over odd sizes at odd offsets."""
    params, grads = _make(SIZES, dtype, 11)
    hyper = (1e-2, (0.9, 0.999), 1e-8, 0.1)
    opt = _optim().AdamW(params, lr=hyper[0], betas=hyper[1], eps=hyper[2], weight_decay=hyper[3],
                         state_bits=bits, master=master)
    gen = torch.Generator(device="cuda").manual_seed(3)
    for t in (1, 2, 3):
        before = _before(opt, params, bits, t == 1)
        norm = R.norm64(grads)
        kept = [g.clone() for g in grads]
        opt.step(max_norm=max_norm)
        if max_norm is None:
            assert opt.total_norm is None
        else:
            assert norm > max_norm and abs(float(opt.total_norm) - norm) <= 1.01 * R.U32 * norm
        assert all(torch.equal(a, b) for a, b in zip(kept, grads))     # gradients stay as they are
        _check_step(opt, params, before, R.clip64(norm, max_norm), t, hyper, bits)
        for g in grads:
            g.copy_(torch.randn(g.shape, generator=gen, device="cuda") * 0.03)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_many_tensors_groups_and_types(bits):
    """More tensors than a launch holds, more groups than list_begin's batch, types mixed, separate
    allocations, one group's lr on the device, some parameters without a gradient."""
    groups, every = [], []
    for i in range(19):
        dtype = (torch.float32, torch.bfloat16, torch.float16)[i % 3]
        params, _ = _make([1 + (37 * i + 11 * j) % 700 for j in range(13)], dtype, i, packed=i % 2 == 0)
        lr = 1e-3 * (i + 1)
        groups.append(dict(params=params, lr=torch.full((), lr, device="cuda") if i == 4 else lr,
                           betas=(0.8 + 0.01 * i, 0.99), weight_decay=0.01 * i, master=i % 2 == 1))
        every.append((params, (float(torch.tensor(lr)) if i == 4 else lr, (0.8 + 0.01 * i, 0.99), 1e-8, 0.01 * i)))
    without = every[3][0][2]
    without.grad = None
    old = without.detach().clone()
    opt = _optim().AdamW(groups, state_bits=bits)
    grads = [p.grad for params, _ in every for p in params if p.grad is not None]
    norm = R.norm64(grads)
    befores = [_before(opt, [p for p in params if p.grad is not None], bits, True) for params, _ in every]
    opt.step(max_norm=1.0)
    assert torch.equal(without.detach(), old) and not opt.state.get(without)
    for (params, hyper), before in zip(every, befores):
        _check_step(opt, [p for p in params if p.grad is not None], before, R.clip64(norm, 1.0), 1, hyper, bits)


def test_adamw_matches_torch_and_exchanges_state():
    """float32, 32-bit moments: four clipped steps beside torch's clip_grad_norm_ + AdamW, the state
    moved from one to the other in between by state_dict().  Both are float32 evaluations of the same
    step: per step each is off by at most ~6 U of a weight and 16 U of an update of <= 10 lr here."""
    params, grads = _make(SIZES, torch.float32, 5)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    a = _optim().AdamW(params, lr=1e-3)
    b = torch.optim.AdamW(twins, lr=1e-3)
    for t in range(4):
        for g, q in zip(grads, twins):
            g.copy_(torch.randn_like(g) * 0.1)
            q.grad = g.clone()
        a.step(max_norm=2.0)
        norm = torch.nn.utils.clip_grad_norm_(twins, 2.0)
        b.step()
        assert abs(float(a.total_norm) - float(norm)) <= 1e-6 * float(norm)
        for p, q in zip(params, twins):
            if p.numel():
                top = float(q.detach().abs().max())
                assert float((p - q).detach().abs().max()) <= (t + 1) * 2 * R.U32 * (6 * top + 16 * 1e-2)
        if t == 1:     # swap the states
            sa, sb = a.state_dict(), b.state_dict()
            a = _optim().AdamW(params, lr=1e-3)
            b = torch.optim.AdamW(twins, lr=1e-3)
            a.load_state_dict(sb)
            b.load_state_dict(sa)
    for p in params:
        assert float(a.state[p]["step"]) == 4.0


@pytest.mark.parametrize("dtype,master", [(torch.float32, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip(bits, dtype, master):
    """A saved and loaded optimizer goes on with the same bits; the state keeps its types."""
    params, grads = _make(SIZES, dtype, 6)
    a = _optim().AdamW(params, state_bits=bits, master=master)
    a.step()
    kept = [p.detach().clone() for p in params]
    types = {k: v.dtype for k, v in a.state[params[4]].items()}
    a.step()
    want = [p.detach().clone() for p in params]
    with torch.no_grad():
        for p, k in zip(params, kept):
            p.copy_(k)
    b = _optim().AdamW(params, state_bits=bits, master=master)
    # (a.state_dict() holds a's own tensors, which its second step moved: the first step's state again)
    fresh, _ = _make(SIZES, dtype, 6)
    d = _optim().AdamW(fresh, state_bits=bits, master=master)
    d.step()
    import copy
    b.load_state_dict(copy.deepcopy(d.state_dict()))
    assert {k: v.dtype for k, v in b.state[params[4]].items()} == types
    b.step()
    assert all(torch.equal(p.detach(), w) for p, w in zip(params, want))


def test_load_state_dict_of_other_adamws():
    """A torch AdamW's 16-bit moments and host step counts become float32 on the device; amsgrad's and
    maximize's are refused; moments of the other form by the next step."""
    p = torch.nn.Parameter(torch.ones(40, device="cuda", dtype=torch.bfloat16))
    q = torch.nn.Parameter(p.detach().clone())
    p.grad, q.grad = torch.full_like(p, 0.5), torch.full_like(p, 0.5)
    torch_opt = torch.optim.AdamW([q])
    torch_opt.step()
    opt = _optim().AdamW([p])
    opt.load_state_dict(torch_opt.state_dict())
    st = opt.state[p]
    assert st["exp_avg"].dtype == torch.float32 and st["step"].is_cuda and float(st["step"]) == 1.0
    assert torch.equal(st["exp_avg"], torch_opt.state[q]["exp_avg"].float())
    opt.step()
    assert float(st["step"]) == 2.0
    for kw in (dict(amsgrad=True), dict(maximize=True)):
        with pytest.raises(ValueError, match="amsgrad or maximize"):
            _optim().AdamW([p]).load_state_dict(torch.optim.AdamW([q], **kw).state_dict())
    other = _optim().AdamW([p], state_bits=8)
    other.load_state_dict(opt.state_dict())
    with pytest.raises(ValueError, match="exp_"):
        other.step()


# ---------------------------------------------------------------------------------- values that are not finite
def test_adamw_nonfinite_gradients():
    """32-bit: as torch (a NaN stays at its value).  8-bit: its block of 256 turns NaN, no other."""
    for bad in (float("nan"), float("inf")):
        p = torch.nn.Parameter(torch.ones(1000, device="cuda"))
        p.grad = torch.full((1000,), 0.1, device="cuda")
        p.grad[300] = bad
        opt = _optim().AdamW([p])
        opt.step()
        assert torch.isfinite(p).sum() == 999 and math.isnan(p.detach()[300])
        q = torch.nn.Parameter(torch.ones(1000, device="cuda"))
        q.grad = p.grad.clone()
        opt = _optim().AdamW([q], state_bits=8)
        opt.step()
        assert torch.isfinite(q).sum() == 999 and math.isnan(q.detach()[300])
        scale = opt.state[q]["exp_avg_scale"]
        assert math.isnan(float(scale[1])) and torch.isfinite(scale).sum() == 3
        q.grad[300] = 0.1
        opt.step()
        nan = torch.isnan(q).cpu()
        assert bool(nan[256:512].all()) and not bool(nan[:256].any()) and not bool(nan[512:].any())
    # the norm of a list with a NaN: every parameter NaN, as clip_grad_norm_ + step; an infinite norm: c = 0
    p = torch.nn.Parameter(torch.ones(8, device="cuda"))
    p.grad = torch.tensor([1.0] * 7 + [float("nan")], device="cuda")
    _optim().AdamW([p]).step(max_norm=1.0)
    assert bool(torch.isnan(p).all())
    p = torch.nn.Parameter(torch.ones(8, device="cuda"))
    p.grad = torch.tensor([1.0] * 7 + [float("inf")], device="cuda")
    opt = _optim().AdamW([p], weight_decay=0.0)
    opt.step(max_norm=1.0)
    assert p[:7].tolist() == [1.0] * 7 and math.isnan(p.detach()[7]) and math.isinf(float(opt.total_norm))


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_zero_tiny_and_huge_values(bits):
    """All-zero gradients and max_norm = 0 (no update but the decay, moments zero), blocks of tiny
    and huge values."""
    for scale, max_norm in ((0.0, None), (1.0, 0.0), (1e-30, None), (1e-18, None), (1e15, None)):
        p = torch.nn.Parameter(torch.linspace(-1, 1, 700, device="cuda"))
        p.grad = torch.linspace(-1, 1, 700, device="cuda") * scale
        opt = _optim().AdamW([p], lr=1e-2, eps=1e-8, state_bits=bits)
        before = _before(opt, [p], bits, True)
        opt.step(max_norm=max_norm)
        assert bool(torch.isfinite(p).all())
        c = R.clip64(R.norm64([p.grad]), max_norm)
        _check_step(opt, [p], before, c, 1, (1e-2, (0.9, 0.999), 1e-8, 1e-2), bits)
    # 8-bit: below 2^-118 a block is held as zeros
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    p.grad = torch.full((300,), 1e-36, device="cuda")
    opt = _optim().AdamW([p], state_bits=8)
    opt.step()
    assert opt.state[p]["exp_avg"].float().abs().max() == 0 and opt.state[p]["exp_avg_scale"].abs().max() == 0


def test_adamw8_rounding_is_unbiased():
    """The mean of what is held over many values equals the mean of what was to be held: 2^20 equal
    gradients (but one larger in each block, which fixes the scale) whose quotient lies a third of
    the way between two codes.  The share s of upper codes has a standard deviation of at most
    1 / (2 * 2^10): five of them are 0.0025; 16-bit draws shift it by at most 2^-16."""
    n = 1 << 20
    lower, unit = 40.0, 4.0                       # e4m3 neighbours 40 and 44
    target = (lower + unit / 3) / 256.0           # of the block's largest
    g = torch.full((n,), target, device="cuda")
    g[::256] = 1.0
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    p.grad = g
    opt = _optim().AdamW([p], state_bits=8)
    opt.step()
    st = opt.state[p]
    for k in ("exp_avg", "exp_rms"):
        q = st[k].float().view(-1, 256)
        assert bool((q[:, 0] == 256).all())
        q = q[:, 1:]
        assert bool(((q == lower) | (q == lower + unit)).all())
        assert abs(float((q > lower).double().mean()) - 1 / 3) <= 0.0025 + 2.0 ** -16, k
    # the draws of exp_avg and exp_rms, and of two steps, are not the same ones
    up = (st["exp_avg"].float() > lower) != (st["exp_rms"].float() > lower)
    assert float(up.double().mean()) > 0.3


def test_adamw8_second_moment_follows_smaller_gradients():
    """After a spike in half of the values, their second moment decays with beta2 towards the rest's,
    in codes whose steps are 6 to 12 %, far above one step's change of 0.05 %: with rounding to the
    nearest it would stay where it is.  Expected after T steps: r^2 = 0.001 * 100 * 0.999^T + (1 -
    0.999^T) (in units of the rest); the noise of the rounding over 2^16 values averages out below
    2 %, and E[r] against sqrt(E[r^2]) differs by the spread of r, at most 25 %."""
    n, T = 1 << 16, 1500
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = _optim().AdamW([p], lr=0.0, state_bits=8, weight_decay=0.0)
    g = torch.ones(n, device="cuda")
    spike = g.clone()
    spike[::2] = 10.0
    p.grad = spike
    for _ in range(30):
        opt.step()
    p.grad = g
    for _ in range(T):
        opt.step()
    st = opt.state[p]
    r = st["exp_rms"].float() * st["exp_rms_scale"].repeat_interleave(256) / 256
    keep = 0.999 ** T
    high = math.sqrt((1 - 0.999 ** 30) * 100 * keep + 1 - keep)
    low = math.sqrt((1 - 0.999 ** 30) * keep + 1 - keep)
    assert abs(float(r[::2].mean()) / high - 1) < 0.25 and abs(float(r[1::2].mean()) / low - 1) < 0.25


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("betas,eps", [((0.9, 0.999), 1e-15), ((0.0, 0.0), 1e-8), ((0.5, 0.9), 0.0), ((0.99, 0.99999), 1e-3)])
def test_adamw_other_hyper_parameters(bits, betas, eps):
    """Betas of 0, an eps of 0 and ones below and above the quick root's bound, no decay: three steps with
    gradients over six decades within a block (none of them 0: eps = 0)."""
    hyper = (1e-3, betas, eps, 0.0)
    gen = torch.Generator().manual_seed(9)
    params = [torch.nn.Parameter((torch.randn(n, generator=gen) * 0.1).cuda()) for n in (700, 45000)]
    opt = _optim().AdamW(params, lr=1e-3, betas=betas, eps=eps, weight_decay=0.0, state_bits=bits)
    for t in (1, 2, 3):
        for p in params:
            g = torch.randn(p.numel(), generator=gen).clamp(min=0.1) * 10.0 ** (-6 * torch.rand(p.numel(), generator=gen))
            p.grad = g.cuda()
        before = _before(opt, params, bits, t == 1)
        opt.step()
        _check_step(opt, params, before, 1.0, t, hyper, bits)


# ---------------------------------------------------------------------------------- streams, graphs, layouts
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_captured_step_replays_as_eager(bits):
    """A captured step (norm, clip, update, counts, a device lr that changes between replays) replayed
    with eager work and synchronizations in between: the bits of eager steps.  Two graphs of two
    optimizers replay beside each other on two streams."""
    sets = []
    for k in range(2):
        params, grads = _make([5, 300, 4096, 777], torch.bfloat16, 20 + k)
        twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
        for p, q in zip(params, twins):
            q.grad = p.grad
        lr = torch.full((), 1e-2, device="cuda")
        a = _optim().AdamW(params, lr=lr, state_bits=bits, master=k == 1)
        b = _optim().AdamW(twins, lr=lr, state_bits=bits, master=k == 1)
        a.step(max_norm=0.5)
        b.step(max_norm=0.5)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            alone = _optim().grad_norm(grads + grads * 20)     # a list of its own, in the long form
            a.step(max_norm=0.5)
        sets.append((params, grads, twins, lr, a, b, graph, (a.total_norm, alone), torch.cuda.Stream()))
    for r in range(4):
        for params, grads, twins, lr, a, b, graph, norm, s in sets:
            lr.fill_(1e-2 / (r + 1))
            for g in grads:
                g.copy_(torch.randn(g.shape, device="cuda") * 0.1)
        torch.cuda.synchronize()
        for x in sets:
            with torch.cuda.stream(x[8]):
                x[6].replay()
        torch.cuda.synchronize()
        for params, grads, twins, lr, a, b, graph, norm, s in sets:
            b.step(max_norm=0.5)
            torch.cuda.synchronize()
            assert torch.equal(norm[0], b.total_norm)
            assert torch.equal(norm[1], _optim().grad_norm(grads + grads * 20))
            for p, q in zip(params, twins):
                assert torch.equal(p, q)
                sa, sb = a.state[p], b.state[q]
                assert all(torch.equal(sa[k].view(torch.uint8) if sa[k].dtype.itemsize == 1 else sa[k],
                                       sb[k].view(torch.uint8) if sb[k].dtype.itemsize == 1 else sb[k]) for k in sa)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_is_deterministic_and_follows_replaced_tensors(bits):
    """The same steps give the same bits, on another stream too; gradients that are strided, and
    parameters and gradients that move to other memory between steps, are followed."""
    runs = []
    for way in range(2):
        params, grads = _make([64 * 48, 1000], torch.float32, 8)
        params[0].data = params[0].data.view(64, 48)
        params[0].grad = grads[0].view(64, 48)
        opt = _optim().AdamW(params, state_bits=bits)
        s = torch.cuda.Stream() if way else torch.cuda.current_stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            opt.step(max_norm=1.0)
            if way:     # the same gradient with other strides, the parameter elsewhere
                params[0].grad = params[0].grad.t().contiguous().t()
                assert not params[0].grad.is_contiguous()
                params[1].data = params[1].data.clone()
                params[1].grad = params[1].grad.clone()
            opt.step(max_norm=1.0)
        torch.cuda.synchronize()
        runs.append([p.detach().clone() for p in params] + [opt.state[p]["exp_avg"].float() for p in params])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_adamw_past_32_bits():
    """A tensor of 2^32 + 515 values: offsets, block numbers and the draws' high word past 32 bits."""
    n = (1 << 32) + 515
    p = torch.nn.Parameter(torch.empty(n, dtype=torch.bfloat16, device="cuda").fill_(0.5))
    p.grad = torch.empty(n, dtype=torch.bfloat16, device="cuda").fill_(2.0 ** -9)
    tail = slice(n - 515 - 1024, n)
    gen = torch.Generator().manual_seed(1)
    p.grad[tail] = (torch.randn(515 + 1024, generator=gen) * 0.01).bfloat16().cuda()
    opt = _optim().AdamW([p], lr=1e-2, state_bits=8)
    opt.step(max_norm=1e9)
    g = p.grad[tail].cpu().double()
    norm = math.sqrt((n - 1539) * 2.0 ** -18 + float(g.square().sum()))
    assert abs(float(opt.total_norm) - norm) <= 1.01 * R.U32 * norm
    zero = torch.zeros(1539, dtype=torch.float64)
    w1, m1, v1, ew, em, ev = R.step64(zero + 0.5, g, zero, zero, 1, 1e-2, (0.9, 0.999), 1e-8, 1e-2, 1.0)
    err = (p.detach()[tail].cpu().double() - w1).abs()
    assert bool((err <= ew + R.HALF_STEP[torch.bfloat16] * (w1.abs() + ew)).all())
    dm, _ = R.draws(1539, 1, first=n - 1539)
    A, q, low, high = R.quantise(m1, dm, 0.0, em)       # n - 1539 is a multiple of 256: blocks as the tensor's
    assert (n - 1539) % 256 == 0
    st = opt.state[p]
    got = st["exp_avg"][tail].cpu().double()
    off = got != q
    assert bool(((got.abs() >= low) & (got.abs() <= high)).all()) and float(off.double().mean()) < 0.02
    assert bool(((st["exp_avg_scale"][-7:].cpu().double() - A).abs() <= 16 * R.U32 * A).all())


# ---------------------------------------------------------------------------------- together, as learn() uses them
def _learn(make_optimizer, use_graphs, use_fused=False, cont=False, mb=256):
    from PPO import PPO
    torch.manual_seed(0)
    D, A = (3, 1) if cont else (4, 2)
    ppo = PPO(cont, D, A, action_scaling=2.0 if cont else None, lr=1e-3, k_epochs=3, batch_size=64, mini_batch_size=mb)
    ppo.show_progress = False
    ppo.use_fused, ppo.use_graphs = use_fused, use_graphs
    if make_optimizer is not None:
        ppo.optimizer = make_optimizer(ppo.policy.parameters())
    gen = torch.Generator(device="cuda").manual_seed(2)
    n = 2000 + 37
    S = torch.randn(n, D, generator=gen, device="cuda")
    act = (torch.randn(n, A, generator=gen, device="cuda") if cont
           else torch.randint(0, A, (n,), generator=gen, device="cuda").float())
    ppo._test_data = (S, act, torch.randn(n, generator=gen, device="cuda"),
                      (torch.rand(n, generator=gen, device="cuda") < 0.01).float())
    ppo.memory.push_device(*ppo._test_data)
    ppo.learn()
    torch.cuda.synchronize()
    return ppo


def test_learn_steps_through_the_list_adamw():
    """PPO.learn() with this AdamW: the update engine takes it with 32-bit moments and leaves it the
    state; with 8-bit moments the per-step paths run (the native gradient step, and autograd captured and
    eager with the same bits), and end near the 32-bit run (24 steps of at most ~lr each could part
    the weights by 2 * 24 * lr)."""
    AdamW = _optim().AdamW
    engine = _learn(lambda p: AdamW(p, lr=1e-3), True, use_fused=True)
    plain = _learn(None, True, use_fused=True)
    assert engine.last_update_path == plain.last_update_path == "fused"
    for p, q in zip(engine.policy.parameters(), plain.policy.parameters()):
        assert torch.equal(p, q)
        assert torch.equal(engine.optimizer.state[p]["exp_avg"], plain.optimizer.state[q]["exp_avg"])
    assert float(engine.optimizer.state[p]["step"]) == 24.0
    # the per-step path goes on from the engine's state
    engine.use_fused = False
    engine.memory.push_device(*engine._test_data)
    engine.learn()
    assert engine.last_update_path == "graph"
    for p, q in zip(engine.policy.parameters(), plain.policy.parameters()):
        assert float(engine.optimizer.state[p]["step"]) == 48.0 and bool(torch.isfinite(p).all())
        assert 0.0 < float((p - q).detach().abs().max()) <= 2 * 24 * 1e-3
    # an optimizer of some of the parameters is not the engine's: the others stay
    part = _learn(lambda p: AdamW(list(p)[:4], lr=1e-3), True, use_fused=True)
    torch.manual_seed(0)
    from PPO import PPO
    start = [p.detach().clone() for p in PPO(False, 4, 2).policy.parameters()]
    moved = [not torch.equal(p, s) for p, s in zip(part.policy.parameters(), start)]
    assert part.last_update_path == "graph" and moved == [i < 4 for i in range(len(start))]
    native = _learn(lambda p: AdamW(p, lr=1e-3, state_bits=8), True, use_fused=True)
    assert native.last_update_path == "graph" and native._last_graphed.wide is not None
    graph = _learn(lambda p: AdamW(p, lr=1e-3, state_bits=8), True)
    eager = _learn(lambda p: AdamW(p, lr=1e-3, state_bits=8), False)
    assert graph.last_update_path == "graph" and graph.last_graph_replays > 0 and eager.last_update_path == "eager"
    for p, q, r, x in zip(*(o.policy.parameters() for o in (graph, eager, plain, native))):
        assert torch.equal(p, q) and bool(torch.isfinite(p).all()) and bool(torch.isfinite(x).all())
        assert float((p - r).detach().abs().max()) <= 2 * 24 * 1e-3
        assert float((x - r).detach().abs().max()) <= 2 * 24 * 1e-3
        for o, w in ((graph, p), (native, x)):
            st = o.optimizer.state[w]
            assert st["exp_avg"].dtype == torch.float8_e4m3fn and float(st["step"]) == 24.0


def test_learn_wide_policy_and_rnd_with_8_bit_moments():
    """The wide step (348 observations, 17 actions) and the RND predictor's update with 8-bit moments."""
    from PPO import PPO
    torch.manual_seed(0)
    ppo = PPO(True, 348, 17, action_scaling=1.0, k_epochs=2, batch_size=64, mini_batch_size=512, use_RND=True)
    ppo.show_progress = False
    AdamW = _optim().AdamW
    ppo.optimizer = AdamW(ppo.policy.parameters(), state_bits=8)
    ppo.rnd.optimizer = AdamW(ppo.rnd.pred_net.parameters(), lr=1e-3, state_bits=8)
    old = [p.detach().clone() for p in list(ppo.policy.parameters()) + list(ppo.rnd.pred_net.parameters())]
    n = 1100
    ppo.memory.push_device(torch.randn(n, 348, device="cuda"), torch.randn(n, 17, device="cuda") * 0.1,
                           torch.randn(n, device="cuda"), (torch.rand(n, device="cuda") < 0.01).float())
    ppo.learn()
    torch.cuda.synchronize()
    for o, steps in ((ppo.optimizer, 6.0), (ppo.rnd.optimizer, 3.0)):
        for g in o.param_groups:
            assert all(float(o.state[p]["step"]) == steps for p in g["params"])
    new = list(ppo.policy.parameters()) + list(ppo.rnd.pred_net.parameters())
    assert all(bool(torch.isfinite(p).all()) and not torch.equal(p, o) for p, o in zip(new, old))


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,master", [(torch.float32, False), (torch.bfloat16, True), (torch.float16, False)])
def test_nothing_around_the_tensors_is_written(bits, dtype, master, long):
    """Parameters, masters, moments, codes and scales as views with other values before and behind them
    (7 of each kind), at every alignment: those stay, in the one-launch form and in the long one."""
    sizes = [1, 2, 3, 4, 5, 63, 255, 256, 257, 258, 1021, 4099] * (3 if long else 1)
    gap, kinds = 7, {}

    def lay(name, lengths, of, fill):
        flat = torch.full((gap + sum(n + gap for n in lengths),), fill, device="cuda").to(of)
        at, views = gap, []
        for n in lengths:
            views.append(flat[at:at + n])
            at += n + gap
        kinds[name] = (flat, lengths, flat.clone())
        return views

    blocks = [-(-n // 256) for n in sizes]
    params = [torch.nn.Parameter(v) for v in lay("param", sizes, dtype, 0.5)]
    opt = _optim().AdamW(params, state_bits=bits, master=master)
    codes = torch.float8_e4m3fn
    state = {"exp_avg": lay("exp_avg", sizes, torch.float32 if bits == 32 else codes, 0.25),
             "exp_avg_sq" if bits == 32 else "exp_rms": lay("second", sizes, torch.float32 if bits == 32 else codes, 2.0)}
    if bits == 8:
        state["exp_avg_scale"] = lay("first scale", blocks, torch.float32, 0.125)
        state["exp_rms_scale"] = lay("second scale", blocks, torch.float32, 0.5)
    if master and dtype != torch.float32:
        state["master"] = lay("master", sizes, torch.float32, 0.5)
    for i, (p, g) in enumerate(zip(params, lay("grad", sizes, dtype, 1.0))):
        p.grad = g
        opt.state[p].update({k: v[i] for k, v in state.items()}, step=torch.full((), 3.0, device="cuda"))
    opt.step(max_norm=1.0)
    torch.cuda.synchronize()
    for name, (flat, lengths, old) in kinds.items():
        at = gap
        inside = torch.zeros(flat.numel(), dtype=torch.bool, device="cuda")
        for n in lengths:
            inside[at:at + n] = True
            at += n + gap
        new, was = flat.float(), old.float()
        assert torch.equal(new[~inside], was[~inside]), name
        if name == "grad":
            assert torch.equal(new, was)
        elif name in ("param", "master", "first scale", "second scale") and flat.dtype == torch.float32:
            # (a 16-bit parameter's step, below lr = 1e-3, may round back to 0.5)
            assert bool((new[inside] != was[inside]).all()), name


def test_empty_lists_and_parameters():
    O = _optim()
    e = torch.nn.Parameter(torch.empty(0, device="cuda"))
    e.grad = torch.empty(0, device="cuda")
    p = torch.nn.Parameter(torch.ones((), device="cuda"))        # 0-dim
    for bits in (32, 8):
        opt = O.AdamW([e, p], state_bits=bits)
        opt.step(max_norm=1.0)                                    # p has no gradient
        assert float(opt.total_norm) == 0.0 and float(opt.state[e]["step"]) == 1.0 and not opt.state.get(p)
        p.grad = torch.full((), 3.0, device="cuda")
        opt.step(max_norm=1.0)
        assert float(opt.total_norm) == 3.0 and float(opt.state[p]["step"]) == 1.0
        p.grad = None
    q = torch.nn.Parameter(torch.ones(5, device="cuda"))
    opt = O.AdamW([q])
    opt.step(max_norm=1.0)
    assert float(opt.total_norm) == 0.0 and not opt.state.get(q) and torch.equal(q.detach(), torch.ones_like(q))
    opt.step()
    assert opt.total_norm is None


def test_replays_and_eager_steps_of_one_optimizer_alternate():
    """A graph's step and eager ones share state and counts; an eager step with other gradients, or with
    a parameter left out, does not disturb the graph's."""
    params, grads = _make([300, 70], torch.float32, 31)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    a, b = _optim().AdamW(params, state_bits=8), _optim().AdamW(twins, state_bits=8)

    def eager(opt, ps, first_only):
        ps[0].grad = grads[0] * 2.0
        ps[1].grad = None if first_only else grads[1] * 0.5
        opt.step(max_norm=1.0)

    for o, ps in ((a, params), (b, twins)):
        for p, g in zip(ps, grads):
            p.grad = g
        o.step(max_norm=1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step(max_norm=1.0)
    for k in range(3):
        graph.replay()
        eager(a, params, k == 1)
        torch.cuda.synchronize()
        for p, g in zip(twins, grads):
            p.grad = g
        b.step(max_norm=1.0)
        eager(b, twins, k == 1)
        for p, q in zip(params, twins):
            assert torch.equal(p, q)
    assert float(a.state[params[0]]["step"]) == 7.0 and float(a.state[params[1]]["step"]) == 6.0


def test_step_runs_torch_hooks_and_shows_in_the_profiler():
    from torch.optim.optimizer import register_optimizer_step_post_hook, register_optimizer_step_pre_hook
    p = torch.nn.Parameter(torch.ones(10, device="cuda"))
    p.grad = torch.ones_like(p)
    opt = _optim().AdamW([p])
    seen = []
    hooks = [opt.register_step_pre_hook(lambda o, a, k: seen.append("pre")),
             opt.register_step_post_hook(lambda o, a, k: seen.append("post")),
             register_optimizer_step_pre_hook(lambda o, a, k: seen.append("global pre")),
             register_optimizer_step_post_hook(lambda o, a, k: seen.append("global post"))]
    for h in hooks:
        opt.step(max_norm=1.0)
        h.remove()
    assert seen.count("pre") == 1 and seen.count("post") == 2
    assert seen.count("global pre") == 3 and seen.count("global post") == 4
    opt.step()
    assert len(seen) == 10 and float(opt.state[p]["step"]) == 5.0
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        opt.step()
    assert any("Optimizer.step#AdamW" in e.key for e in prof.key_averages())
    before = p.detach().clone()
    loss = opt.step(lambda: (p * 2.0).sum().backward() or torch.tensor(3.0))
    assert float(loss) == 3.0 and not torch.equal(p.detach(), before)
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, gamma=0.5)
    opt.step()
    sched.step()
    assert opt.param_groups[0]["lr"] == 0.5e-3


def test_short_and_long_lists_agree():
    """A list at the one-launch form's bounds (160 blocks of 256 values, 32 tensors, 16 groups) and past
    each of them: the same step, up to the norm's summation order (off by one float32 rounding)."""
    O = _optim()
    sizes = [1024] * 39 + [1024 - 3]
    for bits in (32, 8):
        base, bgrads = _make([160 * 256], torch.float32, 4, lead=3)
        over, ograds = _make([160 * 256, 1], torch.float32, 4, lead=3)
        with torch.no_grad():
            over[0].copy_(base[0])
            ograds[0].copy_(bgrads[0])
            ograds[1].zero_()
        a, b = O.AdamW(base, state_bits=bits), O.AdamW(over, state_bits=bits)
        for _ in range(2):
            a.step()
            b.step()
        assert torch.equal(base[0], over[0])
        a.step(max_norm=1.0)
        b.step(max_norm=1.0)
        n = R.norm64(bgrads)
        assert abs(float(a.total_norm) - n) <= 1.01 * R.U32 * n and abs(float(b.total_norm) - n) <= 1.01 * R.U32 * n
        # 33 tensors / 17 groups of the same values
        runs = []
        for split in (lambda ps: [dict(params=ps[:33])], lambda ps: [dict(params=ps[:32]), dict(params=ps[32:33])],
                      lambda ps: [dict(params=[p]) for p in ps[:17]] + [dict(params=ps[17:33])]):
            params, _ = _make(sizes, torch.float32, 4, lead=3)
            opt = O.AdamW(split(params), state_bits=bits)
            opt.step()
            opt.step()
            runs.append([p.detach().clone() for p in params[:33]])
        few, _ = _make(sizes, torch.float32, 4, lead=3)
        opt = O.AdamW(few[:32], state_bits=bits)
        opt.step()
        opt.step()
        for r in runs:
            assert all(torch.equal(x, y) for x, y in zip(r, runs[0]))
            assert all(torch.equal(x, y.detach()) for x, y in zip(r, few[:32]))


def _dp_worker(rank, world, port, out_dir, use_fused):
    import os
    import sys
    from test_distributed_cpu import PATHS, _shard
    sys.path[:0] = PATHS
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    torch.distributed.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from PPO import PPO
        from PPO.optim import AdamW
        torch.cuda.set_device(0)
        torch.manual_seed(0)
        p = PPO(False, 4, 2, lr=1e-3, k_epochs=4, batch_size=1, mini_batch_size=64)
        p.show_progress, p.use_fused = False, use_fused
        p.optimizer = AdamW(p.policy.parameters(), lr=1e-3, state_bits=8)
        S, A, R, D = _shard(rank, 64, 5)
        if rank == 1:      # one minibatch less: its last steps add zero gradients
            S, A, R, D = (x[:-64] for x in (S, A, R, D))
        p.memory.push_device(*(torch.from_numpy(x).cuda() for x in (S, A, R, D)))
        p.learn()
        torch.cuda.synchronize()
        torch.save(dict(params=[q.detach().cpu() for q in p.policy.parameters()], path=p.last_update_path,
                        replays=p.last_graph_replays, step=[float(p.optimizer.state[q]["step"]) for q in p.policy.parameters()],
                        codes=[p.optimizer.state[q]["exp_rms"].float().cpu() for q in p.policy.parameters()]),
                   os.path.join(out_dir, f"rank{rank}.pt"))
    finally:
        torch.distributed.destroy_process_group()


@pytest.mark.parametrize("use_fused", [False, True])
def test_data_parallel_learn_with_8_bit_moments(tmp_path, use_fused):
    """Two ranks on one GPU (gloo) with shards of unequal length: the engine declines, the per-step paths
    (autograd; the native gradient step) clip and step the all-reduced gradient, and both ranks end with
    the same bits, codes included."""
    import os
    import torch.multiprocessing as mp
    mp.spawn(_dp_worker, args=(2, 29671 + int(use_fused), str(tmp_path), use_fused), nprocs=2, join=True)
    a, b = (torch.load(os.path.join(tmp_path, f"rank{r}.pt"), weights_only=True) for r in range(2))
    assert a["path"] == b["path"] == "graph" and a["replays"] > 0
    assert a["step"] == b["step"] == [20.0] * len(a["step"])
    for x, y in zip(a["params"] + a["codes"], b["params"] + b["codes"]):
        assert torch.equal(x, y) and bool(torch.isfinite(x).all())


def test_refusals_on_the_device():
    O = _optim()
    p = torch.nn.Parameter(torch.ones(10, device="cuda"))
    with pytest.raises(ValueError, match="share memory"):
        O.AdamW([p, torch.nn.Parameter(p.detach()[3:5])])
    with pytest.raises(ValueError, match="contiguous"):
        O.AdamW([torch.nn.Parameter(torch.ones(4, 6, device="cuda").t())])
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        O.AdamW([torch.nn.Parameter(torch.ones(4, dtype=torch.float64, device="cuda"))])
    with pytest.raises(ValueError, match="device tensor"):
        O.grad_norm([p, torch.ones(3)])
    with pytest.raises(ValueError, match="at least one"):
        O.grad_norm([])
    opt = O.AdamW([p], state_bits=8)
    p.grad = torch.ones_like(p)
    with pytest.raises(ValueError, match="max_norm"):
        opt.step(max_norm=-1.0)
    with pytest.raises(ValueError, match="max_norm"):
        opt.step(max_norm=float("nan"))
    opt.step()
    opt.state[p]["exp_rms"] = opt.state[p]["exp_rms"].float()
    with pytest.raises(ValueError, match="exp_rms"):
        opt.step()
    del opt.state[p]["exp_rms"]
    with pytest.raises(ValueError, match="no exp_rms"):
        opt.step()
    q = torch.nn.Parameter(torch.ones(10, device="cuda"))
    two = O.AdamW([p, q])
    q.grad = torch.ones_like(q)
    two.step()
    two.state[q]["step"] = two.state[p]["step"]
    with pytest.raises(ValueError, match="same memory"):
        two.step()
    two.state[q]["step"] = two.state[p]["step"].clone()
    two.step()
    two.state[q]["exp_avg_sq"] = two.state[p]["exp_avg_sq"]
    with pytest.raises(ValueError, match="same memory"):
        two.step()
    odd = O.AdamW([q])
    odd.param_groups[0]["betas"] = (0.9, 1.0)
    with pytest.raises(RuntimeError, match="betas"):
        odd.step()
    odd.param_groups[0].update(betas=(0.9, 0.99), lr=torch.ones((), dtype=torch.float64, device="cuda"))
    with pytest.raises(ValueError, match="device lr"):
        odd.step()
    fresh = O.AdamW([q])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="outside it first"):
        with torch.cuda.graph(graph):
            fresh.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_step_raises_the_parameters_versions(bits):
    """A graph kept from before a step is refused by backward() after it, as with torch's AdamW; parameters
    without a gradient keep their version."""
    for make in (lambda ps: _optim().AdamW(ps, state_bits=bits), torch.optim.AdamW):
        p, q, r = (torch.nn.Parameter(torch.randn(5, device="cuda")) for _ in range(3))
        opt = make([p, q, r])
        loss = (p * q).square().sum()
        loss.backward(retain_graph=True)
        for _ in range(2):                   # (the second: the list as it was laid out)
            before = p._version, q._version, r._version
            opt.step()
            assert p._version > before[0] and q._version > before[1] and r._version == before[2]
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                loss.backward(retain_graph=True)


def test_parameters_moved_onto_each_other_are_refused():
    """A step after p.data put a parameter over another's memory: refused before anything is launched."""
    flat = torch.ones(600, device="cuda")
    params = [torch.nn.Parameter(flat[:300]), torch.nn.Parameter(flat[300:])]
    for p in params:
        p.grad = torch.ones_like(p)
    opt = _optim().AdamW(params)
    opt.step()
    params[1].data = flat[299:599]
    old = flat.clone()
    with pytest.raises(ValueError, match="share memory"):
        opt.step()
    assert torch.equal(flat, old) and float(opt.state[params[0]]["step"]) == 1.0
    params[1].data = flat[300:]
    opt.step()
    assert float(opt.state[params[0]]["step"]) == 2.0 and not torch.equal(flat, old)


def test_gradients_cut_short_and_types_changed_in_place():
    """A gradient made shorter at its address is refused; a parameter that became another type at its address
    (and got a gradient of that type) steps as that type."""
    p = torch.nn.Parameter(torch.ones(40, device="cuda"))
    p.grad = torch.full_like(p, 0.5)
    opt = _optim().AdamW([p])
    opt.step()
    old, whole = p.detach().clone(), p.grad.data
    p.grad.data = whole[:3]
    with pytest.raises(ValueError, match="type and size"):
        opt.step()
    assert torch.equal(p.detach(), old) and float(opt.state[p]["step"]) == 1.0
    p.grad.data = whole
    opt.step()
    at = p.data_ptr()
    p.grad = None
    p.data = p.data.view(torch.bfloat16)[:40].fill_(0.25)
    p.grad = torch.full_like(p, 0.125)
    assert p.data_ptr() == at and p.dtype == torch.bfloat16
    before = _before(opt, [p], 32, False)
    opt.step()
    _check_step(opt, [p], before, 1.0, 3, (1e-3, (0.9, 0.999), 1e-8, 1e-2), 32)


# ---------------------------------------------------------------------------------- step counts past 2^24
def test_adamw8_draws_go_on_past_2_to_the_24_steps():
    """float32 counts whole steps up to 2^24.  From there 8-bit moments go on by the next float32, whose bits
    are hashed: the rounding is drawn anew at every step, and a second moment still follows the gradients
    beside a block's decaying largest one (as in test_adamw8_second_moment_follows_smaller_gradients,
    whose bounds these are).  32-bit moments need no
    draws: their count stays, as torch's does."""
    n, T = 1 << 16, 1500
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = _optim().AdamW([p], lr=0.0, state_bits=8, weight_decay=0.0)
    g = torch.ones(n, device="cuda")
    p.grad = g
    opt.step()
    st = opt.state[p]
    spike = torch.ones(n, device="cuda")
    spike[::2] = 10.0
    st["exp_rms_scale"].fill_(10.0)                     # as after many steps of `spike`
    st["exp_rms"].copy_(spike * 25.6)
    st["step"].fill_(2.0 ** 24 - 2)
    counts = []
    for k in range(T):
        opt.step()
        if k < 6:
            counts.append(float(st["step"]))
    assert counts == [2.0 ** 24 - 1, 2.0 ** 24, 2.0 ** 24 + 2, 2.0 ** 24 + 4, 2.0 ** 24 + 6, 2.0 ** 24 + 8]
    r = st["exp_rms"].float() * st["exp_rms_scale"].repeat_interleave(256) / 256
    keep = 0.999 ** T
    high, low = math.sqrt(100 * keep + 1 - keep), 1.0
    assert abs(float(r[::2].mean()) / high - 1) < 0.25 and abs(float(r[1::2].mean()) / low - 1) < 0.25
    q = torch.nn.Parameter(torch.zeros(4, device="cuda"))
    q.grad = torch.ones(4, device="cuda")
    other = _optim().AdamW([q])
    other.step()
    other.state[q]["step"].fill_(2.0 ** 24)
    other.step()
    assert float(other.state[q]["step"]) == 2.0 ** 24


@pytest.mark.parametrize("count,long", [(2.0 ** 24 - 1, False), (2.0 ** 24, False), (2.0 ** 25, True), (2.0 ** 40, True), (2.0 ** 70, False)])
def test_adamw8_large_counts_step_as_defined(count, long):
    """One step from a large count, in the one-launch form and the long one: the draws are those of the count's
    bits past 2^24, the bias corrections 1."""
    import struct
    params, grads = _make([300, 1000] + ([40000] if long else []), torch.float32, 17)
    opt = _optim().AdamW(params, lr=1e-3, state_bits=8)
    opt.step()
    for p in params:
        opt.state[p]["step"].fill_(count)
    before = _before(opt, params, 8, False)
    opt.step()
    for p, (w, g, m, v) in zip(params, before):
        st = opt.state[p]
        t = float(st["step"])
        up = struct.unpack("I", struct.pack("f", count))[0] + 1
        assert t == (count + 1 if count < 2.0 ** 24 else struct.unpack("f", struct.pack("I", up))[0])
        w1, m1, v1, ew, em, ev = R.step64(w, g, m, v, t, 1e-3, (0.9, 0.999), 1e-8, 1e-2, 1.0)
        assert bool(((p.detach().cpu().double() - w1).abs() <= ew).all())
        dm, dr = R.draws(p.numel(), int(t) if t <= 2.0 ** 24 else up)
        r1 = v1.sqrt()
        er = ev / (2 * r1.clamp(min=1e-70)) + 2 * R.U32 * r1
        for k, x, d, least, e in (("exp_avg", m1, dm, 0.0, em), ("exp_rms", r1, dr, 2.0 ** -9, er)):
            _, q, low, high = R.quantise(x, d, least, e)
            got = st[k].cpu().double()
            assert bool(((got.abs() >= low) & (got.abs() <= high)).all()), (k, p.numel())


# ---------------------------------------------------------------------------------- the one-launch form, value by value
SHORT = [1, 3, 4, 5, 255, 256, 257, 1023, 4097, 0, 17411, 777]     # 112 blocks of 256 in 12 tensors


def _one_launch(opt):
    import prl_native
    return prl_native.list_workspace_bytes(opt._plan.table, len(opt.param_groups)) == 0


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,master", [(torch.float32, False), (torch.bfloat16, False),
                                          (torch.bfloat16, True), (torch.float16, False),
                                          (torch.float16, True)])
@pytest.mark.parametrize("max_norm", [None, 0.5])
def test_adamw_steps_in_one_launch(bits, dtype, master, max_norm):
    """Three steps (the first from empty state) of a list that one launch takes, clipped (0 < c < 1) and not."""
    params, grads = _make(SHORT, dtype, 13)
    hyper = (1e-2, (0.9, 0.999), 1e-8, 0.1)
    opt = _optim().AdamW(params, lr=hyper[0], betas=hyper[1], eps=hyper[2], weight_decay=hyper[3],
                         state_bits=bits, master=master)
    gen = torch.Generator(device="cuda").manual_seed(3)
    for t in (1, 2, 3):
        before = _before(opt, params, bits, t == 1)
        norm = R.norm64(grads)
        opt.step(max_norm=max_norm)
        assert _one_launch(opt)
        if max_norm is not None:
            assert norm > max_norm and abs(float(opt.total_norm) - norm) <= 1.01 * R.U32 * norm
        _check_step(opt, params, before, R.clip64(norm, max_norm), t, hyper, bits)
        for g in grads:
            g.copy_(torch.randn(g.shape, generator=gen, device="cuda") * 0.03)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_groups_and_types_in_one_launch(bits):
    """16 groups with hyper-parameters of their own, types and masters mixed, one group's lr on the device."""
    groups, every = [], []
    for i in range(16):
        dtype = (torch.float32, torch.bfloat16, torch.float16)[i % 3]
        params, _ = _make([1 + (37 * i + 11 * j) % 700 for j in range(2)], dtype, i, packed=i % 2 == 0)
        lr = 1e-3 * (i + 1)
        betas = (0.8 + 0.01 * i, 0.99)
        groups.append(dict(params=params, lr=torch.full((), lr, device="cuda") if i == 4 else lr,
                           betas=betas, weight_decay=0.01 * i, master=i % 2 == 1))
        every.append((params, (float(torch.tensor(lr)) if i == 4 else lr, betas, 1e-8, 0.01 * i)))
    opt = _optim().AdamW(groups, state_bits=bits)
    for t in (1, 2):
        norm = R.norm64([p.grad for params, _ in every for p in params])
        befores = [_before(opt, params, bits, t == 1) for params, _ in every]
        opt.step(max_norm=1.0)
        assert _one_launch(opt) and norm > 1.0
        for (params, hyper), before in zip(every, befores):
            _check_step(opt, params, before, R.clip64(norm, 1.0), t, hyper, bits)


@pytest.mark.parametrize("bits", [32, 8])
def test_clipped_step_at_the_one_launch_bound_and_past_it(bits):
    """160 blocks in one launch, 161 in several: both clipped steps against the restatement."""
    for sizes, short in (([160 * 256], True), ([160 * 256, 1], False)):
        params, grads = _make(sizes, torch.float32, 4, lead=3)
        hyper = (1e-3, (0.9, 0.999), 1e-8, 1e-2)
        opt = _optim().AdamW(params, lr=hyper[0], betas=hyper[1], eps=hyper[2], weight_decay=hyper[3], state_bits=bits)
        for t in (1, 2):
            before, norm = _before(opt, params, bits, t == 1), R.norm64(grads)
            opt.step(max_norm=0.25 * norm)
            assert _one_launch(opt) == short
            _check_step(opt, params, before, R.clip64(norm, 0.25 * norm), t, hyper, bits)

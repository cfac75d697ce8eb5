"""The list optimizer without a GPU: its C-ABI (include/prl_optim.h) and that header's symbols, what
it refuses before anything is launched, and the float64 restatement the GPU tests rely on."""
import ctypes
import os
import re
from array import array

import pytest
import torch

import optim_ref as R
from conftest import ROOT


def test_header_symbols_are_exported_and_bound():
    import prl_native
    hdr = open(os.path.join(ROOT, "include", "prl_optim.h")).read()
    syms = sorted(set(re.findall(r"^\s*(?:int|int64_t)\s+(prl_list_\w+)\s*\(", hdr, re.M)))
    assert syms == sorted(prl_native.OPTIM_SIGNATURES)
    assert all(hasattr(prl_native.lib(), s) for s in syms)
    assert len(prl_native.list_entry()) == prl_native.LIST_ENTRY_WORDS
    assert int(re.search(r"#define PRL_LIST_BLOCK (\d+)", hdr).group(1)) == prl_native.LIST_BLOCK


def _adamw(entries, groups=((1e-3, 0.9, 0.999, 1e-8, 0.0, 0),), n_groups=None, ws=1 << 20, norm=None, max_norm=1.0, bytes_=None):
    """prl_list_adamw's status on a list that it must refuse (addresses are never touched)."""
    import struct
    import prl_native
    L = prl_native.lib()
    table = array("q", [w for e in entries for w in e])
    g = b"".join(struct.pack("5dq", *x) for x in groups)
    rc = L.prl_list_adamw(table.buffer_info()[0] if entries else None, len(entries), g, len(groups) if n_groups is None else n_groups,
                          max_norm, norm, ws, 1 << 20 if bytes_ is None else bytes_, None)
    return rc, L.prl_last_error().decode()


def test_c_entry_refuses_bad_lists():
    from prl_native import list_entry
    ok = dict(param=4096, grad=8192, exp_avg=12288, second=16384, step=20480, numel=10)
    cases = [
        (dict(ok, dtype=3), "unknown type"), (dict(ok, dtype=-1), "unknown type"),
        (dict(ok, numel=-1), "bad size"), (dict(ok, numel=1 << 40), "bad size"), (dict(ok, numel=(1 << 34) + 1), "bad size"),
        (dict(ok, bits=16), "moments in 16 bits"), (dict(ok, group=1), "group 1 of 1"), (dict(ok, group=-1), "group -1"),
        (dict(ok, step=0), "null step"), (dict(ok, grad=0), "null grad"), (dict(ok, param=0), "null pointer"),
        (dict(ok, second=0), "null pointer"), (dict(ok, bits=8), "null pointer"),
        (dict(ok, master=4096), "has no master"), (dict(ok, grad=8194), "grad not aligned"),
        (dict(ok, param=4098), "not aligned"), (dict(ok, exp_avg=12289), "not aligned"), (dict(ok, step=20481), "not aligned"),
    ]
    for e, text in cases:
        rc, msg = _adamw([list_entry(**ok), list_entry(**e)])
        assert rc == -1 and text in msg, (e, msg)
    long = [list_entry(**ok)] * 33          # more than the launch of a short list takes: a workspace is needed
    assert _adamw(long, bytes_=64)[0] == -1
    assert _adamw(long, ws=None)[0] == -1
    assert _adamw(long, ws=(1 << 20) + 8)[0] == -1
    assert _adamw([list_entry(**ok)], norm=4096, max_norm=-1.0)[0] == -1
    assert _adamw([list_entry(**ok)], norm=4096, max_norm=float("nan"))[0] == -1
    for bad in ((1e-3, 1.0, 0.9, 0.0, 0.0, 0), (1e-3, 0.9, -0.1, 0.0, 0.0, 0), (-1.0, 0.9, 0.9, 0.0, 0.0, 0), (1e-3, 0.9, 0.9, -1.0, 0.0, 0),
                (1e-3, 0.9, 0.9, 0.0, -1.0, 0), (float("nan"), 0.9, 0.9, 0.0, 0.0, 0), (1e-3, 0.9, float("nan"), 0.0, 0.0, 0)):
        assert _adamw([list_entry(**ok)], groups=(bad,))[0] == -1
    assert _adamw([list_entry(**ok)], n_groups=-1)[0] == -1
    assert _adamw([])[0] == 0          # nothing to do, nothing launched
    import prl_native
    L = prl_native.lib()
    assert L.prl_list_workspace_bytes(None, -1, 1) == -1
    def need(entries, groups=1):
        t = array("q", [w for e in entries for w in e])
        return L.prl_list_workspace_bytes(t.buffer_info()[0], len(entries), groups)
    assert need([list_entry(**ok)] * 32) == 0 and need(long) >= 33 * 56
    assert need([list_entry(**dict(ok, numel=160 * 256))]) == 0 and need([list_entry(**dict(ok, numel=160 * 256 + 1))]) > 0
    assert need([list_entry(**ok)], 17) > 0 and need([list_entry(**dict(ok, numel=-1))]) == -1
    assert L.prl_list_norm(None, 1, 4096, 4096, 1 << 20, None) == -1
    assert L.prl_list_norm(None, -1, 4096, 4096, 1 << 20, None) == -1
    assert L.prl_list_norm(None, 0, None, 4096, 1 << 20, None) == -1
    total = array("q", [w for _ in range(3) for w in list_entry(grad=4096, numel=(1 << 40) - 1)])
    assert L.prl_list_norm(total.buffer_info()[0], 3, 4096, 4096, 1 << 20, None) == -1
    assert "too large" in L.prl_last_error().decode()


def test_c_entry_refuses_unaligned_norm_and_lr():
    from prl_native import list_entry
    import prl_native
    L = prl_native.lib()
    ok = list_entry(param=4096, grad=8192, exp_avg=12288, second=16384, step=20480, numel=10)
    rc, msg = _adamw([ok], norm=4098)
    assert rc == -1 and "norm not aligned" in msg
    rc, msg = _adamw([ok], groups=((0.0, 0.9, 0.999, 1e-8, 0.0, 4097),))
    assert rc == -1 and "lr_dev not aligned" in msg
    table = array("q", ok)
    assert L.prl_list_norm(table.buffer_info()[0], 1, 4097, None, 0, None) == -1
    assert "norm not aligned" in L.prl_last_error().decode()


def test_python_refusals():
    from PPO.optim import AdamW, grad_norm
    p = torch.nn.Parameter(torch.ones(6))
    for kw in (dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=-1.0),
               dict(state_bits=16)):
        with pytest.raises(ValueError):
            AdamW([p], **kw)
    with pytest.raises(ValueError, match="share memory"):
        AdamW([p, torch.nn.Parameter(p.detach()[2:4])])
    opt = AdamW([p])
    with pytest.raises(ValueError, match="share memory"):
        opt.add_param_group(dict(params=[torch.nn.Parameter(p.detach()[:1])]))
    assert len(opt.param_groups) == 1
    p.grad = torch.ones(6)
    with pytest.raises(ValueError, match="device tensor"):
        opt.step()
    with pytest.raises(ValueError, match="device tensor"):
        grad_norm([p.grad])
    assert torch.equal(p.detach(), torch.ones(6)) and not opt.state[p].get("exp_avg", None)


def test_steps_of_nothing():
    """No gradients, or no parameters at all: no step, a norm of 0 in float32 whatever torch's default type is."""
    from PPO.optim import AdamW
    torch.set_default_dtype(torch.float64)
    try:
        for params in ([torch.nn.Parameter(torch.ones(3, dtype=torch.float32))], [dict(params=[])]):
            opt = AdamW(params)
            assert opt.step() is None and opt.total_norm is None
            assert opt.step(max_norm=1.0) is None
            assert opt.total_norm.dtype == torch.float32 and opt.total_norm.shape == () and float(opt.total_norm) == 0.0
    finally:
        torch.set_default_dtype(torch.float32)


def test_learn_keeps_its_step_for_other_optimizers():
    """clip_and_step is clip_grad_norm_ + step() for any optimizer that is not this AdamW."""
    from PPO.optim import clip_and_step
    p = torch.nn.Parameter(torch.ones(4))
    q = torch.nn.Parameter(torch.ones(4))
    p.grad, q.grad = torch.full((4,), 3.0), torch.full((4,), 3.0)
    clip_and_step(torch.optim.SGD([p], lr=0.1), [p], 2.0)
    torch.nn.utils.clip_grad_norm_([q], 2.0)
    torch.optim.SGD([q], lr=0.1).step()
    assert torch.equal(p, q) and torch.equal(p.grad, q.grad)


@pytest.mark.parametrize("held,fused", [((0, 1, 2), True), ((2, 0, 1), True), ((0, 1, 2, 4), True), ((0, 1, 2, 3), False), ((0, 1), False)])
def test_clip_and_step_takes_one_call_only_for_exactly_these_gradients(monkeypatch, held, fused):
    """The list AdamW clips by the norm of all it holds: parameters 0 - 2 are clipped in its step only if these
    are all that have a gradient in it (4 has none); else their gradients are, by their own norm."""
    from PPO.optim import AdamW, clip_and_step
    params = [torch.nn.Parameter(torch.ones(4)) for _ in range(5)]
    for i, p in enumerate(params[:4]):
        p.grad = torch.full((4,), 3.0 + i)
    opt = AdamW([params[i] for i in held])
    calls = []
    monkeypatch.setattr(opt, "step", lambda **kw: calls.append(kw))
    clip_and_step(opt, params[:3], 2.0)
    assert calls == [{"max_norm": 2.0} if fused else {}]
    want = [torch.full((4,), 3.0 + i) for i in range(4)]
    if not fused:
        c = 2.0 / (sum(4 * (3.0 + i) ** 2 for i in range(3)) ** 0.5 + 1e-6)
        want[:3] = [g * c for g in want[:3]]
    assert all(torch.allclose(p.grad, w, rtol=1e-6, atol=0.0) for p, w in zip(params, want))


def test_flat_state_looks_at_the_state():
    """The engine is offered float32 moments only: state of the other form, of another size or incomplete is not
    its business, whatever state_bits says; a parameter may have none yet."""
    from PPO.optim import AdamW
    p, q = torch.nn.Parameter(torch.ones(6)), torch.nn.Parameter(torch.ones(3))
    opt = AdamW([p, q])
    good = dict(step=torch.zeros(()), exp_avg=torch.zeros(6), exp_avg_sq=torch.zeros(6))
    assert opt.flat_state([p, q])
    opt.state[p] = dict(good)
    assert opt.flat_state([p, q]) and not opt.flat_state([q, p]) and not opt.flat_state([p])
    codes = torch.zeros(6, dtype=torch.float8_e4m3fn)
    for bad in (dict(step=torch.zeros(()), exp_avg=codes, exp_rms=codes), dict(good, exp_avg=codes),
                dict(good, exp_avg_sq=torch.zeros(5)), dict(good, exp_avg_sq=torch.zeros(6, dtype=torch.float64)),
                {k: v for k, v in good.items() if k != "step"}):
        opt.state[p] = bad
        assert not opt.flat_state([p, q])


def _laid_out(monkeypatch, opt):
    """What a step checks before anything is launched, for parameters on the CPU."""
    import PPO.optim as O
    monkeypatch.setattr(O, "_dense", lambda tensors, device, name: tensors)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    params = [p for g in opt.param_groups for p in g["params"]]
    return O._Plan(opt, opt.param_groups, params, [p.grad for p in params])


@pytest.mark.parametrize("bits", [32, 8])
def test_a_list_whose_written_tensors_overlap_is_not_laid_out(monkeypatch, bits):
    """Parameters moved onto each other after the optimizer was made, and state that overlaps state or a
    parameter in any part, are refused; neighbours without a gap are not."""
    from PPO.optim import AdamW

    def make():
        flat = torch.ones(600)
        params = [torch.nn.Parameter(flat[:300]), torch.nn.Parameter(flat[300:])]
        for p in params:
            p.grad = torch.ones(300)
        opt = AdamW(params, state_bits=bits)
        _laid_out(monkeypatch, opt)                  # makes the state
        return opt, params, flat

    opt, params, flat = make()
    _laid_out(monkeypatch, opt)
    params[1].data = flat[299:599]
    with pytest.raises(ValueError, match="share memory"):
        _laid_out(monkeypatch, opt)
    params[1].data = flat[300:]
    _laid_out(monkeypatch, opt)
    second = "exp_avg_sq" if bits == 32 else "exp_rms"
    whole = torch.zeros(600).to(opt.state[params[0]]["exp_avg"].dtype)
    for one, two in (((0, "exp_avg"), (1, "exp_avg")), ((0, "exp_avg"), (0, second)), ((1, second), (0, "exp_avg"))):
        for at, shared in ((299, True), (300, False)):
            opt, params, flat = make()
            for (i, k), lo in ((one, 0), (two, at)):
                opt.state[params[i]][k] = whole[lo:lo + 300]
            if shared:
                with pytest.raises(ValueError, match="same memory"):
                    _laid_out(monkeypatch, opt)
            else:
                _laid_out(monkeypatch, opt)
    opt, params, flat = make()
    opt.state[params[0]]["step"] = flat[10:11].view(())
    with pytest.raises(ValueError, match="a parameter and a state tensor are"):
        _laid_out(monkeypatch, opt)
    opt, params, flat = make()
    opt.state[params[0]]["step"] = opt.state[params[1]]["step"]
    with pytest.raises(ValueError, match="same memory"):
        _laid_out(monkeypatch, opt)


def test_a_laid_out_list_does_not_serve_other_sizes_or_types(monkeypatch):
    """Gradients that were cut short or changed their type where they lie: the list is to be laid out, and
    checked, again."""
    from PPO.optim import AdamW
    p, q = torch.nn.Parameter(torch.ones(10)), torch.nn.Parameter(torch.ones(4))
    p.grad, q.grad = torch.ones(10), torch.ones(4)
    opt = AdamW([p, q])
    plan = _laid_out(monkeypatch, opt)
    grads = [p.grad, q.grad]
    for _ in range(2):
        table, keep = plan.fill(grads)
        assert [table[1], table[12]] == [g.data_ptr() for g in grads]
    at, whole = p.grad.data_ptr(), p.grad.data
    p.grad.data = whole[:3]
    assert p.grad.data_ptr() == at and plan.holds(opt.param_groups, [p, q], grads, opt.state)
    assert plan.fill(grads) is None
    with pytest.raises(ValueError, match="type and size"):
        _laid_out(monkeypatch, opt)
    assert plan.fill([whole.view(torch.bfloat16)[:10], q.grad]) is None
    assert plan.fill([whole, q.grad]) is not None


def test_clip_and_step_takes_what_clip_grad_norm_takes(monkeypatch):
    """An iterator of parameters, or one tensor."""
    from PPO.optim import AdamW, clip_and_step
    for of, given in ((1, lambda ps: iter(ps)), (2, lambda ps: iter(ps)), (2, lambda ps: ps[0]), (1, lambda ps: ps[0])):
        params = [torch.nn.Parameter(torch.ones(4)) for _ in range(2)]
        for p in params:
            p.grad = torch.full((4,), 3.0)
        opt = AdamW(params[:of])
        calls = []
        monkeypatch.setattr(opt, "step", lambda **kw: calls.append(kw))
        one = torch.is_tensor(given(params))
        clip_and_step(opt, given(params), 2.0)
        fused = (of == 1) == one
        assert calls == [{"max_norm": 2.0} if fused else {}]
        norm = (36.0 if one else 72.0) ** 0.5
        want = 3.0 if fused else 3.0 * 2.0 / (norm + 1e-6)
        assert torch.allclose(params[0].grad, torch.full((4,), want), rtol=1e-6, atol=0.0)


# ---------------------------------------------------------------------------------- the restatement itself
def test_restatement_is_torch_adamw():
    gen = torch.Generator().manual_seed(0)
    w = torch.randn(50, generator=gen, dtype=torch.float64)
    p = torch.nn.Parameter(w.clone())
    opt = torch.optim.AdamW([p], lr=1e-2, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.1)
    m = v = torch.zeros(50, dtype=torch.float64)
    for t in (1, 2, 3):
        g = torch.randn(50, generator=gen, dtype=torch.float64)
        p.grad = g.clone()
        norm = float(torch.nn.utils.clip_grad_norm_([p], 0.5))
        opt.step()
        assert abs(R.norm64([g]) - norm) < 1e-12 * norm
        w, m, v, *_ = R.step64(w, g, m, v, t, 1e-2, (0.8, 0.95), 1e-6, 0.1, R.clip64(norm, 0.5))
        assert torch.allclose(w, p.detach(), rtol=1e-12, atol=1e-14)


def test_restatement_rounds_to_neighbours_on_the_e4m3_grid():
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(1000, generator=gen, dtype=torch.float64) * 10.0 ** torch.linspace(-8, 0, 1000, dtype=torch.float64)
    d, _ = R.draws(1000, 5)
    assert int(d.min()) >= 0 and int(d.max()) < 65536 and abs(float(d.double().mean()) / 32768 - 1) < 0.1
    A, q, low, high = R.quantise(x, d, 0.0)
    assert torch.equal(q.float().to(torch.float8_e4m3fn).double(), q)             # on the grid
    y = x / A.repeat_interleave(256)[:1000] * 256
    unit = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    assert bool(((q - y).abs() < unit).all())
    lowest = R.quantise(x, d * 0, 2.0 ** -9)[1]
    assert bool((lowest.abs() >= 2.0 ** -9).all())                                  # nothing becomes 0
    # two values may be held where, and only where, the error reaches over a border
    assert float((low < high).double().mean()) < 0.01
    _, q, low, high = R.quantise(x, d, 0.0, x.abs() * 1e-3)
    assert bool(((low <= q.abs()) & (q.abs() <= high)).all())
    assert 0.001 < float((low < high).double().mean()) < 0.1

"""adamw_step and the AdamW solver: against the formula in 64 bits, and the 8-bit
codes against the torch implementation, code for code."""

import math

import pytest
import torch

from npairloss_amd.engine import AdamW, CaffeSGD, build_optimizer
from npairloss_amd.config.params import SolverConfig
from npairloss_amd.ops import adamw_state, adamw_step
from transformer_util import DEVICES, TYPES, U, assert_within, half_step, least, replays

HYPER = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)
SIZES = [(1,), (7,), (8,), (255,), (256,), (257,), (33, 65), (4096,), (4097,), (3, 5, 7, 11), (0,), (20000,)]


def make(sizes, dtype, device, bits, master, seed=0):
    g = torch.Generator().manual_seed(seed)
    params = [torch.randn(s, generator=g).to(dtype).to(device) for s in sizes]
    grads = [(0.1 * torch.randn(s, generator=g)).to(dtype).to(device) for s in sizes]
    states = [adamw_state(p, bits=bits, master=master) for p in params]
    return params, grads, states


def call(params, grads, states, seed=0, **more):
    get = lambda n: [s[n] for s in states]  # noqa: E731
    adamw_step(params, grads, get("exp_avg"), get("exp_avg_sq"), get("step"), masters=get("master") if "master" in states[0] else None,
               scales=get("scales") if "scales" in states[0] else None, seed=seed, **{**HYPER, **more})


def exact_step(p, g, m, v, t, lr, betas, eps, weight_decay):
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    update = lr * (m / (1 - betas[0] ** t)) / (torch.sqrt(v / (1 - betas[1] ** t)) + eps)
    return p * (1 - lr * weight_decay) - update, m, v, update


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("master", [False, True])
def test_32_bits(dtype, master, device):
    params, grads, states = make(SIZES, dtype, device, 32, master)
    wide = [p.double().cpu() for p in params]
    moments = [(torch.zeros_like(w), torch.zeros_like(w)) for w in wide]
    for t in range(1, 4):
        call(params, grads, states)
        for i, (p, g, s) in enumerate(zip(params, grads, states)):
            w, m, v, update = exact_step(wide[i], g.double().cpu(), *moments[i], t, **HYPER)
            # coefficients, products and sums: under 8 U a step of the moments' magnitudes (no term cancels more than
            # the other: both are kept with their error), and under 40 U of the update (two expm1, a root, three quotients)
            mags = sum(0.9 ** k * 0.1 for k in range(t)) * g.double().cpu().abs()
            assert_within(s["exp_avg"], m, 8 * t * U * mags + 1e-44, "m")
            assert_within(s["exp_avg_sq"], v, 8 * t * U * v + 1e-44, "v")
            kept = s.get("master", p)
            tol = 4 * U * w.abs() + 40 * t * U * update.abs()
            if kept.dtype == torch.float32:
                assert_within(kept, w, tol + least(torch.float32), "weights")
            assert_within(p, w, tol + half_step(dtype) * (w.abs() + tol) + least(dtype), "parameters")
            if "master" in s:
                assert torch.equal(p, s["master"].to(dtype))
            assert int(s["step"]) == t
            # go on from what is stored, so that errors do not add up over steps
            wide[i], moments[i] = kept.double().cpu(), (s["exp_avg"].double().cpu(), s["exp_avg_sq"].double().cpu())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_8_bits_against_the_formula(dtype, device):
    params, grads, states = make(SIZES, dtype, device, 8, True)
    for t in range(1, 4):
        before = []
        for p, s in zip(params, states):
            n = p.numel()
            spread = torch.repeat_interleave(s["scales"].double().cpu(), 256, 0)[:n]
            before.append((s.get("master", p).double().cpu(), s["exp_avg"].double().cpu() * spread[:, 0].view(p.shape),
                           (s["exp_avg_sq"].double().cpu() * spread[:, 1].view(p.shape)) ** 2))
        call(params, grads, states, seed=t)
        for p, g, s, (w0, m0, v0) in zip(params, grads, states, before):
            w, m, v, update = exact_step(w0, g.double().cpu(), m0, v0, t, **HYPER)
            kept = s.get("master", p).double().cpu()
            tol = 4 * U * w.abs() + 40 * U * (update.abs() + HYPER["lr"] * 0.1 * (m0.abs() + g.double().cpu().abs()) / (v.sqrt() + 1e-6) * 20)
            assert_within(kept, w, tol + least(torch.float32), "weights")
            n = p.numel()
            blocks = -(-n // 256)
            pad = lambda x: torch.nn.functional.pad(x.flatten(), (0, blocks * 256 - n)).view(blocks, 256)  # noqa: E731
            for i, (codes, x) in enumerate(((s["exp_avg"], pad(m)), (s["exp_avg_sq"], pad(v.sqrt())))):
                scale = s["scales"][:, i].double().cpu()
                assert_within(scale, (x.abs().amax(1) / 448).clamp_min(2.0 ** -126) if blocks else scale, scale * 20 * U, "scales")
                value = pad(codes.double().cpu()) * scale[:, None]
                step = torch.exp2(torch.floor(torch.log2((x.abs() / scale[:, None]).clamp_min(2.0 ** -6))) - 3) * scale[:, None]
                # up or down: within a whole step (the next power's where x is just under it)
                assert_within(value, x, step * (1 + 1e-5) + x.abs() * 20 * U, "codes")
                if i:
                    assert ((value > 0) == (x > 0)).all()


def test_8_bits_are_unbiased():
    """Over 400 seeds the mean of m is m, and that of v is v.  A value lies between two
    neighbours a step apart, so its variance is at most a quarter of the step squared:
    the mean of 400 is off by over 5 deviations (step / 8) in one of 10^6 values."""
    seeds, n = 400, 512
    g = torch.Generator().manual_seed(1)
    grad = torch.randn(n, generator=g)
    sums = torch.zeros(2, n, dtype=torch.float64)
    for seed in range(seeds):
        p = torch.zeros(n)
        s = adamw_state(p, bits=8)
        call([p], [grad], [s], seed=seed * 7919)
        spread = torch.repeat_interleave(s["scales"].double(), 256, 0)
        sums[0] += s["exp_avg"].double() * spread[:, 0]
        sums[1] += (s["exp_avg_sq"].double() * spread[:, 1]) ** 2
    m, v = 0.1 * grad.double(), 0.01 * grad.double() ** 2
    top = torch.repeat_interleave(torch.stack([m.view(-1, 256).abs().amax(1), v.view(-1, 256).sqrt().amax(1)], 1) / 448, 256, 0)
    for i, x in enumerate((m.abs(), v.sqrt())):
        step = torch.exp2(torch.floor(torch.log2((x / top[:, i]).clamp_min(2.0 ** -6))) - 3) * top[:, i]
        want, width = (m, step) if i == 0 else (v, (x + step) ** 2 - (x - 0) ** 2)
        # the least root that is kept: what lies under it is rounded up, by at most its square
        more = 0 if i == 0 else (2.0 ** -9 * top[:, 1]) ** 2
        assert_within(sums[i] / seeds, want, width / 8 + more + 1e-6 * want.abs(), "mean %d" % i)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_8_bits_code_for_code(dtype):
    """GPU and CPU: equal codes and scales, over steps; masters to 8 roundings."""
    cpu = make(SIZES, dtype, "cpu", 8, True, seed=5)
    gpu = make(SIZES, dtype, "cuda", 8, True, seed=5)
    for t in range(3):
        call(*cpu, seed=77)
        call(*gpu, seed=77)
        for i, (a, b) in enumerate(zip(cpu[2], gpu[2])):
            for n in ("exp_avg", "exp_avg_sq", "scales", "step"):
                assert torch.equal(a[n].float(), b[n].float().cpu()), (t, SIZES[i], n)
            x, y = (s[2][i].get("master", s[0][i]) for s in (cpu, gpu))
            assert_within(y.float(), x.float(), 8 * U * x.double().abs() + 100 * U * HYPER["lr"] * 10 + (half_step(dtype) * 2 * x.double().abs() if "master" not in a and dtype != torch.float32 else 0), "weights")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
def test_not_finite(bits, device):
    """A gradient that is not finite costs its own element and no other."""
    params, grads, states = make([(600,)], torch.float32, device, bits, False)
    other = make([(600,)], torch.float32, device, bits, False)
    for i, x in ((3, float("nan")), (300, float("inf"))):
        grads[0][i] = x
        other[1][0][i] = 0.0
    for _ in range(2):
        call(params, grads, states)
        call(*other)
    lost = torch.zeros(600, dtype=torch.bool)
    lost[[3, 300]] = True
    assert params[0][3].isnan() and params[0][300].isnan()
    assert torch.equal(params[0].cpu()[~lost], other[0][0].cpu()[~lost])
    for n in ("exp_avg", "exp_avg_sq"):
        assert torch.equal(states[0][n].float().cpu()[~lost], other[2][0][n].float().cpu()[~lost])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
def test_layouts(bits, device):
    """channels_last parameters, gradients in another order or off the 16-byte border."""
    g = torch.Generator().manual_seed(3)
    p = torch.randn(8, 5, 3, 3, generator=g).to(device)
    grad = torch.randn(8, 5, 3, 3, generator=g).to(device)
    last = p.clone(memory_format=torch.channels_last)
    flat = torch.empty(p.numel() + 1, device=device)[1:]
    view = flat.as_strided(last.shape, last.stride(), flat.storage_offset()).copy_(grad)
    for gr in (grad, grad.contiguous(memory_format=torch.channels_last), view):
        x = last.clone(memory_format=torch.channels_last)
        s = adamw_state(x, bits=bits)
        assert s["exp_avg"].stride() == x.stride()
        call([x], [gr], [s])
        want = exact_step(p.double().cpu(), grad.double().cpu(), 0.0, 0.0, 1, **HYPER)
        assert_within(x, want[0], 4 * U * want[0].abs() + 60 * U * want[3].abs() + least(torch.float32))


@pytest.mark.parametrize("device", DEVICES)
def test_many_tensors(device):
    """More tensors than one launch takes, with counts of steps that differ."""
    sizes = [(1 + 13 * i % 700,) for i in range(470)]
    params, grads, states = make(sizes, torch.float32, device, 32, False)
    for i, s in enumerate(states):
        s["step"].fill_(i % 5)
    start = [p.double().cpu() for p in params]
    call(params, grads, states)
    for i, (p, g, s) in enumerate(zip(params, grads, states)):
        w, _, _, update = exact_step(start[i], g.double().cpu(), 0.0, 0.0, i % 5 + 1, **HYPER)
        assert_within(p, w, 4 * U * w.abs() + 60 * U * update.abs() + least(torch.float32))
        assert int(s["step"]) == i % 5 + 1


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    params, grads, states = make([(300,), (20,)], torch.float32, device, 32, False)
    eight = make([(300,), (20,)], torch.float32, device, 8, False)
    get = lambda n, s=states: [x[n] for x in s]  # noqa: E731
    ok = dict(params=params, grads=grads, exp_avgs=get("exp_avg"), exp_avg_sqs=get("exp_avg_sq"), steps=get("step"), **HYPER)
    bad = [dict(grads=grads[:1]), dict(grads=[grads[0], grads[1][:19]]), dict(grads=[x.half() for x in grads]), dict(lr=-1.0), dict(betas=(1.0, 0.9)),
           dict(eps=-1.0), dict(weight_decay=float("nan")), dict(exp_avgs=[x.half() for x in get("exp_avg")]), dict(steps=[x.float() for x in get("step")]),
           dict(params=[params[0], params[1].half()]), dict(scales=get("scales", eight[2])), dict(exp_avgs=get("exp_avg", eight[2])),
           dict(masters=[x.half() for x in params]), dict(params=[torch.zeros(600, device=device)[::2], params[1]])]
    before = [p.clone() for p in params]
    for change in bad:
        with pytest.raises((ValueError, TypeError)):
            adamw_step(**{**ok, **change})
    assert all(torch.equal(a, b) for a, b in zip(before, params))
    short = [x[:1] for x in get("scales", eight[2])]
    with pytest.raises(ValueError):
        adamw_step(**{**ok, "exp_avgs": get("exp_avg", eight[2]), "exp_avg_sqs": get("exp_avg_sq", eight[2]), "scales": short})
    with pytest.raises(ValueError):
        adamw_state(params[0], bits=4)
    with pytest.raises(TypeError):
        adamw_state(params[0].double())
    with pytest.raises(ValueError):
        adamw_state(params[0][::2])
    adamw_step([], [], [], [], [], lr=0.1)


@pytest.mark.gpu
def test_the_same_tensor_twice_is_refused():
    params, grads, states = make([(300,)], torch.float32, "cuda", 32, False)
    with pytest.raises(RuntimeError, match="twice"):
        call(params * 2, grads * 2, states * 2)
    more = make([(300,)], torch.float32, "cuda", 32, False)
    more[2][0]["step"] = states[0]["step"]
    with pytest.raises(RuntimeError, match="twice"):
        call(params + more[0], grads + more[1], states + more[2])
    for name in ("exp_avg", "exp_avg_sq"):
        more = make([(300,)], torch.float32, "cuda", 32, False)
        more[2][0][name] = states[0][name]
        with pytest.raises(RuntimeError, match="twice"):
            call(params + more[0], grads + more[1], states + more[2])


@pytest.mark.parametrize("device", DEVICES)
def test_a_graph_that_saved_a_parameter_learns_of_the_step(device):
    w = torch.randn(40, device=device, requires_grad=True)
    loss = (w * w).sum()
    state = adamw_state(w)
    adamw_step([w], [torch.ones_like(w)], [state["exp_avg"]], [state["exp_avg_sq"]], [state["step"]], lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
def test_solver_state_goes_on(bits, device):
    """A run that is saved and loaded in its middle ends where one that is not does."""
    def run(stop):
        torch.manual_seed(0)
        model = torch.nn.Linear(40, 30).to(device).to(torch.bfloat16)
        x = torch.randn(16, 40, generator=torch.Generator().manual_seed(1)).to(device).to(torch.bfloat16)
        opt = AdamW(model.parameters(), lr=1e-2, master_weights=True, state_bits=bits, seed=3)
        for i in range(6):
            if i == stop:
                saved = opt.state_dict()
                opt = AdamW(model.parameters(), lr=5.0, master_weights=True, state_bits=bits)
                opt.load_state_dict(saved)
                st = opt.state[model.weight]
                assert st["master"].dtype == torch.float32 and st["exp_avg"].dtype == (torch.float8_e4m3fn if bits == 8 else torch.float32)
                assert st["step"].dtype == torch.int32 and int(st["step"]) == i
            opt.zero_grad()
            model(x).float().square().mean().backward()
            opt.step()
        return [p.detach().clone() for p in model.parameters()] + [opt.state[model.weight]["master"]]

    for a, b in zip(run(-1), run(3)):
        assert torch.equal(a, b)


def test_solver_skips_what_has_no_gradient():
    a, b = (torch.nn.Parameter(torch.ones(5)) for _ in range(2))
    opt = AdamW([a, b], lr=0.1)
    a.grad = torch.ones(5)
    opt.step()
    assert (b == 1).all() and b not in opt.state and int(opt.state[a]["step"]) == 1
    opt.set_lr(0.0)
    assert opt.param_groups[0]["lr"] == 0.0
    for bad in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0)):
        with pytest.raises(ValueError):
            AdamW([a], **bad)


def test_solver_from_prototxt():
    solver = SolverConfig.from_prototxt('type: "AdamW" base_lr: 0.002 momentum: 0.8 momentum2: 0.95 delta: 1e-7 weight_decay: 0.3 state_bits: 8 random_seed: 4')
    opt = build_optimizer(torch.nn.Linear(3, 3), solver, master_weights=True)
    g = opt.param_groups[0]
    assert isinstance(opt, AdamW) and (g["lr"], g["betas"], g["eps"], g["weight_decay"], g["state_bits"], g["seed"]) == (0.002, (0.8, 0.95), 1e-7, 0.3, 8, 4)
    assert isinstance(build_optimizer(torch.nn.Linear(3, 3), SolverConfig()), CaffeSGD)


def test_trainer_refuses_sgd_snapshots(tmp_path):
    from npairloss_amd import NPairLossConfig, NPairMultiClassLoss
    from npairloss_amd.engine import Trainer
    trainer = Trainer(torch.nn.Linear(4, 4), NPairMultiClassLoss(NPairLossConfig()), SolverConfig(type="AdamW"), [], device=torch.device("cpu"))
    with pytest.raises(RuntimeError, match="AdamW"):
        trainer.snapshot_caffe(str(tmp_path / "x"))
    with pytest.raises(RuntimeError, match="AdamW"):
        trainer.restore_caffe(str(tmp_path / "x"))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_captured_steps_count_on(bits):
    """Replays of a captured step against the same number of eager ones."""
    sizes = [(5000,), (77,), (300, 20)]
    params, grads, states = make(sizes, torch.bfloat16, "cuda", bits, True)
    other = make(sizes, torch.bfloat16, "cuda", bits, True)
    call(*other)  # replays() runs once before it captures
    for _ in replays(lambda: call(params, grads, states)):
        call(*other)
        for a, b in zip(states, other[2]):
            for n in a:
                assert torch.equal(a[n].float(), b[n].float()), n
    solver = AdamW([torch.nn.Parameter(torch.ones(4, device="cuda"))])
    solver.param_groups[0]["params"][0].grad = torch.ones(4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(graph):
            solver.step()


@pytest.mark.gpu
def test_another_stream():
    params, grads, states = make([(70000,)], torch.float32, "cuda", 8, False)
    other = make([(70000,)], torch.float32, "cuda", 8, False)
    call(*other)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(params, grads, states)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(params[0], other[0][0])


def test_hash_is_even():
    """16 low and 16 high bits over elements, blocks and steps: mean and neighbours' product.
    Uniform on [0, 1): the mean of n is within 6 / sqrt(12 n) of 1/2, the products' within 6 / (12 sqrt(n)) of 1/4."""
    from npairloss_amd.ops.adamw import _bits
    for step in (1, 2, 1000):
        bits = _bits(0, step, 3, 400).double()
        for u in ((bits % 65536) / 65536, torch.floor(bits / 65536) / 65536):
            n = u.numel()
            assert abs(float(u.mean()) - 0.5) < 6 / math.sqrt(12 * n)
            c = u - 0.5
            for a, b in ((c[:, 1:], c[:, :-1]), (c[1:], c[:-1])):
                assert abs(float((a * b).mean())) < 6 / (12 * math.sqrt(n))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", ["param", "exp_avg", "exp_avg_sq", "step", "part"])
def test_what_shares_memory_is_refused(which, device):
    """Whole or in part, before anything is changed."""
    params, grads, states = make([(300,), (300,)], torch.float32, device, 32, False)
    if which == "param":
        params[1] = params[0]
    elif which == "part":
        both = torch.randn(500, device=device)
        params = [both[:300], both[200:]]
    else:
        states[1][which] = states[0][which]
    before = [p.clone() for p in params]
    with pytest.raises(RuntimeError, match="twice"):
        call(params, grads, states)
    assert all(torch.equal(a, b) for a, b in zip(params, before)) and int(states[0]["step"]) == 0
    both = torch.randn(600, device=device)
    call([both[:300], both[300:]], *make([(300,), (300,)], torch.float32, device, 32, False)[1:])

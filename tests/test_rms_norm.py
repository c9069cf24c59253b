"""rms_norm and rms_norm_fp8 against the formulas in 64 bits."""

import pytest
import torch

from npairloss_amd.ops import RMSNorm, rms_norm, rms_norm_fp8
from transformer_util import DEVICES, TYPES, U, assert_within, half_step, least, replays

SHAPES = [(1, 1), (3, 7), (5, 8), (4, 100), (2, 512), (3, 513), (300, 768), (2, 1024), (2, 1025), (2, 2056), (3, 4096), (2, 5000),
          (2, 8192), (1, 8193), (2, 16384), (1, 16383)]
EPS = 1e-6
FP8_MAX = 448.0


def inputs(n, d, dtype, device, residual, wide=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, d, generator=g).to(dtype).to(device)
    r = (3 * torch.randn(n, d, generator=g)).to(dtype).to(device) if residual else None
    w = (1 + 0.3 * torch.randn(d, generator=g)).to(torch.float32 if wide else dtype).to(device)
    dy = torch.randn(n, d, generator=g).to(dtype).to(device)
    ds = torch.randn(n, d, generator=g).to(dtype).to(device) if residual else None
    return x, w, r, dy, ds


def formula(s, w, dy=None, ds=None):
    s, w = s.double().cpu(), w.double().cpu()
    inv = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + EPS)
    y = s * inv * w
    if dy is None:
        return y
    dy = dy.double().cpu()
    g, n = dy * w, s * inv
    mean = (g * n).mean(-1, keepdim=True)
    dx = inv * (g - n * mean) + (0 if ds is None else ds.double().cpu())
    return y, dx, (dy * n).reshape(-1, n.shape[-1]).sum(0), (inv, g, n, dy)


# A sum of D products of one sign: each thread adds at most 8 * 4 of them in a
# row and ten levels of joining follow (torch's CPU sums are pairwise, fewer), so
# it is off by at most 45 U; its root, the quotients and the two products add 6.
SUM = 45
CHAIN = (SUM + 6) * U


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_formula(shape, dtype, residual, device):
    n, d = shape
    x, w, r, dy, ds = inputs(n, d, dtype, device, residual, wide=d % 2 == 1)
    leaves = [t.requires_grad_() for t in (x, w, r) if t is not None]
    got = rms_norm(x, w, r, eps=EPS)
    y, s = got if residual else (got, x)
    if residual:
        assert torch.equal(s, (x.float() + r.float()).to(dtype))
    grads = torch.autograd.grad([y, s] if residual else [y], leaves, [dy, ds] if residual else [dy])
    want, dx, dw, (inv, g, nrm, dyf) = formula(s.detach(), w.detach(), dy, ds)
    e = half_step(dtype)
    assert_within(y, want, want.abs() * (e + CHAIN) + least(dtype), "y")
    # the mean of g n is off by the sum's error of its magnitudes; 3 more roundings
    mags = inv * (g.abs() + nrm.abs() * (g * nrm).abs().mean(-1, keepdim=True) * 2) + (0 if ds is None else ds.double().cpu().abs())
    assert_within(grads[0], dx, dx.abs() * e + mags * 2 * CHAIN + least(dtype), "dx")
    if residual:
        assert torch.equal(grads[2], grads[0])
    total = (dyf * nrm).abs().sum(0)
    assert_within(grads[1], dw, dw.abs() * half_step(w.dtype) + total * (CHAIN + (min(n, 8) + 40) * U) + least(w.dtype), "dweight")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(13000, 24), (5000, 2500)])
def test_weight_gradient_of_many_rows(shape, dtype, device):
    """Summed over as many workgroups as there are: a wave adds up to 4 of 13000 rows or 10 of
    5000, 3 joins follow, then up to 1024 partial sums 32 at a time (32 and 31 additions): 76."""
    x, w, _, dy, _ = inputs(*shape, dtype, device, False)
    got = torch.autograd.grad(rms_norm(x, w.requires_grad_(), eps=EPS), w, dy)[0]
    _, _, dw, (_, _, nrm, dyf) = formula(x, w.detach(), dy)
    total = (dyf * nrm).abs().sum(0)
    assert_within(got, dw, dw.abs() * half_step(dtype) + total * (CHAIN + 76 * U) + least(dtype), "dweight")


@pytest.mark.parametrize("device", DEVICES)
def test_gradient_against_differences(device):
    """<gradient, u> against central differences of the formula in 64 bits."""
    x, w, r, dy, ds = inputs(6, 40, torch.float32, device, True, seed=3)
    for t in (x, w, r):
        t.requires_grad_()
    y, s = rms_norm(x, w, r, eps=EPS)
    grads = torch.autograd.grad([y, s], (x, w, r), [dy, ds])

    def loss(x, w, r):
        t = x + r
        return float((formula(t, w) * dy.double().cpu()).sum() + (t.cpu() * ds.double().cpu()).sum())

    g = torch.Generator().manual_seed(9)
    at = [t.detach().double().cpu() for t in (x, w, r)]
    for i in range(3):
        u = torch.randn(at[i].shape, generator=g).double()
        h = 1e-5
        up, down = [list(at) for _ in range(2)]
        up[i], down[i] = at[i] + h * u, at[i] - h * u
        fd = (loss(*up) - loss(*down)) / (2 * h)
        mine = float((grads[i].double().cpu() * u).sum())
        # fp32 gradients: CHAIN of their magnitudes (terms up to 4 times the result); differences: h^2 of third derivatives
        tol = 8 * CHAIN * float((grads[i].double().cpu().abs() * u.abs()).sum() + u.abs().sum()) + 1e-6
        assert abs(fd - mine) <= tol, (i, fd, mine)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,group", [((3, 7), 0), ((1, 4096), 0), ((5, 768), 0), ((4, 768), 16), ((3, 1024), 64), ((2, 4096), 128),
                                         ((2, 8192), 512), ((1, 16384), 256), ((2, 16383), 0), ((300, 256), 32)])
def test_fp8(shape, group, dtype, device):
    x, w, r, _, _ = inputs(*shape, dtype, device, True)
    for res in (None, r):
        got = rms_norm_fp8(x, w, res, eps=EPS, group=group)
        s = x if res is None else (x.float() + r.float()).to(dtype)
        if res is not None:
            assert torch.equal(got[2], s)
        codes, scales = got[0], got[1]
        n, d = shape
        assert codes.dtype == torch.float8_e4m3fn and codes.shape == x.shape and scales.shape == (n, d // group if group else 1)
        y = formula(s, w).view(n, -1, group or d)
        top = y.abs().amax(-1) / FP8_MAX
        assert_within(scales, top, top * (CHAIN + U), "scales")
        value = (codes.double().cpu().view(n, -1, group or d) * scales.double().cpu().unsqueeze(-1))
        # nearest code: 2^-4 of the value, or half the least step (2^-10) of the scale; fp32 arithmetic in front of it
        tol = y.abs() * (2.0 ** -4 + 2 * CHAIN) + scales.double().cpu().unsqueeze(-1) * 2.0 ** -10
        assert_within(value, y, tol, "values")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("group", [0, 64])
def test_fp8_rows_of_zeros_and_nan(device, group):
    x, w, _, _, _ = inputs(4, 256, torch.bfloat16, device, False)
    x[1] = 0
    x[2, 17] = float("nan")
    codes, scales = rms_norm_fp8(x, w, eps=EPS, group=group)
    assert (codes[1].float() == 0).all() and (scales[1] == 2.0 ** -126).all()
    assert codes[2].float().isnan().all() and scales[2].isnan().all()
    assert codes[[0, 3]].float().isfinite().all() and scales[[0, 3]].isfinite().all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_views_and_shapes(dtype, device):
    """Three dimensions, other orders, rows off the 16-byte border, no rows."""
    base = torch.randn(2, 96, 5, generator=torch.Generator().manual_seed(1)).to(dtype).to(device)
    w = torch.ones(96, dtype=dtype, device=device)
    x = base.transpose(1, 2)
    y = rms_norm(x, w)
    assert y.shape == x.shape
    assert torch.equal(y, rms_norm(x.contiguous(), w))
    flat = torch.randn(1 + 6 * 96, generator=torch.Generator().manual_seed(2)).to(dtype).to(device)
    off = flat[1:].view(6, 96)
    # the same arithmetic in another order of summation
    want = formula(off, w)
    assert_within(rms_norm(off, w), want, want.abs() * (half_step(dtype) + CHAIN) + least(dtype))
    codes, scales = rms_norm_fp8(off, w, group=32)
    other = rms_norm_fp8(off.clone(), w, group=32)
    assert torch.equal(codes.float(), other[0].float()) and torch.equal(scales, other[1])
    empty = torch.empty(0, 96, dtype=dtype, device=device, requires_grad=True)
    wl = w.clone().requires_grad_()
    out = rms_norm(empty, wl)
    assert out.shape == (0, 96)
    out.sum().backward()
    assert (wl.grad == 0).all() and rms_norm_fp8(empty.detach(), w)[0].shape == (0, 96)


@pytest.mark.parametrize("device", DEVICES)
def test_parts_of_the_gradient(device):
    x, w, r, dy, ds = inputs(5, 64, torch.float32, device, True)
    for t in (x, w, r):
        t.requires_grad_()
    _, s = rms_norm(x, w, r)
    gx, gr = torch.autograd.grad(s, (x, r), ds)
    assert torch.equal(gx, ds) and torch.equal(gr, ds)
    y, _ = rms_norm(x, w, r)
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    _, dx, _, (inv, g, n, _) = formula((x + r).detach(), w.detach(), dy, None)
    assert_within(gx, dx, inv * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True) * 2) * 2 * CHAIN)
    # a gradient that is one number broadcast
    y = rms_norm(x, w)
    y.sum().backward()
    assert x.grad.shape == x.shape


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x, w, r, _, _ = inputs(4, 64, torch.bfloat16, device, True)
    for args, kind in [((x, w[:63]), ValueError), ((x, w, r[:3]), ValueError), ((x, w, r.float()), ValueError), ((x.double(), w.double()), TypeError),
                       ((x, w.half()), TypeError), ((x[:, :0], w[:0]), ValueError), ((x.long(), w), TypeError),
                       ((torch.zeros(1, 16385, device=device), torch.ones(16385, device=device)), ValueError)]:
        with pytest.raises(kind):
            rms_norm(*args)
    for group in (-1, 8, 24, 1024, 128):
        with pytest.raises(ValueError):
            rms_norm_fp8(x, w, group=group)
    with pytest.raises(RuntimeError):
        rms_norm_fp8(x.clone().requires_grad_(), w)
    with torch.no_grad():
        rms_norm_fp8(x.clone().requires_grad_(), w)


def test_module():
    m = RMSNorm(32)
    x = torch.randn(3, 32, generator=torch.Generator().manual_seed(0))
    assert torch.equal(m(x), rms_norm(x, m.weight))
    y, s = m(x, x)
    assert torch.equal(s, x + x)


@pytest.mark.gpu
def test_another_stream_and_repeated():
    x, w, r, dy, ds = inputs(2000, 768, torch.bfloat16, "cuda", True)
    for t in (x, w, r):
        t.requires_grad_()

    def run():
        y, s = rms_norm(x, w, r)
        return (y, s) + torch.autograd.grad([y, s], (x, w, r), [dy, ds])

    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, again):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_captured():
    x, w, r, dy, ds = inputs(333, 768, torch.bfloat16, "cuda", True)
    with torch.no_grad():
        want = rms_norm(x, w, r) + rms_norm_fp8(x, w, r, group=128)

        def make():
            return rms_norm(x, w, r) + rms_norm_fp8(x, w, r, group=128)

        for out in replays(make):
            for a, b in zip(out, want):
                assert torch.equal(a.float(), b.float())
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, r)]

    def train():
        y, s = rms_norm(*leaves)
        return torch.autograd.grad([y, s], leaves, [dy, ds])

    want = [g.clone() for g in train()]
    for out in replays(train):
        for a, b in zip(out, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape", [(16,), (6, 16), (2, 3, 16)])
def test_outputs_changed_in_place(shape, device):
    """y is not kept for the backward pass and may be changed; the sum is, which then says so."""
    g = torch.Generator().manual_seed(0)
    x, r = (torch.randn(*shape, generator=g).to(device) for _ in range(2))
    w = torch.ones(16, device=device, requires_grad=True)
    want = rms_norm(x, w)
    (grad,) = torch.autograd.grad(want, w, x)
    y = rms_norm(x, w)
    y *= 2
    assert torch.equal(y.detach(), want.detach() * 2)
    y.backward(x / 2)
    assert torch.equal(w.grad, grad)
    y, s = rms_norm(x, w, r)
    s += 1
    assert torch.equal(s.detach(), x + r + 1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(x)


@pytest.mark.gpu
def test_more_rows_than_a_launch_takes_across():
    """2^24 blocks of four rows are 2^32 threads, which a launch does not take along one axis."""
    x = torch.full((2 ** 26 + 8, 8), 2.0, dtype=torch.bfloat16, device="cuda")
    w = torch.full((8,), 3.0, dtype=torch.bfloat16, device="cuda")
    y = rms_norm(x, w)
    assert (y == 3).all()
    del y
    codes, scales = rms_norm_fp8(x, w)
    assert (codes.view(torch.uint8) == 0x7E).all()  # 448: the largest of its row
    assert_within(scales[-1], torch.tensor([3 / FP8_MAX]), 3 / FP8_MAX * (CHAIN + U))

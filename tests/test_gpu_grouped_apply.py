"""grouped_linear with an activation and a residual on the GPU against its definition in 64 bits: widths and
sizes of both kernels, rows of no group, gradients, extremes of the activations, strides, refusals.

Tolerances, EPS = 2^-24.  z errs by (k + 2) EPS of its terms' magnitudes (32-bit sums), which the
activations' slopes (at most 1.13) pass on; a value of its own errs by 8 EPS and, where the argument of an
exponential or of erfc is rounded, by z^2 (gelu) or |z| (silu) EPS of itself, twice that with the function's
own; the sum with the residual by EPS.  dz likewise with slopes' slopes (at most 0.8), and is rounded to the
type; its error goes through the other products as their operand does.  bfloat16: 2^-8 of a result."""
import math

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from dynamis_amd import dynamis_state as ds
from oracle import operators as oracle

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
ACTS = pytest.mark.parametrize("act", ["silu", "gelu"])


def _f(act, z):
    """(f, f', the relative error's growth with z)."""
    if act is None:
        return z, np.ones_like(z), np.zeros_like(z)
    if act == "silu":
        s = np.exp(-np.logaddexp(0, -z))
        t = np.exp(-np.logaddexp(0, z))  # 1 - s
        return z * s, s * (1 + z * t), 2 * np.abs(z)
    share = 0.5 * np.vectorize(math.erfc)(-z / math.sqrt(2))
    return z * share, share + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi), 2 * z * z


def _near(name, got, want, tol, dtype):
    got = got.detach().double().cpu().numpy()
    tol = tol + (2.0 ** -8 * np.abs(want) if dtype == torch.bfloat16 else 0)
    bad = ~(np.abs(got - want) <= tol + 1e-37)
    assert got.shape == want.shape and not bad.any(), \
        f"{name}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - want)[bad]):.3g} at {np.argwhere(bad)[0]}"


def _make(sizes, k, n, dtype, bias, residual, seed, rows=None):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    rows = sum(sizes) if rows is None else rows
    return (rand(rows, k).to(dtype), (2 * rand(len(sizes), n, k) / math.sqrt(k)).to(dtype),
            rand(len(sizes), n).to(dtype) if bias else None, rand(rows, n).to(dtype) if residual else None, rand(rows, n).to(dtype))


def _check(sizes, k, n, dtype, act, bias=True, residual=True, seed=0):
    print(f"\n[case] apply {sizes[:12]} k={k} n={n} {dtype} {act} bias={bias} residual={residual}", flush=True)
    x, w, b, res, grad = _make(sizes, k, n, dtype, bias, residual, seed)
    xd, wd, bd, rd = (None if t is None else t.cuda().requires_grad_(True) for t in (x, w, b, res))
    leaves = [t for t in (xd, wd, bd, rd) if t is not None]
    s = torch.tensor(sizes).cuda()

    def step():
        y = ds.grouped_linear(xd, wd, s, bd, activation=act, residual=rd)
        return [y, *torch.autograd.grad(y, leaves, grad.cuda())]

    got = step()
    x64, w64, b64, r64, g64 = (None if t is None else t.double().numpy() for t in (x, w, b, res, grad))
    r, m = oracle.grouped_linear(x64, w64, sizes, b64)
    z, z_err = r["y"], (k + 3) * EPS * m["y"]
    f, slope, growth = _f(act, z)
    y = f + (0 if res is None else r64)
    own = (8 + growth) * EPS
    tol = 1.13 * z_err + own * np.abs(f) + EPS * np.abs(y)
    _near("y", got[0], y, tol, dtype)
    dz = g64 * slope
    d_err = np.abs(g64) * (0.8 * z_err + own * (np.abs(slope) + 1)) + (2.0 ** -8 * np.abs(dz) if dtype == torch.bfloat16 and act else 0)
    if act is None:
        d_err = np.zeros_like(dz)
    r, m = oracle.grouped_linear(x64, w64, sizes, b64, dz)
    _, e = oracle.grouped_linear(x64, w64, sizes, None, d_err)
    longest = max(list(sizes) + [1])
    for name, t, terms in zip(("dx", "dweight", "dbias"), got[1:], (n, longest, longest)):
        if name == "dbias" and not bias:
            break
        _near(name, t, r[name], (terms + 2) * EPS * (m[name] + e[name]) + e[name], dtype)
    if residual:
        assert torch.equal(got[-1].cpu(), grad)
    assert all(torch.equal(p, q) for p, q in zip(got, step()))
    with torch.no_grad():
        assert torch.equal(ds.grouped_linear(xd, wd, sizes, bd, act, rd), got[0])


@TYPES
@ACTS
@pytest.mark.parametrize("k,n", [(1, 1), (3, 5), (8, 8), (32, 64), (33, 65), (64, 128), (100, 164), (127, 129), (128, 128),
                                 (200, 40), (256, 512), (520, 136), (64, 24), (512, 264)])
def test_widths(cuda, k, n, act, dtype):
    _check([5, 0, 130, 1, 64], k, n, dtype, act, seed=k)


@TYPES
@ACTS
@pytest.mark.parametrize("bias,residual", [(True, False), (False, True), (False, False)])
def test_with_and_without(cuda, bias, residual, act, dtype):
    for k, n in ((64, 96), (50, 70)):
        _check([33, 100, 0, 300], k, n, dtype, act, bias, residual, seed=n)


@TYPES
@pytest.mark.parametrize("k,n", [(64, 128), (33, 65)])
def test_a_residual_alone(cuda, k, n, dtype):
    _check([33, 100, 0, 300], k, n, dtype, None, seed=n)


@TYPES
@pytest.mark.parametrize("sizes", [[1], [0, 0, 3], [255, 256, 257, 0], [1000, 0, 2, 1], [3] * 300, [20000], [9000] * 4],
                         ids=lambda s: f"{len(s)}_{sum(s)}")
def test_sizes(cuda, sizes, dtype):
    """Panels of 32, 64 and 128 columns of the streaming kernel, and the other one."""
    _check(sizes, 72, 96, dtype, "silu", seed=len(sizes))
    _check(sizes, 24, 200, dtype, "gelu", seed=len(sizes))
    _check(sizes, 20, 50, dtype, "silu", seed=len(sizes))


@TYPES
@ACTS
def test_rows_of_no_group(cuda, act, dtype):
    """They give their residual (zeros without one), and no gradient but the residual's."""
    for k, n in ((48, 56), (45, 55)):
        print(f"\n[case] rest {dtype} {act} {k} {n}", flush=True)
        x, w, b, res, grad = (t.cuda().requires_grad_(True) for t in _make([30, 40], k, n, dtype, True, True, 4, rows=400))
        sizes = torch.tensor([30, 40]).cuda()
        y = ds.grouped_linear(x, w, sizes, b, act, res)
        assert torch.equal(y[70:], res[70:])
        assert not ds.grouped_linear(x, w, sizes, b, act)[70:].any()
        got = torch.autograd.grad(y, [x, w, b, res], grad)
        short = [x[:70].detach().requires_grad_(True), w, b]
        y2 = ds.grouped_linear(*short[:2], sizes, b, act, res[:70])
        assert torch.equal(y2, y[:70])
        want = torch.autograd.grad(y2, short, grad[:70])
        assert torch.equal(got[0][:70], want[0]) and not got[0][70:].any() and torch.equal(got[1], want[1])
        assert torch.equal(got[2], want[2]) and torch.equal(got[3], grad)


@TYPES
@ACTS
def test_extremes(cuda, act, dtype):
    """Far below zero the digits are there; far above f is z; nothing becomes a NaN before an infinity does."""
    print(f"\n[case] extremes {dtype} {act}", flush=True)
    z = torch.tensor([0.0, -0.0, 1e-20, -1e-20, 0.5, -1.0, 3.0, -4.0, 8.0, -8.0, 12.0, -12.0, 88.0, -88.0, 200.0, -200.0, 1e4, -1e4,
                      3e38, -3e38]).to(dtype)
    z = torch.cat([z, z[-4:]])  # (24 columns: the streaming kernel's chunks)
    for n in (24, 23):
        w = torch.zeros(1, n, 8, dtype=dtype)
        x = torch.zeros(3, 8, dtype=dtype)
        b = z[None, :n].clone()
        leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
        y = ds.grouped_linear(*leaves[:2], [3], leaves[2], act)
        v = b[0].double().numpy()
        f, slope, growth = _f(act, v)
        with np.errstate(all="ignore"):
            tol = (8 + growth) * EPS * np.abs(f)
        # (below 2^-126 32 bits lose digits: those count as nothing)
        far = np.abs(f) < 2.0 ** -120
        got = y[0].detach().double().cpu().numpy()
        assert (np.abs(got[far]) < 2.0 ** -119).all()
        _near("y", y[0][~torch.from_numpy(far)], f[~far], tol[~far], dtype)
        # the slope, through the bias's gradient: one row's dy of 1, rounded to the type
        g = torch.zeros(3, n, dtype=dtype, device="cuda")
        g[1] = 1
        db, = torch.autograd.grad(y, leaves[2], g)
        with np.errstate(all="ignore"):
            tol = (8 + np.minimum(growth, 1e6)) * EPS * (np.abs(slope) + np.abs(v) * np.exp(-np.minimum(np.abs(v), 80)))
        _near("slope", db[0], slope, tol + 2.0 ** -120, dtype)


@TYPES
def test_what_is_not_finite_stays_in_its_row(cuda, dtype):
    for k, n in ((40, 104), (41, 101)):
        print(f"\n[case] nan {dtype} {k} {n}", flush=True)
        x, w, b, res, _ = (t.cuda() for t in _make([50, 60], k, n, dtype, True, True, 5))
        want = ds.grouped_linear(x, w, [50, 60], b, "gelu", res)
        x2, res2 = x.clone(), res.clone()
        x2[55, 3], res2[7, 9] = float("nan"), -float("inf")
        got = ds.grouped_linear(x2, w, [50, 60], b, "gelu", res2)
        keep = (torch.arange(110) != 55) & (torch.arange(110) != 7)
        assert got[55].isnan().all() and torch.equal(got[keep], want[keep]) and got[7, 9] == -float("inf")
        got[7, 9] = want[7, 9]
        assert torch.equal(got[7], want[7])


@TYPES
def test_strides_alignment_streams(cuda, dtype):
    print(f"\n[case] strides {dtype}", flush=True)
    sizes = [33, 100, 7]
    x, w, b, res, grad = (t.cuda() for t in _make(sizes, 64, 72, dtype, True, True, 6))
    want = ds.grouped_linear(x, w, sizes, b, "silu", res)
    odd = torch.empty(res.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(res).copy_(res)
    assert torch.equal(ds.grouped_linear(x, w, sizes, b, "silu", odd), want)
    assert torch.equal(ds.grouped_linear(x, w, sizes, b, "silu", res.t().contiguous().t()), want)
    assert torch.equal(ds.grouped_linear(x, w, sizes, b, "silu", torch.cat([res, res], 1)[:, :72]), want)
    one = res[:1].expand(140, 72)
    assert torch.equal(ds.grouped_linear(x, w, sizes, b, "silu", one), ds.grouped_linear(x, w, sizes, b, "silu", one.contiguous()))
    p = one.clone()[:1].requires_grad_(True)
    y = ds.grouped_linear(x, w, sizes, b, "silu", p.expand(140, 72))
    assert torch.equal(torch.autograd.grad(y, p, grad)[0], grad.sum(0, keepdim=True))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ds.grouped_linear(x, w, sizes, b, "silu", res)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # the residual may be the rows themselves
    w2 = w[:, :64].contiguous()
    xs = x.clone().requires_grad_(True)
    y = ds.grouped_linear(xs, w2, sizes, None, "silu", xs)
    a = torch.autograd.grad(y, xs, grad[:, :64].contiguous())[0]
    other = x.clone().requires_grad_(True)
    c, d = torch.autograd.grad(ds.grouped_linear(xs, w2, sizes, None, "silu", other), [xs, other], grad[:, :64].contiguous())
    assert torch.equal(a, c + d)


@ACTS
def test_gradients_against_differences(cuda, act):
    sizes = [20, 0, 45]
    x, w, b, res, grad = _make(sizes, 24, 40, torch.float32, True, True, 7)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b, res)]
    y = ds.grouped_linear(leaves[0], leaves[1], sizes, leaves[2], act, leaves[3])
    grads = torch.autograd.grad(y, leaves, grad.cuda())
    p = [t.double().numpy() for t in (x, w, b, res)]
    rng = np.random.default_rng(8)

    def loss(q):
        return ((_f(act, oracle.grouped_linear(q[0], q[1], sizes, q[2])[0]["y"])[0] + q[3]) * grad.double().numpy()).sum()

    for i, g in enumerate(grads):
        d, h = rng.standard_normal(p[i].shape), 1e-5
        up, down = ([*p[:i], p[i] + e * h * d, *p[i + 1:]] for e in (1, -1))
        diff = (loss(up) - loss(down)) / (2 * h)
        g = g.double().cpu().numpy()
        assert abs(diff - (g * d).sum()) < 1e-5 * (1 + np.abs(g * d).sum()), i


def test_only_what_is_asked(cuda):
    sizes = [20, 45]
    leaves = [t.cuda() for t in _make(sizes, 24, 40, torch.float32, True, True, 9)]
    grad = leaves.pop()
    all_of = [t.clone().requires_grad_(True) for t in leaves]
    want = torch.autograd.grad(ds.grouped_linear(*all_of[:2], sizes, all_of[2], "silu", all_of[3]), all_of, grad)
    for i in range(4):
        args = [t.clone().requires_grad_(i == j) for j, t in enumerate(leaves)]
        got, = torch.autograd.grad(ds.grouped_linear(*args[:2], sizes, args[2], "silu", args[3]), args[i], grad)
        assert torch.equal(got, want[i])


def test_no_rows(cuda):
    x, w = torch.empty(0, 24, device="cuda", requires_grad=True), torch.ones(3, 16, 24, device="cuda", requires_grad=True)
    res = torch.empty(0, 16, device="cuda", requires_grad=True)
    y = ds.grouped_linear(x, w, torch.zeros(3, dtype=torch.long, device="cuda"), None, "gelu", res)
    dx, dw, dr = torch.autograd.grad(y, (x, w, res), torch.empty(0, 16, device="cuda"))
    assert y.shape == dr.shape == (0, 16) and dx.shape == x.shape and not dw.any()


def test_refusals(cuda):
    x, w = torch.zeros(10, 8, device="cuda"), torch.zeros(2, 4, 8, device="cuda")
    bad = lambda match, *a, **kw: pytest.raises(RuntimeError, ds.grouped_linear, *a, **kw).match(match)  # noqa: E731
    bad("activation", x, w, [5, 5], None, "relu")
    bad("activation", x, w, [5, 5], None, 1)
    res = torch.zeros(10, 4, device="cuda")
    bad("residual", x, w, [5, 5], residual=res[:9])
    bad("residual", x, w, [5, 5], residual=res.bfloat16())
    bad("residual", x, w, [5, 5], residual=res.cpu())
    bad("residual", x, w, [5, 5], residual=1.0)
    with forward_ad.dual_level():
        bad("forward-mode", x, w, [5, 5], residual=forward_ad.make_dual(res, res))

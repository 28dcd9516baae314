"""grouped_linear on the GPU against its definition in 64 bits (oracle/operators.py), forward
and backward: sizes around the kernels' tiles, slabs and items, empty groups, odd widths, rows
of no group, NaN beside a group, and bit-equal repeats.

Tolerances.  A sum of n products in 32 bits errs by at most (n + 2) eps times the sum of the
products' magnitudes; bfloat16 results are rounded once (2^-8 of themselves)."""
import numpy as np
import pytest
import torch

from dynamis_amd import dynamis_state as ds
from oracle import operators as oracle

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


def _near(name, got, want, mag, n, dtype):
    got = got.detach().double().cpu().numpy()
    tol = (n + 2) * EPS * mag + (2.0 ** -8 * np.abs(want) if dtype == torch.bfloat16 else 0)
    bad = ~(np.abs(got - want) <= tol + 1e-30)
    assert not bad.any(), f"{name}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - want)[bad]):.3g}"


def _make(sizes, k, n, dtype, bias, seed, rows=None):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    rows = sum(sizes) if rows is None else rows
    return rand(rows, k), rand(len(sizes), n, k), rand(len(sizes), n) if bias else None, rand(rows, n)


def _check(sizes, k, n, dtype, bias=True, seed=0):
    print(f"\n[case] grouped {sizes[:12]} k={k} n={n} {dtype} bias={bias}", flush=True)
    x, w, b, grad = _make(sizes, k, n, dtype, bias, seed)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b) if t is not None]
    s = torch.tensor(sizes)

    def step():
        y = ds.grouped_linear(leaves[0], leaves[1], s.cuda(), leaves[2] if bias else None)
        return [y, *torch.autograd.grad(y, leaves, grad.cuda())]

    got = step()
    np64 = [None if t is None else t.double().numpy() for t in (x, w, b, grad)]
    r, m = oracle.grouped_linear(np64[0], np64[1], sizes, np64[2], np64[3])
    longest = max(list(sizes) + [1])
    for name, t, terms in zip(("y", "dx", "dweight", "dbias"), got, (k + 1, n, longest, longest)):
        _near(name, t, r[name], m[name], terms, dtype)
    assert all(torch.equal(p, q) for p, q in zip(got, step()))
    with torch.no_grad():
        assert torch.equal(ds.grouped_linear(leaves[0], leaves[1], sizes, leaves[2] if bias else None), got[0])


@TYPES
@pytest.mark.parametrize("k,n", [(1, 1), (3, 5), (8, 8), (32, 64), (33, 65), (64, 128), (100, 164), (127, 129), (128, 128),
                                 (200, 40), (256, 512), (520, 136)])
def test_widths(cuda, k, n, dtype):
    _check([5, 0, 130, 1, 64], k, n, dtype, seed=k)


@TYPES
@pytest.mark.parametrize("sizes", [[1], [0, 0, 3], [127, 128, 129], [255, 256, 257, 0], [1000, 0, 2, 1], [3] * 300,
                                   [0] * 700 + [5, 9], [63, 64, 65, 31, 32, 33]], ids=lambda s: f"{len(s)}_{sum(s)}")
def test_sizes(cuda, sizes, dtype):
    _check(sizes, 72, 96, dtype, seed=len(sizes))
    _check(sizes, 24, 200, dtype, bias=False, seed=len(sizes))


@TYPES
def test_items_of_long_groups(cuda, dtype):
    """Groups whose weight gradient is summed in several items, beside ones that take a single one."""
    _check([4000, 0, 17, 6001, 256, 257], 40, 136, dtype, seed=3)


@TYPES
def test_rows_of_no_group_and_sizes_that_reach_past(cuda, dtype):
    print(f"\n[case] rest {dtype}", flush=True)
    x, w, b, grad = _make([30, 40], 48, 56, dtype, True, 4, rows=400)
    r, m = oracle.grouped_linear(x[:70].double().numpy(), w.double().numpy(), [30, 40], b.double().numpy(),
                                 grad[:70].double().numpy())
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y = ds.grouped_linear(leaves[0], leaves[1], torch.tensor([30, 40]).cuda(), leaves[2])
    dx, dw, db = torch.autograd.grad(y, leaves, grad.cuda())
    assert not y[70:].any() and not dx[70:].any()
    for name, t, terms in (("y", y[:70], 49), ("dx", dx[:70], 56), ("dweight", dw, 40), ("dbias", db, 40)):
        _near(name, t, r[name], m[name], terms, dtype)
    # the second group reaches past the rows: it ends with them; a negative size is an empty group
    for sizes, same in (([30, 10 ** 12], [30, 370]), ([-5, 400], [0, 400])):
        got = ds.grouped_linear(leaves[0], leaves[1], torch.tensor(sizes).cuda(), leaves[2])
        assert torch.equal(got, ds.grouped_linear(leaves[0], leaves[1], torch.tensor(same).cuda(), leaves[2]))
        for p, q in zip(*(torch.autograd.grad(ds.grouped_linear(leaves[0], leaves[1], torch.tensor(z).cuda(), leaves[2]),
                                              leaves, grad.cuda()) for z in (sizes, same))):
            assert torch.equal(p, q)


@TYPES
def test_a_nan_stays_in_its_group(cuda, dtype):
    print(f"\n[case] nan {dtype}", flush=True)
    sizes = [50, 60, 70]
    x, w, b, grad = (t.cuda() for t in _make(sizes, 40, 100, dtype, True, 5))
    want = ds.grouped_linear(x, w, sizes, b)
    y = x.clone()
    y[55, 3] = float("nan")
    got = ds.grouped_linear(y, w, sizes, b)
    keep = torch.arange(180) != 55
    assert torch.isnan(got[55]).all() and torch.equal(got[keep], want[keep])
    v = w.clone()
    v[1] = float("inf")
    got = ds.grouped_linear(x, v, sizes, b)
    assert torch.equal(got[:50], want[:50]) and torch.equal(got[110:], want[110:])
    leaves = [y.requires_grad_(True), w.requires_grad_(True)]
    dw = torch.autograd.grad(ds.grouped_linear(*leaves, sizes), leaves, grad)[1]
    assert torch.isfinite(dw[0]).all() and torch.isfinite(dw[2]).all() and torch.isnan(dw[1][:, 3]).all()
    assert torch.isfinite(dw[1][:, torch.arange(40) != 3]).all()


@TYPES
def test_strides_alignment_streams(cuda, dtype):
    print(f"\n[case] strides {dtype}", flush=True)
    sizes = [33, 100, 7]
    x, w, b, _ = (t.cuda() for t in _make(sizes, 64, 72, dtype, True, 6))
    want = ds.grouped_linear(x, w, sizes, b)
    odd = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(x).copy_(x)
    assert torch.equal(ds.grouped_linear(odd, w, sizes, b), want)
    assert torch.equal(ds.grouped_linear(x.t().contiguous().t(), w.transpose(1, 2).contiguous().transpose(1, 2), sizes, b), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ds.grouped_linear(x, w, sizes, b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_gradients_against_differences(cuda):
    sizes = [20, 0, 45]
    x, w, b, grad = _make(sizes, 24, 40, torch.float32, True, 7)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(ds.grouped_linear(leaves[0], leaves[1], sizes, leaves[2]), leaves, grad.cuda())
    p = [t.double().numpy() for t in (x, w, b)]
    rng = np.random.default_rng(8)
    loss = lambda q: (oracle.grouped_linear(q[0], q[1], sizes, q[2])[0]["y"] * grad.double().numpy()).sum()  # noqa: E731
    for i, g in enumerate(grads):
        d, h = rng.standard_normal(p[i].shape), 1e-4  # (the loss is linear in each: no h^2)
        up, down = ([*p[:i], p[i] + e * h * d, *p[i + 1:]] for e in (1, -1))
        diff = (loss(up) - loss(down)) / (2 * h)
        g = g.double().cpu().numpy()
        assert abs(diff - (g * d).sum()) < 1e-6 * (1 + np.abs(g * d).sum()), i


def test_only_what_is_asked(cuda):
    sizes = [20, 45]
    x, w, b, grad = (t.cuda() for t in _make(sizes, 24, 40, torch.float32, True, 9))
    want = torch.autograd.grad(ds.grouped_linear(*(ls := [t.clone().requires_grad_(True) for t in (x, w)]), sizes,
                                                 lb := b.clone().requires_grad_(True)), [*ls, lb], grad)
    for i in range(3):
        args = [t.clone().requires_grad_(i == j) for j, t in enumerate((x, w, b))]
        got, = torch.autograd.grad(ds.grouped_linear(args[0], args[1], sizes, args[2]), args[i], grad)
        assert torch.equal(got, want[i])


def test_no_rows(cuda):
    print("\n[case] no rows", flush=True)
    x, w, b = torch.empty(0, 24, device="cuda", requires_grad=True), torch.ones(3, 16, 24, device="cuda", requires_grad=True), \
        torch.ones(3, 16, device="cuda", requires_grad=True)
    y = ds.grouped_linear(x, w, torch.zeros(3, dtype=torch.long, device="cuda"), b)
    assert y.shape == (0, 16)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(0, 16, device="cuda"))
    assert dx.shape == x.shape and not dw.any() and not db.any()


def test_refusals(cuda):
    x, w = torch.zeros(10, 8, device="cuda"), torch.zeros(2, 4, 8, device="cuda")
    bad = lambda match, *a: pytest.raises(RuntimeError, ds.grouped_linear, *a).match(match)  # noqa: E731
    bad("CUDA tensor", x.cpu(), w, [5, 5])
    bad("shape", x[0], w, [5, 5])
    bad("float32 or bfloat16", x.double(), w.double(), [5, 5])
    bad("weight must have shape", x, w[:, :, :4], [5, 5])
    bad("weight must be", x, w.bfloat16(), [5, 5])
    bad("weight must be on", x, w.cpu(), [5, 5])
    bad("sizes", x, w, [5, 5, 0])
    bad("sizes", x, w, torch.tensor([5, 5], dtype=torch.int32, device="cuda"))
    bad("add up", x, w, [5, 4])
    bad("add up", x, w, [11, -1])
    bad("bias", x, w, [5, 5], torch.zeros(2, 5, device="cuda"))
    bad("bias", x, w, [5, 5], torch.zeros(2, 4, device="cuda").bfloat16())

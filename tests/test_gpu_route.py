"""route_rows, dispatch_rows and combine_rows on the GPU against their definitions in 64 bits
(oracle/layers.py), forward and backward: numbers of experts and choices around the kernels' lanes, groups,
ties, masked experts, rows of padding, what is not finite, strides, streams, graphs, refusals.

What is chosen, the sizes and the places are equal.  Tolerances of the rest, in units of EPS = 2^-24 of a
result or of the sum of its terms' magnitudes: a weight's exponentials err by the difference of their
logits (up to D in a row) and 4, a sum by its n terms, quotients and products by 8 in all: 2 D + n + 12,
as much again and k for a gradient.  A row's sum errs by its k terms and 2, a product of rows by the width
and 2.  bfloat16 results are rounded once, 2^-8 of themselves."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from dynamis_amd import dynamis_state as ds
from oracle import layers as oracle

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
INF = float("inf")


def _near(name, got, want, mag, n, rounded):
    got = got.detach().double().cpu().numpy()
    tol = n * EPS * mag + (2.0 ** -8 * np.abs(want) if rounded else 0)
    bad = ~((np.abs(got - want) <= tol + 1e-37) | (np.isnan(got) & np.isnan(want)))
    assert got.shape == want.shape and not bad.any(), \
        f"{name}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - want)[bad]):.3g} at {np.argwhere(bad)[0]}"


def _logits(rows, n, dtype, seed, spread=2.0, masked=0.1, padding=True):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(rows, n, generator=g)
    x[torch.rand(rows, n, generator=g) < masked] = -INF
    if padding and rows > 2:
        x[rows // 3] = -INF
        x[-1, 1:] = -INF
    return x.to(dtype), torch.randn(rows, n, generator=g)


def _check_route(x, k, seed=0, **how):
    rows, n = x.shape
    print(f"\n[case] route {rows}x{n} k={k} {x.dtype} {({a: b for a, b in how.items() if a != 'bias'})} "
          f"bias={how.get('bias') is not None}", flush=True)
    grad = torch.randn(rows, k, generator=torch.Generator().manual_seed(seed + 1))
    want = oracle.route_rows(x.double().numpy(), k, grad=grad.numpy(),
                             **{a: b.double().numpy() if a == "bias" and b is not None else b for a, b in how.items()})
    xd = x.cuda().requires_grad_(True)
    how_d = {a: b.cuda() if a == "bias" and b is not None else b for a, b in how.items()}

    def step():
        r = ds.route_rows(xd, k, **how_d)
        return [r.weights, r.experts, r.sizes, r.places, torch.autograd.grad(r.weights, xd, grad.cuda())[0]], r

    got, r = step()
    assert (r.rows, r.k, r.num_experts) == (rows, k, n)
    for name, t in zip(("experts", "sizes", "places"), got[1:4]):
        t = t.cpu().numpy()
        assert np.array_equal(t, want[name]), (name, np.argwhere(t != want[name])[:4])
    finite = np.where(np.isfinite(x.double().numpy()), x.double().numpy(), np.nan)
    spread = 0.0 if np.isnan(finite).all() else np.nanmax(finite) - np.nanmin(finite)
    value = 2 * spread + n + 12
    _near("weights", got[0], want["weights"], np.abs(want["weights"]), value, False)
    _near("dlogits", got[4], want["dlogits"], want["mag"], 2 * value + k, x.dtype == torch.bfloat16)
    again, _ = step()
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    with torch.no_grad():
        r = ds.route_rows(xd, k, **how_d)
        assert torch.equal(r.weights, got[0]) and torch.equal(r.places, got[3])
    return r


@TYPES
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("n,k", [(1, 1), (2, 2), (3, 1), (4, 4), (8, 2), (15, 3), (16, 16), (33, 5), (60, 6), (64, 8), (100, 7),
                                 (128, 8), (200, 33), (256, 8), (257, 64), (512, 10), (1000, 2), (1024, 64)])
def test_experts_and_choices(cuda, n, k, renormalize, scoring, dtype):
    x, _ = _logits(37, n, dtype, n, masked=0.1 if n > 4 else 0.3)
    _check_route(x, k, scoring=scoring, renormalize=renormalize, scale=2.5 if renormalize else 1.0)


@TYPES
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("n,k", [(5, 2), (64, 6), (100, 9), (256, 8), (1024, 4)])
def test_bias(cuda, n, k, scoring, dtype):
    """The bias moves the choice alone; an expert whose bias is -inf takes no row."""
    x, noise = _logits(65, n, dtype, n)
    bias = 0.2 * noise[0]
    bias[n // 2] = -INF
    r = _check_route(x, k, scoring=scoring, bias=bias, renormalize=True)
    assert r.sizes[n // 2] == 0
    # none at all moves nothing: the order of the scores is that of the logits
    plain = ds.route_rows(x.cuda(), k, scoring=scoring)
    zero = ds.route_rows(x.cuda(), k, scoring=scoring, bias=torch.zeros(n, device="cuda", dtype=torch.float64))
    assert torch.equal(plain.experts, zero.experts) and torch.equal(plain.weights, zero.weights)


@TYPES
@pytest.mark.parametrize("group_best", [1, 2])
@pytest.mark.parametrize("biased", [True, False])
@pytest.mark.parametrize("n,groups,top,k", [(8, 8, 3, 2), (12, 3, 1, 4), (60, 5, 2, 7), (64, 8, 4, 6), (64, 64, 10, 8),
                                            (256, 8, 4, 8), (1024, 64, 1, 20), (1024, 4, 4, 3), (130, 2, 1, 3)])
def test_groups(cuda, n, groups, top, k, biased, group_best, dtype):
    x, noise = _logits(50, n, dtype, n + top, masked=0.3)
    for scoring in ("softmax", "sigmoid"):
        _check_route(x, k, scoring=scoring, bias=0.2 * noise[0] if biased else None, groups=groups, top_groups=top,
                     group_best=group_best)


def test_a_group_may_hold_less_than_k(cuda):
    """The chosen groups' experts run out: the other choices are of none."""
    x, _ = _logits(20, 12, torch.float32, 1, masked=0.0, padding=False)
    r = _check_route(x, 5, groups=6, top_groups=1)
    assert (r.experts[:, 2:] == -1).all() and (r.weights[:, 2:] == 0).all() and (r.experts[:, :2] >= 0).all()


@TYPES
def test_ties_go_to_the_lowest(cuda, dtype):
    for n, k in ((8, 3), (64, 9), (300, 20)):
        x = torch.randint(-2, 3, (70, n), generator=torch.Generator().manual_seed(n)).to(dtype)
        x[3] = 0.0
        x[4, ::2] = -0.0
        x[4, 1::2] = 0.0
        for how in (dict(), dict(scoring="sigmoid", bias=torch.zeros(n)), dict(groups=min(n // 4, 60), top_groups=2, group_best=2),
                    dict(bias=torch.full((n,), 0.5), groups=4, top_groups=3)):
            r = _check_route(x, k, **how)
        assert r.experts[3, :3].tolist() == r.experts[4, :3].tolist() == [0, 1, 2]


def test_neighbours_that_32_bits_would_merge(cuda):
    """Scores plus a bias that differ in their last bits of 32 and beyond are chosen as 64 have them."""
    n, k = 32, 6
    g = torch.Generator().manual_seed(5)
    x = torch.randn(200, n, generator=g)
    bias = torch.zeros(n)
    # pairs whose sigmoid plus bias lie 2^-30 to 2^-40 apart: the second logit makes up for the bias to 32 bits
    bias[1::2] = 0.25
    s = torch.sigmoid(x[:, ::2].double()) * 0.5 + 0.3
    x[:, ::2] = torch.log(s / (1 - s)).float()
    t = torch.sigmoid(x[:, ::2].double()) - 0.25
    x[:, 1::2] = torch.log(t / (1 - t)).float()
    v = torch.sigmoid(x.double()) + bias.double()
    gap = (v[:, ::2] - v[:, 1::2]).abs()
    assert gap.max() < 2e-7 and (gap > 0).any() and ((v[:, ::2] > v[:, 1::2]).any() and (v[:, ::2] < v[:, 1::2]).any())
    _check_route(x, k, scoring="sigmoid", bias=bias)
    _check_route(x, k, scoring="sigmoid", bias=bias, groups=4, top_groups=2, group_best=2)


@TYPES
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_what_is_not_finite_and_extremes(cuda, renormalize, scoring, dtype):
    print(f"\n[case] extremes {scoring} {renormalize} {dtype}", flush=True)
    low = torch.finfo(dtype).min
    x, _ = _logits(12, 20, dtype, 7, masked=0.0, padding=False)
    x[1, 3] = float("nan")
    x[2, 4] = INF
    x[3] = low                     # the type's lowest value is a value
    x[4, :18] = low
    x[5] = -200.0                  # every sigmoid vanishes in 32 bits
    x[5, 7] = -199.0
    x[6] = 200.0
    x[7] = -INF
    x[8, 1:] = -INF
    x[9, 2:] = -INF
    grad = torch.randn(12, 4, generator=torch.Generator().manual_seed(8))
    want = oracle.route_rows(x.double().numpy(), 4, scoring, renormalize=renormalize, grad=grad.numpy())
    xd = x.cuda().requires_grad_(True)
    r = ds.route_rows(xd, 4, scoring=scoring, renormalize=renormalize)
    assert np.array_equal(r.experts.cpu().numpy(), want["experts"])
    assert np.array_equal(r.places.cpu().numpy(), want["places"])
    rows = [0, 3, 4, 5, 6, 7, 8, 9, 10, 11]
    value = 2 * 8 + 20 + 12 + 2 * 220  # (D of the rows at 200 and -200: what is at `low` is 0)
    # (numbers below 1e-37, where 32 bits lose digits, count as nothing)
    w = r.weights.detach().double().cpu().numpy()
    assert np.allclose(w[rows], want["weights"][rows], rtol=value * EPS, atol=1e-37)
    dx, = torch.autograd.grad(r.weights, xd, grad.cuda())
    _near("dlogits", dx[rows], want["dlogits"][rows], want["mag"][rows], 2 * value + 4, dtype == torch.bfloat16)
    if scoring == "softmax":  # a NaN or an infinity is in every weight of its row
        assert r.weights[1].isnan().all() and r.weights[2].isnan().all()
    else:
        assert r.weights[1].isnan().any() and r.experts[1, 0] == 3 and r.experts[2, 0] == 4
        if not renormalize:
            assert r.weights[1].isnan().sum() == 1 and r.weights[2, 0] == 1
    assert torch.isfinite(r.weights[rows]).all() and not dx[7].any()


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 255, 257, 1000, 16384, 16385, 40001])
def test_rows_and_places(cuda, rows):
    """Around the workgroups' rows: sizes and places of the stable order; choices of none come last."""
    print(f"\n[case] places {rows}", flush=True)
    for n, k in ((8, 2), (40, 5), (1024, 3)):
        x, _ = _logits(rows, n, torch.float32, rows, masked=0.6)
        r = ds.route_rows(x.cuda(), k)
        e = r.experts.cpu().numpy()
        sizes, places = oracle.places_of(e, n)
        assert np.array_equal(r.sizes.cpu().numpy(), sizes) and np.array_equal(r.places.cpu().numpy(), places)
        top = torch.sort(x, dim=1, descending=True, stable=True)
        want = torch.where(top.values[:, :k] == -INF, -1, top.indices[:, :k])
        assert torch.equal(r.experts.cpu().long(), want)


def test_many_workgroups(cuda):
    print("\n[case] 700,000 rows", flush=True)
    x = torch.randn(700_001, 16, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    r = ds.route_rows(x, 2)
    e = r.experts.flatten().long()
    order = torch.argsort(e, stable=True)
    assert torch.equal(r.places.flatten()[order], torch.arange(e.numel(), device="cuda", dtype=torch.int32))
    assert torch.equal(r.sizes, torch.bincount(e, minlength=16))


@TYPES
def test_strides_of_logits(cuda, dtype):
    x, _ = _logits(90, 3 * 24, dtype, 3)
    x = x.cuda()
    part = x[:, 24:48]
    want = ds.route_rows(part.contiguous(), 4)
    for t in (part, part.t().contiguous().t(), x.view(90, 24, 3)[:, :, 0]):
        got = ds.route_rows(t, 4)
        same = ds.route_rows(t.contiguous(), 4)
        assert torch.equal(got.weights, same.weights) and torch.equal(got.places, same.places)
    assert torch.equal(ds.route_rows(part, 4).weights, want.weights)
    one = part[:1].expand(90, 24)
    assert torch.equal(ds.route_rows(one, 4).weights, ds.route_rows(one.contiguous(), 4).weights)
    p = part.clone().requires_grad_(True)
    a, = torch.autograd.grad(ds.route_rows(p, 4, renormalize=False).weights.sum(), p)
    b, = torch.autograd.grad(ds.route_rows(p, 4, renormalize=False).weights, p, torch.ones(90, 4, device="cuda"))
    assert torch.equal(a, b)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_gradient_against_differences(cuda, scoring, renormalize):
    x, _ = _logits(9, 14, torch.float32, 11, masked=0.2)
    grad = torch.randn(9, 3, generator=torch.Generator().manual_seed(2))
    xd = x.cuda().requires_grad_(True)
    r = ds.route_rows(xd, 3, scoring=scoring, renormalize=renormalize, scale=1.5)
    g, = torch.autograd.grad(r.weights, xd, grad.cuda())
    there = torch.isfinite(x).numpy()
    d, h, p = np.where(there, np.random.default_rng(3).standard_normal(x.shape), 0), 1e-6, x.double().numpy()
    loss = lambda v: (oracle.route_rows(v, 3, scoring, renormalize=renormalize, scale=1.5)["weights"] * grad.numpy()).sum()  # noqa: E731
    diff = (loss(p + h * d) - loss(p - h * d)) / (2 * h)
    g = g.double().cpu().numpy()
    assert abs(diff - (g * d).sum()) < 1e-5 * (1 + np.abs(g * d).sum())


# ---------------------------------------------------------------- rows into the experts' order and back


def _routing(rows, n, k, masked=0.5, seed=0, padding=True):
    return ds.route_rows(_logits(rows, n, torch.float32, seed, masked=masked, padding=padding)[0].cuda(), k)


def _check_exchange(rows, n, k, width, dtype, residual=True, seed=0):
    print(f"\n[case] exchange {rows} n={n} k={k} width={width} {dtype} {residual}", flush=True)
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    logits = _logits(rows, n, torch.float32, seed, masked=0.5)[0].cuda().requires_grad_(True)
    r = ds.route_rows(logits, k, scale=1.5)
    places, rounded = r.places.cpu().numpy(), dtype == torch.bfloat16
    x, go = rand(rows, width), rand(rows * k, width)
    xd = x.cuda().requires_grad_(True)
    want, dx, mag = oracle.dispatch_rows(x.double().numpy(), places, go.double().numpy())

    def there_and_back():
        out = ds.dispatch_rows(xd, r)
        return [out, *torch.autograd.grad(out, xd, go.cuda())]

    got = there_and_back()
    sent = got[0]
    assert np.array_equal(got[0].detach().double().cpu().numpy(), want)
    _near("dx", got[1], dx, mag, k + 2, rounded)
    assert all(torch.equal(a, b) for a, b in zip(got, there_and_back()))
    assert int(r.sizes.sum()) == int((r.experts >= 0).sum())
    # what lies behind the last expert's rows is not read
    y, res, gr = rand(rows * k, width), rand(rows, width) if residual else None, rand(rows, width)
    taken = int(r.sizes.sum())
    y[taken:] = float("nan")
    leaves = [y.cuda().requires_grad_(True)] + ([res.cuda().requires_grad_(True)] if residual else [])

    def combine():
        out = ds.combine_rows(leaves[0], r, leaves[1] if residual else None)
        return [out, *torch.autograd.grad(out, [leaves[0], r.weights, *leaves[1:]], gr.cuda())]

    got = combine()
    clean = y.clone()
    clean[taken:] = 0
    np64 = lambda t: None if t is None else t.detach().double().cpu().numpy()  # noqa: E731
    want, mag = oracle.combine_rows(np64(clean), places, np64(r.weights), np64(res), np64(gr))
    _near("out", got[0], want["out"], mag["out"], k + 2, rounded)
    _near("dy", got[1], want["dy"], np.abs(want["dy"]), 1, rounded)
    _near("dweights", got[2], want["dweights"], mag["dweights"], width + 2, False)
    if residual:
        assert torch.equal(got[3].cpu(), gr)
    assert not got[1][taken:].any()
    assert all(torch.equal(a, b) for a, b in zip(got, combine()))
    with torch.no_grad():
        assert torch.equal(ds.combine_rows(leaves[0], r, leaves[1] if residual else None), got[0])
        assert torch.equal(ds.dispatch_rows(xd, r), sent)


@TYPES
@pytest.mark.parametrize("width", [1, 2, 7, 8, 16, 100, 128, 130, 256, 512, 520, 1024, 1111, 4096])
def test_widths(cuda, width, dtype):
    _check_exchange(45, 9, 3, width, dtype, seed=width)


@TYPES
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 8, 8), (2, 4, 1), (300, 5, 5), (301, 64, 6), (70, 40, 33), (70, 100, 64)])
def test_rows_and_choices(cuda, rows, n, k, dtype):
    _check_exchange(rows, n, k, 72, dtype, seed=rows)
    _check_exchange(rows, n, k, 37, dtype, residual=False, seed=rows)


@TYPES
def test_strides_and_alignment_of_rows(cuda, dtype):
    r = _routing(50, 6, 2)
    g = torch.Generator().manual_seed(4)
    wide = torch.randn(50, 3 * 64, generator=g).to(dtype).cuda()
    y = torch.randn(100, 64, generator=g).to(dtype).cuda()
    part = wide[:, 64:128]
    odd = torch.empty(50 * 64 + 1, dtype=dtype, device="cuda")[1:].view(50, 64).copy_(part)
    turned, one = part.t().contiguous().t(), part[:1].expand(50, 64)
    for t in (part, odd, turned):
        assert torch.equal(ds.dispatch_rows(t, r), ds.dispatch_rows(part.contiguous(), r))
        assert torch.equal(ds.combine_rows(y, r, t), ds.combine_rows(y, r, part.contiguous()))
    assert torch.equal(ds.dispatch_rows(one, r), ds.dispatch_rows(one.contiguous(), r))
    odd_y = torch.empty(100 * 64 + 1, dtype=dtype, device="cuda")[1:].view(100, 64).copy_(y)
    assert torch.equal(ds.combine_rows(odd_y, r), ds.combine_rows(y, r))
    # gradients that are broadcast
    p, o = part.clone().requires_grad_(True), y.clone().requires_grad_(True)
    one = torch.ones(100, 64, dtype=dtype, device="cuda")
    a, b = torch.autograd.grad(ds.dispatch_rows(p, r).sum(), p)[0], torch.autograd.grad(ds.dispatch_rows(p, r), p, one)[0]
    assert torch.equal(a, b)
    a, b = torch.autograd.grad(ds.combine_rows(o, r).sum(), o)[0], torch.autograd.grad(ds.combine_rows(o, r), o, one[:50])[0]
    assert torch.equal(a, b)


@TYPES
def test_infinities_and_nan_stay_in_their_rows(cuda, dtype):
    r = _routing(60, 6, 2, masked=0.0, seed=9)
    x = torch.randn(60, 40, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    x[5, 3], x[6, 4] = float("nan"), -INF
    out = ds.dispatch_rows(x, r)
    assert torch.equal(out[r.places[6].long()], x[6].expand(2, 40))
    assert torch.isnan(out).sum() == 2 and torch.isinf(out).sum() == 2
    back = ds.combine_rows(out, r)
    assert torch.isnan(back).sum() == 1 and torch.isinf(back).sum() == 1 and back[5, 3].isnan() and back[6, 4] == -INF


def test_offsets_past_32_bits(cuda):
    """6 GB in the experts' order: rows whose offsets pass 2^31 elements, in whole chunks and one by one."""
    for width in (1 << 15, (1 << 15) + 1):
        print(f"\n[case] far rows {width}", flush=True)
        rows, k = 35_000, 2
        r = _routing(rows, 4, k, masked=0.0, padding=False)
        x = torch.arange(rows, device="cuda").remainder(251).bfloat16()[:, None].expand(rows, width)
        out = ds.dispatch_rows(x, r)
        order = torch.argsort(r.places.flatten()) // k
        assert out.numel() > 2 ** 31 and torch.equal(out[:, 0], x[order, 0]) and torch.equal(out[:, -1], x[order, 0])
        back = ds.combine_rows(out, r)
        del out
        # (the weights of a row add up to one, but for 4 EPS)
        assert ((back[:, -1].double() - x[:, 0].double()).abs() <= (2.0 ** -8 + 8 * EPS) * x[:, 0].double()).all()
        del back


def test_no_rows(cuda):
    logits = torch.empty(0, 8, device="cuda", requires_grad=True)
    r = ds.route_rows(logits, 2)
    assert r.weights.shape == (0, 2) and r.sizes.tolist() == [0] * 8
    x, y = torch.empty(0, 16, device="cuda", requires_grad=True), torch.empty(0, 16, device="cuda", requires_grad=True)
    assert ds.dispatch_rows(x, r).shape == (0, 16) and ds.combine_rows(y, r, x).shape == (0, 16)
    grads = torch.autograd.grad(ds.combine_rows(ds.dispatch_rows(x, r), r, y).sum(), [x, y, logits])
    assert all(g.numel() == 0 for g in grads)


def test_all_padding(cuda):
    r = ds.route_rows(torch.full((70, 8), -INF, device="cuda"), 3)
    assert (r.experts == -1).all() and not r.sizes.any() and not r.weights.any()
    x = torch.randn(70, 24, device="cuda")
    assert not ds.dispatch_rows(x, r).any()
    assert torch.equal(ds.combine_rows(torch.full((210, 24), float("nan"), device="cuda"), r, x), x)


def test_streams_and_graphs(cuda):
    """On a side stream, and the whole of a layer of experts replayed from two graphs in turn."""
    print("\n[case] streams and graphs", flush=True)
    g = torch.Generator("cuda").manual_seed(3)
    logits, x = torch.randn(3000, 16, device="cuda", generator=g), torch.randn(3000, 64, device="cuda", generator=g).bfloat16()
    w = (torch.randn(16, 64, 64, device="cuda", generator=g) / 8).bfloat16()

    def layer(logits, x):
        r = ds.route_rows(logits, 2, scoring="sigmoid", bias=None)
        return ds.combine_rows(ds.grouped_linear(ds.dispatch_rows(x, r), w, r.sizes), r, x), r.experts

    want = layer(logits, x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer(logits, x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs, ins = [], [], [(logits.clone(), x.clone()) for _ in range(2)]
    for pair in ins:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(layer(*pair))
    for i in range(4):
        for pair, graph, out in zip(ins, graphs, outs):
            pair[0].copy_(torch.randn(3000, 16, device="cuda", generator=g))
            graph.replay()
            eager = layer(*pair)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, eager)), i


def test_refusals(cuda):
    x = torch.zeros(10, 8, device="cuda")
    bad = lambda match, f, *a, **kw: pytest.raises(RuntimeError, f, *a, **kw).match(match)  # noqa: E731
    route = ds.route_rows
    bad("CUDA tensor", route, x.cpu(), 2)
    bad("CUDA tensor", route, [1.0], 2)
    bad("must have shape", route, x[0], 2)
    bad("float32 or bfloat16", route, x.double(), 2)
    bad("k must be", route, x, 0)
    bad("k must be", route, x, 9)
    bad("k must be", route, torch.zeros(2, 100, device="cuda"), 65)
    bad("1 to 1024", route, torch.zeros(2, 1025, device="cuda"), 2)
    bad("1 to 1024", route, torch.zeros(2, 0, device="cuda"), 1)
    bad("below 2\\^31", route, x[:1].expand(1 << 30, 8), 2)
    bad("scoring", route, x, 2, scoring="relu")
    bad("groups must", route, x, 2, groups=3)
    bad("groups must", route, x, 2, groups=0)
    bad("top_groups", route, x, 2, groups=4, top_groups=5)
    bad("group_best", route, x, 2, groups=4, top_groups=2, group_best=3)
    bad("scale", route, x, 2, scale=float("nan"))
    bad("bias", route, x, 2, bias=torch.zeros(7, device="cuda"))
    bad("bias", route, x, 2, bias=torch.zeros(8))
    bad("bias", route, x, 2, bias=torch.zeros(8, device="cuda", dtype=torch.int64))
    r = route(x, 2)
    bad("Routing", ds.dispatch_rows, x, None)
    bad("shape", ds.dispatch_rows, x[:9], r)
    bad("CUDA tensor", ds.dispatch_rows, x.cpu(), r)
    bad("float32 or bfloat16", ds.dispatch_rows, x.half(), r)
    bad("width", ds.dispatch_rows, x[:, :0], r)
    bad("shape", ds.combine_rows, x, r)
    y = torch.zeros(20, 8, device="cuda")
    bad("residual must", ds.combine_rows, y, r, x.bfloat16())
    bad("residual must", ds.combine_rows, y, r, x[:, :4])
    bad("residual must", ds.combine_rows, y, r, y)
    with forward_ad.dual_level():
        bad("forward-mode", route, forward_ad.make_dual(x, x), 2)
        bad("forward-mode", ds.dispatch_rows, forward_ad.make_dual(x, x), r)
        bad("forward-mode", ds.combine_rows, y, r, forward_ad.make_dual(x, x))


@pytest.mark.parametrize("renormalize", [True, False])
def test_logits_past_32_bits(cuda, renormalize):
    """Rows that lie 2^20 elements apart: the bits of the same rows side by side, forward and backward."""
    print("\n[case] far logits", flush=True)
    close = torch.randn(4200, 24, device="cuda", generator=torch.Generator("cuda").manual_seed(8)).requires_grad_(True)
    apart = torch.empty(4200, 1 << 20, device="cuda")[:, 5:29]
    with torch.no_grad():
        apart.copy_(close)
    apart.requires_grad_(True)
    bias = torch.linspace(-0.2, 0.2, 24, device="cuda")
    a, b = (ds.route_rows(x, 3, bias=bias, renormalize=renormalize) for x in (close, apart))
    for name in ("weights", "experts", "sizes", "places"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name
    g = torch.arange(4200 * 3, device="cuda").float().cos().view(4200, 3)
    assert torch.equal(torch.autograd.grad(a.weights, close, g)[0], torch.autograd.grad(b.weights, apart, g)[0])

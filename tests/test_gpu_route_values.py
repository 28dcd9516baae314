"""route_rows where its 32-bit arithmetic has little room: biases near the largest numbers, logits that lie far
apart, sigmoids that vanish; and choices that a caller drops.

Tolerances, EPS = 2^-24 of a weight.  An exponential of a difference of logits, which is taken in two parts: 2 for
the exponential and 1 for the second part.  A sigmoid's denominator 4 more (2 for its exponential, a sum and a quotient).  The
sum over a row's choices has errors of its terms (7) and of 6 additions of lanes; the quotient and the scale 1 each: 22
in all.  Without renormalisation the sum of a softmax has up to 16 additions in a lane and 6 of lanes, and terms whose
error, 2 + 2 d for one at a distance d, counts for exp(-d), so 3: 25, with the exponential, quotient and scale 30.  Below
2^-126 numbers are steps of 2^-149."""
import numpy as np
import pytest
import torch

from dynamis_amd import dynamis_state as ds
from oracle import layers as oracle

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24
SCORINGS = pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
RENORMALIZE = pytest.mark.parametrize("renormalize", [True, False])


def _choices(x, k, **how):
    want = oracle.route_rows(x.double().numpy(), k, **{a: b.double().numpy() if a == "bias" else b for a, b in how.items()})
    got = ds.route_rows(x.cuda(), k, **{a: b.cuda() if a == "bias" else b for a, b in how.items()})
    for name in ("experts", "sizes", "places"):
        t = getattr(got, name).cpu().numpy()
        assert np.array_equal(t, want[name]), (name, np.argwhere(t != want[name])[:4], how)


@SCORINGS
def test_groups_whose_sums_pass_32_bits(cuda, scoring):
    """The sum of a group's two largest is no 32-bit number; of two such groups the larger is taken."""
    print(f"\n[case] four experts {scoring}", flush=True)
    x = torch.zeros(5, 4)
    for bias in ([3e38, 2e38, 2.9e38, 2.5e38], [3e38, 2e38, 3.1e38, 1e38], [-3e38, -2e38, -2.9e38, -2.0e38], [1e38, 2.5e38, -1e38, -3e38]):
        for k in (1, 2):
            _choices(x, k, scoring=scoring, bias=torch.tensor(bias), groups=2, top_groups=1, group_best=2)


@SCORINGS
@pytest.mark.parametrize("group_best", [1, 2])
@pytest.mark.parametrize("n,groups,top", [(64, 8, 4), (64, 8, 1), (60, 5, 2), (12, 3, 1), (130, 2, 1), (256, 8, 4), (1024, 64, 3), (1024, 4, 2)])
def test_large_finite_biases(cuda, n, groups, top, group_best, scoring):
    """Biases up to the largest numbers, of both signs, alone among small ones or in every group."""
    print(f"\n[case] large biases {n} {groups} {top} {group_best} {scoring}", flush=True)
    g = torch.Generator().manual_seed(n + top)
    x = 2 * torch.randn(40, n, generator=g)
    x[torch.rand(40, n, generator=g) < 0.1] = -float("inf")
    for spread in (1.0, 0.05):
        for low, high in ((2e38, 3.4e38), (-3.4e38, -2e38), (-3.4e38, 3.4e38), (-1e5, -1e4)):
            bias = 0.2 * torch.randn(n, generator=g)
            large = torch.rand(n, generator=g) < spread
            bias[large] = (low + (high - low) * torch.rand(n, generator=g).double()).float()[large]
            _choices(x, 3, scoring=scoring, bias=bias, groups=groups, top_groups=top, group_best=group_best)
            _choices(x, 8, scoring=scoring, bias=bias)


def _near(name, got, want, mag, n, beneath=1.0):
    got = got.detach().double().cpu().numpy()
    bad = ~(np.abs(got - want) <= n * EPS * mag + 2.0 ** -148 * beneath)
    assert not bad.any(), (f"{name}: {bad.sum()} of {bad.size} off, worst {(np.abs(got - want)[bad] / mag[bad] / EPS).max():.3g} EPS at "
                           f"{np.argwhere(bad)[0]}")


@RENORMALIZE
@SCORINGS
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("n,k", [(8, 4), (64, 8), (100, 33), (1024, 10)])
def test_weights_of_logits_far_apart(cuda, n, k, biased, scoring, renormalize):
    """The digits are there whatever the distance of a logit to the largest."""
    print(f"\n[case] far apart {n} {k} {biased} {scoring} {renormalize}", flush=True)
    g = torch.Generator().manual_seed(n)
    x = 25 * torch.randn(60, n, generator=g)
    x[::2] = -30 * torch.rand(30, n, generator=g) ** 2 - 5
    bias = 0.01 * torch.randn(n, generator=g) if biased else None
    grad = torch.randn(60, k, generator=g)
    how = dict(scoring=scoring, renormalize=renormalize, scale=1.5)
    want = oracle.route_rows(x.double().numpy(), k, bias=None if bias is None else bias.double().numpy(), grad=grad.numpy(), **how)
    xd = x.cuda().requires_grad_(True)
    r = ds.route_rows(xd, k, bias=None if bias is None else bias.cuda(), **how)
    assert np.array_equal(r.experts.cpu().numpy(), want["experts"])
    w = want["weights"]
    _near("weights", r.weights, w, np.abs(w), 22 if renormalize else 30)
    # what is differentiated is what was returned: the gradient by the returned weights (u = w / scale)
    dx, = torch.autograd.grad(r.weights, xd, grad.cuda())
    u, e, gs = r.weights.detach().double().cpu().numpy() / 1.5, want["experts"], 1.5 * grad.double().numpy()
    c = np.take_along_axis(x.double().numpy(), e, 1)
    slope = np.exp(-np.logaddexp(0, c)) if scoring == "sigmoid" else 1.0
    if renormalize:
        d, mag = u * (gs - (gs * u).sum(1, keepdims=True)) * slope, u * (np.abs(gs) + np.abs(gs * u).sum(1, keepdims=True)) * slope
    else:
        d, mag = u * gs * slope, u * np.abs(gs) * slope
    if scoring == "sigmoid" or renormalize:
        # (its factors: the weight, whose sum and quotient are the forward pass's, 2; the dot product k and 6; 1 - s by 6; products 4)
        # (1 - s is a number of 32 bits: beneath 2^-126 off by a step, 2^-149, of its exponential and half a step of
        # its own, which what it multiplies, mag / slope, takes with it; the product's own rounding is the other half)
        _near("dlogits", torch.gather(dx, 1, torch.from_numpy(e).cuda()), d, mag, k + 18, 1 + mag / slope)
        rest = dx.clone()
        rest.scatter_(1, torch.from_numpy(e).cuda(), 0)
        assert not rest.any()


def test_sigmoids_that_vanish_beside_others(cuda):
    """Chosen together, -29 and -90 keep their ratio, and so do sigmoids beneath what 32 bits hold."""
    print("\n[case] vanishing sigmoids", flush=True)
    x = torch.tensor([[-29.0, -90.0, -60.0, -100.0], [-120.0, -100.0, -101.0, -130.0], [-31.0, -88.5, -95.0, -103.0], [0.0, -90.0, -80.0, 40.0],
                      [-29.5, -88.0, -86.0, -104.0], [5.0, -60.0, -87.5, -3.0]])
    grad = torch.tensor([[0.5, -1.0, 2.0, 1.0]]).expand(6, 4)
    for scale in (1.0, 1e30):
        for renormalize in (True, False):
            want = oracle.route_rows(x.double().numpy(), 4, "sigmoid", renormalize=renormalize, scale=scale, grad=grad.numpy())
            xd = x.cuda().requires_grad_(True)
            r = ds.route_rows(xd, 4, scoring="sigmoid", renormalize=renormalize, scale=scale)
            assert np.array_equal(r.experts.cpu().numpy(), want["experts"])
            w = want["weights"]
            # (a weight is a number of 32 bits before the scale)
            lost = 2.0 ** -149 * scale * np.ones_like(w)
            got = r.weights.detach().double().cpu().numpy()
            assert (np.abs(got - w) <= 24 * EPS * np.abs(w) + 2 * lost).all(), (renormalize, scale, got, w)
            dx, = torch.autograd.grad(r.weights, xd, grad.cuda())
            dx = dx.double().cpu().numpy()
            assert (np.abs(dx - want["dlogits"]) <= 60 * EPS * want["mag"] + 16 * lost).all(), (renormalize, scale, dx, want["dlogits"])


def test_a_dropped_choice_keeps_the_permutation(cuda):
    """Its place p as -1 - p: its row is zeros, it adds nothing, and nothing is left unwritten."""
    r = ds.route_rows(torch.randn(12, 4, device="cuda", generator=torch.Generator("cuda").manual_seed(1)), 2)
    x = torch.randn(12, 24, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).requires_grad_(True)
    places, weights = r.places.clone(), r.weights.detach().clone().requires_grad_(True)
    places[5, 1] = -1 - places[5, 1]
    few = ds.Routing(4, weights, r.experts, r.sizes, places)
    rows = ds.dispatch_rows(x, few)
    want = ds.dispatch_rows(x, r).detach().clone()
    want[int(r.places[5, 1])] = 0
    assert torch.equal(rows, want)
    y = want.clone().requires_grad_(True)
    out = ds.combine_rows(y, few)
    assert torch.equal(out[5], weights[5, 0] * x[5])
    dy, dw = torch.autograd.grad(out, [y, weights], torch.ones_like(out))
    assert not dy[int(r.places[5, 1])].any() and dw[5, 1] == 0 and torch.isfinite(dy).all()
    dx, = torch.autograd.grad(rows, x, torch.ones_like(rows))
    assert (dx[5] == 1).all() and (dx[:5] == 2).all()

"""A layer of all operators on a built graph, as a model runs it, and what no test of a single one holds: training
steps replayed from graphs, two graphs in turn, rows chosen with a bias that are not finite, places that point
nowhere."""
import math

import numpy as np
import pytest
import torch

from dynamis_amd import configs
from dynamis_amd import dynamis_state as ds
from dynamis_amd.dynamis_state import dynamis_state_impl as impl
from oracle import layers as oracle

pytestmark = pytest.mark.gpu
INF = float("inf")
HEADS, DIM, EXPERTS, K = 4, 16, 6, 2


def _weights(seed=0):
    g = torch.Generator().manual_seed(seed)
    new = lambda *s: torch.randn(*s, generator=g) / math.sqrt(s[-1])  # noqa: E731
    w = HEADS * DIM
    return {"x": math.sqrt(w) * new(256, w), "qkv": new(1, 3 * w, w), "qn": 1 + 0.1 * new(DIM), "kn": 1 + 0.1 * new(DIM),
            "table": new(16, HEADS), "out": new(1, w, w), "router": 3 * new(1, EXPERTS, w), "up": new(EXPERTS, 2 * w, w),
            "up_bias": new(EXPERTS, 2 * w), "down": new(EXPERTS, w, 2 * w)}


def _graph():
    """256 atoms of a jittered crystal: edges as the build gives them, distances, positions."""
    box = configs.fcc(cells=4, seed=5)
    pos = torch.from_numpy(box.pos).cuda()
    ei, _, _, _, _, dist = impl.radius_graph_pbc_vectors(pos, torch.from_numpy(box.cell), torch.tensor(box.pbc), 4.0)
    return pos.float(), ei, dist, torch.linspace(0.0, 4.0, 17, device="cuda")[1:-1]


def _layer(p, pos, plan, freq):
    x, rows = p["x"], torch.full((1,), 256, device="cuda")
    qkv = ds.grouped_linear(x, p["qkv"], rows)
    q, k, v = (t.unflatten(1, (HEADS, DIM)) for t in qkv.chunk(3, 1))
    q, k = ds.rotate_heads(q, k, pos, freq, None, p["qn"], p["kn"])
    y = ds.neighbor_attention(q, k, v, plan, p["table"])
    x = ds.grouped_linear(y.flatten(1), p["out"], rows, residual=x)
    r = ds.route_rows(ds.grouped_linear(x, p["router"], rows), K)
    h = ds.grouped_linear(ds.dispatch_rows(x, r), p["up"], r.sizes, p["up_bias"], activation="silu")
    return ds.combine_rows(ds.grouped_linear(h, p["down"], r.sizes), r, x), r.experts


def _plain(p, pos, src, dst, bucket, freq):
    """The same in 64 bits out of elementary steps, each expert by itself."""
    x = p["x"]
    q, k, v = ((x @ w.T).unflatten(1, (HEADS, DIM)) for w in p["qkv"][0].chunk(3, 0))
    theta = (pos[:, [0, 0, 1, 1, 2, 2]] * freq)[:, None]
    heads = []
    for t, w in ((q, p["qn"]), (k, p["kn"])):
        t = t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * w
        a, b = t[..., :6], t[..., 6:12]
        heads.append(torch.cat([a * theta.cos() - b * theta.sin(), a * theta.sin() + b * theta.cos(), t[..., 12:]], -1))
    logit = (heads[0][dst] * heads[1][src]).sum(-1) / math.sqrt(DIM) + p["table"][bucket]
    w = torch.exp(logit - logit.max())
    total = torch.zeros(256, HEADS, dtype=torch.float64).index_add(0, dst, w)
    y = torch.zeros(256, HEADS, DIM, dtype=torch.float64).index_add(0, dst, (w / total[dst])[..., None] * v[src])
    x = y.flatten(1) @ p["out"][0].T + x
    logits = x @ p["router"][0].T
    top = torch.sort(logits.detach(), dim=1, descending=True)
    share = torch.softmax(torch.gather(logits, 1, top.indices[:, :K]), 1)
    out = x
    for e in range(EXPERTS):
        z = x @ p["up"][e].T + p["up_bias"][e]
        f = (z * torch.sigmoid(z)) @ p["down"][e].T
        out = out + (share * (top.indices[:, :K] == e)).sum(1)[:, None] * f
    return out, top


def test_a_layer_forward_and_backward(cuda):
    """float32 against 64 bits.  Some ten operators follow each other, each within 200 2^-24 of its terms'
    magnitudes, which the next ones add up over no more than 128 terms of either sign: 2e-4 of the largest."""
    print("\n[case] layer", flush=True)
    pos, ei, dist, bounds = _graph()
    plan = ds.neighbor_plan(ei, 256, distances=dist, boundaries=bounds.to(dist.dtype))
    freq = torch.tensor([1.0, 0.5, 1.1, 0.6, 0.9, 0.4], device="cuda")
    p = {k: t.cuda().requires_grad_(True) for k, t in _weights().items()}
    at = pos.clone().requires_grad_(True)
    out, experts = _layer(p, at, plan, freq)
    grad = torch.randn(256, HEADS * DIM, generator=torch.Generator().manual_seed(1))
    leaves = [*p.values(), at]
    got = torch.autograd.grad(out, leaves, grad.cuda())

    p64 = {k: t.double().requires_grad_(True) for k, t in _weights().items()}
    at64 = pos.cpu().double().requires_grad_(True)
    bucket = torch.bucketize(dist.cpu(), bounds.to(dist.dtype).cpu(), right=True)
    want, top = _plain(p64, at64, ei[0].cpu(), ei[1].cpu(), bucket, freq.cpu().double())
    # (no choice hangs on a rounding)
    assert (top.values[:, :K] - top.values[:, 1:K + 1]).min() > 2e-5
    assert torch.equal(experts.cpu().long(), top.indices[:, :K])
    want_grads = torch.autograd.grad(want, [*p64.values(), at64], grad.double())
    for name, a, b in zip(["out", *p, "pos"], [out, *got], [want, *want_grads]):
        a, b = a.detach().double().cpu(), b.detach()
        assert (a - b).abs().max() <= 2e-4 * b.abs().max(), (name, float((a - b).abs().max() / b.abs().max()))
    again, _ = _layer(p, at, plan, freq)
    assert torch.equal(again, out) and all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(again, leaves, grad.cuda())))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_training_steps_replayed_from_two_graphs(cuda, dtype):
    """Forward and backward of the whole layer, captured twice with their own leaves: each replay the eager bits."""
    print(f"\n[case] graphs {dtype}", flush=True)
    pos, ei, dist, bounds = _graph()
    plan = ds.neighbor_plan(ei, 256, distances=dist, boundaries=bounds.to(dist.dtype))
    freq = torch.tensor([1.0, 0.5, 1.1, 0.6, 0.9, 0.4], device="cuda")
    grad = torch.randn(256, HEADS * DIM, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(dtype)

    def leaves_of(seed):
        p = {k: (t if k == "table" else t.to(dtype)).cuda().requires_grad_(True) for k, t in _weights(seed).items()}
        return p, pos.clone().requires_grad_(True)

    def step(p, at):
        out, experts = _layer(p, at, plan, freq)
        return [out.detach(), experts, *torch.autograd.grad(out, [*p.values(), at], grad)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*leaves_of(0))
    torch.cuda.current_stream().wait_stream(side)
    sets, graphs, outs = [leaves_of(s) for s in (1, 2)], [], []
    for p, at in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(p, at))
    for i in range(4):
        for (p, at), graph, out in zip(sets, graphs, outs):
            with torch.no_grad():
                p["x"].copy_(torch.randn(256, HEADS * DIM, device="cuda"))
                at.add_(0.01)
            graph.replay()
            fresh = {k: t.detach().clone().requires_grad_(True) for k, t in p.items()}
            eager = step(fresh, at.detach().clone().requires_grad_(True))
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, eager)), i


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_chosen_with_a_bias_and_not_finite(cuda, scoring, groups):
    print(f"\n[case] bias, not finite {scoring} {groups}", flush=True)
    g = torch.Generator().manual_seed(3)
    x, bias = torch.randn(40, 32, generator=g), 0.3 * torch.randn(32, generator=g)
    x[1, 5], x[2, 6], x[3, 7], x[4], x[5, 1:] = float("nan"), INF, -INF, -INF, -INF
    x[6, 30], x[6, 31] = float("nan"), INF
    for b in (bias, torch.where(torch.arange(32) == 5, -INF, bias), torch.where(torch.arange(32) == 9, INF, bias),
              torch.where(torch.arange(32) == 11, float("nan"), bias)):
        for best in (1, 2):
            for renormalize in (True, False):
                how = dict(scoring=scoring, groups=groups, top_groups=max(1, groups // 2), group_best=best, renormalize=renormalize)
                r = ds.route_rows(x.cuda(), 4, bias=b.cuda(), **how)
                want = oracle.route_rows(x.double().numpy(), 4, bias=b.double().numpy(), **how)
                assert np.array_equal(r.experts.cpu().numpy(), want["experts"]), (b[5], how)
                assert np.array_equal(r.places.cpu().numpy(), want["places"])
                w = r.weights.cpu().double().numpy()
                assert np.array_equal(np.isnan(w), np.isnan(want["weights"]))
                # (32 terms, logits up to 8 apart: 2 * 8 + 32 + 12 roundings)
                assert np.allclose(w, want["weights"], rtol=60 * 2.0 ** -24, atol=1e-37, equal_nan=True)


@pytest.mark.parametrize("width", [64, 33])
def test_places_that_point_nowhere_are_left_out(cuda, width):
    """A routing whose places were changed: what lies past the last row is neither read nor written."""
    r = ds.route_rows(torch.randn(10, 4, device="cuda", generator=torch.Generator("cuda").manual_seed(1)), 2)
    x = torch.randn(10, width, device="cuda")
    good = ds.dispatch_rows(x, r)
    for far in (20, 2 ** 31 - 1, -2 ** 31, -21):
        bad = ds.Routing(4, r.weights, r.experts, r.sizes, r.places.clone())
        lost = int(bad.places[3, 1])
        bad.places[3, 1] = far
        out = ds.dispatch_rows(x, bad)
        keep = torch.arange(20, device="cuda") != lost
        assert torch.equal(out[keep], good[keep])
        weights = r.weights.clone().requires_grad_(True)
        bad.weights = weights
        y = good.clone().requires_grad_(True)
        back = ds.combine_rows(y, bad)
        want = r.weights[3, 0] * x[3]
        assert torch.equal(back[3], want)
        dy, dw = torch.autograd.grad(back, [y, weights], torch.ones_like(back))
        assert dw[3, 1] == 0 and torch.equal(dy[int(r.places[3, 0])], r.weights[3, 0].expand(width))


def test_weights_of_another_make_are_refused(cuda):
    r = ds.route_rows(torch.randn(10, 4, device="cuda"), 2)
    y = torch.zeros(20, 8, device="cuda")
    for w in (r.weights.bfloat16(), r.weights[:, :1], r.weights.double()):
        with pytest.raises(RuntimeError, match="routing.weights must be"):
            ds.combine_rows(y, ds.Routing(4, w, r.experts, r.sizes, r.places))
    turned = r.weights.t().contiguous().t()
    assert torch.equal(ds.combine_rows(y + 1, ds.Routing(4, turned, r.experts, r.sizes, r.places)), ds.combine_rows(y + 1, r))


def test_a_changed_routing_is_refused(cuda):
    """Weights elsewhere, places of another type, more or fewer rows than the operands have."""
    r = ds.route_rows(torch.randn(10, 4, device="cuda"), 2)
    x, y = torch.zeros(10, 8, device="cuda"), torch.zeros(20, 8, device="cuda")
    for w in (r.weights.cpu(), None):
        with pytest.raises(RuntimeError, match="routing.weights must be"):
            ds.combine_rows(y, ds.Routing(4, w, r.experts, r.sizes, r.places))
    for places in (r.places.long(), r.places.cpu(), r.places.float(), r.places.flatten()):
        bad = ds.Routing(4, r.weights, r.experts, r.sizes, places)
        with pytest.raises(RuntimeError, match="routing.places must be"):
            ds.dispatch_rows(x, bad)
        with pytest.raises(RuntimeError, match="routing.places must be"):
            ds.combine_rows(y, bad)
    for rows in (9, 11):
        bad = ds.Routing(4, r.weights, r.experts, r.sizes, r.places)
        bad.places = torch.zeros(rows, 2, dtype=torch.int32, device="cuda")
        with pytest.raises(RuntimeError, match="x must have shape"):
            ds.dispatch_rows(x, bad)
        with pytest.raises(RuntimeError, match="y must have shape"):
            ds.combine_rows(y, bad)


def test_dispatched_bits_are_those_of_the_rows(cuda):
    """Every bit pattern of bfloat16, NaNs with their payloads, in whole chunks and one by one."""
    bits = torch.arange(-2 ** 15, 2 ** 15, device="cuda", dtype=torch.int32).to(torch.int16)
    for width in (64, 1):
        x = bits.view(torch.bfloat16).view(-1, width)
        r = ds.route_rows(torch.randn(x.size(0), 4, device="cuda"), 1)
        out = ds.dispatch_rows(x, r)
        assert torch.equal(out.view(torch.int16)[r.places[:, 0].long()], x.view(torch.int16))


def test_operators_run_at_once_on_two_streams(cuda):
    g = torch.Generator("cuda").manual_seed(2)
    sets = [(torch.randn(20000, 64, device="cuda", generator=g), torch.randn(20000, 96, device="cuda", generator=g)) for _ in range(2)]
    bias = torch.randn(64, device="cuda", generator=g) * 0.1

    def work(pair):
        r = ds.route_rows(pair[0], 6, scoring="sigmoid", bias=bias, groups=8, top_groups=4, group_best=2)
        return [r.experts, r.sizes, ds.combine_rows(ds.dispatch_rows(pair[1], r), r, pair[1])]

    want = [work(pair) for pair in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for s, pair in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append(work(pair))
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))


def test_gradients_are_taken_once(cuda):
    """A graph of the gradients may be asked for; differentiating them raises, instead of calling them constants."""
    g = torch.Generator("cuda").manual_seed(4)
    new = lambda *s: torch.randn(*s, device="cuda", generator=g).requires_grad_(True)  # noqa: E731
    q, k, at, logits, x, w = new(9, 2, 16), new(9, 2, 16), new(9, 2), new(9, 4), new(9, 8), new(1, 8, 8)
    r = ds.route_rows(logits, 2)
    calls = {"rotate_heads": (ds.rotate_heads(q, k, at, torch.ones(4, device="cuda"))[0], q),
             "route_rows": (r.weights, logits), "dispatch_rows": (ds.dispatch_rows(x, r), x),
             "combine_rows": (ds.combine_rows(ds.dispatch_rows(x.detach(), r).requires_grad_(True), r, x), x),
             "grouped_linear": (ds.grouped_linear(x, w, [9], None, "silu", x), w)}
    for name, (out, leaf) in calls.items():
        want, = torch.autograd.grad(out, leaf, torch.ones_like(out), retain_graph=True)
        again, = torch.autograd.grad(out, leaf, torch.ones_like(out), create_graph=True)
        assert torch.equal(want, again), name
        with pytest.raises(RuntimeError, match=f"twice {name}"):
            again.square().sum().backward()


def test_hooks_and_anomalies(cuda):
    """Saved tensors that a hook moves to the host and back, and the mode that looks for NaN: the same gradients."""
    g = torch.Generator("cuda").manual_seed(5)
    new = lambda *s: torch.randn(*s, device="cuda", generator=g).requires_grad_(True)  # noqa: E731
    logits, x, w = new(40, 6), new(40, 16), new(6, 16, 16)

    def step():
        r = ds.route_rows(logits, 2)
        y = ds.combine_rows(ds.grouped_linear(ds.dispatch_rows(x, r), w, r.sizes, activation="gelu"), r, x)
        return torch.autograd.grad(y, [logits, x, w], torch.ones_like(y))

    want = step()
    with torch.autograd.graph.save_on_cpu():
        assert all(torch.equal(a, b) for a, b in zip(step(), want))
    with torch.autograd.detect_anomaly(check_nan=True):
        assert all(torch.equal(a, b) for a, b in zip(step(), want))


def test_hooks_that_lay_saved_tensors_out_anew(cuda):
    """Rows that lie apart come back whole, whole ones apart or transposed: the same gradients."""
    g = torch.Generator("cuda").manual_seed(6)
    new = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    wide, scores, table = new(33, 400), new(33, 50), new(2, 33)
    q = wide[:, :96].unflatten(1, (6, 16)).requires_grad_(True)
    k = wide[:, 96:128].unflatten(1, (2, 16)).requires_grad_(True)
    at, qw, kw = table.t().requires_grad_(True), new(16).requires_grad_(True), new(16).requires_grad_(True)
    logits, x = scores[:, :6].requires_grad_(True), new(33, 32).requires_grad_(True)
    w, b = new(6, 32, 32).requires_grad_(True), new(6, 32).requires_grad_(True)
    freq = torch.linspace(0.1, 1.0, 6, device="cuda")
    leaves = [q, k, at, qw, kw, logits, x, w, b]

    def step():
        a, c = ds.rotate_heads(q, k, at, freq, None, qw, kw)
        r = ds.route_rows(logits, 2, renormalize=False)
        y = ds.combine_rows(ds.grouped_linear(ds.dispatch_rows(x, r), w, r.sizes, b, activation="silu"), r, x)
        out = [a, c, y]
        return torch.autograd.grad(out, leaves, [torch.cos(torch.arange(t.numel(), device="cuda").float()).view_as(t) for t in out])

    want = step()
    turned = lambda t: t.movedim(0, -1).contiguous().movedim(-1, 0)  # noqa: E731
    apart = lambda t: torch.stack([t, t], -1)[..., 0]  # noqa: E731
    for back in (lambda t: t.contiguous(), lambda t: t.clone(memory_format=torch.contiguous_format), turned, apart):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
            assert all(torch.equal(m, n) for m, n in zip(step(), want))
    with torch.autograd.graph.save_on_cpu():
        assert all(torch.equal(m, n) for m, n in zip(step(), want))


def test_hooks_that_change_saved_tensors_are_refused(cuda):
    new = lambda *s: torch.randn(*s, device="cuda").requires_grad_(True)  # noqa: E731
    logits, x, w = new(10, 4), new(10, 16), new(4, 16, 16)
    r = ds.route_rows(logits, 2)
    calls = {"rotate_heads": lambda: ds.rotate_heads(x.view(10, 1, 16), x.view(10, 1, 16), x[:, :2], torch.ones(8, device="cuda"))[0],
             "route_rows": lambda: ds.route_rows(logits, 2).weights, "dispatch_rows": lambda: ds.dispatch_rows(x, r),
             "combine_rows": lambda: ds.combine_rows(torch.cat([x, x]), r, x),
             "grouped_linear": lambda: ds.grouped_linear(x, w, torch.tensor([1, 2, 3, 4], device="cuda"), None, "gelu")}
    for change in (lambda t: t[:-1], lambda t: t.double(), lambda t: t.cpu()):
        for name, call in calls.items():
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
                out = call()
            with pytest.raises(RuntimeError, match=f"{name}: a saved tensor came back"):
                torch.autograd.grad(out, [x, w, logits], torch.ones_like(out), allow_unused=True)


def test_an_input_changed_in_place_is_noticed(cuda):
    x = torch.randn(10, 8, device="cuda")
    w = torch.randn(1, 8, 8, device="cuda", requires_grad=True)
    y = ds.grouped_linear(x, w, [10], None, "silu")
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()

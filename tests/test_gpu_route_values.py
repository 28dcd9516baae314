"""route_rows where its 32-bit arithmetic has little room: biases near the largest numbers."""
import numpy as np
import pytest
import torch

from dynamis_amd import dynamis_state as ds
from oracle import layers as oracle

pytestmark = pytest.mark.gpu
SCORINGS = pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])


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

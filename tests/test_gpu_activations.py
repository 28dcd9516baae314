"""grouped_linear's activations over all of their arguments: f is z far above, and its slope 1; digits are kept far below.

z is the bias (the rows are zeros), so what is off is the activation's own.  Tolerances, EPS = 2^-24, in absolute terms: an
exponential's argument is rounded two or three times, so it errs by 2 |z| (silu) or 2 z^2 (gelu) of itself, and what it
goes into by 14 more (the exponential, reciprocals, the fit and its products); that counts with the exponential's part in the
result alone, m = min(s, 1 - s) for silu, the normal distribution's share beyond |z| and |z| times its density for
gelu.  The rest, 1 or z, errs by 4.  Beneath 2^-120 the hardware's reciprocal and exponential lose digits: that is nothing.
bfloat16: 2^-8 of the result."""
import math

import numpy as np
import pytest
import torch

from dynamis_amd import dynamis_state as ds

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


def _parts(act, z):
    """(f, f', tolerance of f, of f')."""
    with np.errstate(all="ignore"):
        if act == "silu":
            s, t = np.exp(-np.logaddexp(0, -z)), np.exp(-np.logaddexp(0, z))
            m, growth, rest = np.minimum(s, t), 2 * np.abs(z) + 14, 4.0 * (z > 0)
            f, slope = z * s, s * (1 + z * t)
            tail = growth * m * (1 + np.abs(z))
        else:
            beyond = 0.5 * np.vectorize(math.erfc)(np.abs(z) / math.sqrt(2))
            density = np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
            m, growth, rest = beyond, 2 * z * z + 14, 4.0 * (z > 0)
            share = np.where(z < 0, beyond, 1 - beyond)
            f, slope = z * share, share + z * density
            tail = growth * (beyond + np.abs(z) * density)
        own = np.where(m == 0, 0, growth * m)
        tail = np.where(m == 0, 0, tail)
        return f, slope, EPS * (rest + own) * np.abs(z) + 2.0 ** -119, EPS * (rest + tail) + 2.0 ** -119


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("pad", [0, 1])
def test_over_all_arguments(cuda, pad, act, dtype):
    """pad: columns of the streaming kernel, or of the other one."""
    print(f"\n[case] {act} {dtype} {pad}", flush=True)
    most = torch.finfo(dtype).max
    far = torch.tensor([0.0, 1e-30, 1e-10, 16.0, 20.0, 40.0, 87.0, 90.0, 200.0, 1e4, 1e10, 1e19, 1e20, 3e38, most])
    z = torch.cat([torch.linspace(-14, 14, 4097), far, -far])
    z = z[:(len(z) - 8) // 8 * 8 + pad].to(dtype)
    z = torch.cat([z, (far if len(z) % 2 else -far)[-8:].to(dtype)])
    n = len(z)
    assert (n % 8 == 0) == (pad == 0) and (z.double().abs() >= 3e38).any()
    w, x = torch.zeros(1, n, 8, dtype=dtype, device="cuda"), torch.zeros(3, 8, dtype=dtype, device="cuda")
    b = z[None].cuda().requires_grad_(True)
    y = ds.grouped_linear(x, w, [3], b, act)
    g = torch.zeros(3, n, dtype=dtype, device="cuda")
    g[1] = 1
    db, = torch.autograd.grad(y, b, g)
    f, slope, tol, tol_slope = _parts(act, z.double().numpy())
    for name, got, want, t in (("f", y[0], f, tol), ("slope", db[0], slope, tol_slope)):
        got = got.detach().double().cpu().numpy()
        t = t + (2.0 ** -8 * np.abs(want) if dtype == torch.bfloat16 else 0)
        bad = ~(np.abs(got - want) <= t)
        assert not bad.any(), f"{name}: {bad.sum()} off, at z = {z[torch.from_numpy(bad)][:5].tolist()}: {got[bad][:5]} for {want[bad][:5]}"
    up = z.double().numpy() > 20
    exact = z[torch.from_numpy(up)].cuda()
    assert torch.allclose(y[0][torch.from_numpy(up)], exact, rtol=4 * EPS, atol=0) and torch.allclose(
        db[0][torch.from_numpy(up)].float(), torch.ones(1, device="cuda"), rtol=0, atol=4 * EPS)

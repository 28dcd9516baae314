"""neighbor_attention and grouped_linear whose saved tensors a hook lays out anew: the same gradients, whatever their
strides; another shape, type or device is refused before anything is launched."""
import pytest
import torch

from dynamis_amd import dynamis_state as ds

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


def _attention(dtype):
    """A step over q, k and v that are views of one product, and its leaves."""
    g = torch.Generator("cuda").manual_seed(1)
    new = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    src = torch.randint(0, 40, (300,), device="cuda", generator=g)
    dst = torch.sort(torch.randint(0, 30, (300,), device="cuda", generator=g)).values
    plan = ds.neighbor_plan(torch.stack([src, dst]), 40, num_targets=30, distances=4 * torch.rand(300, device="cuda", generator=g),
                            boundaries=torch.tensor([1.0, 2.0, 3.0], device="cuda"))
    qkv = new(40, 8 * 16).to(dtype).requires_grad_(True)
    table = new(4, 4).requires_grad_(True)
    grad = new(30, 4, 16).to(dtype)

    def step():
        q, k, v = qkv[:30, :64].unflatten(1, (4, 16)), qkv[:, 64:96].unflatten(1, (2, 16)), qkv[:, 96:].unflatten(1, (2, 16))
        return torch.autograd.grad(ds.neighbor_attention(q, k, v, plan, table), [qkv, table], grad)

    return step


def _grouped(dtype):
    g = torch.Generator("cuda").manual_seed(2)
    new = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    leaves = [t.requires_grad_(True) for t in (new(50, 24), new(3, 40, 24), new(3, 40))]
    sizes, grad = torch.tensor([20, 0, 30], device="cuda"), new(50, 40)
    return lambda: torch.autograd.grad(ds.grouped_linear(leaves[0], leaves[1], sizes, leaves[2]), leaves, grad)


@TYPES
@pytest.mark.parametrize("make", [_attention, _grouped])
def test_laid_out_anew(cuda, make, dtype):
    print(f"\n[case] {make.__name__} {dtype}", flush=True)
    step = make(dtype)
    want = step()
    turned = lambda t: t.movedim(0, -1).contiguous().movedim(-1, 0)  # noqa: E731
    apart = lambda t: torch.stack([t, t], -1)[..., 0]  # noqa: E731
    wide = lambda t: torch.cat([t, t], -1)[..., :t.size(-1)]  # noqa: E731
    for back in (lambda t: t.contiguous(), lambda t: t.clone(memory_format=torch.contiguous_format), turned, apart, wide):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
            assert all(torch.equal(a, b) for a, b in zip(step(), want))
    with torch.autograd.graph.save_on_cpu():
        assert all(torch.equal(a, b) for a, b in zip(step(), want))


@TYPES
@pytest.mark.parametrize("make", [_attention, _grouped])
def test_another_make_is_refused(cuda, make, dtype):
    step = make(dtype)
    for back in (lambda t: t[:-1], lambda t: t.double(), lambda t: t.cpu(), lambda t: t.flatten()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
            with pytest.raises(RuntimeError, match="a saved tensor came back"):
                step()

"""A batch with more atoms than a launch of a wave each holds along one axis."""
import pytest
import torch

from dynamis_amd.dynamis_state import dynamis_state_impl as impl

pytestmark = pytest.mark.gpu


def test_a_batch_of_more_than_2_to_the_26_atoms(cuda):
    """1,048,576 chains of 65 atoms, one apart, each atom next to one or two others."""
    structures, atoms = 2 ** 20, 65
    print(f"\n[case] {structures * atoms} atoms", flush=True)
    chain = torch.zeros(atoms, 3, device="cuda")
    chain[:, 0] = torch.arange(atoms)
    pos = chain.repeat(structures, 1)
    cells = (torch.eye(3, device="cuda") * 200.0).expand(structures, 3, 3).contiguous()
    natoms = torch.full((structures,), atoms, device="cuda")
    edges, offsets, per_structure = impl.build_batch(pos, cells, natoms, torch.tensor([False] * 3), 1.5)
    assert (per_structure == 2 * (atoms - 1)).all()
    assert edges.shape == (2, 2 * (atoms - 1) * structures) and not offsets.any()
    one = torch.tensor([(s, t) for t in range(atoms) for s in (t - 1, t + 1) if 0 <= s < atoms], device="cuda").T
    for first in (0, 1000, structures - 1000):
        at = torch.arange(first, first + 1000, device="cuda")
        want = (one[:, None, :] + atoms * at[None, :, None]).flatten(1)
        assert torch.equal(edges[:, one.size(1) * first:one.size(1) * (first + 1000)], want)

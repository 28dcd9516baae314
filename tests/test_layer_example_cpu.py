"""The batches of examples/structure_energies.py, which need no GPU."""
import importlib.util
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    path = os.path.join(ROOT, "examples", "structure_energies.py")
    spec = importlib.util.spec_from_file_location("structure_energies", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_a_lattice_has_a_site_for_each_atom(example, monkeypatch):
    """Structures of every number of atoms up to 1,100, 217 and 344 (cubes and one) among them."""
    numbers = torch.arange(2, 1101)
    monkeypatch.setattr(example.torch, "randint", lambda lo, hi, size, generator=None, keep=torch.randint:
                        numbers if size == (len(numbers),) else keep(lo, hi, size, generator=generator))
    batch = example.make_batch(len(numbers), 1100, device="cpu")
    assert torch.equal(batch.natoms, numbers) and len(batch.pos) == len(batch.species) == int(numbers.sum())
    for n, cell, pos in zip(numbers.tolist(), batch.cell, batch.pos.split(numbers.tolist())):
        side = float(cell[0, 0])
        assert (pos >= 0).all() and (pos < side).all()
        assert abs(side ** 3 / n - 10) < 1e-3 * 10  # 0.1 atoms per cubic Angstrom

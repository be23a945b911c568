"""The example of the operators on nodes together: examples/structure_transformer.py."""

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


def _example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "structure_transformer.py")
    spec = importlib.util.spec_from_file_location("structure_transformer", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_whole_structures_and_atom_by_atom_agree():
    ex = _example()
    torch.manual_seed(0)
    model = ex.StructureTransformer(layers=2).cuda().eval()
    batch = ex.random_structures([5, 1, 17, 30, 2], species=8, cutoff=model.cutoff, seed=3)
    with torch.no_grad():
        whole = model(*batch)
    one_by_one = ex.read_one_by_one(model, *batch)
    # the same sums in float32 in another order: some 1e3 rounding errors of 6e-8 of scores of order one
    assert (whole - one_by_one).abs().max() <= 1e-4 * max(1.0, whole.abs().max().item())


def test_training_learns_and_structures_do_not_mix():
    ex = _example()
    torch.manual_seed(0)
    model = ex.StructureTransformer(channels=32, heads=4, key_heads=1, layers=1).cuda()
    batch = ex.random_structures([12, 20, 3], species=4, cutoff=model.cutoff, seed=5)
    optimizer = torch.optim.AdamW(model.parameters(), lr=1e-2)
    losses = []
    for _ in range(40):
        optimizer.zero_grad()
        loss = model.loss(*batch)
        loss.backward()
        assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
        optimizer.step()
        losses.append(loss.item())
    assert sum(losses[-5:]) < 0.8 * sum(losses[:5])
    model.eval()
    with torch.no_grad():
        before = model(*batch)
        species, xyz, ptr, rows, cols = batch
        xyz = xyz.clone()
        xyz[12:32] += 0.1 * torch.randn_like(xyz[12:32])
        after = model(species, xyz, ptr, rows, cols)
    assert torch.equal(before[:12], after[:12]) and torch.equal(before[32:], after[32:])
    assert not torch.equal(before[12:32], after[12:32])

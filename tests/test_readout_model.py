"""The readout ops together: a RelationalGNN with an ObjectReadout on top, trained by Muon."""

from __future__ import annotations

import pytest
import torch

from relmo_amd.consumers import RelationalGNN, synthetic_c4
from relmo_amd.readout import Muon, ObjectReadout, readout_train_step

GRAPHS, OBJECTS = 6, 200


def _setup(device, dtype):
    torch.manual_seed(0)
    batch = synthetic_c4("cpu", seed=1, num_graphs=GRAPHS)
    batch.atoms = {p: a.to(device) for p, a in batch.atoms.items()}
    model = RelationalGNN(16, 2, batch.relations, 0).to(device=device, dtype=dtype)
    readout = ObjectReadout(16, heads=4, kv_heads=2, queries=3).to(device=device, dtype=dtype)
    # the objects start from nothing in the network: the atoms' routing tells them apart
    offsets = torch.arange(GRAPHS + 1, device=device) * OBJECTS
    targets = torch.randn(GRAPHS, 3, generator=torch.Generator().manual_seed(4)).to(device=device, dtype=dtype)
    params = [*model.parameters(), *readout.parameters()]
    matrices = [p for p in params if p.dim() == 2 and min(p.shape) > 1]
    others = [p for p in params if not (p.dim() == 2 and min(p.shape) > 1)]
    optimisers = [Muon(matrices, lr=0.02), torch.optim.SGD(others, lr=0.05)]
    return model, readout, optimisers, batch, model.routing(batch), readout.plan(offsets), targets


def _losses(device, dtype, steps=12):
    setup = _setup(device, dtype)
    return [float(readout_train_step(*setup)) for _ in range(steps)], setup


def test_training_on_the_cpu_lowers_the_loss() -> None:
    losses, _ = _losses("cpu", torch.float64, steps=50)  # at a constant rate the loss falls in a band
    assert min(losses) < 0.7 * losses[0]


def test_muon_takes_matrices_only() -> None:
    with pytest.raises(ValueError, match="matrices only"):
        Muon([torch.nn.Parameter(torch.zeros(3))])


def test_muon_steps_past_empty_matrices() -> None:
    """A relation without features: nothing to step, and the others are stepped as without it."""

    def params():
        return [torch.nn.Parameter(torch.ones(*s)) for s in ((3, 0), (0, 4), (4, 3))]

    some, alone = params(), params()[2:]
    for group in (some, alone):
        for p in group:
            p.grad = torch.arange(float(p.numel())).view(p.shape) + 1.0
        Muon(group).step()
    assert torch.equal(some[2], alone[0]) and not torch.equal(some[2], torch.ones(4, 3))


def test_readout_ignores_masked_objects_and_empty_graphs() -> None:
    torch.manual_seed(1)
    readout = ObjectReadout(8, heads=2, queries=2).double()
    offsets = torch.tensor([0, 3, 3, 7])
    x = torch.randn(7, 8, dtype=torch.float64)
    mask = torch.tensor([True, False, True, True, True, False, True])
    values = readout(x, readout.plan(offsets), mask)
    kept = torch.tensor([0, 2, 2, 5])
    torch.testing.assert_close(values, readout(x[mask], readout.plan(kept)))
    assert values.shape == (3, 2)


def _autocast_step(device):
    """Values and gradients of a float32 readout, plain and under autocast to bfloat16."""

    torch.manual_seed(2)
    readout = ObjectReadout(32, heads=4, kv_heads=2, queries=3).to(device)
    x = torch.randn(20, 32, generator=torch.Generator().manual_seed(3)).to(device)
    plan = readout.plan(torch.tensor([0, 7, 7, 20], device=device))
    results = []
    for enabled in (False, True):
        states = x.clone().requires_grad_()
        with torch.autocast(device, dtype=torch.bfloat16, enabled=enabled):
            values = readout(states, plan)
        grads = torch.autograd.grad(values.float().square().sum(), (states, *readout.parameters()))
        results.append((values.detach(), grads))
    (want, want_grads), (got, grads) = results
    assert got.isfinite().all() and [g.dtype for g in grads] == [g.dtype for g in want_grads]
    # a few roundings of 2^-8 on a path of sums of 32 terms
    assert float((got.float() - want).abs().max()) <= 0.1 * float(want.abs().max()) + 0.02
    for a, b in zip(grads, want_grads):
        assert float((a - b).norm()) <= 0.15 * float(b.norm()) + 1e-3


def test_autocast_on_the_cpu() -> None:
    _autocast_step("cpu")


@pytest.mark.gpu
def test_autocast_on_the_gpu() -> None:
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")
    _autocast_step("cuda")


@pytest.mark.gpu
def test_training_on_the_gpu_follows_the_64_bit_steps() -> None:
    """The same steps in float32 on the GPU and in float64 on the CPU: equal losses up to what float32 gradients and
    the orthogonalised steps' growth of their error (below 1e-4 of a step) make of 12 steps of 0.02."""

    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")
    torch.manual_seed(0)
    want, cpu = _losses("cpu", torch.float64)
    setup = _setup("cuda", torch.float32)
    with torch.no_grad():  # the same start
        fresh = _setup("cpu", torch.float64)
        for a, b in zip((*setup[0].parameters(), *setup[1].parameters()), (*fresh[0].parameters(), *fresh[1].parameters())):
            a.copy_(b)
    got = [float(readout_train_step(*setup)) for _ in range(12)]
    assert got[-1] < got[0]
    for a, b in zip(got, want):
        assert abs(a - b) <= 2e-2 * max(abs(b), 1e-3) + 1e-3, (got, want)

"""GPU tests of calls that the readout ops have no answer for: they raise, and do not return something else."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")


@pytest.mark.parametrize("which", [0, 1, 2])
def test_forward_mode_derivatives_are_refused(which) -> None:
    """A tangent on any argument: an op without a forward-mode formula raises, as the message-passing ops do."""
    from relmo_amd import mp

    o = torch.tensor([0, 4, 8], device=DEV)
    plan = mp.attention_plan(o, o, 2)
    x = [torch.randn(8, 2, 16, device=DEV) for _ in range(3)]
    rows = [torch.randn(8, 16, device=DEV), torch.randn(8, 16, device=DEV), torch.rand(16, device=DEV)]
    with fwd.dual_level():
        duals = [fwd.make_dual(t, torch.ones_like(t)) if i == which else t for i, t in enumerate(x)]
        assert not any(t.requires_grad for t in duals)
        norm = [fwd.make_dual(t, torch.ones_like(t)) if i == which else t for i, t in enumerate(rows)]
        calls = [lambda: mp.cross_attention(*duals, plan), lambda: mp.add_rms_norm(*norm), lambda: mp.add_rms_norm_fp8(*norm),
                 lambda: mp.orthogonalise([duals[0][0], duals[1][0], duals[2][0]])]
        if which != 1:
            calls.append(lambda: mp.rms_norm(norm[0], norm[2]))
            calls.append(lambda: mp.add_rms_norm(norm[0], None, norm[2]))
        for call in calls:
            with pytest.raises(RuntimeError, match="forward"):
                call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward"):  # which does not turn forward mode off
            mp.cross_attention(*duals, plan)
    # and none of it outside of a level
    mp.cross_attention(*x, plan), mp.add_rms_norm(*rows), mp.orthogonalise(x[0][0])


def test_forward_mode_over_the_backward_is_refused() -> None:
    from relmo_amd import mp

    o = torch.tensor([0, 4, 8], device=DEV)
    plan = mp.attention_plan(o, o, 2)
    x = torch.randn(8, 2, 16, device=DEV, requires_grad=True)
    w = torch.rand(16, device=DEV)
    for out in (mp.cross_attention(x, x, x, plan), mp.rms_norm(x, w), mp.add_rms_norm(x, x, w)[0]):
        with fwd.dual_level():
            grad = fwd.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(RuntimeError, match="forward"):
                torch.autograd.grad(out, x, grad, retain_graph=True)
        torch.autograd.grad(out, x, torch.ones_like(out))


def test_steps_past_32_bits_are_refused() -> None:
    from relmo_amd import mp

    for steps in (5 - (1 << 32), 5 + (1 << 32), -(1 << 62)):
        with pytest.raises(RuntimeError, match="steps"):
            mp.orthogonalise(torch.ones(4, 8, device=DEV), steps=steps)

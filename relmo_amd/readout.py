"""A readout over the object states of a relational batch and the step that trains it.

What runs the readout ops together: :class:`ObjectReadout` attends with a few queries per
graph to the object states that a RelationalGNN leaves (``mp.cross_attention`` between
``mp.rms_norm`` and ``mp.add_rms_norm``) and gives values per query; :class:`Muon` steps
matrices by their orthogonalised momentum (``mp.orthogonalise``), all of them at once.

    model, readout = RelationalGNN(128, 10, relations, 0), ObjectReadout(128, heads=4)
    step = Muon([p for p in (*model.parameters(), *readout.parameters()) if p.dim() == 2], lr=0.02)
    plan = readout.plan(object_offsets)                    # once per batch
    values = readout(model(batch, routing), plan)          # [graphs, queries]
"""

from __future__ import annotations

import torch
from torch import Tensor, nn

from . import mp


class ObjectReadout(nn.Module):
    """``queries`` learned queries per graph over the graph's object states, in a block with a residual
    stream: ``h = r + attention(norm(r), norm(x))``, then a value per query from ``norm(h)``."""

    def __init__(self, embedding_size: int, heads: int = 4, kv_heads: int | None = None, queries: int = 1):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if embedding_size % heads != 0 or heads % kv_heads != 0:
            raise ValueError("embedding_size must be a multiple of heads, and heads of kv_heads")
        self.heads, self.kv_heads, self.queries = heads, kv_heads, queries
        self.dim = embedding_size // heads
        self.query = nn.Parameter(torch.randn(queries, embedding_size))
        self.object_norm = nn.Parameter(torch.ones(embedding_size))
        self.query_norm = nn.Parameter(torch.ones(embedding_size))
        self.out_norm = nn.Parameter(torch.ones(embedding_size))
        self.to_q = nn.Linear(embedding_size, embedding_size, bias=False)
        self.to_kv = nn.Linear(embedding_size, 2 * kv_heads * self.dim, bias=False)
        self.out = nn.Linear(embedding_size, embedding_size, bias=False)
        self.value = nn.Linear(embedding_size, 1)

    def plan(self, object_offsets: Tensor):
        """The attention's plan of a batch (graph ``b`` holds the objects ``object_offsets[b]:object_offsets[b +
        1]``): made once and kept while the batch is used."""

        graphs = object_offsets.numel() - 1
        q_offsets = torch.arange(graphs + 1, device=object_offsets.device) * self.queries
        return mp.attention_plan(q_offsets, object_offsets, self.heads, self.kv_heads)

    def forward(self, x: Tensor, plan, object_mask: Tensor | None = None) -> Tensor:
        """Values [graphs, queries] from object states ``x`` [objects, embedding_size]; objects whose
        ``object_mask`` is False are not read."""

        graphs = plan.q_offsets.numel() - 1
        kv = self.to_kv(mp.rms_norm(x, self.object_norm)).view(-1, 2, self.kv_heads, self.dim)
        r = self.query.repeat(graphs, 1)
        q = self.to_q(mp.rms_norm(self.query, self.query_norm)).repeat(graphs, 1).view(-1, self.heads, self.dim)
        read = mp.cross_attention(q, kv[:, 0], kv[:, 1], plan, key_mask=object_mask)
        # under autocast the projections are 16-bit; the residual stream stays in its parameters' type
        y, _h = mp.add_rms_norm(self.out(read.flatten(1)).to(r.dtype), r, self.out_norm)
        return self.value(y).view(graphs, self.queries)


class Muon(torch.optim.Optimizer):
    """Matrices stepped along their orthogonalised momentum (Nesterov): ``p -= lr * sqrt(max(1, rows /
    cols)) * orthogonalise(g + momentum * m)``, ``m = momentum * m + g``.  Every parameter is a matrix; biases, norms
    and single columns go to another optimiser."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, steps: int = 5):
        super().__init__(params, {"lr": lr, "momentum": momentum, "steps": steps})
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() != 2:
                    raise ValueError("Muon steps matrices only")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            kinds: dict[tuple, list[Tensor]] = {}
            for p in group["params"]:
                if p.grad is not None:
                    kinds.setdefault((p.dtype, p.device), []).append(p)
            for params in kinds.values():
                grads = [p.grad for p in params]
                for p, g in zip(params, grads):
                    if "momentum" not in self.state[p]:
                        self.state[p]["momentum"] = torch.zeros_like(g)
                momenta = [self.state[p]["momentum"] for p in params]
                torch._foreach_mul_(momenta, group["momentum"])
                torch._foreach_add_(momenta, grads)
                updates = torch._foreach_add(grads, momenta, alpha=group["momentum"])
                results = mp.orthogonalise(updates, steps=group["steps"])
                rates = [-group["lr"] * max(1.0, p.size(0) / max(1, p.size(1))) ** 0.5 for p in params]
                torch._foreach_mul_(results, rates)
                torch._foreach_add_(params, results)
        return loss


def readout_train_step(model: nn.Module, readout: ObjectReadout, optimisers, batch, routing, plan, targets: Tensor) -> Tensor:
    """One step on the squared error of the readout's values against ``targets`` [graphs, queries]."""

    for o in optimisers:
        o.zero_grad(set_to_none=True)
    with mp.plan_scope():
        loss = (readout(model(batch, routing), plan) - targets).square().mean()
        loss.backward()
    for o in optimisers:
        o.step()
    return loss.detach()


__all__ = ["Muon", "ObjectReadout", "readout_train_step"]

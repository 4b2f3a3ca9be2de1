"""A retriever's catalogue, its answers and its training, on one GPU.

    python quiver-ae_amd/examples/dense_retrieval.py [--rows N] [--queries N] [--steps N]

1. A catalogue of normalised float vectors (the benchmark's mixture) is kept in 8
   bits and scored exhaustively: each query's distribution over all rows, the log
   probability of the row it was made from, how sure it is (entropy), its ten best
   rows, and how often the exact nearest row is among them.  The same in 4 bits.
2. A linear map of distorted queries is trained with the contrastive loss over a
   batch and the catalogue's hardest rows, by autograd through ``log_probs``.
3. The same with a tower that ends in a layer norm, whose weight and bias are
   trained too.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import quiver  # noqa: E402
from quiver import scoring  # noqa: E402

TEMPERATURE = 0.05


def answers(catalogue: scoring.DenseCatalogue, vectors: torch.Tensor, queries: torch.Tensor,
            targets: torch.Tensor) -> dict:
    """The queries' distributions over the catalogue."""
    r = catalogue.log_probs(queries, targets, top_k=10, temperature=TEMPERATURE)
    nearest = (queries @ vectors.T).argmax(1)
    found = (r.top_ids.long() == nearest[:, None]).any(1).float().mean().item()
    return {"log_prob": r.target.mean().item(), "entropy": r.entropy.mean().item(), "recall": found}


def train(catalogue: scoring.DenseCatalogue, vectors: torch.Tensor, queries: torch.Tensor, targets: torch.Tensor,
          steps: int, rate: float = 0.02) -> list[float]:
    """Contrastive losses of the steps: every row of the batch and the catalogue's eight hardest rows against each query."""
    n, dim = queries.shape
    weight = torch.eye(dim, device=queries.device).requires_grad_()
    optimizer = torch.optim.Adam([weight], lr=rate)
    labels = torch.arange(n, dtype=torch.int32, device=queries.device)
    losses = []
    for _ in range(steps):
        mapped = torch.nn.functional.normalize(queries @ weight, dim=1)
        hard = catalogue.log_probs(mapped.detach(), top_k=8, temperature=TEMPERATURE).top_ids.long()
        in_batch = mapped @ vectors[targets.long()].T
        others = (mapped[:, None, :] * vectors[hard]).sum(2)
        others = others.masked_fill(hard == targets.long()[:, None], -torch.inf)  # the answer itself is no negative
        logits = torch.cat([in_batch, others], 1)
        loss = -scoring.log_probs(logits, labels, temperature=TEMPERATURE).target.mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    return losses


def tower_loss(queries: torch.Tensor, vectors: torch.Tensor, labels: torch.Tensor, weight: torch.Tensor,
               gain: torch.Tensor, offset: torch.Tensor) -> torch.Tensor:
    """The contrastive loss of queries through a linear map and a layer norm, every row of the batch against each."""
    hidden = scoring.layer_norm(queries @ weight, gain, offset)
    logits = hidden @ vectors.T
    # a normalised row has the length sqrt(dim): the temperature grows with it
    return -scoring.log_probs(logits, labels, temperature=TEMPERATURE * queries.shape[1] ** 0.5).target.mean()


def train_tower(vectors: torch.Tensor, queries: torch.Tensor, targets: torch.Tensor, steps: int,
                rate: float = 0.02) -> list[float]:
    """Contrastive losses of the steps."""
    n, dim = queries.shape
    leaves = [torch.eye(dim, device=queries.device), torch.ones(dim, device=queries.device),
              torch.zeros(dim, device=queries.device)]
    for leaf in leaves:
        leaf.requires_grad_()
    optimizer = torch.optim.Adam(leaves, lr=rate)
    labels = torch.arange(n, dtype=torch.int32, device=queries.device)
    answers_of = vectors[targets.long()]
    losses = []
    for _ in range(steps):
        loss = tower_loss(queries, answers_of, labels, *leaves)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    return losses


def main(rows: int = 100_000, queries: int = 512, steps: int = 30, dim: int = 96) -> dict:
    base = torch.from_numpy(quiver.mixture(rows, dim, data_type="float", num_centers=max(16, rows // 64), sigma=1.0,
                                           seed=5)).cuda()
    g = torch.Generator(device="cuda").manual_seed(1)
    targets = torch.randperm(rows, generator=g, device="cuda")[:queries].to(torch.int32)
    near = base[targets.long()] + 0.03 * torch.randn((queries, dim), generator=g, device="cuda")
    near = torch.nn.functional.normalize(near, dim=1)
    catalogue = scoring.DenseCatalogue(base)
    result = answers(catalogue, base, near, targets)
    print(f"{queries} queries over {rows} rows: log probability of the answer {result['log_prob']:.3f}, "
          f"entropy {result['entropy']:.3f}, nearest row among the ten best {result['recall']:.3f}")
    short = answers(scoring.DenseCatalogue(base, bits=4), base, near, targets)
    print(f"in 4 bits: log probability {short['log_prob']:.3f}, entropy {short['entropy']:.3f}, nearest row among the ten "
          f"best {short['recall']:.3f}")
    distortion = torch.eye(dim, device="cuda") + 1.5 * torch.randn((dim, dim), generator=g, device="cuda") / dim ** 0.5
    losses = train(catalogue, base, near @ distortion, targets, steps)
    print(f"contrastive loss over {steps} steps: {losses[0]:.4f} -> {losses[-1]:.4f}")
    tower = train_tower(base, near @ distortion, targets, steps)
    print(f"with a layer norm over {steps} steps: {tower[0]:.4f} -> {tower[-1]:.4f}")
    return {**result, "losses": losses, "in_4_bits": short, "tower_losses": tower}


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--rows", type=int, default=100_000)
    parser.add_argument("--queries", type=int, default=512)
    parser.add_argument("--steps", type=int, default=30)
    args = parser.parse_args()
    main(args.rows, args.queries, args.steps)

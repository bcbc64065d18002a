"""Train a small potential with the training blocks: element embedding, gated feed-forward and
irreps dropout together, next to the stock layers.

    python examples/training_blocks.py [--steps 20] [--molecules 32] [--dropout 0.05]

Seeded random-walk molecules with random energy labels; prints the loss of the first and last
step and the time per step of both models.
"""

import argparse
import copy
import os
import statistics
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from flashcart_b200.model.flashcart import FlashCartPotential  # noqa: E402
from flashcart_b200.nn.blocks import use_training_blocks  # noqa: E402
from flashcart_b200.ops import check_device_status  # noqa: E402
from flashcart_b200.training import ELEMENTS, batch_graph, make_optimizer, synthetic_molecules  # noqa: E402


def train(model, graph, labels, steps):
    """Energy-only training; (first loss, last loss, median milliseconds per step)."""
    main, aux = make_optimizer(model, lr=2e-3)
    losses, times = [], []
    for _ in range(steps):
        torch.cuda.synchronize()
        start = time.perf_counter()
        for opt in (main, *aux):
            opt.zero_grad(set_to_none=True)
        energy = torch.zeros_like(labels).index_add(0, graph["batch"], model(graph))
        loss = ((energy - labels) / graph["n_atoms"]).square().mean()
        loss.backward()
        for opt in (main, *aux):
            opt.step()
        torch.cuda.synchronize()
        times.append((time.perf_counter() - start) * 1e3)
        losses.append(loss.detach())
    return losses[0].item(), losses[-1].item(), statistics.median(times)


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--molecules", type=int, default=32)
    ap.add_argument("--channels", type=int, default=64)
    ap.add_argument("--dropout", type=float, default=0.05)
    args = ap.parse_args()
    device = torch.device("cuda")
    graph = batch_graph(synthetic_molecules(args.molecules), 5.0, device)
    torch.manual_seed(0)
    stock = FlashCartPotential(ELEMENTS, r_max=5.0, n_hidden_feats=args.channels, l_max_hidden_feats=2,
                               l_max_edge_attrs=2, n_interactions=2, correlation=2, nonlinearity=True,
                               layer_norm=True, element_agnostic_interaction=False,
                               element_agnostic_product=False, avg_neighbors=20.0).to(device)
    blocks = use_training_blocks(copy.deepcopy(stock), dropout=args.dropout)
    labels = torch.randn(args.molecules, device=device) * graph["n_atoms"]
    for name, model in (("stock layers", stock), (f"training blocks, dropout {args.dropout}", blocks)):
        first, last, ms = train(model, graph, labels, args.steps)
        print(f"{name}: loss {first:.4f} -> {last:.4f}, {ms:.1f} ms per step")
    check_device_status(device)


if __name__ == "__main__":
    main()

"""A move-sequence policy trained with the operators of ``alphazero_b200.ops``:
an embedding of the last moves of a game, residual layers, and the cross
entropy over the moves, each forward and backward pass by this package's
kernels.

    python -m alphazero_b200.move_model [--board 9] [--steps 200]
    python -m alphazero_b200.move_model --records DIR     (self-play records)

Without records it learns the moves that the evaluation engine prefers (a
seeded network, evaluated by ``CudaEngine``) in seeded random positions; with
them it learns the search's moves (record files of ``selfplay_cuda --records``
in the reference's format, src/main_selfplay.cpp:17-32; each target is drawn
from the record's policy, so the gradient's expectation is that of the whole
distribution).  Weights are kept in fp32 and copied to bf16 for each step.
"""
from __future__ import annotations

import argparse
import glob
import math
import os

import numpy as np
import torch

from . import ops

HISTORY = 8  # boards in the input planes, hence one move fewer


def tokens_from_planes(planes, board: int) -> np.ndarray:
    """[n, 17 * board^2] encoded positions -> [n, 7] the last moves, latest
    first: a point, board^2 for a pass, -1 before the first stone.  The move
    between two boards of the history is the point that gained a stone."""
    p = np.asarray(planes, np.float32).reshape(-1, 17, board * board)
    stones = p[:, :HISTORY] + p[:, HISTORY:2 * HISTORY] > 0
    gained = stones[:, :-1] & ~stones[:, 1:]
    moves = np.where(gained.any(2), gained.argmax(2), board * board)
    return np.where(stones[:, :-1].any(2), moves, -1).astype(np.int64)


def read_records(directory: str, board: int):
    """(planes, policies) of every record file in a directory."""
    planes, policies = [], []
    for path in sorted(glob.glob(os.path.join(directory, "*.bin"))):
        raw = np.fromfile(path, np.uint8)
        count, at = int(raw[:4].view("<i4")[0]), 4
        for _ in range(count):
            for out in (planes, policies):
                size = int(raw[at:at + 4].view("<i4")[0])
                out.append(raw[at + 4:at + 4 + 4 * size].view("<f4"))
                at += 4 + 4 * size
            at += 4  # the value
    if not planes:
        raise FileNotFoundError(f"no records in {directory}")
    if policies[0].size != board * board + 1:
        raise ValueError(f"records are not of a {board}x{board} board")
    return np.stack(planes), np.stack(policies)


class MoveModel:
    """logits = head(blocks(in(embed(moves)))), a block being
    h + gelu(h W^T + b)."""

    def __init__(self, board: int, dim: int = 64, hidden: int = 256, blocks: int = 2, seed: int = 0,
                 device: str = "cuda"):
        self.moves = board * board + 1
        self.scale = math.sqrt(dim)
        g = torch.Generator().manual_seed(seed)

        def normal(rows, cols, gain=1.0):
            return (torch.randn(rows, cols, generator=g) * gain * cols ** -0.5).to(device)

        wide = (HISTORY - 1) * dim
        self.weights = {"table": normal(self.moves, dim), "in.w": normal(hidden, wide),
                        "in.b": torch.zeros(hidden, device=device), "head.w": normal(self.moves, hidden),
                        "head.b": torch.zeros(self.moves, device=device)}
        self.blocks = blocks
        for i in range(blocks):
            self.weights[f"{i}.w"] = normal(hidden, hidden, 0.5)
            self.weights[f"{i}.b"] = torch.zeros(hidden, device=device)

    def half(self):
        return {k: v.to(torch.bfloat16) for k, v in self.weights.items()}

    def _features(self, p, tokens, keep: bool):
        """(h, what the backward pass needs)."""
        e = ops.embed(tokens, p["table"], self.scale).flatten(1)
        out = ops.linear(e, p["in.w"], p["in.b"], activation="gelu", keep_preactivation=keep)
        h, z = out if keep else (out, None)
        kept = [(e, z)]
        for i in range(self.blocks):
            out = ops.linear(h, p[f"{i}.w"], p[f"{i}.b"], residual=h, activation="gelu",
                             keep_preactivation=keep)
            nxt, z = out if keep else (out, None)
            kept.append((h, z))
            h = nxt
        return h, kept

    def gradients(self, tokens, targets):
        """(loss, gradient of every weight) of one batch."""
        p = self.half()
        h, kept = self._features(p, tokens, True)
        g = {}
        loss, _, dh, g["head.w"], g["head.b"] = ops.linear_cross_entropy_grad(h, p["head.w"], targets, p["head.b"])
        for i in reversed(range(self.blocks)):
            x, z = kept[i + 1]
            dx, g[f"{i}.w"], g[f"{i}.b"] = ops.linear_backward(dh, x, p[f"{i}.w"], z, "gelu")
            dh = dx + dh  # the residual's gradient
        e, z = kept[0]
        de, g["in.w"], g["in.b"] = ops.linear_backward(dh, e, p["in.w"], z, "gelu")
        g["table"] = ops.embed_backward(de.view(*tokens.shape, -1), tokens, self.moves, self.scale)
        return loss, g

    def step(self, tokens, targets, rate: float):
        """One step of gradient descent; the loss before it, on the device."""
        loss, g = self.gradients(tokens, targets)
        for k, v in self.weights.items():
            v.add_(g[k].float(), alpha=-rate)
        return loss

    def score(self, tokens, targets):
        """(mean, per-row) losses, without gradients."""
        p = self.half()
        h, _ = self._features(p, tokens, False)
        return ops.linear_cross_entropy(h, p["head.w"], targets, p["head.b"])

    def logits(self, tokens):
        """[n, moves], for playing: one row is enough."""
        p = self.half()
        h, _ = self._features(p, tokens, False)
        return ops.linear(h, p["head.w"], p["head.b"])


def engine_targets(planes, board: int, seed: int) -> np.ndarray:
    """The move a seeded network prefers in each position, by CudaEngine."""
    from . import weights
    from .engine import CudaEngine

    e = CudaEngine(0, max_batch=min(1024, len(planes)))
    try:
        e.load_state_dict(weights.make_state_dict(board, 64, 2, seed=seed, variant="perturbed"))
        return e.forward(planes, want_logits=False)[0].argmax(1).astype(np.int64)
    finally:
        e.close()


def main(argv=None) -> float:
    a = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    a.add_argument("--board", type=int, default=9)
    a.add_argument("--positions", type=int, default=4096)
    a.add_argument("--batch", type=int, default=512)
    a.add_argument("--steps", type=int, default=200)
    a.add_argument("--rate", type=float, default=0.2)
    a.add_argument("--seed", type=int, default=0)
    a.add_argument("--records", help="directory of self-play record files")
    a = a.parse_args(argv)
    rng = np.random.default_rng(a.seed)
    if a.records:
        planes, policies = read_records(a.records, a.board)
    else:
        from . import host_lib

        planes = host_lib.random_positions(a.board, a.positions, a.seed + 1, 60 if a.board <= 9 else 250)
        targets = engine_targets(planes, a.board, a.seed)
    tokens = torch.from_numpy(tokens_from_planes(planes, a.board)).cuda()
    model = MoveModel(a.board, seed=a.seed)
    for i in range(a.steps):
        pick = rng.integers(0, len(planes), a.batch)
        if a.records:
            edges = policies[pick].cumsum(1)
            t = (edges < rng.random((a.batch, 1)) * edges[:, -1:]).sum(1).clip(max=model.moves - 1)
        else:
            t = targets[pick]
        loss = model.step(tokens[pick], torch.from_numpy(t).cuda(), a.rate)
        if i % 20 == 0 or i == a.steps - 1:
            print(f"step {i}: loss {loss.item():.4f}", flush=True)
    ops.synchronize()
    return loss.item()


if __name__ == "__main__":
    main()

"""Train a gated-recurrence stack with Muon, put its projections into 4 bits, and decode with it.

The task is delayed recall with forgetting: a token's target mixes the values of the document so far,
each weighted down by its age, so the states must carry information over many tokens and must be
dropped where a new document begins in a packed sequence.

    python examples/train_quantize_decode.py                  # on a GPU: the sm_100a kernels
    python examples/train_quantize_decode.py --device cpu --width 32 --steps 5

On a GPU the decode loop runs as a CUDA graph of one token: projections on 4-bit weights, states
updated in place.
"""

from __future__ import annotations

import argparse
import time
from pathlib import Path
import sys

import torch
from torch.nn import functional as F

if __package__ in (None, ""):
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from mamba3_b200 import GatedRecurrence, Muon, quantize_projections


def batch_of_documents(batch: int, length: int, width: int, generator: torch.Generator, device):
    """Packed documents: inputs, the flags of first tokens, and the targets."""
    x = torch.randn(batch, length, width, generator=generator)
    first = torch.rand(batch, length, generator=generator) < 0.02
    first[:, 0] = True
    decay = torch.linspace(0.5, 0.95, width)
    target, memory = torch.empty_like(x), torch.zeros(batch, width)
    for t in range(length):
        memory = torch.where(first[:, t, None], 0.0, memory) * decay + (1.0 - decay) * x[:, t]
        target[:, t] = memory
    return x.to(device), first.to(device), (target / target.std()).to(device)


def train(model: GatedRecurrence, args, generator) -> list[float]:
    matrices = [p for p in model.parameters() if p.dim() == 2]
    others = [p for p in model.parameters() if p.dim() != 2]
    optimizers = [Muon(matrices, lr=args.lr), torch.optim.AdamW(others, lr=args.lr, weight_decay=0.0)]
    device = matrices[0].device
    losses = []
    for step in range(args.steps):
        x, first, target = batch_of_documents(args.batch, args.length, args.width, generator, device)
        with torch.autocast(device.type, torch.bfloat16, enabled=device.type == "cuda"):
            y = model(x, reset=first)
        loss = F.mse_loss(y.float(), target)
        loss.backward()
        for optimizer in optimizers:
            optimizer.step()
            optimizer.zero_grad(set_to_none=True)
        losses.append(float(loss.detach()))
        if step % max(1, args.steps // 10) == 0:
            print(f"step {step:4d}  loss {losses[-1]:.4f}")
    return losses


class Decoder:
    """One token a call; on a GPU a captured graph with the states in place."""

    def __init__(self, model: GatedRecurrence, cache, example: torch.Tensor) -> None:
        self.model, self.cache = model, cache
        self.graph = None
        if example.is_cuda:
            self.x = example.clone()
            saved = [state.clone() for state in cache]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                model.step(self.x, cache, in_place=True)
            torch.cuda.current_stream().wait_stream(side)
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self.y, _ = model.step(self.x, cache, in_place=True)
            for state, was in zip(cache, saved):
                state.copy_(was)

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        if self.graph is None:
            y, _ = self.model.step(x, self.cache, in_place=True)
            return y
        self.x.copy_(x)
        self.graph.replay()
        return self.y.clone()


@torch.no_grad()
def decode(model: GatedRecurrence, x: torch.Tensor, prefix: int) -> tuple[torch.Tensor, float]:
    """The outputs of ``x [B, L, width]``: a prefilled prefix, then one token at a time."""
    y, cache = model.prefill(x[:, :prefix])
    decoder = Decoder(model, cache, x[:, :1])
    tokens = []
    if x.is_cuda:
        torch.cuda.synchronize()
    start = time.perf_counter()
    for t in range(prefix, x.shape[1]):
        tokens.append(decoder(x[:, t:t + 1]))
    if x.is_cuda:
        torch.cuda.synchronize()
    seconds = (time.perf_counter() - start) / max(1, len(tokens))
    return torch.cat([y, *tokens], dim=1), seconds


def main(argv=None) -> dict:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    parser.add_argument("--width", type=int, default=512)
    parser.add_argument("--depth", type=int, default=2)
    parser.add_argument("--batch", type=int, default=8)
    parser.add_argument("--length", type=int, default=256)
    parser.add_argument("--steps", type=int, default=100)
    parser.add_argument("--lr", type=float, default=0.02)
    parser.add_argument("--group-size", type=int, default=64, choices=(32, 64, 128))
    args = parser.parse_args(argv)

    device = torch.device(args.device)
    generator = torch.Generator().manual_seed(0)
    torch.manual_seed(0)
    model = GatedRecurrence(args.width, depth=args.depth).to(device)
    losses = train(model, args, generator)

    model = model.to(torch.bfloat16 if device.type == "cuda" else torch.float32).eval()
    dtype = next(model.parameters()).dtype
    x, _, _ = batch_of_documents(1, 64, args.width, generator, device)
    x = x.to(dtype)
    with torch.no_grad():
        reference = model(x)
    quantize_projections(model, group_size=args.group_size, zeros=True)
    with torch.no_grad():
        whole = model(x)
    tokens, seconds = decode(model, x, prefix=16)

    def off(a, b):
        return float((a.float() - b.float()).norm() / b.float().norm())

    result = dict(first_loss=losses[0], last_loss=losses[-1], quantization=off(whole, reference), decoding=off(tokens, whole),
                  seconds_per_token=seconds)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f}; 4-bit projections move the output by {result['quantization']:.3f} of its "
          f"size, decoding by tokens by {result['decoding']:.2g}; {seconds * 1e6:.0f} us a token")
    return result


if __name__ == "__main__":
    main()

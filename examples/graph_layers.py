"""A gated layer pair on an aggregated graph, trained and served in 8-bit blocks.

    python examples/graph_layers.py [--graph c2] [--hidden 256] [--classes 47] [--steps 20]

The sparse product aggregates INT8 features of a synthetic graph; its FP32 rows go through BlockLinear, a gated
block_activation and a second BlockLinear, all with their gradients; then the layers' weights are quantized once and
answer for single nodes with linear_blocks and activation_blocks. What a training step keeps for its backward pass is
a byte an element.
"""
import argparse
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch

from tcc_spmm_amd import convert_csr_to_sw32, synth_csr, synth_features
from tcc_spmm_amd.blocks import BlockLinear, activation_blocks, block_activation, linear_blocks
from tcc_spmm_amd.device import TorchDeviceMatrix, quantize_pack_features_int8


def aggregate(graph: str, features: int = 128) -> torch.Tensor:
    """Rows of the graph's sparse product with random features, scaled to a mean square of one."""
    csr = synth_csr(graph)
    matrix = TorchDeviceMatrix(convert_csr_to_sw32(csr.rows, csr.cols, csr), features)
    x = torch.from_numpy(synth_features(csr.cols, features, 1)).cuda()
    y = matrix.spmm(*quantize_pack_features_int8(x))
    return y / y.square().mean().sqrt()


class Layers(torch.nn.Module):
    def __init__(self, features: int, hidden: int, classes: int):
        super().__init__()
        self.up = BlockLinear(features, 2 * hidden)
        self.down = BlockLinear(hidden, classes)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.down(block_activation(self.up(x), "silu", gated=True))

    def server(self):
        """A function of rows of x with the weights as they are now, quantized once."""
        up, down = self.up.serving(), self.down.serving()

        def answer(x: torch.Tensor) -> torch.Tensor:
            h, _ = activation_blocks(linear_blocks(x, *up), "silu", gated=True, codes=None)
            return linear_blocks(h, *down)
        return answer


def train(rows: torch.Tensor, hidden: int, classes: int, steps: int):
    """(layers, loss of each step): labels are those of a random linear map of the rows."""
    torch.manual_seed(3)
    labels = (rows @ torch.randn(rows.shape[1], classes, device=rows.device)).argmax(1)
    layers = Layers(rows.shape[1], hidden, classes).cuda()
    optimizer = torch.optim.Adam(layers.parameters(), lr=3e-3)
    losses = []
    for _ in range(steps):
        optimizer.zero_grad()
        loss = torch.nn.functional.cross_entropy(layers(rows), labels)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return layers, [float(v) for v in losses]


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--graph", default="c2", help="synthetic graph: c1 to c5 or t<rows>_<degree>_<seed>")
    parser.add_argument("--hidden", type=int, default=256)
    parser.add_argument("--classes", type=int, default=47)
    parser.add_argument("--steps", type=int, default=20)
    args = parser.parse_args()
    rows = aggregate(args.graph)
    train(rows, args.hidden, args.classes, 2)  # first calls
    torch.cuda.synchronize()
    start = time.perf_counter()
    layers, losses = train(rows, args.hidden, args.classes, args.steps)
    torch.cuda.synchronize()
    took = time.perf_counter() - start
    print(f"{rows.shape[0]} nodes, {args.steps} steps of {took / args.steps * 1e3:.2f} ms: "
          f"loss {losses[0]:.3f} -> {losses[-1]:.3f}")
    answer, calls = layers.server(), 200
    answer(rows[:1])
    torch.cuda.synchronize()
    start = time.perf_counter()
    for i in range(calls):
        scores = answer(rows[i:i + 1])
    torch.cuda.synchronize()
    print(f"one node: {(time.perf_counter() - start) / calls * 1e6:.1f} us, class {int(scores.argmax())}")


if __name__ == "__main__":
    main()

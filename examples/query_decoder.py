"""A decoder over a feature pyramid, trained for some steps on synthetic data.

The parts as a detector's decoder uses them:

  PyramidGroupNorm   normalises each level of a backbone's maps and flattens
                     them into the values that the queries sample
  AxialRotary        turns queries and keys of the queries' self-attention by
                     their reference points, which are learned
  MSDA2D             lets each query sample the pyramid around its reference
                     point
  AdamW              updates bf16 parameters over fp32 master copies, with
                     moments in 8 bits

    python examples/query_decoder.py --steps 200
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from msda_triton_b200 import MSDA2D, AdamW, AxialRotary, PyramidGroupNorm  # noqa: E402


class DecoderLayer(nn.Module):
    """Self-attention of the queries with rotary positions, then sampling of the pyramid."""

    def __init__(self, embed: int, heads: int, levels: int, points: int) -> None:
        super().__init__()
        self.heads = heads
        self.qkv = nn.Linear(embed, 3 * embed)
        self.out = nn.Linear(embed, embed)
        self.rotary = AxialRotary(embed // heads, num_axes=2)
        self.sample = MSDA2D(embed, heads, levels, points, dropout=0.0, batch_first=True)
        self.norms = nn.ModuleList(nn.LayerNorm(embed) for _ in range(3))
        self.ffn = nn.Sequential(nn.Linear(embed, 4 * embed), nn.GELU(), nn.Linear(4 * embed, embed))

    def forward(self, x, positions, reference, value, shapes):
        B, Q, E = x.shape
        qkv = self.qkv(self.norms[0](x)).view(B, Q, 3 * self.heads, E // self.heads)
        q, k, v = qkv.split(self.heads, dim=2)
        q, k = self.rotary(q, k, positions)  # read in place out of the one projection
        a = nn.functional.scaled_dot_product_attention(*(t.transpose(1, 2) for t in (q, k, v)))
        x = x + self.out(a.transpose(1, 2).reshape(B, Q, E))
        x = self.sample(self.norms[1](x), value=value, identity=x, reference_points=reference,
                        spatial_shapes=shapes)
        return x + self.ffn(self.norms[2](x))


class QueryDecoder(nn.Module):
    """Backbone maps (B, C, H, W), finest first, to one output per query."""

    def __init__(self, shapes, channels: int = 64, heads: int = 4, queries: int = 100,
                 layers: int = 2, points: int = 4, outputs: int = 8) -> None:
        super().__init__()
        self.register_buffer("shapes", torch.tensor(shapes), persistent=False)
        self.host_shapes = torch.tensor(shapes)
        self.norm = PyramidGroupNorm(8, channels, num_levels=len(shapes), activation="silu")
        self.queries = nn.Parameter(torch.randn(queries, channels) * 0.2)
        self.places = nn.Parameter(torch.randn(queries, 2))  # of the reference points, as logits
        self.layers = nn.ModuleList(DecoderLayer(channels, heads, len(shapes), points)
                                    for _ in range(layers))
        for layer in self.layers:
            layer.sample.init_weights()
        self.head = nn.Linear(channels, outputs)

    def forward(self, maps):
        # channels last: a view of maps in torch's channels_last memory format
        value = self.norm([m.movedim(1, -1) for m in maps], self.host_shapes)
        B, L = value.shape[0], len(maps)
        reference = self.places.sigmoid()  # (x, y) in [0, 1]
        positions = reference.float() * self.shapes[0].flip(0)  # in cells of the finest level
        reference = reference[None, :, None].expand(B, -1, L, -1)
        x = self.queries.expand(B, -1, -1)
        for layer in self.layers:
            x = layer(x, positions, reference, value, self.host_shapes)
        return self.head(x)


def train(steps: int = 200, batch: int = 4, seed: int = 0, device: str = "cuda") -> list[float]:
    """Losses of fitting fixed random targets."""
    torch.manual_seed(seed)
    shapes = [(24, 32), (12, 16), (6, 8)]
    model = QueryDecoder(shapes).to(device=device, dtype=torch.bfloat16)
    maps = [torch.randn(batch, 64, h, w, device=device, dtype=torch.bfloat16)
            .contiguous(memory_format=torch.channels_last) for h, w in shapes]
    target = torch.randn(batch, 100, 8, device=device)
    slow = [p for n, p in model.named_parameters() if "sampling_offsets" in n or n == "places"]
    rest = [p for p in model.parameters() if all(p is not s for s in slow)]
    optimizer = AdamW([{"params": rest}, {"params": slow, "lr": 5e-4}], lr=3e-3, weight_decay=1e-4,
                      state_bits=8, master_weights=True, seed=seed)
    losses = []
    for _ in range(steps):
        optimizer.zero_grad()
        loss = (model(maps).float() - target).square().mean()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--batch", type=int, default=4)
    args = ap.parse_args()
    history = train(args.steps, args.batch)
    for i in range(0, len(history), max(1, len(history) // 10)):
        print(f"step {i:5d}  loss {history[i]:.4f}")
    print(f"last        loss {history[-1]:.4f}")

"""Attention, rotary positions and neighbour masks together, as a program uses them.

1. Trains one causal attention layer with rotary positions to continue repeating sequences.
2. Runs a sequence token by token over a cache of keys and values and checks the outputs against one
   call over the whole sequence.
3. Smooths noisy labels over the neighbour graph of a point set: a radius mask as attention's mask.

    python examples/attention.py [--device cuda] [--steps 150]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import torchpairwise as tp  # noqa: E402


class Layer(torch.nn.Module):
    """Shared-key-head causal attention over token embeddings, with a read-out to tokens."""

    def __init__(self, tokens=16, width=64, heads=4, key_heads=2, head_width=32):
        super().__init__()
        self.heads, self.key_heads, self.head_width = heads, key_heads, head_width
        self.embed = torch.nn.Embedding(tokens, width)
        self.q = torch.nn.Linear(width, heads * head_width, bias=False)
        self.k = torch.nn.Linear(width, key_heads * head_width, bias=False)
        self.v = torch.nn.Linear(width, key_heads * head_width, bias=False)
        self.out = torch.nn.Linear(heads * head_width, tokens)
        frequencies, self.scale = tp.rotary_frequencies(head_width, 100.0)
        self.register_buffer("frequencies", frequencies)

    def project(self, tokens, positions):
        """Queries, keys and values [batch, heads, n, head_width], queries and keys turned."""
        x = self.embed(tokens)
        q, k, v = (f(x).unflatten(-1, (h, self.head_width)).transpose(1, 2)
                   for f, h in ((self.q, self.heads), (self.k, self.key_heads), (self.v, self.key_heads)))
        turn = lambda y: tp.rotary_embedding(y, positions, self.frequencies, scale=self.scale)  # noqa: E731
        return turn(q), turn(k), v

    def read(self, o):
        return self.out(o.transpose(1, 2).flatten(-2))

    def forward(self, tokens):
        q, k, v = self.project(tokens, torch.arange(tokens.shape[1], device=tokens.device))
        return self.read(tp.attention(q, k, v, causal=True))


def sequences(batch, length, tokens, generator, device):
    """Sequences that repeat a random period of 7: from the eighth on, each token follows from the past."""
    period = torch.randint(0, tokens, (batch, 7), generator=generator)
    return period.repeat(1, length // 7 + 1)[:, :length].to(device)


def train(layer, steps, generator, device):
    opt = torch.optim.Adam(layer.parameters(), 5e-3)
    losses = []
    for _ in range(steps):
        x = sequences(32, 48, 16, generator, device)
        logits = layer(x)
        loss = torch.nn.functional.cross_entropy(logits[:, 7:-1].flatten(0, 1), x[:, 8:].flatten())
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())
    return losses


@torch.no_grad()
def decode(layer, tokens, capacity=64):
    """The logits of every position, one token at a time over a cache with room for `capacity`."""
    b, n = tokens.shape
    cache = tokens.new_zeros((2, b, layer.key_heads, capacity, layer.head_width), dtype=torch.float32)
    lengths = tokens.new_zeros(b)
    logits = []
    for i in range(n):
        q, k, v = layer.project(tokens[:, i:i + 1], lengths.view(b, 1))
        cache[0, :, :, i:i + 1], cache[1, :, :, i:i + 1] = k, v
        lengths += 1
        logits.append(layer.read(tp.attention(q, cache[0], cache[1], lengths=lengths)))
    return torch.cat(logits, 1)


def smooth(generator, device, n=400):
    """Share of right labels before and after one pass over the graph of neighbours within 0.5."""
    centre = torch.randint(0, 2, (n,), generator=generator)
    x = torch.randn(n, 2, generator=generator) * 0.4 + 3.0 * centre[:, None]
    noisy = torch.where(torch.rand(n, generator=generator) < 0.2, 1 - centre, centre)
    x, centre, noisy = x.to(device), centre.to(device), noisy.to(device)
    mask = tp.radius_neighbors_mask(x, epsilon=0.5)
    votes = tp.attention(x, x, torch.nn.functional.one_hot(noisy, 2).float(), mask, scale=0.0)
    return (noisy == centre).float().mean().item(), (votes.argmax(-1) == centre).float().mean().item()


def main(device="cuda", steps=150):
    generator = torch.Generator().manual_seed(0)
    torch.manual_seed(0)
    layer = Layer().to(device)
    losses = train(layer, steps, generator, device)
    x = sequences(4, 40, 16, generator, device)
    with torch.no_grad():
        gap = (decode(layer, x) - layer(x)).abs().max().item()
    before, after = smooth(generator, device)
    return {"first_loss": losses[0], "last_loss": losses[-1], "decode_gap": gap, "labels_before": before,
            "labels_after": after}


if __name__ == "__main__":
    p = argparse.ArgumentParser()
    p.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    p.add_argument("--steps", type=int, default=150)
    a = p.parse_args()
    for key, value in main(a.device, a.steps).items():
        print(f"{key}: {value:.4g}")

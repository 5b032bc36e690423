"""The attention half of a decoder layer over packed weights and an 8-bit cache, as a serving loop runs it: prompts of
several sequences together, then decode steps of one token each, captured once and replayed.

    python examples/decoder_attention.py [--tokens 2048] [--steps 64] [--sequences 4]

Weights are random 4-bit affine packs.
"""
import argparse
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch  # noqa: E402

from ishizuki_amd import attention, synth  # noqa: E402
from ishizuki_amd.linear import PackedLinear  # noqa: E402


def packed(rows, width, seed):
    codes, scales, biases = synth.affine_pack_bits(rows, width, 4, group=64, seed=seed)
    return PackedLinear(*(torch.from_numpy(t).cuda() for t in (codes.view("int32"), scales, biases)), group_size=64, bits=4)


class Attention:
    """x [rows, width] -> [rows, width]: norm, qkv projection, per-head norms and rotation, cache, attention, output
    projection, added to x. One launch each from the projection to the projection."""

    def __init__(self, width=2048, heads=16, kv_heads=4, dim=128, base=1e6, seed=0):
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.qkv = packed((heads + 2 * kv_heads) * dim, width, seed)
        self.out = packed(width, heads * dim, seed + 1)
        self.turns = attention.turns(dim, base)
        self.norm = torch.ones(width, device="cuda")
        self.q_norm, self.k_norm = torch.full((dim,), 1.5, device="cuda"), torch.full((dim,), 1.5, device="cuda")

    def heads_of(self, x):
        """The projection's q, k and v heads, parts of one tensor."""
        h = x.float()
        h = (h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * self.norm).to(x.dtype)
        return self.qkv(h).view(x.shape[0], -1, self.dim).split([self.heads, self.kv_heads, self.kv_heads], 1)

    def __call__(self, x, cache, batch, positions):
        q, k, v = self.heads_of(x)
        q = attention.append(k, v, cache, batch, q=q, positions=positions, turns=self.turns, q_weight=self.q_norm, k_weight=self.k_norm)
        y = attention.attend(q, cache, batch)
        return x + self.out(y.reshape(x.shape[0], -1))


class Sequences:
    """A pool shared by sequences of up to `most` tokens, blocks handed out in turn as they grow."""

    def __init__(self, layer, lengths, most, dtype=torch.int8):
        each = -(-most // attention.BLOCK)
        n = len(lengths)
        self.cache = attention.new_cache(n * each, layer.kv_heads, layer.dim, dtype)
        self.table = torch.arange(n * each, dtype=torch.int32, device="cuda").view(each, n).t().contiguous()
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        self.most = most

    def prompt(self, lengths):
        """(batch, positions) of all tokens of all sequences."""
        starts = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
        positions = torch.cat([torch.arange(n, dtype=torch.int32) for n in lengths]).cuda()
        return attention.Batch(self.table, self.lengths, starts, max(lengths), max(lengths)), positions

    def step(self):
        """(batch, positions) of one more token of each: what a captured step reads as it grows."""
        n = self.lengths.shape[0]
        return attention.Batch(self.table, self.lengths, torch.arange(n + 1, dtype=torch.int32, device="cuda"), 1, self.most), self.lengths.clone()


def capture(layer, x, seqs, batch, positions):
    """A graph of one step: the lengths and positions move on, then the layer; `x` and the output are its own."""
    def step():
        batch.lengths.add_(1)
        y = layer(x, seqs.cache, batch, positions)
        positions.add_(1)
        return y
    lengths, at = batch.lengths.clone(), positions.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # warms up; it wrote where the first replay writes again
    torch.cuda.current_stream().wait_stream(side)
    batch.lengths.copy_(lengths), positions.copy_(at)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    return graph, y


def main():
    p = argparse.ArgumentParser(description=__doc__)
    p.add_argument("--tokens", type=int, default=2048, help="of the longest prompt")
    p.add_argument("--steps", type=int, default=64)
    p.add_argument("--sequences", type=int, default=4)
    a = p.parse_args()
    layer = Attention()
    lengths = [max(1, a.tokens - 100 * s) for s in range(a.sequences)]
    seqs = Sequences(layer, lengths, a.tokens + a.steps + 1)
    g = torch.Generator().manual_seed(0)
    x = torch.randn(sum(lengths), 2048, generator=g).bfloat16().cuda()
    batch, positions = seqs.prompt(lengths)
    for _ in range(2):
        torch.cuda.synchronize()
        t = time.perf_counter()
        y = layer(x, seqs.cache, batch, positions)
        torch.cuda.synchronize()
    print(f"prompts: {sum(lengths)} tokens in {1e3 * (time.perf_counter() - t):.2f} ms")
    x = torch.stack([y[n - 1] for n in batch.starts[1:].tolist()])
    batch, positions = seqs.step()
    graph, y = capture(layer, x, seqs, batch, positions)
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(a.steps):
        graph.replay()
        x.copy_(y)
    torch.cuda.synchronize()
    t = time.perf_counter() - t
    print(f"decode: {a.steps} steps of {a.sequences} sequences, {1e6 * t / a.steps:.1f} us a step; "
          f"lengths now {batch.lengths.tolist()}, |x| {x.float().abs().mean().item():.3f}")


if __name__ == "__main__":
    main()

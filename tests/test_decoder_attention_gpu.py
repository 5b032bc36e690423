"""examples/decoder_attention.py: the layer against the same layer in plain operations, and a captured step against eager
ones."""
import importlib.util
import os

import pytest
import torch

from ishizuki_amd import attention

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("decoder_attention", os.path.join(ROOT, "examples", "decoder_attention.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def plain(layer, x, seqs, batch, positions):
    """The layer's output with norms, rotation and attention in 64 bits on the CPU, the projections and the cache's values as
    the layer has them; and the attention's own output."""
    q, _, _ = (t.cpu().double() for t in layer.heads_of(x))
    q = q / (q.square().mean(-1, keepdim=True) + 1e-6).sqrt() * layer.q_norm.cpu().double()
    half = layer.dim // 2
    angle = positions.cpu().double()[:, None, None] * 1e6 ** (-2.0 * torch.arange(half, dtype=torch.float64) / layer.dim)
    a, b = q[..., :half], q[..., half:]
    q = torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1)
    keys, values = (t.cpu().double() for t in attention.read(seqs.cache, batch, dtype=torch.float32))
    out, starts, lengths = torch.empty_like(q), batch.starts.tolist(), batch.lengths.tolist()
    group, most = layer.heads // layer.kv_heads, keys.shape[1]
    for s, n in enumerate(lengths):
        rows = slice(starts[s], starts[s + 1])
        for h in range(layer.heads):
            k, v = keys[s, most - n:, h // group], values[s, most - n:, h // group]
            logit = q[rows, h] @ k.T * layer.dim ** -0.5
            at = n - (starts[s + 1] - starts[s]) + torch.arange(starts[s + 1] - starts[s])
            out[rows, h] = torch.softmax(logit.masked_fill(torch.arange(n) > at[:, None], -torch.inf), -1) @ v
    return out


def test_layer_and_captured_steps(example):
    layer = example.Attention(width=512, heads=4, kv_heads=2, dim=128)
    lengths = [130, 1, 64]
    seqs = example.Sequences(layer, lengths, 200)
    x = torch.randn(195, 512, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    batch, positions = seqs.prompt(lengths)
    y = layer(x, seqs.cache, batch, positions)
    want = plain(layer, x, seqs, batch, positions)
    q, k, v = layer.heads_of(x)
    q = attention.append(k, v, seqs.cache, batch, q=q, positions=positions, turns=layer.turns, q_weight=layer.q_norm, k_weight=layer.k_norm)
    got = attention.attend(q, seqs.cache, batch)
    # q and the output rounded to bf16 (2^-9 each; q's moves a logit of size |q||k| by 2^-9 of it, under 2^-9 * 1.5^2 * 128
    # ^0.5 = 0.05, and each weight by twice that at most), weights to fp16
    bound = want.abs().amax()
    assert torch.all((got.cpu().double() - want).abs() <= 2.0 ** -9 * want.abs() + 2 * 0.05 * bound)
    assert (got.cpu().double() - want).norm() <= 0.01 * want.norm()
    assert torch.equal(y, x + layer.out(got.reshape(195, -1)))

    first = torch.stack([y[n - 1] for n in batch.starts[1:].tolist()])
    kept, eager = [t.clone() for t in seqs.cache], []
    batch, positions = seqs.step()
    at = first.clone()
    for _ in range(5):
        batch.lengths.add_(1)
        at = layer(at, seqs.cache, batch, positions)
        positions.add_(1)
        eager.append(at)
    for a, b in zip(seqs.cache, kept):
        a.copy_(b)
    batch.lengths.sub_(5), positions.sub_(5)
    at = first.clone()
    graph, out = example.capture(layer, at, seqs, batch, positions)
    for a, b in zip(seqs.cache, kept):  # the capture's warming step wrote a token
        a.copy_(b)
    for want in eager:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        at.copy_(out)

"""A language model over sampled walks: ``python -m nextdoor_amd.walk_model``.

Walks are its sentences, vertices its words.  The engine samples one walk from every vertex, once; a step takes some of them,
packs them one after another (a walk ends where a vertex has no edges), and trains a small transformer to predict each next
vertex: embeddings with dropout, causal attention within each walk, softmax cross entropy over all vertices
(nextdoor_amd/ops.py).  It shows the operators as a training program uses them; nothing is tuned for accuracy.
"""
import argparse
import time

import numpy as np
import torch
from torch import nn
from torch.nn import functional as F

from . import Graph, Sampler, ops


def pack_walks(roots, samples, n_vertices):
    """Walks as one packed batch: (tokens, targets, starts), int32 arrays.

    ``roots``: [walks], ``samples``: [walks, steps] as ``Sampler.final_samples`` gives them.  A walk is its root and the
    vertices up to the first that is none (the value ``n_vertices``).  The target of a token is the vertex
    after it; the last one's is ``n_vertices``, which :func:`ops.vocabulary_loss` takes as no target."""
    walks = np.concatenate([np.asarray(roots, np.int32).reshape(-1, 1), np.asarray(samples, np.int32)], axis=1)
    ended = walks >= n_vertices
    length = np.where(ended.any(1), ended.argmax(1), walks.shape[1])
    inside = np.arange(walks.shape[1]) < length[:, None]
    starts = np.concatenate([[0], np.cumsum(length)]).astype(np.int32)
    after = np.concatenate([walks[:, 1:], np.full((len(walks), 1), n_vertices, np.int32)], axis=1)
    last = np.arange(walks.shape[1]) == length[:, None] - 1
    return walks[inside], np.where(last, n_vertices, after)[inside].astype(np.int32), starts


class Block(nn.Module):
    def __init__(self, width, heads, kv_heads, p):
        super().__init__()
        self.heads, self.kv_heads, self.dim, self.p = heads, kv_heads, width // heads, p
        self.norm1, self.norm2 = nn.LayerNorm(width), nn.LayerNorm(width)
        self.qkv = nn.Linear(width, (heads + 2 * kv_heads) * self.dim, bias=False)
        self.out = nn.Linear(width, width, bias=False)
        self.up, self.down = nn.Linear(width, 4 * width), nn.Linear(4 * width, width)

    def forward(self, x, sequences, seed, step):
        # (q, k and v are slices of one projection: the kernels read them in place)
        qkv = self.qkv(self.norm1(x)).view(x.shape[0], -1, self.dim)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], dim=1)
        attended = ops.packed_attention(q, k, v, sequences).reshape(x.shape)
        x = ops.dropout(self.out(attended), self.p, seed, step, residual=x)
        return ops.dropout(self.down(F.gelu(self.up(self.norm2(x)))), self.p, seed, step + 1, residual=x)


class WalkModel(nn.Module):
    """Next-vertex prediction; the embeddings of the vertices are the classes' vectors too."""

    def __init__(self, n_vertices, width=64, heads=2, kv_heads=1, layers=2, longest=128, dropout=0.1):
        super().__init__()
        self.p = dropout
        self.vertices = nn.Embedding(n_vertices, width)
        self.places = nn.Embedding(longest, width)
        nn.init.normal_(self.vertices.weight, std=width ** -0.5)
        nn.init.normal_(self.places.weight, std=width ** -0.5)
        self.blocks = nn.ModuleList(Block(width, heads, kv_heads, dropout) for _ in range(layers))
        self.norm = nn.LayerNorm(width)

    def forward(self, tokens, places, targets, sequences, seed):
        """The loss of each token; tokens without a next vertex have 0.  ``seed`` chooses what is dropped: another one each
        step."""
        x = self.vertices(tokens) + self.places(places)
        x = ops.dropout(x, self.p, seed, 0)
        for i, block in enumerate(self.blocks):
            x = block(x, sequences, seed, 1 + 2 * i)
        return ops.vocabulary_loss(self.norm(x), self.vertices.weight, targets)


def batch_of(tokens, targets, starts, device="cuda"):
    """A packed batch on the GPU: (tokens, places, targets, sequences)."""
    places = np.arange(len(tokens)) - np.repeat(starts[:-1], np.diff(starts))
    sequences = ops.PackedSequences(starts, device=device)
    on_gpu = [torch.from_numpy(np.ascontiguousarray(a)).to(device) for a in (tokens, places, targets)]
    return (*on_gpu, sequences)


def train(graph, steps=20, walks=1024, seed=42, log=print, **model_args):
    """Trains on walks from ``graph``; returns (model, the mean loss of each step)."""
    torch.manual_seed(seed)
    sampler = Sampler("DeepWalkPerVertex", graph, seed=seed)
    sampler.do_transit_parallel()
    samples, roots = sampler.final_samples(), sampler.initial_contents
    model = WalkModel(graph.n_vertices, longest=samples.shape[1] + 1, **model_args).to("cuda", torch.bfloat16)
    optimizer = torch.optim.AdamW(model.parameters(), lr=2e-3)
    order, losses = np.random.default_rng(seed), []
    for step in range(steps):
        some = order.choice(len(roots), min(walks, len(roots)), replace=False)
        tokens, places, targets, sequences = batch_of(*pack_walks(roots[some], samples[some], graph.n_vertices))
        begin = time.perf_counter()
        each = model(tokens, places, targets, sequences, (seed * 1000003 + step) % (1 << 64))
        loss = each.sum() / (targets < graph.n_vertices).sum()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
        if log:
            log("step %3d: %6d tokens, loss %.4f, %.1f ms" % (step, len(tokens), losses[-1],
                                                              1e3 * (time.perf_counter() - begin)))
    sampler.close()
    return model, losses


def main(argv=None):
    p = argparse.ArgumentParser(prog="python -m nextdoor_amd.walk_model", description=__doc__.splitlines()[0])
    p.add_argument("-g", "--graph-file", help="binary edge list; default: a synthetic graph of 10000 vertices")
    p.add_argument("-n", "--steps", type=int, default=20)
    p.add_argument("--walks", type=int, default=1024, help="walks in a batch")
    p.add_argument("--width", type=int, default=64)
    p.add_argument("--layers", type=int, default=2)
    p.add_argument("--seed", type=int, default=42)
    args = p.parse_args(argv)
    graph = Graph.load(args.graph_file) if args.graph_file else Graph.chung_lu(10000, 150000, 2.2, seed=args.seed)
    train(graph, args.steps, args.walks, args.seed, width=args.width, layers=args.layers)


if __name__ == "__main__":
    main()

"""One attention layer served from a paged cache: prompts, then decode steps, behind a prefix that all requests share.

    python examples/paged_decode.py [--requests 4] [--steps 8] [--prefix 50]

A step of the layer, for the new tokens of every request at once:

    q, k, v = x Wq^T, x Wk^T, x Wv^T          gguf_linear, Q4_K weights
    offsets, lengths, positions, slots, table  paged_slots: pages taken from a free list where a request needs one
    q, cache <- rotary(q), rotary(k), v        rotary_store
    a = attention(q, cache)                    paged_attention
    y = a Wo^T                                 gguf_linear

Nothing of it waits for the GPU: lengths, tables and the free list stay in device memory from step to step.  The
weights are random; the attention of every token is compared with the formula in 64 bits.
"""

from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import tensor_amd.torch as tensor_torch
from tensor_amd.gguf.quant import sample_weight
from tensor_amd.kernels.paged import rotary_angles
from tensor_amd.torch.session import session


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Layer:
    """Weights, cache and free list; `state` is what a step passes to the next."""

    def __init__(self, *, hidden, heads, kv, dim, page, pages, reach, seed=0):
        self.heads, self.kv, self.dim = heads, kv, dim
        rows = {"q": heads * dim, "k": kv * dim, "v": kv * dim}
        self.weights = {name: torch.from_numpy(sample_weight(n, hidden, "q4_k", seed=seed + i, std=hidden ** -0.5)).cuda()
                        for i, (name, n) in enumerate(rows.items())}
        self.weights["o"] = torch.from_numpy(sample_weight(hidden, heads * dim, "q4_k", seed=seed + 3)).cuda()
        self.angles = torch.from_numpy(rotary_angles(reach, dim)).cuda()
        self.k_cache = torch.zeros((pages, kv, page, dim), dtype=torch.float16, device="cuda")
        self.v_cache = torch.zeros_like(self.k_cache)
        self.free, self.left = torch.randperm(pages).to(torch.int32).cuda(), ints([pages])
        self.linear = tensor_torch.load("gguf_linear", encoding="q4_k", out_dtype="float16")
        self.slots = tensor_torch.load("paged_slots", page_size=page)
        self.store = tensor_torch.load("rotary_store", layout="half")
        self.attention = tensor_torch.load("paged_attention")
        self.workspace = None  # of the attention, as large as a step has needed

    def project(self, x):
        return [self.linear(x, self.weights[name]).view(x.shape[0], -1, self.dim) for name in "qkv"]

    def step(self, x, counts, lengths, start, table, prefix_pages):
        """(y, attention, lengths, table) after the new tokens x, counts of them for each request."""
        tokens, requests = x.shape[0], counts.shape[0]
        q, k, v = self.project(x)
        offsets, lengths, positions, slots, table, self.left = self.slots(
            lengths, counts, start, self.free, self.left, table, tokens)
        turned = torch.empty_like(q)
        self.store.raw(q, k, v, positions, slots, self.angles, turned, self.k_cache, self.v_cache)
        need = session(x.device.index).attention_workspace(tokens, requests, self.heads, self.kv, self.dim)
        if self.workspace is None or self.workspace.numel() < need:
            self.workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
        a = self.attention(turned, self.k_cache, self.v_cache, offsets, lengths, table, prefix_pages, start, self.workspace)
        return self.linear(a.view(tokens, -1), self.weights["o"]), a, lengths, table


def turn(x, angles, at):
    """Rotary positions of x [n, heads, dim] in 64 bits."""
    x, half = x.double(), x.shape[-1] // 2
    cos, sin = angles[at, None, :half].double(), angles[at, None, half:].double()
    return torch.cat([x[..., :half] * cos - x[..., half:] * sin, x[..., half:] * cos + x[..., :half] * sin], -1)


def formula(layer, x, new):
    """(attention of the last `new` of a sequence's tokens x, what an fp16 result may differ by)."""
    q, k, v = layer.project(x)
    at, n = torch.arange(x.shape[0], device=x.device), x.shape[0]
    share = layer.heads // layer.kv
    q = turn(q, layer.angles, at)[-new:].transpose(0, 1)
    k, v = (t.transpose(0, 1).repeat_interleave(share, 0) for t in (turn(k, layer.angles, at), v.double()))
    seen = at[None, :] <= at[-new:, None]
    scale = layer.dim ** -0.5
    scores = (q[:, :, None, :] * k[:, None, :, :]).sum(-1) * scale
    a = (torch.softmax(scores.masked_fill(~seen, -torch.inf), -1)[..., None] * v[:, None]).sum(2)
    # queries and keys are kept in fp16 (2^-11 of each, and 2^-12 for their fp32 rotation): scores move by `off`, weights by
    # e^(2 off); weights and the output are rounded to fp16
    off = 2.0 ** -9 * scale * (q.abs()[:, :, None, :] * k.abs()[:, None, :, :]).sum(-1).amax(-1, keepdim=True)
    bound = (torch.expm1(2 * off) + 2.0 ** -9) * v.abs().amax(1, keepdim=True) + 2.0 ** -20
    return a.transpose(0, 1), bound.transpose(0, 1)


def run(*, requests=4, steps=8, prefix=50, hidden=1024, heads=8, kv=2, dim=128, page=16, seed=0):
    """The largest |difference| / bound over every token's attention; prints a line a step."""
    rng = np.random.default_rng(seed)
    prompts = [int(n) for n in rng.integers(1, 60, requests)]
    columns = -(-(max(prompts) + steps) // page)
    layer = Layer(hidden=hidden, heads=heads, kv=kv, dim=dim, page=page, pages=requests * columns + prefix // page + 3,
                  reach=prefix + max(prompts) + steps, seed=seed)

    def tokens(n):
        return torch.from_numpy(rng.standard_normal((n, hidden)).astype(np.float16)).cuda()

    # the prefix is stored once, as a request of its own at position 0; its page list then stands for it
    shared, none = tokens(prefix), torch.full((1, -(-prefix // page)), -1, dtype=torch.int32, device="cuda")
    _, _, _, row = layer.step(shared, ints([prefix]), ints([0]), ints([0]), none, ints([-1]))
    prefix_pages, start = row[0].contiguous(), ints([prefix])

    histories = [shared] * requests
    lengths, table = ints([0] * requests), torch.full((requests, columns), -1, dtype=torch.int32, device="cuda")
    worst = 0.0
    for step in range(steps + 1):
        counts = prompts if step == 0 else [1] * requests
        x = tokens(sum(counts))
        _, a, lengths, table = layer.step(x, ints(counts), lengths, start, table, prefix_pages)
        at = 0
        for b, new in enumerate(counts):
            histories[b] = torch.cat([histories[b], x[at:at + new]])
            want, bound = formula(layer, histories[b], new)
            error = float(((a[at:at + new].double() - want).abs() / bound).max())
            worst = max(worst, error if math.isfinite(error) else math.inf)  # (max would pass a NaN by)
            at += new
        print(f"step {step}: {len(x)} tokens, own lengths {lengths.tolist()}, {int(layer.left)} pages left, "
              f"largest difference {worst:.3f} of its bound", flush=True)
    return worst


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("requests", 4), ("steps", 8), ("prefix", 50)):
        parser.add_argument(f"--{name}", type=int, default=value)
    sys.exit(0 if run(**vars(parser.parse_args())) <= 1.0 else 1)

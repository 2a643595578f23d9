"""One decoder layer with its linears in 8 bits, served from a paged cache: prompts, then decode steps.

    python examples/fp8_layer.py [--requests 4] [--steps 6]

A step of the layer, for the new tokens of every request at once (r is the residual stream, in fp32):

    r, x8 = r + y, norm(r + y)                 rms_norm_fp8 with the residual's addition
    q, k, v = x8 Wq^T, x8 Wk^T, x8 Wv^T        fp8_linear
    q, k = norm(q), norm(k)                    rms_norm, a row for each head
    q, cache <- rotary(q), rotary(k), v        rotary_store
    a = attention(q, cache)                    paged_attention
    y = quantize(a) Wo^T                       quantize_fp8, fp8_linear
    r, x8 = r + y, norm(r + y)                 rms_norm_fp8
    y = quantize(silu(gate) up) Wd^T           fp8_linear, quantize_fp8 with gates, fp8_linear

Nothing of it waits for the GPU.  The weights are random; every step's y is compared with the same layer in 64 bits on the
weights as the codes hold them, without the activations' rounding to 8 bits.
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
from tensor_amd.kernels.fp8 import e4m3_values, quantize_weight
from tensor_amd.kernels.paged import rotary_angles
from tensor_amd.torch.session import session


# Four times an activation is rounded to 8 bits on the way, by 2^-4 of it at most, and what that adds to a result stays.
LIMIT = 4 * 2.0 ** -4


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Layer:
    """Weights, cache and free list; `step` takes and returns what one step passes to the next."""

    def __init__(self, *, hidden, inner, heads, kv, dim, page, pages, reach, seed=0, eps=1e-6):
        rng = np.random.default_rng(seed)
        self.heads, self.kv, self.dim, self.eps = heads, kv, dim, eps
        rows = {"q": (heads * dim, hidden), "k": (kv * dim, hidden), "v": (kv * dim, hidden), "o": (hidden, heads * dim),
                "gate_up": (2 * inner, hidden), "down": (hidden, inner)}
        self.weights = {name: tuple(torch.from_numpy(t).cuda() for t in quantize_weight(
            (rng.standard_normal(shape) * shape[1] ** -0.5).astype(np.float32))) for name, shape in rows.items()}
        self.norms = {name: torch.from_numpy(rng.uniform(0.5, 1.5, width).astype(np.float32)).cuda()
                      for name, width in (("attention", hidden), ("mlp", hidden), ("q", dim), ("k", dim))}
        self.angles = torch.from_numpy(rotary_angles(reach, dim)).cuda()
        self.k_cache = torch.zeros((pages, kv, page, dim), dtype=torch.float16, device="cuda")
        self.v_cache = torch.zeros_like(self.k_cache)
        self.free, self.left = torch.randperm(pages).to(torch.int32).cuda(), ints([pages])
        self.prefix = ints([-1]), ints([0])  # no shared prefix
        load = tensor_torch.load
        self.linear = load("fp8_linear", out_dtype="float16")
        self.norm = load("rms_norm_fp8", residual="float32", eps=eps)
        self.head_norm = load("rms_norm", eps=eps)
        self.quantize, self.gated = load("quantize_fp8"), load("quantize_fp8", gated=True)
        self.slots = load("paged_slots", page_size=page)
        self.store = load("rotary_store", layout="half")
        self.attention = load("paged_attention")
        self.workspace = None  # of the attention, as large as a step has needed

    def project(self, name, codes, scales):
        return self.linear(codes, scales, *self.weights[name])

    def step(self, y, r, counts, lengths, table):
        """(y, r, lengths, table) after the new tokens, whose layer input is r + y."""
        tokens, requests = y.shape[0], counts.shape[0]
        codes, scales, r = self.norm(y, r, self.norms["attention"])
        q, k, v = (self.project(name, codes, scales).view(tokens, -1, self.dim) for name in "qkv")
        q, k = (self.head_norm(x.view(-1, self.dim), self.norms[name]).view_as(x) for x, name in ((q, "q"), (k, "k")))
        offsets, lengths, positions, slots, table, self.left = self.slots(
            lengths, counts, self.prefix[1], self.free, self.left, table, tokens)
        turned = torch.empty_like(q)
        self.store.raw(q, k, v, positions, slots, self.angles, turned, self.k_cache, self.v_cache)
        need = session(y.device.index).attention_workspace(tokens, requests, self.heads, self.kv, self.dim)
        if self.workspace is None or self.workspace.numel() < need:
            self.workspace = torch.empty(need, dtype=torch.uint8, device=y.device)
        a = self.attention(turned, self.k_cache, self.v_cache, offsets, lengths, table, *self.prefix, self.workspace)
        y = self.project("o", *self.quantize(a.view(tokens, -1)))
        codes, scales, r = self.norm(y, r, self.norms["mlp"])
        y = self.project("down", *self.gated(self.project("gate_up", codes, scales)))
        return y, r, lengths, table


def weight_of(layer, name):
    """The matrix that a weight's codes and scales stand for, in 64 bits."""
    codes, scales = layer.weights[name]
    values = torch.from_numpy(e4m3_values()).cuda().double()[codes.long()]
    spread = scales.double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    return values * spread[:codes.shape[0], :codes.shape[1]]


def formula(layer, x, new):
    """y and r of the last `new` of a sequence's tokens x [n, hidden], in 64 bits."""
    def norm(t, name):
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + layer.eps) * layer.norms[name].double()

    r, n = x.double(), x.shape[0]
    at = torch.arange(n, device=x.device)
    h = norm(r, "attention")
    q, k, v = ((h @ weight_of(layer, name).T).view(n, -1, layer.dim) for name in "qkv")
    half = layer.dim // 2
    cos, sin = layer.angles[at, None, :half].double(), layer.angles[at, None, half:].double()

    def turn(t):
        return torch.cat([t[..., :half] * cos - t[..., half:] * sin, t[..., half:] * cos + t[..., :half] * sin], -1)

    q, k = turn(norm(q, "q"))[-new:], turn(norm(k, "k"))
    k, v = (t.repeat_interleave(layer.heads // layer.kv, 1) for t in (k, v))
    scores = torch.stack([q[:, h] @ k[:, h].T for h in range(layer.heads)]) * layer.dim ** -0.5
    scores = scores.masked_fill(at[None, None, :] > at[None, -new:, None], -torch.inf)
    a = torch.stack([torch.softmax(scores[h], -1) @ v[:, h] for h in range(layer.heads)], 1).reshape(new, -1)
    r = r[-new:] + a @ weight_of(layer, "o").T
    gate, up = (norm(r, "mlp") @ weight_of(layer, "gate_up").T).chunk(2, -1)
    return (gate * torch.sigmoid(gate) * up) @ weight_of(layer, "down").T, r


def run(*, requests=4, steps=6, hidden=512, inner=1280, heads=8, kv=2, dim=64, page=16, seed=0):
    """The largest difference of a step's y from the 64-bit layer, relative in the 2-norm; prints a line a step."""
    rng = np.random.default_rng(seed)
    prompts = [int(n) for n in rng.integers(1, 40, requests)]
    columns = -(-(max(prompts) + steps) // page)
    layer = Layer(hidden=hidden, inner=inner, heads=heads, kv=kv, dim=dim, page=page, pages=requests * columns + 3,
                  reach=max(prompts) + steps, seed=seed)
    histories = [torch.empty((0, hidden), device="cuda") for _ in range(requests)]
    lengths, table = ints([0] * requests), torch.full((requests, columns), -1, dtype=torch.int32, device="cuda")
    worst = 0.0
    for step in range(steps + 1):
        counts = prompts if step == 0 else [1] * requests
        y = torch.from_numpy(rng.standard_normal((sum(counts), hidden)).astype(np.float16)).cuda()
        r = torch.from_numpy((3 * rng.standard_normal((sum(counts), hidden))).astype(np.float32)).cuda()
        x = r.double() + y.double()
        out, stream, lengths, table = layer.step(y, r, ints(counts), lengths, table)
        at = 0
        for b, new in enumerate(counts):
            histories[b] = torch.cat([histories[b], x[at:at + new].float()])
            want, want_r = formula(layer, histories[b], new)
            for got, exact in ((out, want), (stream, want_r)):
                error = float((got[at:at + new].double() - exact).norm() / exact.norm())
                worst = max(worst, error if math.isfinite(error) else math.inf)  # (max would pass a NaN by)
            at += new
        print(f"step {step}: {len(y)} tokens, lengths {lengths.tolist()}, {int(layer.left)} pages left, "
              f"largest difference {worst:.4f}", flush=True)
    return worst


def main(arguments=None):
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("requests", 4), ("steps", 6)):
        parser.add_argument(f"--{name}", type=int, default=value)
    return 0 if run(**vars(parser.parse_args(arguments))) < LIMIT else 1


if __name__ == "__main__":
    sys.exit(main())

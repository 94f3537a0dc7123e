"""The attention block of a W8A8 decoder over a paged, budgeted key-value cache, one token per sequence and step.

    python examples/decode_paged_cache.py --batch 16 --budget 1024 --steps 64 [--int8-cache | --int4-cache] [--layer] [--graph]

Random weights and prompts.  Per step: npu_dynamic_quant, npu_quant_matmul (qkv), PagedKVCache.append, attend and evict,
npu_dynamic_quant, npu_quant_matmul (output).  With --layer the step also has a decoder layer's norms and positions:
npu_add_rms_norm_dynamic_quant in place of the first npu_dynamic_quant, PagedKVCache.rotate before append, and npu_add_rms_norm,
which adds the residual, at the end.  With --graph the steps are replays of one captured step.
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

import pytorch_amd as pa  # noqa: E402
from pytorch_amd.contrib.module import PagedKVCache  # noqa: E402


def linear(features_in, features_out, generator):
    """int8 weight, stored [out, in] and passed as its transposed view, and a scale per output."""
    weight = torch.randint(-127, 128, (features_out, features_in), generator=generator, dtype=torch.int8).cuda()
    return pa.prepare_quant_matmul_weight(weight.t()), torch.full((features_out,), 1.0 / (74 * features_in ** 0.5), device="cuda")


def project(layer, x):
    return project_codes(layer, *pa.npu_dynamic_quant(x))


def project_codes(layer, codes, scale):
    return pa.npu_quant_matmul(codes, layer[0], layer[1], pertoken_scale=scale, output_dtype=torch.bfloat16)


class DecodeAttention:
    def __init__(self, hidden, heads, cache, generator):
        self.heads, self.cache = heads, cache
        self.kv_heads, self.head_dim = cache.key_cache.shape[2], hidden // heads
        self.qkv = linear(hidden, (heads + 2 * self.kv_heads) * self.head_dim, generator)
        self.o = linear(heads * self.head_dim, hidden, generator)

    def split(self, x):
        """Queries, keys and values as views of the projection."""
        qkv = project(self.qkv, x).view(x.shape[0], self.heads + 2 * self.kv_heads, self.head_dim)
        return qkv.split((self.heads, self.kv_heads, self.kv_heads), 1)

    def prefill(self, sequence, x):
        _, k, v = self.split(x)
        self.cache.prefill(sequence, k, v)

    def step(self, x):
        q, k, v = self.split(x)
        self.cache.append(k, v)
        out = self.cache.attend(q)
        self.cache.evict()
        return x + project(self.o, out.flatten(1))


class DecodeLayer(DecodeAttention):
    """With the norms on both sides and rotary positions; a step returns what the MLP reads."""

    def __init__(self, hidden, heads, cache, generator, positions):
        super().__init__(hidden, heads, cache, generator)
        self.gamma = [(1 + 0.1 * torch.randn(hidden, generator=generator)).to(torch.bfloat16).cuda() for _ in range(2)]
        angles = torch.arange(float(positions))[:, None] * 10000.0 ** (-torch.arange(0, self.head_dim, 2) / self.head_dim)
        self.cos_sin = torch.cat((angles.cos(), angles.sin()), 1).cuda()

    def split(self, x):
        codes, scale, _ = pa.npu_add_rms_norm_dynamic_quant(x, None, self.gamma[0])
        qkv = project_codes(self.qkv, codes, scale).view(x.shape[0], self.heads + 2 * self.kv_heads, self.head_dim)
        return qkv.split((self.heads, self.kv_heads, self.kv_heads), 1)

    def prefill(self, sequence, x):
        q, k, v = self.split(x)
        _, k = pa.npu_mrope(torch.arange(x.shape[0], device=x.device), q, k, self.cos_sin, self.head_dim)
        self.cache.prefill(sequence, k, v)

    def step(self, x):
        q, k, v = self.split(x)
        q, k = self.cache.rotate(q, k, self.cos_sin)
        self.cache.append(k, v)
        out = self.cache.attend(q)
        self.cache.evict()
        return pa.npu_add_rms_norm(x, project(self.o, out.flatten(1)), self.gamma[1])[0]


def main(argv=None):
    p = argparse.ArgumentParser()
    for name, value in (("batch", 16), ("hidden", 4096), ("heads", 32), ("kv-heads", 8), ("budget", 1024), ("prompt", 1000), ("steps", 64)):
        p.add_argument("--" + name, type=int, default=value)
    codes = p.add_mutually_exclusive_group()
    codes.add_argument("--int8-cache", action="store_true")
    codes.add_argument("--int4-cache", action="store_true")
    p.add_argument("--layer", action="store_true")
    p.add_argument("--graph", action="store_true")
    a = p.parse_args(argv)
    g = torch.Generator().manual_seed(0)
    room = max(a.prompt, a.budget) + 1
    cache = PagedKVCache(a.batch, room, a.kv_heads, a.hidden // a.heads, budget=a.budget, quantized=a.int8_cache or a.int4_cache, bits=4 if a.int4_cache else 8,
                         device="cuda")
    block = DecodeLayer(a.hidden, a.heads, cache, g, a.prompt + a.steps + 2) if a.layer else DecodeAttention(a.hidden, a.heads, cache, g)
    for b in range(a.batch):
        block.prefill(b, torch.randn(a.prompt - b % 2, a.hidden, generator=g).to(torch.bfloat16).cuda())
    x = torch.randn(a.batch, a.hidden, generator=g).to(torch.bfloat16).cuda()
    step = lambda: block.step(x)  # noqa: E731
    y = step()
    if a.graph:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = block.step(x)
        step = graph.replay
    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(a.steps):
        out = step()
    torch.cuda.synchronize()
    y = y if a.graph else out
    ms = (time.perf_counter() - start) / a.steps * 1e3
    print(f"{a.batch} sequences, {int(cache.context_lens.max())} of {cache.capacity} tokens held, {ms:.3f} ms per step, "
          f"{a.batch / ms * 1e3:.0f} tokens/s of one {'layer without its MLP' if a.layer else 'attention block'}")
    return y, cache


if __name__ == "__main__":
    main()

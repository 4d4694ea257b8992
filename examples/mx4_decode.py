"""A transformer block's attention on MX4: prompts in, tokens decoded in a batch.

    python examples/mx4_decode.py [--hidden 4096 --heads 32 --kv-heads 8 --batch 8 --prompt 1000 --tokens 64]

Random weights. Each prompt is written to the paged cache in chunks (its keys and
values are read back for the chunk's own attention); then all sequences decode
together, one token a step, as one CUDA graph replayed. The last step's output is
compared with the same block in float32 without any quantization.

Two times a step are given: the whole step, from the scheduler's page lists and the
copies of tables, lengths and inputs to the step's end, and the graph alone.
"""
import argparse
import os
import sys
import time

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "comfyui-int4-convrot-rdna4_b200"))

from _int4.mx4_layers import Mx4ConvRotLinear, Mx4KVCache, Mx4SelfAttention  # noqa: E402


def float_block(x, w_qkv, w_out, heads, kv_heads, head_dim):
    """The block's causal attention of whole sequences x [T, hidden] in float32."""
    y = (x.float() @ w_qkv.t()).unflatten(-1, (heads + 2 * kv_heads, head_dim))
    q, k, v = y.split((heads, kv_heads, kv_heads), dim=-2)
    y = torch.nn.functional.scaled_dot_product_attention(
        q.transpose(0, 1)[None], k.transpose(0, 1)[None], v.transpose(0, 1)[None], is_causal=True, enable_gqa=True)
    return y[0].transpose(0, 1).reshape(x.shape[0], -1) @ w_out.t()


@torch.inference_mode()
def run(hidden=4096, heads=32, kv_heads=8, head_dim=128, batch=8, prompt=1000, chunk=512, tokens=64, page=64, seed=0):
    """Returns {"us_per_step", "us_graph", "tokens_per_s", "rel"}: a decode step's time, that of its
    graph alone, the tokens a second of whole steps, and the distance from float32."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = (heads + 2 * kv_heads) * head_dim
    w_qkv = torch.randn(width, hidden, generator=g, device="cuda") / hidden ** 0.5
    w_out = torch.randn(hidden, heads * head_dim, generator=g, device="cuda") / hidden ** 0.5
    block = Mx4SelfAttention(hidden, heads, kv_heads, head_dim, device="cuda")
    for linear, w in ((block.qkv, w_qkv), (block.out, w_out)):
        source = torch.nn.Linear(w.shape[1], w.shape[0], bias=False, device="meta")
        source.weight = torch.nn.Parameter(w, requires_grad=False)
        quantized = Mx4ConvRotLinear.from_linear(source)
        linear.weight, linear.weight_scale = quantized.weight, quantized.weight_scale

    # prompts of different lengths
    lengths = [max(1, prompt - 37 * i) for i in range(batch)]
    x = [torch.randn(n + tokens, hidden, generator=g, device="cuda").bfloat16() for n in lengths]
    pages = sum(-(-(n + tokens) // page) for n in lengths)
    cache = Mx4KVCache(pages, kv_heads, head_dim, page)
    seqs = [cache.add() for _ in lengths]
    for s, n, xs in zip(seqs, lengths, x):
        for at in range(0, n, chunk):
            block.prefill(xs[at:min(n, at + chunk)], cache, s)

    # decoding: buffers of a step are filled, the step is a graph
    slots = torch.zeros(batch, dtype=torch.int64, device="cuda")
    table = torch.full((batch, max(-(-(n + tokens) // page) for n in lengths)), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(batch, dtype=torch.int32, device="cuda")
    inp = torch.zeros(batch, 1, hidden, dtype=torch.bfloat16, device="cuda")

    def fill(step):
        new = [cache.extend(s, 1)[0] for s in seqs]
        slots.copy_(torch.tensor(new))
        t, n = cache.tables(seqs)
        table[:, :t.shape[1]] = t
        lens.copy_(n)
        inp.copy_(torch.stack([xs[n0 + step] for xs, n0 in zip(x, lengths)])[:, None])

    fill(0)
    out = block(inp, cache, slots, table, lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(inp, cache, slots, table, lens)
    spent, whole = [], []
    torch.cuda.synchronize()
    for step in range(tokens):
        start = time.perf_counter()
        if step:
            fill(step)
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        graph.replay()
        end.record()
        end.synchronize()
        spent.append(begin.elapsed_time(end) * 1e3)
        if step or tokens == 1:                                   # (the first step was filled ahead of the capture)
            whole.append((time.perf_counter() - start) * 1e6)
    want = torch.stack([float_block(xs, w_qkv, w_out, heads, kv_heads, head_dim)[-1] for xs in x])
    rel = float((out[:, 0].float() - want).norm() / want.norm())
    us = sorted(whole)[len(whole) // 2]
    return {"us_per_step": us, "us_graph": sorted(spent)[len(spent) // 2], "tokens_per_s": batch / us * 1e6, "rel": rel}


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("hidden", 4096), ("heads", 32), ("kv-heads", 8), ("head-dim", 128), ("batch", 8), ("prompt", 1000),
                        ("chunk", 512), ("tokens", 64), ("page", 64), ("seed", 0)):
        ap.add_argument("--" + name, type=int, default=value)
    r = run(**{k.replace("-", "_"): v for k, v in vars(ap.parse_args()).items()})
    print(f"decode step {r['us_per_step']:.0f} us (its graph alone {r['us_graph']:.1f} us), {r['tokens_per_s']:.0f} tokens/s, "
          f"relative distance from float32 {r['rel']:.3f}")


if __name__ == "__main__":
    main()

"""An attention block served from quantised weights over the 4-bit cache.

Quantises the four projections of a random attention block (EXL3, K = 4 bits a
weight), decodes them from their stored form, and serves a few requests with
them: one prompt step of ragged lengths, then single tokens, each step planned
on the GPU, its keys and values appended in 4 bits, its queries attending over
the cache. Prints how far the outputs are from the block's exact attention with
the same decoded weights.

    python examples/serve_quantized.py [--tokens 8]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from exl3_intel_arc_quantizer_amd.kv_cache import (append_tokens, cache_attention,  # noqa: E402
                                                   cache_pages, plan_step)
from exl3_intel_arc_quantizer_amd.layer_quant import (hessian_from_activations,  # noqa: E402
                                                      quantize_linear_module)
from exl3_intel_arc_quantizer_amd.rotary import apply_rotary, rotary_frequencies  # noqa: E402
from exl3_intel_arc_quantizer_amd.serialization import (decode_weight_from_storage,  # noqa: E402
                                                        pack_module_trellis)

HIDDEN, Q_HEADS, KV_HEADS, HEAD_DIM, PAGE, BITS = 512, 4, 2, 128, 64, 4


def quantized_block(device, generator) -> dict:
    """Decoded bfloat16 weights (in, out) of the projections, through their
    packed storage."""
    x = torch.randn(2048, HIDDEN, device=device, generator=generator).to(torch.bfloat16)
    hessian, _ = hessian_from_activations(x)
    weights = {}
    for name, rows in (("qkv", (Q_HEADS + 2 * KV_HEADS) * HEAD_DIM), ("o", HIDDEN)):
        w = torch.randn(rows, HIDDEN, device=device, generator=generator) * HIDDEN ** -0.5
        r = quantize_linear_module(name, w, hessian, K=BITS)
        stored = decode_weight_from_storage(pack_module_trellis(r.encoded, BITS), r.su, r.sv, BITS, r.cb)
        weights[name] = stored.to(torch.bfloat16)
    return weights


def exact_attention(q, k, v, first):
    """Causal attention in float64 of queries at positions first.. over all
    keys; (tokens, heads, head_dim) each."""
    k, v = (x.double().repeat_interleave(Q_HEADS // KV_HEADS, 1).transpose(0, 1) for x in (k, v))
    scores = q.double().transpose(0, 1) @ k.transpose(1, 2).contiguous() * HEAD_DIM ** -0.5
    at = torch.arange(first, first + q.shape[0], device=q.device)[:, None]
    scores = scores.masked_fill(torch.arange(k.shape[1], device=q.device)[None] > at, float("-inf"))
    return (torch.softmax(scores, -1) @ v).transpose(0, 1)


def serve(tokens: int = 8, lengths=(70, 1, 130), device: str = "cuda", seed: int = 0) -> float:
    """Relative error of all served outputs against exact attention."""
    device = torch.device(device, torch.cuda.current_device())
    g = torch.Generator(device=device).manual_seed(seed)
    weights = quantized_block(device, g)
    frequencies, magnitude = rotary_frequencies(HEAD_DIM, scaling="linear", factor=2.0, device=device)
    requests, width = len(lengths), -(-(max(lengths) + tokens) // PAGE)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=device)

    pages = cache_pages(requests * width, PAGE, KV_HEADS, HEAD_DIM, device)
    tables = torch.full((requests, width), -1, dtype=torch.int32, device=device)
    free, taken = torch.randperm(requests * width, device=device, generator=g).to(torch.int32), ints([0])
    cached = ints([0] * requests)
    history = [[] for _ in lengths]
    off = total = 0.0
    for step in range(1 + tokens):
        new = list(lengths) if step == 0 else [1] * requests
        x = torch.randn(sum(new), HIDDEN, device=device, generator=g).to(torch.bfloat16)
        qkv = (x @ weights["qkv"]).view(-1, Q_HEADS + 2 * KV_HEADS, HEAD_DIM)
        q, k, v = qkv.split([Q_HEADS, KV_HEADS, KV_HEADS], 1)

        plan = plan_step(cached, ints(new), tables, free, taken, page_size=PAGE, max_tokens=len(x))
        turned = append_tokens(pages, k, v, plan.slots, q=q, positions=plan.positions,
                               frequencies=frequencies, magnitude=magnitude)
        out = cache_attention(turned, pages, tables, plan.starts, plan.lengths, max_new=max(new))
        served = out.flatten(1) @ weights["o"]
        cached, taken = plan.lengths, plan.taken

        plan.check()
        exact_k = apply_rotary(k, None, plan.positions, frequencies, magnitude=magnitude)[0]
        starts = plan.starts.tolist()
        for r, past in enumerate(history):
            rows = slice(starts[r], starts[r + 1])
            past.append((exact_k[rows], v[rows]))
            keys, values = (torch.cat(y) for y in zip(*past))
            want = exact_attention(turned[rows], keys, values, len(keys) - new[r])
            want = want.flatten(1) @ weights["o"].double()
            off += float((served[rows].double() - want).square().sum())
            total += float(want.square().sum())
    return (off / total) ** 0.5


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=8, help="single tokens that each request decodes")
    args = ap.parse_args()
    print(f"relative error of the 4-bit cache: {serve(args.tokens):.4f}")

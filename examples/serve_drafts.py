"""Greedy decoding of drafted trees with weights that stay in their stored form.

Quantises the projections of a small random model (one attention block over the
4-bit cache and a head, EXL3, 4 bits a weight) and decodes a few requests with it,
every product taken from the stored words. Tokens have three positions (time,
height, width; here text, whose three are alike). Each step drafts a tree after the
last chosen token: the two tokens that the head ranks highest without the
attention block, and after each of them one more. All drafted tokens go through the
model at once; those that it would have chosen are kept, and the pages of the rest
go back. The operators wait for nothing; the example reads each step's tokens.

    python examples/serve_drafts.py [--tokens 24]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from exl3_intel_arc_quantizer_amd.kv_cache import (accept_drafts, append_tokens, cache_attention,  # noqa: E402
                                                   cache_pages, keep_tokens, plan_step, plan_tree,
                                                   release_pages)
from exl3_intel_arc_quantizer_amd.layer_quant import (hessian_from_activations,  # noqa: E402
                                                      quantize_linear_module)
from exl3_intel_arc_quantizer_amd.quantized_linear import quantized_linear  # noqa: E402
from exl3_intel_arc_quantizer_amd.rotary import rotary_axes, rotary_frequencies  # noqa: E402
from exl3_intel_arc_quantizer_amd.serialization import pack_module_trellis  # noqa: E402

HIDDEN, VOCABULARY, Q_HEADS, KV_HEADS, HEAD_DIM, PAGE, BITS = 256, 512, 4, 2, 64, 32, 4
SECTIONS = (8, 12, 12)                   # pairs of each position
PARENTS = (-1, 0, 0, 1, 2)               # the chosen token, two after it, one after each


class Model:
    def __init__(self, device, generator):
        self.embedding = torch.randn(VOCABULARY, HIDDEN, device=device, generator=generator).half()
        hessian, _ = hessian_from_activations(self.embedding.to(torch.bfloat16))
        self.stored = {}
        for name, rows, inputs in (("qkv", (Q_HEADS + 2 * KV_HEADS) * HEAD_DIM, HIDDEN),
                                   ("o", HIDDEN, Q_HEADS * HEAD_DIM), ("head", VOCABULARY, HIDDEN)):
            w = torch.randn(rows, inputs, device=device, generator=generator) * inputs ** -0.5
            r = quantize_linear_module(name, w, hessian, K=BITS)
            self.stored[name] = (pack_module_trellis(r.encoded, BITS), r.su, r.sv, BITS, r.cb)
        self.frequencies, self.magnitude = rotary_frequencies(HEAD_DIM, device=device)
        self.axes = rotary_axes(SECTIONS, device=device)

    def product(self, name, x):
        return quantized_linear(x, *self.stored[name])

    def ranked(self, hidden):
        """The head's two highest tokens."""
        return self.product("head", hidden).topk(2, dim=-1).indices

    def choices(self, tokens, plan, positions, pages, tables, most, masks=None):
        """The token that follows each of the step's tokens."""
        x = self.embedding[tokens.long()]
        q, k, v = self.product("qkv", x).view(-1, Q_HEADS + 2 * KV_HEADS, HEAD_DIM).split([Q_HEADS, KV_HEADS, KV_HEADS], 1)
        turned = append_tokens(pages, k, v, plan.slots, q=q, positions=positions.expand(3, -1).contiguous(),
                               frequencies=self.frequencies, magnitude=self.magnitude, axes=self.axes)
        out = cache_attention(turned, pages, tables, plan.starts, plan.lengths, max_new=most, trees=masks)
        return self.ranked(x + self.product("o", out.flatten(1)))[:, 0].int()


def serve(tokens: int = 24, lengths=(40, 3, 75), device: str = "cuda", seed: int = 0) -> tuple:
    """The chosen tokens of every request, `tokens` or more, and the steps taken."""
    device = torch.device(device, torch.cuda.current_device())
    g = torch.Generator(device=device).manual_seed(seed)
    model = Model(device, g)
    requests, drafted = len(lengths), len(PARENTS)
    width = -(-(max(lengths) + 3 * tokens + drafted) // PAGE)    # a step keeps three at most

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=device)

    pages = cache_pages(requests * width, PAGE, KV_HEADS, HEAD_DIM, device)
    tables = torch.full((requests, width), -1, dtype=torch.int32, device=device)
    free, taken = torch.arange(requests * width, dtype=torch.int32, device=device), ints([0])
    parents, new = ints(PARENTS * requests), ints([drafted] * requests)

    prompt = torch.randint(VOCABULARY, (sum(lengths),), device=device, generator=g).int()
    plan = plan_step(ints([0] * requests), ints(lengths), tables, free, taken, page_size=PAGE, max_tokens=len(prompt))
    plan.check()
    after = model.choices(prompt, plan, plan.positions, pages, tables, max(lengths))
    chosen = after[plan.starts[1:].long() - 1]
    cached, taken, steps = plan.lengths, plan.taken, 0
    answers = [[int(t)] for t in chosen]
    while min(map(len, answers)) < tokens:
        second = model.ranked(model.embedding[chosen.long()])
        third = model.ranked(model.embedding[second.flatten()])[:, 0].view(requests, 2)
        tree = torch.cat([chosen[:, None], second.int(), third.int()], 1).flatten()
        plan = plan_step(cached, new, tables, free, taken, page_size=PAGE, max_tokens=len(tree))
        shape = plan_tree(parents, plan.starts, plan.lengths, max_new=drafted)
        after = model.choices(tree, plan, shape.positions, pages, tables, drafted, shape.masks)
        kept = accept_drafts(tree, after, parents, plan.starts, plan.lengths, max_new=drafted)
        keep_tokens(pages, plan.slots, plan.starts, kept.places)
        taken = release_pages(plan.lengths, kept.lengths, tables, free, plan.taken, page_size=PAGE)
        cached, chosen, steps = kept.lengths, kept.next, steps + 1

        plan.check()
        places, given = kept.places.view(requests, drafted).tolist(), tree.view(requests, drafted).tolist()
        for answer, place, token, last in zip(answers, places, given, chosen.tolist()):
            follow = sorted((p, t) for p, t in zip(place, token) if p > 0)
            answer += [t for _, t in follow] + [last]
    return answers, steps


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=24, help="tokens that a request decodes")
    args = ap.parse_args()
    answers, steps = serve(args.tokens)
    for answer in answers:
        print(*answer)
    print(f"{sum(map(len, answers)) - len(answers)} tokens in {steps} steps of {len(answers)} requests")

"""Serves a few requests through a small stack of selective-attention layers.

Prompts of different lengths enter packed, one after another; then every request gets one token at
a time, until some end and others take over their pages. All attention state lives in a
``PagedSelectiveCache`` (8-bit pages, grouped heads, log-gates), and no step waits for the GPU
but to read the tokens.

    python examples/serve_selective.py [--steps 24] [--code int8|e4m3]
"""
from __future__ import annotations

import argparse
import os
import sys
from collections import deque

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import selective_attention_b200 as sab  # noqa: E402

CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


class Stack:
    """Random weights: embedding, ``layers`` of selective attention with residuals, head."""

    def __init__(self, vocab=512, layers=2, heads=8, groups=2, dim=64, dtype=torch.bfloat16, seed=0, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)
        width = heads * dim
        self.layers, self.heads, self.groups, self.dim = layers, heads, groups, dim

        def weight(*shape):
            return (torch.randn(shape, generator=g, device=device) / shape[0] ** 0.5).to(dtype)

        self.embed = weight(vocab, width) * vocab ** 0.5
        self.head = weight(width, vocab)
        self.qkv = [weight(width, (heads + 2 * groups) * dim) for _ in range(layers)]
        self.gate = [weight(width, groups) for _ in range(layers)]
        self.out = [weight(width, width) for _ in range(layers)]

    def project(self, i, x):
        """Queries, keys and values as slices of one product, and the log-gates."""
        x = torch.nn.functional.rms_norm(x, x.shape[-1:])
        qkv = (x @ self.qkv[i]).view(x.shape[0], self.heads + 2 * self.groups, self.dim)
        q, k, v = qkv.split((self.heads, self.groups, self.groups), dim=1)
        return q, k, v, torch.nn.functional.logsigmoid((x @ self.gate[i]).float() + 2.0)

    def forward(self, tokens, attend):
        """``attend(layer, q, k, v, log_gate)``; the next token of every row."""
        x = self.embed[tokens]
        for i in range(self.layers):
            x = x + attend(i, *self.project(i, x)).flatten(1) @ self.out[i]
        return (torch.nn.functional.rms_norm(x, x.shape[-1:]) @ self.head).argmax(dim=-1)


def serve(prompts, budgets, rows=4, steps=24, code=torch.int8, stack=None, page_size=16, max_tokens=256):
    """Token lists of all ``prompts`` continued by up to ``budgets`` tokens each, ``rows`` at a time."""
    stack = stack or Stack()
    dev = stack.embed.device
    cache = sab.PagedSelectiveCache(stack.layers, rows, max_tokens, rows * -(-max_tokens // page_size), stack.groups,
                                    stack.dim, page_size, code, device=dev)
    waiting, running, done = deque(range(len(prompts))), {}, {i: list(p) for i, p in enumerate(prompts)}
    left = list(budgets)
    for _ in range(steps):
        # prompts into free rows
        entering = {}
        for row in range(rows):
            if row not in running and waiting:
                entering[row] = running[row] = waiting.popleft()
        if entering:
            new = torch.zeros(rows, dtype=torch.int32)
            for row, i in entering.items():
                new[row] = len(prompts[i])
            tokens = torch.tensor([t for row in sorted(entering) for t in prompts[entering[row]]], device=dev)
            cu, slots, _ = cache.plan(new.to(dev), tokens.numel())

            def attend(i, q, k, v, log_gate):
                cache.append(i, k, v, slots, log_gate)
                return sab.sattn_prefill_packed(q, k, v, cu, log_gate)

            following = stack.forward(tokens, attend)[cu[1:].long().clamp(min=1) - 1].tolist()
            for row, i in entering.items():
                done[i].append(following[row])
                left[i] -= 1
        # finished requests out
        ended = [row for row, i in running.items() if left[i] <= 0]
        if ended:
            cache.release(torch.tensor(ended, device=dev))
            for row in ended:
                del running[row]
        if not running:
            if not waiting:
                break
            continue
        # one token for every running request; the rows of the others are empty
        active = sorted(running)
        new = torch.zeros(rows, dtype=torch.int32)
        new[active] = 1
        tokens = torch.tensor([done[running[row]][-1] for row in active], device=dev)
        _, slots, _ = cache.plan(new.to(dev), len(active))
        index = torch.tensor(active, device=dev)

        def attend(i, q, k, v, log_gate):
            cache.append(i, k, v, slots, log_gate)
            wide = q.new_zeros(rows, *q.shape[1:])
            wide[index] = q
            return cache.decode(i, wide)[index]

        for row, token in zip(active, stack.forward(tokens, attend).tolist()):
            done[running[row]].append(token)
            left[running[row]] -= 1
    sab.check_device_error()
    return done, cache


def main():
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--steps", type=int, default=24)
    p.add_argument("--code", choices=sorted(CODES), default="int8")
    args = p.parse_args()
    g = torch.Generator().manual_seed(1)
    lengths = (5, 70, 1, 33, 16, 120)
    prompts = [torch.randint(512, (n,), generator=g).tolist() for n in lengths]
    done, cache = serve(prompts, [6, 4, 9, 3, 5, 7], steps=args.steps, code=CODES[args.code])
    for i, tokens in done.items():
        print(f"request {i}: {lengths[i]} prompt tokens, then {tokens[lengths[i]:]}")
    head, tail = cache.free_state.tolist()
    print(f"pages handed out {head}, returned {tail - cache.free_pages.numel()}")


if __name__ == "__main__":
    main()

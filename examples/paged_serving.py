# SPDX-License-Identifier: Apache-2.0
"""Continuous batching over a paged KV cache.

A random-weight decoder of a few attention layers serves more requests than
it has batch slots: prompts are admitted as slots and pages come free, run
through causal ``attention`` and stored by ``append``; every generation step is
one replay of a CUDA graph (reserve a slot for the new token, then per layer
append-and-attend, then the next token), which reads lengths and tables on the
GPU; finished requests release their pages.  At the end each request is
recomputed without any cache and compared.  With rotary positions on request,
and with the cache in 16 bits or in 8.

    python examples/paged_serving.py [--rotary] [--kv e4m3|int8]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from kotflash_b200 import PagedKVCache, PagedKVCache8, apply_rotary, attention, rotary_frequencies  # noqa: E402


class Decoder:
    """Embedding, `layers` of attention each with a residual and a norm, output."""

    def __init__(self, vocab, layers, hq, hkv, d, *, seed, device, dtype, rotary=False):
        g = torch.Generator(device=device).manual_seed(seed)
        width = hq * d

        def weight(*shape):
            return (torch.randn(*shape, generator=g, device=device) * shape[0] ** -0.5).to(dtype)

        self.hq, self.hkv, self.d = hq, hkv, d
        self.frequencies = rotary_frequencies(d, device=device)[0] if rotary else None
        self.embed = torch.randn(vocab, width, generator=g, device=device).to(dtype)
        self.qkv = [weight(width, (hq + 2 * hkv) * d) for _ in range(layers)]
        self.out = [weight(width, width) for _ in range(layers)]
        self.unembed = weight(width, vocab)

    def heads(self, x, layer, positions):
        """[N, S, width] -> q [N, Hq, S, D], k and v [N, Hkv, S, D] (views of one
        product), q and k rotated by positions [N, S] or [S]."""
        y = (x @ self.qkv[layer]).view(*x.shape[:2], -1, self.d).transpose(1, 2)
        q, k, v = y.split([self.hq, self.hkv, self.hkv], 1)
        if self.frequencies is not None:
            q, k = apply_rotary(q, k, positions, self.frequencies)
        return q, k, v

    def residual(self, x, o, layer):
        # random attention averages its values away: a gain keeps it audible
        x = x + 4 * (o.transpose(1, 2).reshape(x.shape) @ self.out[layer])
        return torch.nn.functional.rms_norm(x, x.shape[-1:])

    def logits(self, x):
        return (x @ self.unembed).float()

    def forward(self, tokens):
        """Logits of the last position, all positions recomputed."""
        x = self.embed[tokens][None]
        positions = torch.arange(len(tokens), device=x.device)
        for layer in range(len(self.qkv)):
            q, k, v = self.heads(x, layer, positions)
            x = self.residual(x, attention(q, k, v, causal=True), layer)
        return self.logits(x[0, -1])


@torch.inference_mode()
def serve(prompts, new_tokens, *, vocab=500, layers=2, hq=8, hkv=2, d=64, page_size=16, num_pages=64, slots=4,
          seed=0, device="cuda", dtype=torch.bfloat16, rotary=False, kv=None):
    """Generate new_tokens tokens behind each prompt (a list of token lists),
    with rotary positions or none, and the cache in dtype or in 8 bits (kv:
    "e4m3" or "int8").

    Returns the generated tokens of each request, the last logits of each, and
    the model.
    """
    model = Decoder(vocab, layers, hq, hkv, d, seed=seed, device=device, dtype=dtype, rotary=rotary)
    longest = max(map(len, prompts)) + new_tokens
    kind, held = (PagedKVCache, dtype) if kv is None else (PagedKVCache8, {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}[kv])
    cache = kind(num_pages, page_size, hkv, d, slots, -(-longest // page_size), layers=layers, device=device, dtype=held)
    tokens = torch.zeros(slots, dtype=torch.long, device=device)        # each slot's newest token
    active = torch.zeros(slots, dtype=torch.int32, device=device)       # 1 where a slot generates
    logits = torch.zeros(slots, vocab, device=device)

    def step():
        rows, _ = cache.reserve(active, tokens_per_request=1)
        positions = (cache.lengths - 1)[:, None]
        x = model.embed[tokens][:, None]
        for layer in range(layers):
            q, k, v = model.heads(x, layer, positions)
            x = model.residual(x, cache.append_and_attend(q, k, v, rows, layer=layer), layer)
        logits.copy_(model.logits(x[:, 0]))
        tokens.copy_(logits.argmax(-1))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()  # warm-up; nothing is active, so nothing is stored
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()

    waiting = list(range(len(prompts)))
    running = [None] * slots
    generated = [[] for _ in prompts]
    last = [None] * len(prompts)
    while waiting or any(r is not None for r in running):
        # admit: first come, first served, while a slot and the pages for the whole answer are there
        claimed = sum(-(-(len(prompts[r]) + new_tokens) // page_size) for r in running if r is not None)
        for slot in range(slots):
            if running[slot] is None and waiting:
                prompt = prompts[waiting[0]]
                need = -(-(len(prompt) + new_tokens) // page_size)
                if claimed + need > num_pages:
                    break
                claimed += need
                running[slot] = request = waiting.pop(0)
                added = torch.zeros(slots, dtype=torch.int32, device=device)
                added[slot] = len(prompt)
                rows, _ = cache.reserve(added, num_tokens=len(prompt))
                x = model.embed[torch.tensor(prompt, device=device)][None]
                positions = torch.arange(len(prompt), device=device)
                for layer in range(layers):
                    q, k, v = model.heads(x, layer, positions)
                    cache.append(k, v, rows, layer=layer)
                    x = model.residual(x, attention(q, k, v, causal=True), layer)
                last[request] = model.logits(x[0, -1])
                tokens[slot] = last[request].argmax()
                generated[request].append(int(tokens[slot]))
                active[slot] = 1
        if not any(r is not None for r in running):
            raise RuntimeError("a prompt needs more pages than the pool has")
        graph.replay()
        newest = tokens.tolist()
        finished = [False] * slots
        for slot, request in enumerate(running):
            if request is None:
                continue
            if len(generated[request]) < new_tokens:
                generated[request].append(newest[slot])
                last[request] = logits[slot].clone()
            if len(generated[request]) == new_tokens:
                finished[slot], running[slot] = True, None
        if any(finished):
            done = torch.tensor(finished, device=device)
            cache.release(done)
            active.masked_fill_(done, 0)
    assert int(cache.free_count) == num_pages, "every page came back"
    del graph
    return generated, last, model


def main():
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--rotary", action="store_true", help="rotary positions")
    ap.add_argument("--kv", choices=["e4m3", "int8"], help="hold the cache in 8 bits")
    args = ap.parse_args()
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(500, (n,), generator=g).tolist() for n in (5, 130, 16, 64, 1, 77, 200, 33)]
    generated, last, model = serve(prompts, 24, rotary=args.rotary, kv=args.kv)
    for prompt, answer, got in zip(prompts, generated, last):
        with torch.inference_mode():
            want = model.forward(torch.tensor(prompt + answer[:-1], device="cuda"))
        print(f"prompt of {len(prompt):3d}: {answer[:6]} ...  largest difference of the last logits from a "
              f"recomputation: {(got - want).abs().max():.4f} (logits up to {want.abs().max():.1f})")


if __name__ == "__main__":
    main()

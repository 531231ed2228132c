#!/usr/bin/env python3
"""Generate several tokens a step from a streamed, compressed model with fp8 weights.

Writes a small random Llama-architecture model, its projections in e4m3 with a scale for each block of 128 by 128, as a .bs
container. Drafts are looked up in the text so far: what followed the last two tokens where they last stood side by side. A
step computes all drafts at once, keeps those that the model agrees with, and the cache takes the others back.

    python examples/draft_generate.py [--layers 4] [--tokens 48] [--drafts 4] [--temperature 0.0]
"""
import argparse
import sys
import tempfile
import time
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import torch
from transformers import LlamaConfig

import bigsmall_amd
from bigsmall_amd.paged_llama import PagedLlama


def fp8_blocks(w):
    """w in e4m3 codes and a scale for each block of 128 by 128."""
    n, k = w.shape
    blocks = w.view(n // 128, 128, k // 128, 128)
    scale = (blocks.abs().amax((1, 3)) / 448).clamp(min=1e-12)
    return (blocks / scale[:, None, :, None]).view(n, k).to(torch.float8_e4m3fn), scale


def random_model(config, seed=0):
    g = torch.Generator().manual_seed(seed)
    h, d = config.hidden_size, config.hidden_size // config.num_attention_heads
    kv, ff = config.num_key_value_heads * d, config.intermediate_size

    def matrix(rows, cols):
        return torch.randn(rows, cols, generator=g) * cols ** -0.5

    sd = {"model.embed_tokens.weight": matrix(config.vocab_size, h).bfloat16(), "lm_head.weight": matrix(config.vocab_size, h).bfloat16(),
          "model.norm.weight": torch.ones(h).bfloat16()}
    for i in range(config.num_hidden_layers):
        p = f"model.layers.{i}."
        for name, rows, cols in (("self_attn.q_proj", h, h), ("self_attn.k_proj", kv, h), ("self_attn.v_proj", kv, h),
                                 ("self_attn.o_proj", h, h), ("mlp.gate_proj", ff, h), ("mlp.up_proj", ff, h), ("mlp.down_proj", h, ff)):
            sd[p + name + ".weight"], sd[p + name + ".weight_scale_inv"] = fp8_blocks(matrix(rows, cols))
        for name in ("input_layernorm", "post_attention_layernorm"):
            sd[p + name + ".weight"] = torch.ones(h).bfloat16()
    return sd


def lookup(tokens, lengths, n):
    """The n tokens after the last place where the text's last two stood before; the last token again where they never did."""
    b, width = tokens.shape
    row, end = torch.arange(b, device=tokens.device), lengths.long()
    two = torch.stack([tokens[row, (end - 2).clamp(min=0)], tokens[row, end - 1]], 1)
    at = torch.arange(width - 1, device=tokens.device)
    same = (tokens[:, :-1] == two[:, :1]) & (tokens[:, 1:] == two[:, 1:]) & (at < end[:, None] - 2)
    last = torch.where(same, at, -1).amax(1)
    follow = last[:, None] + 2 + torch.arange(n, device=tokens.device)
    found = (last[:, None] >= 0) & (follow < end[:, None])
    return torch.where(found, tokens[row[:, None], follow.clamp(0, width - 1)], two[:, 1:]), None


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=48)
    ap.add_argument("--drafts", type=int, default=4)
    ap.add_argument("--temperature", type=float, default=0.0)
    args = ap.parse_args()
    config = LlamaConfig(hidden_size=1024, intermediate_size=2816, num_hidden_layers=args.layers, num_attention_heads=8,
                         num_key_value_heads=2, vocab_size=8192, max_position_embeddings=4096)
    with tempfile.TemporaryDirectory() as tmp:
        path = str(Path(tmp) / "model.bs")
        bigsmall_amd.compress(random_model(config), path)
        with bigsmall_amd.StreamingLoader(path, device="cuda", prefetch=1) as loader:
            model = PagedLlama(loader, config, pages=512, sequences=8)
            g = torch.Generator().manual_seed(1)
            prompts = [torch.randint(config.vocab_size, (n,), generator=g) for n in (5, 64, 200, 777)]
            steps = []

            def draft(tokens, lengths, n):
                steps.append(n)
                return lookup(tokens, lengths, n)

            for name, what in (("one token a step", {}), ("drafts", {"draft": draft, "drafts": args.drafts})):
                torch.cuda.synchronize()
                t = time.perf_counter()
                out = model.generate(prompts, args.tokens, temperature=args.temperature, **what)
                torch.cuda.synchronize()
                print(f"{name}: {args.tokens} tokens of {len(prompts)} sequences in {time.perf_counter() - t:.3f} s")
            print(f"{len(steps)} steps with drafts")
            for p, o in zip(prompts, out):
                print(f"prompt of {len(p)} tokens -> {o.tolist()}")


if __name__ == "__main__":
    main()

#!/usr/bin/env python3
"""Generate with a paged 8-bit KV cache from a streamed, compressed model.

Writes a small random Llama-architecture model as a .bs container, generates for a few prompts of different lengths in
one batch, parks a conversation in the compressed store and brings it back.

    python examples/paged_generate.py [--layers 4] [--tokens 16] [--fp8]
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


def random_model(config, seed=0):
    g = torch.Generator().manual_seed(seed)
    h, d = config.hidden_size, config.hidden_size // config.num_attention_heads
    kv, ff = config.num_key_value_heads * d, config.intermediate_size

    def matrix(rows, cols):
        return (torch.randn(rows, cols, generator=g) * cols ** -0.5).bfloat16()

    sd = {"model.embed_tokens.weight": matrix(config.vocab_size, h), "lm_head.weight": matrix(config.vocab_size, h),
          "model.norm.weight": torch.ones(h).bfloat16()}
    for i in range(config.num_hidden_layers):
        p = f"model.layers.{i}."
        for name, rows, cols in (("self_attn.q_proj", h, h), ("self_attn.k_proj", kv, h), ("self_attn.v_proj", kv, h),
                                 ("self_attn.o_proj", h, h), ("mlp.gate_proj", ff, h), ("mlp.up_proj", ff, h), ("mlp.down_proj", h, ff)):
            sd[p + name + ".weight"] = matrix(rows, cols)
        for name in ("input_layernorm", "post_attention_layernorm"):
            sd[p + name + ".weight"] = torch.ones(h).bfloat16()
    return sd


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=16)
    ap.add_argument("--fp8", action="store_true", help="e4m3 pages instead of int8")
    args = ap.parse_args()
    config = LlamaConfig(hidden_size=1024, intermediate_size=2816, num_hidden_layers=args.layers, num_attention_heads=8,
                         num_key_value_heads=2, vocab_size=8192, max_position_embeddings=4096)
    kind = torch.float8_e4m3fn if args.fp8 else torch.int8
    with tempfile.TemporaryDirectory() as tmp:
        path = str(Path(tmp) / "model.bs")
        bigsmall_amd.compress(random_model(config), path)
        with bigsmall_amd.StreamingLoader(path, device="cuda", prefetch=1) as loader:
            model = PagedLlama(loader, config, pages=512, sequences=8, kind=kind)
            g = torch.Generator().manual_seed(1)
            prompts = [torch.randint(config.vocab_size, (n,), generator=g) for n in (5, 64, 200, 777)]
            torch.cuda.synchronize()
            t = time.perf_counter()
            for p, out in zip(prompts, model.generate(prompts, args.tokens)):
                print(f"prompt of {len(p)} tokens -> {out.tolist()}")
            torch.cuda.synchronize()
            print(f"{args.tokens} steps of {len(prompts)} sequences in {time.perf_counter() - t:.3f} s")

            seq = model.cache.add()
            logits = model.forward({seq: prompts[2]})
            store = bigsmall_amd.CompressedKVCache(device="cuda")
            model.park(seq, store)
            print(store, f"{model.cache.free_pages()} pages free")
            seq = model.resume(seq, store)
            logits = model.forward({seq: logits.argmax(-1)})
            print("the parked conversation goes on with token", int(logits.argmax(-1)))


if __name__ == "__main__":
    main()

"""PagedLlama: a Llama-architecture model that generates from a paged KV cache,
its layers streamed from a BigSmall container.

The reference streams layers through the HuggingFace module and keeps its
bf16 cache (bigsmall/streaming_inference.py:77-347); here a step takes the new
tokens of any number of sequences at once (whole prompts, parts of prompts and
single tokens side by side), and K and V go rotated into a PagedKVCache in 8
bits, from which attention reads them.

The rest of a layer is the architecture's own arithmetic in torch: RMS norm,
projections without bias, SwiGLU. Tensor names follow the HuggingFace layout:
`model.embed_tokens`, `model.layers.<i>.*`, `model.norm`, `lm_head`. Models that
need anything else are refused (`check_model`).
"""
from __future__ import annotations

import torch
from torch.nn.functional import linear, silu

from .paged_kv import PagedKVCache, Rope


_TOP = {"model.embed_tokens.weight", "model.norm.weight", "lm_head.weight"}
_LAYER = {"input_layernorm.weight", "post_attention_layernorm.weight"} | \
    {f"self_attn.{n}_proj.weight" for n in "qkvo"} | {f"mlp.{n}_proj.weight" for n in ("gate", "up", "down")}
_UNUSED = "rotary_emb.inv_freq"       # a buffer that old checkpoints hold


def check_model(config, loader, rope=None) -> None:
    """ValueError if PagedLlama does not compute this model: another architecture, activation or rotation than it has,
    a sliding window, or tensors (biases, further norms) that it would pass over."""
    kind = getattr(config, "model_type", "llama")
    if kind not in ("llama", "mistral"):
        raise ValueError(f"PagedLlama does not compute models of type {kind!r}")
    window = getattr(config, "sliding_window", None)
    if window is not None and window < config.max_position_embeddings:
        raise ValueError(f"PagedLlama attends to all tokens; the model has a sliding window of {window}")
    if getattr(config, "hidden_act", "silu") not in ("silu", "swish"):
        raise ValueError(f"PagedLlama's activation is silu, the model's {config.hidden_act}")
    for bias in ("attention_bias", "mlp_bias"):
        if getattr(config, bias, False):
            raise ValueError(f"PagedLlama has no biases; the model has {bias}")
    if rope is None:
        given = getattr(config, "rope_parameters", None) or getattr(config, "rope_scaling", None) or {}
        variant = given.get("rope_type") or given.get("type") or "default"
        part = given.get("partial_rotary_factor") or getattr(config, "partial_rotary_factor", None) or 1.0
        if variant != "default" or part != 1.0:
            raise ValueError(f"the model's rotation is {variant!r} over {part} of a head; pass its angles as `rope`")
    layers = loader.layer_count()
    if layers != getattr(config, "num_hidden_layers", layers):
        raise ValueError(f"the config has {config.num_hidden_layers} layers, the container {layers}")
    groups = [("", set(loader.non_layer_tensor_names()), _TOP, _TOP - {"lm_head.weight"})]
    groups += [(f"model.layers.{i}.", set(loader.layer_tensor_names(i)), _LAYER, _LAYER) for i in range(layers)]
    for prefix, names, known, needed in groups:
        missing = {prefix + n for n in needed} - names
        other = {n for n in names if not n.endswith(_UNUSED)} - {prefix + n for n in known}
        if missing or other:
            raise ValueError("PagedLlama: " + "; ".join(f"{what}: {', '.join(sorted(x)[:4])}" for what, x in
                                                        (("missing tensors", missing), ("tensors it does not use", other)) if x))


class PagedLlama:
    """loader: a StreamingLoader on a GPU; its `prefetch` sets how many layers decode ahead.
    config: the model's transformers.LlamaConfig (plain rotation; scaled or partial ones: pass `rope`).
    pages, sequences: what the cache holds at most; kind: torch.int8 or torch.float8_e4m3fn."""

    def __init__(self, loader, config, pages: int, sequences: int, kind=torch.int8, rope: Rope | None = None):
        check_model(config, loader, rope)
        self.loader, self.config = loader, config
        self.heads, self.kv_heads = config.num_attention_heads, config.num_key_value_heads
        self.dim = getattr(config, "head_dim", None) or config.hidden_size // self.heads
        top = loader.load_non_layer_tensors()
        self.embed, self.norm = top["model.embed_tokens.weight"], top["model.norm.weight"]
        self.head = top.get("lm_head.weight", self.embed)
        self.device = self.embed.device
        self.cache = PagedKVCache(loader.layer_count(), self.kv_heads, self.dim, pages, sequences, kind, self.device)
        if rope is None:
            theta = getattr(config, "rope_theta", None) or config.rope_parameters["rope_theta"]
            rope = Rope.from_theta(self.dim, config.max_position_embeddings, theta, device=self.device)
        self.rope = rope

    def _norm(self, x, weight):
        y = x.float()
        return weight * (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + self.config.rms_norm_eps)).to(x.dtype)

    @torch.no_grad()
    def forward(self, new: dict) -> torch.Tensor:
        """new: {sequence: its new token ids (1-D)}; sequences come from `self.cache.add()`. Returns the
        logits [sequences, vocab] after each sequence's last new token, in the dict's order. If it raises, the
        sequences are as they were before."""
        ids = [torch.as_tensor(t).to(self.device) for t in new.values()]
        step = self.cache.step({seq: len(t) for seq, t in zip(new, ids)})
        try:
            return self._forward(step, torch.cat(ids))
        except BaseException:         # the cache would claim tokens that some layer never got
            self.cache.undo(step)
            raise

    def _forward(self, step, ids):
        x = self.embed[ids]
        t = x.shape[0]
        for i, layer in self.loader.iter_layers(progress=False):
            p = f"model.layers.{i}."
            y = self._norm(x, layer[p + "input_layernorm.weight"])
            q, k, v = (linear(y, layer[p + f"self_attn.{n}_proj.weight"]).view(t, -1, self.dim) for n in "qkv")
            q = self.cache.append(i, step, q, k, v, self.rope)
            y = self.cache.attend(i, step, q)
            x = x + linear(y.view(t, -1), layer[p + "self_attn.o_proj.weight"])
            y = self._norm(x, layer[p + "post_attention_layernorm.weight"])
            y = silu(linear(y, layer[p + "mlp.gate_proj.weight"])) * linear(y, layer[p + "mlp.up_proj.weight"])
            x = x + linear(y, layer[p + "mlp.down_proj.weight"])
        last = step.cu[1:].long() - 1
        return linear(self._norm(x[last], self.norm), self.head)

    def generate(self, prompts: list, max_new_tokens: int) -> list:
        """Greedy continuations of prompts (1-D token ids), all in one batch."""
        seqs = []
        try:
            for _ in prompts:
                seqs.append(self.cache.add())
            logits, out = self.forward(dict(zip(seqs, prompts))), []
            for n in range(max_new_tokens):
                out.append(logits.argmax(-1))
                if n + 1 < max_new_tokens:
                    logits = self.forward({s: out[-1][j:j + 1] for j, s in enumerate(seqs)})
            return list(torch.stack(out, 1)) if out else [torch.empty(0, dtype=torch.int64) for _ in prompts]
        finally:
            for s in seqs:
                self.cache.drop(s)

    def park(self, seq: int, store) -> None:
        """Move a sequence's K and V, as bf16, into a CompressedKVCache under (seq, layer) and drop it here.
        A sequence without tokens has nothing to keep: ValueError."""
        if not self.cache.length(seq):
            raise ValueError(f"sequence {seq} has no tokens to park")
        for i in range(len(self.cache.pools)):
            store.set((seq, i), *self.cache.read(i, seq))
        self.cache.drop(seq)

    def resume(self, seq: int, store) -> int:
        """Bring a parked sequence back: its K and V are already rotated. Returns its new number."""
        new, step = self.cache.add(), None
        try:
            for i in range(len(self.cache.pools)):
                k, v = (x.transpose(0, 1).to(self.device) for x in store.get((seq, i)))
                step = step or self.cache.step({new: k.shape[0]})
                self.cache.append(i, step, None, k, v)
        except BaseException:
            self.cache.drop(new)
            raise
        return new


__all__ = ["PagedLlama"]

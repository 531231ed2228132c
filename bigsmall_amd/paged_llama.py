"""PagedLlama: a Llama-architecture model that generates from a paged KV cache,
its layers streamed from a BigSmall container.

The reference streams layers through the HuggingFace module and keeps its
bf16 cache (bigsmall/streaming_inference.py:77-347); here a step takes the new
tokens of any number of sequences at once (whole prompts, parts of prompts and
single tokens side by side), and K and V go rotated into a PagedKVCache in 8
bits, from which attention reads them.

The rest of a layer is the architecture's own arithmetic in torch: RMS norm,
projections without bias, SwiGLU. Projections whose weight is e4m3, with a
`weight_scale_inv` beside it (f32, one scale for each block of 128 by 128), are
products of fp8 (`fp8_linear`). Tensor names follow the HuggingFace layout:
`model.embed_tokens`, `model.layers.<i>.*`, `model.norm`, `lm_head`. Models that
need anything else are refused (`check_model`).

`generate` takes drafts: a guess at the next few tokens of each sequence, all of
which one step then computes; `draft_verify` keeps as many as agree with the model,
and the cache's tables on the GPU (`KVTables`) take the others back.
"""
from __future__ import annotations

import torch
from torch.nn.functional import linear, silu

from .device import StatusWord
from .draft import MOST_DRAFTS, draft_verify
from .fp8 import BLOCK, Fp8Weight, fp8_linear, fp8_quantise
from .paged_kv import PAGE, PagedKVCache, Rope


_TOP = {"model.embed_tokens.weight", "model.norm.weight", "lm_head.weight"}
_PROJECTIONS = {f"self_attn.{n}_proj.weight" for n in "qkvo"} | {f"mlp.{n}_proj.weight" for n in ("gate", "up", "down")}
_LAYER = {"input_layernorm.weight", "post_attention_layernorm.weight"} | _PROJECTIONS
_SCALES = {n + "_scale_inv" for n in _PROJECTIONS}        # of fp8 weights
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
    groups += [(f"model.layers.{i}.", set(loader.layer_tensor_names(i)), _LAYER | _SCALES, _LAYER) for i in range(layers)]
    scaled = any(n.endswith("_scale_inv") for _, names, _, _ in groups for n in names)
    quantised = getattr(config, "quantization_config", None)
    if scaled and quantised is not None:
        q = quantised if isinstance(quantised, dict) else quantised.to_dict()
        if q.get("quant_method") != "fp8" or list(q.get("weight_block_size") or ()) != [BLOCK, BLOCK] or q.get("activation_scheme") != "dynamic":
            raise ValueError(f"PagedLlama computes fp8 weights with a scale for each block of {BLOCK} by {BLOCK}; the model is quantised otherwise: {q}")
    if scaled and getattr(loader, "dtype", None) is not None:
        raise ValueError("PagedLlama: fp8 weights and their scales are taken as they are stored; the loader casts them to " + str(loader.dtype))
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
        x = self._hidden(step, ids)
        return self._logits(x[step.cu[1:].long() - 1])

    def _logits(self, x):
        return linear(self._norm(x, self.norm), self.head)

    @staticmethod
    def _project(x, layer, *names):
        """x through the projections `names`, whatever their weights are held in; quantised once for all of fp8."""
        out, rows = [], None
        for name in names:
            w = layer[name + ".weight"]
            if w.dtype == torch.float8_e4m3fn:
                if name + ".weight_scale_inv" not in layer:
                    raise ValueError(f"PagedLlama: {name} is held in fp8 without {name}.weight_scale_inv")
                rows = (x if len(names) == 1 else fp8_quantise(x)) if rows is None else rows
                out.append(fp8_linear(rows, Fp8Weight(w, layer[name + ".weight_scale_inv"])))
            else:
                out.append(linear(x, w))
        return out

    def _hidden(self, step, ids):
        """The last layer's output for a step's rows."""
        x = self.embed[ids]
        t = x.shape[0]
        for i, layer in self.loader.iter_layers(progress=False):
            p = f"model.layers.{i}."
            y = self._norm(x, layer[p + "input_layernorm.weight"])
            q, k, v = (z.view(t, -1, self.dim) for z in self._project(y, layer, *(p + f"self_attn.{n}_proj" for n in "qkv")))
            q = self.cache.append(i, step, q, k, v, self.rope)
            y = self.cache.attend(i, step, q)
            x = x + self._project(y.view(t, -1), layer, p + "self_attn.o_proj")[0]
            y = self._norm(x, layer[p + "post_attention_layernorm.weight"])
            gate, up = self._project(y, layer, p + "mlp.gate_proj", p + "mlp.up_proj")
            x = x + self._project(silu(gate) * up, layer, p + "mlp.down_proj")[0]
        return x

    def generate(self, prompts: list, max_new_tokens: int, draft=None, drafts: int = 4, temperature: float = 0.0, generator=None) -> list:
        """Continuations of prompts (1-D token ids), all in one batch; greedy, or drawn at `temperature` (generator: a
        torch.Generator of the device).

        draft: a callable (tokens, lengths, n) -> (ids, probabilities) that guesses the next n tokens of each sequence from
        tokens int64 [sequences, ...], of which row i begins with the lengths[i] (int32) tokens so far; ids int64
        [sequences, n], and the probabilities [sequences, n, vocab] (f32) that they were drawn from, or None if they were
        not drawn. Up to `drafts` of them, and 1,024, are computed in one step; what comes out is distributed as without drafts (greedy:
        the same tokens, as far as steps of more rows round alike). RuntimeError where a row that a token is drawn from has no
        probability at all, or the cache has too few pages free; what the sequences do not need stays free meanwhile."""
        if draft is not None or temperature:
            return self._generate_drafted(prompts, max_new_tokens, draft, drafts, temperature, generator)
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

    def _probabilities(self, logits, temperature):
        if temperature:
            x = logits.float()         # (the largest first taken off: no temperature makes it an infinity)
            return torch.softmax((x - x.amax(-1, keepdim=True)) / max(temperature, 1e-30), -1)
        one = torch.zeros(logits.shape, dtype=torch.float32, device=logits.device)
        return one.scatter_(1, logits.argmax(-1, keepdim=True), 1.0)

    @torch.no_grad()
    def _generate_drafted(self, prompts, max_new_tokens, draft, drafts, temperature, generator):
        if draft is None:
            drafts = 0
        if drafts < 0 or not 0.0 <= temperature < float("inf"):
            raise ValueError(f"drafts {drafts} and temperature {temperature} must not be negative or infinite")
        drafts = min(drafts, MOST_DRAFTS)
        if not prompts or max_new_tokens < 1:
            return [torch.empty(0, dtype=torch.int64) for _ in prompts]
        b, dev = len(prompts), self.device
        ids = [torch.as_tensor(t).to(dev).long() for t in prompts]
        if min(len(t) for t in ids) < 1:
            raise ValueError("a prompt needs at least one token")
        flat = torch.cat(ids)
        if not 0 <= int(flat.min()) <= int(flat.max()) < self.embed.shape[0]:
            raise ValueError("a prompt holds ids that are no tokens")
        longest = max(len(t) for t in ids) + max_new_tokens
        # the last token is not cached, and drafts that are taken back complete no page: the rest of the pages stays with the cache
        pages = max(1, sum((len(t) + max_new_tokens - 1) // PAGE for t in ids))
        places = torch.arange(b, dtype=torch.int32, device=dev)
        status, drawn = StatusWord(dev), StatusWord(dev)

        def i32(x):
            return torch.tensor(x, dtype=torch.int32, device="cpu").to(dev)

        def rand(n):
            return torch.rand(n, generator=generator, dtype=torch.float32, device=dev)

        def run(tables, new, sure, rows, widest, reach):
            step, at = tables.step(places, new, sure, rows=rows, max_new=widest, max_len=reach, status=status)
            if int(status.t):
                raise RuntimeError(f"PagedLlama.generate: {tables.free.shape[0]} pages do not hold {b} sequences of up to {longest} tokens")
            return step, at

        def numbers(counts):
            *n, nothing = torch.cat([counts, drawn.t]).tolist()
            if nothing:
                raise RuntimeError("PagedLlama.generate: the model's logits leave no probability to draw from (they hold a NaN or an infinity)")
            return n

        with self.cache.tables(b, longest, pages) as tables:
            tokens = torch.zeros(b, tables.longest + drafts + 1, dtype=torch.int64, device=dev)   # (room for what is cut off at the end)
            row = torch.arange(b, device=dev)
            lens = [len(t) for t in ids]
            step, at = run(tables, i32(lens), None, sum(lens), max(lens), max(lens))
            tokens[at.owner, at.position] = flat
            x = self._hidden(step, flat)
            tables.keep(step)
            p = self._probabilities(self._logits(x[step.cu[1:].long() - 1]), temperature)
            every = torch.arange(b + 1, dtype=torch.int32, device=dev)
            new, counts = draft_verify(p, torch.zeros(b, dtype=torch.int64, device=dev), every, rand(b), rand(b), max_drafts=0, status=drawn)
            lengths = i32(lens)                         # tokens so far, the last of which is not in the cache yet
            tokens[row, lengths.long()] = new[:, 0]
            lengths = lengths + 1
            made = numbers(counts)
            while min(made) < max_new_tokens:
                left = [max_new_tokens - m for m in made]
                n = min(drafts, max(left) - 1)
                guess, q = draft(tokens, lengths, n) if n else (torch.empty(b, 0, dtype=torch.int64, device=dev), None)
                if guess.shape != (b, n) or (q is not None and q.shape != (b, n, self.head.shape[0])):
                    raise ValueError(f"draft returned {tuple(guess.shape)} ids" + (f" and {tuple(q.shape)} probabilities" if q is not None else ""))
                if n and not 0 <= int(guess.min()) <= int(guess.max()) < self.embed.shape[0]:
                    raise ValueError("draft returned ids that are no tokens")
                # a sequence that has all of its tokens takes no part, and none guesses past its end
                wanted = i32([min(1 + n, m) for m in left])
                sure = i32([min(1, m) for m in left])
                reach = max(a + m - 1 + min(1 + n, k) for a, m, k in zip(lens, made, left))
                step, at = run(tables, wanted, sure, b * (1 + n), 1 + n, reach)
                given = torch.cat([tokens[row, lengths.long() - 1][:, None], guess.long(), torch.zeros(b, 1, dtype=torch.int64, device=dev)], 1)
                covered = at.owner >= 0
                owner = torch.where(covered, at.owner, 0).long()
                place = torch.where(covered, at.position - step.start[owner], 0).long()       # of a row among its sequence's
                x = self._hidden(step, given[owner, place])
                p = self._probabilities(self._logits(x), temperature)
                q = q[owner, place.clamp(max=n - 1)].float() if q is not None else None
                new, counts = draft_verify(p, given[owner, place + 1], step.cu, rand(len(owner)), rand(b), q=q, max_drafts=n, status=drawn)
                tables.keep(step, counts)               # the last token and the drafts that were taken
                to = lengths[:, None].long() + torch.arange(1 + n, device=dev)
                kept = torch.arange(1 + n, device=dev) < counts[:, None]
                tokens[row[:, None].expand_as(to)[kept], to[kept]] = new[kept]
                lengths = lengths + counts
                made = [min(max_new_tokens, m + c) for m, c in zip(made, numbers(counts))]
            return [tokens[i, k:k + max_new_tokens].clone() for i, k in enumerate(lens)]

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

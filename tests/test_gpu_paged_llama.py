"""PagedLlama against HuggingFace's own module on the same weights."""
from __future__ import annotations

import runpy
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    from transformers import LlamaConfig, LlamaForCausalLM

    import bigsmall_amd
    config = LlamaConfig(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                         vocab_size=500, max_position_embeddings=512, attn_implementation="eager", tie_word_embeddings=False)
    torch.manual_seed(0)
    hf = LlamaForCausalLM(config).to(torch.bfloat16).eval()
    with torch.no_grad():
        for p in hf.parameters():           # scores that tell keys apart
            if p.dim() == 2:
                p.mul_(4.0)
    path = tmp_path_factory.mktemp("llama") / "model.bs"
    bigsmall_amd.compress({k: v.contiguous() for k, v in hf.state_dict().items()}, str(path))
    return path, config, hf.float()


# What separates the two: K and V in 8 bits, and activations in bf16 where the module computes in f32. A value is off by
# half a step at most: int8 pages 1/254 of the page's largest, about 4.5 standard deviations, so 1 % of a value's size in
# the mean square; e4m3 1/16 of itself, 2.6 %. Activations add about ten roundings of 2^-9 a layer. Bound: three times the sum.
@pytest.mark.parametrize("kind,bound", [(torch.int8, 0.06), (torch.float8_e4m3fn, 0.12)])
def test_logits_match_the_module(model, kind, bound):
    import bigsmall_amd
    from bigsmall_amd.paged_llama import PagedLlama
    path, config, hf = model
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(config.vocab_size, (n,), generator=g) for n in (150, 37, 64)]
    with bigsmall_amd.StreamingLoader(str(path), device="cuda") as loader:
        m = PagedLlama(loader, config, pages=16, sequences=4, kind=kind)
        seqs = [m.cache.add() for _ in prompts]
        logits = m.forward(dict(zip(seqs, prompts)))
        for step in range(3):
            for j, ids in enumerate(prompts):
                with torch.no_grad():
                    want = hf(ids[None]).logits[0, -1]
                got = logits[j].float().cpu()
                assert float((got - want).norm() / want.norm()) < bound, (step, j)
            nxt = [torch.randint(config.vocab_size, (n,), generator=g) for n in ((1, 1, 1), (1, 30, 1), (2, 1, 70))[step]]
            prompts = [torch.cat([p, t]) for p, t in zip(prompts, nxt)]
            logits = m.forward(dict(zip(seqs, nxt)))
        # parked in the compressed store and brought back, a sequence goes on as before: its bf16 values are the cache's
        store = bigsmall_amd.CompressedKVCache(device="cuda")
        kept = [m.cache.read(i, seqs[0]) for i in range(2)]
        m.park(seqs[0], store)
        for i, (k, v) in enumerate(kept):
            k2, v2 = store.get((seqs[0], i))
            assert torch.equal(k, k2) and torch.equal(v, v2)
        back = m.resume(seqs[0], store)
        token = torch.tensor([7])
        got = m.forward({back: token})[0].float().cpu()
        with torch.no_grad():
            want = hf(torch.cat([prompts[0], token])[None]).logits[0, -1]
        assert float((got - want).norm() / want.norm()) < bound


def test_generate_takes_and_returns_pages(model):
    import bigsmall_amd
    from bigsmall_amd.paged_llama import PagedLlama
    path, config, _ = model
    with bigsmall_amd.StreamingLoader(str(path), device="cuda") as loader:
        m = PagedLlama(loader, config, pages=10, sequences=2)
        a = torch.arange(70) % config.vocab_size
        one, two = m.generate([a, a[:9]], 5)
        assert len(one) == len(two) == 5 and m.cache.free_pages() == 10
        assert torch.equal(m.generate([a], 5)[0], one)                     # alone or beside another
        with pytest.raises(RuntimeError, match="pages"):
            m.generate([torch.zeros(400, dtype=torch.int64)] * 2, 1)      # 12 pages
        assert m.cache.free_pages() == 10


def test_example_runs(monkeypatch, capsys):
    monkeypatch.setattr(sys, "argv", ["paged_generate.py", "--layers", "2", "--tokens", "3", "--fp8"])
    runpy.run_path(str(ROOT / "examples" / "paged_generate.py"), run_name="__main__")
    assert "goes on with token" in capsys.readouterr().out

"""PagedLlama with fp8 weights and with drafts; the cache's tables with its append and attention."""
from __future__ import annotations

import runpy
import sys
from pathlib import Path

import pytest
import torch

import fp8_reference as ref
from test_gpu_paged_llama import model  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]
PAGE = 64


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---- the tables with the cache

@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
def test_what_is_taken_back_leaves_no_trace(kind):
    """Two sequences in steps of some certain tokens and drafts that are partly taken back, across page borders: what the
    cache holds is bit for bit what one append of the kept tokens gives, and attention sees nothing else."""
    import bigsmall_amd as bs
    hk, hq, d, g = 2, 4, 64, torch.Generator().manual_seed(5)
    cache = bs.PagedKVCache(1, hk, d, pages=40, sequences=4, kind=kind)
    rope = bs.Rope.from_theta(d, 700)
    whole = [[torch.randn(700, h, d, generator=g).bfloat16().cuda() for h in (hq, hk, hk)] for _ in range(2)]
    have, y_parts = [0, 0], [[], []]
    with cache.tables(2, 640) as tables:
        assert cache.free_pages() == 0
        for i in range(60):
            new = [1 + (i * 7 + s * 3) % 6 if i else (50, 120)[s] for s in range(2)]
            sure = [1 + (i % 3 == 0) if i else n for n in new]
            sure = [min(a, b) for a, b in zip(sure, new)]
            rows = sum(new) + 3
            step, at = tables.step(_i32(0, 1), _i32(*new), _i32(*sure), rows=rows, max_new=max(new))
            cu, start = step.cu.tolist(), step.start.tolist()
            assert start == have
            q, k, v = (torch.full((rows, h, d), float("nan"), dtype=torch.bfloat16, device="cuda") for h in (hq, hk, hk))
            for s in range(2):
                n = cu[s + 1] - cu[s]
                sel = slice(cu[s], cu[s + 1])
                for x, w in zip((q, k, v), whole[s]):
                    x[sel] = w[have[s]:have[s] + n]
                wrong = have[s] + sure[s]                       # drafts that will be taken back hold other values
                keep = sure[s] + (i + s) % (n - sure[s] + 1)
                for x in (k, v):
                    x[cu[s] + keep:cu[s + 1]] = 100.0
                assert wrong <= have[s] + keep <= have[s] + n
            kept = _i32(*(sure[s] + (i + s) % (cu[s + 1] - cu[s] - sure[s] + 1) for s in range(2)))
            qr = cache.append(0, step, q, k, v, rope)
            y = cache.attend(0, step, qr)
            tables.keep(step, kept)
            for s, n in enumerate(kept.tolist()):
                y_parts[s].append(y[cu[s]:cu[s] + n].clone())
                have[s] += n
            assert tables.length.tolist() == have
        stored = []
        for s in range(2):
            tail = (tables.tails[s] + tables.which[s]).view(1)
            stored.append(bs.kv_read(cache.pools[0], tables.table[s], have[s], tail))
    assert cache.free_pages() == 40
    for s in range(2):
        seq = cache.add()
        step = cache.step({seq: have[s]})
        q, k, v = (w[:have[s]] for w in whole[s])
        qr = cache.append(0, step, q, k, v, rope)
        for a, b in zip(stored[s], cache.read(0, seq)):
            assert torch.equal(a, b)
        # the same keys in steps of other lengths: weights of 11 bits and an output of 8 round apart by half a step each
        # (values are below 5 standard deviations, a weighted mean of them below the largest)
        one = cache.attend(0, step, qr).float()
        got = torch.cat(y_parts[s]).float()
        # a token still in the tail when it was seen first was seen in bf16, later in 8 bits: off by half a code of the page's largest
        # (int8 1/254 of it, e4m3 1/16 of the value), weighted by probabilities that move by twice the scores' change
        big = float(whole[s][2][:have[s]].float().abs().max())
        assert float((one - got).abs().max()) < big * (2 ** -7 + (3 / 254 if kind == torch.int8 else 3 / 16))
        cache.drop(seq)


def test_lending():
    import bigsmall_amd as bs
    cache = bs.PagedKVCache(1, 1, 64, pages=6, sequences=3)
    a = cache.add()
    x = torch.randn(130, 1, 64, device="cuda").bfloat16()
    cache.append(0, cache.step({a: 130}), None, x, x)
    for sequences, pages in ((3, None), (0, 1), (1, 5), (1, 0)):
        with pytest.raises(RuntimeError, match="free"):
            cache.tables(sequences, 100, pages)
    one = cache.tables(1, 200, 3)
    assert cache.free_pages() == 1 and one.longest == 256
    two = cache.tables(1, 64, 1)
    with pytest.raises(RuntimeError):
        cache.add()
    step, _ = one.step(_i32(0), _i32(130), rows=130)
    cache.append(0, step, None, -x, -x)
    one.keep(step)
    used = one.table[0, :2].tolist()
    assert set(used).isdisjoint(cache._books.seqs[a][1]) and set(used).isdisjoint(two.free.tolist())
    k, v = cache.read(0, a)
    k2, v2 = bs.kv_read(cache.pools[0], one.table[0], 130, one.tails + one.which)
    assert torch.equal(k, -k2) and torch.equal(v, -v2)
    one.close()
    one.close()
    two.close()
    assert cache.free_pages() == 4
    with pytest.raises(ValueError, match="closed"):
        one.step(_i32(0), _i32(1), rows=1)
    b, c = cache.add(), cache.add()
    cache.append(0, cache.step({b: 64, c: 192}), None, x[:1].expand(256, 1, 64), x[:1].expand(256, 1, 64))
    for s in (a, b, c):
        cache.drop(s)
    assert cache.free_pages() == 6 and sorted(cache._books.free) == list(range(6)) and sorted(cache._books.free_tails) == [0, 2, 4]


def test_a_chain_captured():
    """A step's tables, append, attention, verification and what stays of it in one graph, again and again: every replay as
    the same calls without a graph."""
    import bigsmall_amd as bs
    hk, hq, d, vocab, b, n = 2, 4, 64, 500, 3, 4
    g = torch.Generator(device="cuda").manual_seed(3)
    out_w = torch.randn(hq * d, vocab, generator=g, device="cuda") * 0.1
    embed = torch.randn(vocab, (hq + 2 * hk), d, generator=g, device="cuda").bfloat16()
    rope = bs.Rope.from_theta(d, 512)
    seqs, new, sure = _i32(0, 1, 2), _i32(*[1 + n] * b), _i32(1, 1, 1)

    def world():
        cache = bs.PagedKVCache(1, hk, d, pages=24, sequences=b)
        tables = cache.tables(b, 448)
        step, at = tables.step(seqs, _i32(60, 5, 64), rows=129)
        rows = embed[torch.arange(129, device="cuda") % vocab]
        cache.append(0, step, None, rows[:, hq:hq + hk], rows[:, hq + hk:], rope)
        tables.keep(step)
        return cache, tables

    def chain(cache, tables, last, guess, accept, pick):
        step, at = tables.step(seqs, new, sure, rows=b * (1 + n), max_new=1 + n)
        given = torch.cat([last[:, None], guess, last[:, None]], 1)
        owner = torch.where(at.owner >= 0, at.owner, 0).long()
        place = torch.where(at.owner >= 0, at.position - step.start[owner], 0).long()
        x = embed[given[owner, place]]
        q = cache.append(0, step, x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:], rope)
        y = cache.attend(0, step, q)
        y = torch.where((at.owner >= 0)[:, None], y.view(-1, hq * d).float(), 0.0)
        p = torch.softmax(y @ out_w, 1)
        tokens, counts = bs.draft_verify(p, given[owner, place + 1], step.cu, accept, pick, max_drafts=n)
        tables.keep(step, counts)
        return tokens, counts, step.cu, tables.length

    inputs = []
    for i in range(12):
        inputs.append((torch.randint(vocab, (b,), generator=g, device="cuda"), torch.randint(vocab, (b, n), generator=g, device="cuda"),
                       torch.rand(b * (1 + n), generator=g, device="cuda") * 0.01, torch.rand(b, generator=g, device="cuda")))
    eager = world()
    want = [[t.clone() for t in chain(*eager, *x)] for x in inputs]
    static = [t.clone() for t in inputs[0]]
    lent = world()
    side = torch.cuda.Stream()                      # (the products' library sets itself up outside the capture)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.softmax(torch.zeros(b * (1 + n), hq * d, device="cuda") @ out_w, 1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain(*lent, *static)
    for x, w in zip(inputs, want):
        for s, t in zip(static, x):
            s.copy_(t)
        graph.replay()
        for a, e in zip(out, w):
            assert torch.equal(a, e)
        torch.cuda.synchronize()
    assert sum(int(c.sum()) for _, c, _, _ in want) > 12 * b                    # some drafts were taken


# ---- the model

@pytest.fixture(scope="module")
def fp8_model(tmp_path_factory):
    from transformers import LlamaConfig, LlamaForCausalLM

    import bigsmall_amd
    config = LlamaConfig(hidden_size=256, intermediate_size=640, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                         vocab_size=500, max_position_embeddings=512, attn_implementation="eager", tie_word_embeddings=False,
                         quantization_config={"quant_method": "fp8", "weight_block_size": [128, 128], "activation_scheme": "dynamic"})
    torch.manual_seed(0)
    plain = LlamaConfig(**{k: v for k, v in config.to_dict().items() if k != "quantization_config"}, attn_implementation="eager")
    hf = LlamaForCausalLM(plain).to(torch.bfloat16).eval()
    sd = {}
    with torch.no_grad():
        for name, p in hf.named_parameters():
            if p.dim() == 2:
                p.mul_(4.0)
            if "_proj" in name:
                n, k = p.shape
                blocks = p.float().view(n // 128, 128, k // 128, 128)
                scale = blocks.abs().amax((1, 3)) / 448
                codes = (blocks / scale[:, None, :, None]).view(n, k).to(torch.float8_e4m3fn)
                sd[name], sd[name + "_scale_inv"] = codes, scale
                p.copy_(codes.float() * ref.spread(ref.spread(scale, n, 0), k, 1))
            else:
                sd[name] = p.detach().clone()
    path = tmp_path_factory.mktemp("fp8") / "model.bs"
    bigsmall_amd.compress(sd, str(path))
    return path, config, hf.float()


def test_fp8_logits(fp8_model, monkeypatch):
    """Against the same model with its fp8 products made in 64 bits, and against the architecture's own module."""
    import bigsmall_amd
    from bigsmall_amd import paged_llama
    path, config, hf = fp8_model
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(config.vocab_size, (n,), generator=g) for n in (150, 3, 64)]
    follow = [torch.randint(config.vocab_size, (n,), generator=g) for n in (1, 2, 1)]

    def logits():
        with bigsmall_amd.StreamingLoader(str(path), device="cuda") as loader:
            m = paged_llama.PagedLlama(loader, config, pages=16, sequences=4)
            seqs = [m.cache.add() for _ in prompts]
            return [m.forward(dict(zip(seqs, x))).float().cpu() for x in (prompts, follow)]

    got = logits()

    def exact(x, weight):
        codes, scales = ref.quantise(x.cpu().view(-1, x.shape[-1]))
        y = codes * ref.spread(scales, x.shape[-1], 1)
        w = weight.codes.cpu().float().double() * ref.spread(ref.spread(weight.scales.cpu(), weight.outer, 0), weight.inner, 1)
        return (y @ w.T).to(x.dtype).cuda()

    monkeypatch.setattr(paged_llama, "fp8_quantise", lambda x: x)
    monkeypatch.setattr(paged_llama, "fp8_linear", exact)
    want = logits()
    for a, b in zip(got, want):
        # Sums that round to bf16 differently are 2^-9 of a value apart. One that is quantised next lies on the other side of a
        # border with a chance of 2^-9 over a code's step (2^-3.5 of it in the middle), so 2^-5.5, and is then a step apart: in the mean
        # square 2^-2.75 2^-3.5 = 2^-6.25 for each of a layer's seven products, sqrt(14) of that in all. Bound: twice.
        assert float((a - b).norm() / b.norm()) < 2 * 14 ** 0.5 * 2 ** -6.25
    with torch.no_grad():
        for j in range(3):
            ids = torch.cat([prompts[j], follow[j]])
            own = hf(ids[None]).logits[0, -1]
            # x in e4m3: off by 2^-4 / sqrt(3) of a value in the mean square at most, seven times a layer; K and V in int8 1 %
            assert float((got[1][j] - own).norm() / own.norm()) < 2 * (14 ** 0.5 * 2 ** -4 / 3 ** 0.5 + 0.02)


def _greedy_enough(m, prompt, out, bound):
    """Each token's logit is near its row's largest: the model's own choice up to what rounding moves."""
    ids = torch.cat([prompt, out.cpu()])
    seq = m.cache.add()
    try:
        step = m.cache.step({seq: len(ids)})
        with torch.no_grad():
            logits = m._logits(m._hidden(step, ids.cuda())).float()
    finally:
        m.cache.drop(seq)
    rows = logits[len(prompt) - 1:-1]
    lack = rows.amax(1) - rows[torch.arange(len(out)), out]
    assert float((lack / rows.std(1)).max()) < bound, lack


@pytest.mark.parametrize("which", ["bf16", "fp8"])
@pytest.mark.parametrize("drafts", [1, 4])
def test_drafts_that_agree_and_drafts_that_do_not(model, fp8_model, which, drafts):  # noqa: F811
    import bigsmall_amd
    from bigsmall_amd.paged_llama import PagedLlama
    path, config, _ = model if which == "bf16" else fp8_model
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(config.vocab_size, (n,), generator=g) for n in (60, 1, 127)]
    with bigsmall_amd.StreamingLoader(str(path), device="cuda") as loader:
        m = PagedLlama(loader, config, pages=20, sequences=3)
        plain = m.generate(prompts, 24)
        calls = []

        def known(tokens, lengths, n):
            calls.append(n)
            out = torch.zeros(3, n, dtype=torch.int64, device="cuda")
            for i, (p, o) in enumerate(zip(prompts, plain)):
                done = int(lengths[i]) - len(p)
                part = o[done:done + n]
                out[i, :len(part)] = part
            return out, None

        def wrong(tokens, lengths, n):
            calls.append(n)
            return (known(tokens, lengths, n)[0] + 1 + torch.arange(n, device="cuda")) % config.vocab_size, None

        for draft in (known, wrong):
            calls.clear()
            out = m.generate(prompts, 24, draft=draft, drafts=drafts)
            assert [len(o) for o in out] == [24] * 3 and m.cache.free_pages() == 20
            if draft is known:
                assert len(calls) < 24              # (a token that rounding moved ends the agreement, at worst for good)
            for p, o in zip(prompts, out):
                # K and V in 8 bits or bf16 by when they were seen, and roundings: the bound of the logits' own test, twice
                _greedy_enough(m, p, o, 2 * (0.06 if which == "bf16" else 0.3))
        for n in (0, 1):
            assert [len(o) for o in m.generate(prompts, n, draft=known)] == [n] * 3
        assert m.generate([], 3, draft=known) == []


def test_drawn_tokens(model):  # noqa: F811
    import bigsmall_amd
    from bigsmall_amd.paged_llama import PagedLlama
    path, config, _ = model
    prompts = [torch.arange(70) % config.vocab_size, torch.arange(3)]

    def draft(tokens, lengths, n):
        g = torch.Generator(device="cuda").manual_seed(int(lengths.sum()))
        q = torch.softmax(torch.randn(2, n, config.vocab_size, generator=g, device="cuda"), -1)
        return torch.multinomial(q.view(2 * n, -1), 1, generator=g).view(2, n), q

    with bigsmall_amd.StreamingLoader(str(path), device="cuda") as loader:
        m = PagedLlama(loader, config, pages=12, sequences=2)

        def run(seed, **what):
            return [o.tolist() for o in m.generate(prompts, 20, temperature=0.8, generator=torch.Generator(device="cuda").manual_seed(seed), **what)]

        for what in ({}, {"draft": draft, "drafts": 3}):
            one = run(1, **what)
            assert [len(o) for o in one] == [20, 20] and all(0 <= t < config.vocab_size for o in one for t in o)
            assert run(1, **what) == one and run(2, **what) != one
        assert m.cache.free_pages() == 12


def test_refusals(model, fp8_model):  # noqa: F811
    import bigsmall_amd
    from bigsmall_amd.paged_llama import PagedLlama
    path, config, _ = model
    with bigsmall_amd.StreamingLoader(str(path), device="cuda") as loader:
        m = PagedLlama(loader, config, pages=4, sequences=2)
        prompts = [torch.arange(30)] * 2
        for draft in (lambda t, l, n: (torch.zeros(2, n + 1, dtype=torch.int64, device="cuda"), None),
                      lambda t, l, n: (torch.full((2, n), config.vocab_size, device="cuda"), None),
                      lambda t, l, n: (torch.full((2, n), -1, device="cuda"), None),
                      lambda t, l, n: (torch.zeros(2, n, dtype=torch.int64, device="cuda"), torch.zeros(2, n, 7, device="cuda"))):
            with pytest.raises(ValueError, match="draft returned"):
                m.generate(prompts, 8, draft=draft)
            assert m.cache.free_pages() == 4
        ok = lambda t, l, n: (torch.zeros(2, n, dtype=torch.int64, device="cuda"), None)     # noqa: E731
        for what in ({"drafts": -1}, {"temperature": -1.0}, {"temperature": float("inf")}):
            with pytest.raises(ValueError):
                m.generate(prompts, 8, draft=ok, **what)
        with pytest.raises(ValueError, match="at least one token"):
            m.generate([torch.arange(3), torch.arange(0)], 8, draft=ok)
        with pytest.raises(RuntimeError, match="pages"):
            m.generate([torch.zeros(200, dtype=torch.int64)] * 2, 8, draft=ok)
        with pytest.raises(RuntimeError, match="free"):
            m.generate(prompts * 2, 8, draft=ok)
        assert m.cache.free_pages() == 4
    path, config, _ = fp8_model
    with bigsmall_amd.StreamingLoader(str(path), device="cuda", dtype=torch.bfloat16) as loader, pytest.raises(ValueError, match="casts"):
        PagedLlama(loader, config, pages=4, sequences=2)


def test_prompts_are_tokens(model):  # noqa: F811
    """(an id past the embedding is refused before anything reads it)"""
    import bigsmall_amd
    from bigsmall_amd.paged_llama import PagedLlama
    path, config, _ = model
    with bigsmall_amd.StreamingLoader(str(path), device="cuda") as loader:
        m = PagedLlama(loader, config, pages=4, sequences=2)
        for bad in (-1, config.vocab_size, 1 << 40):
            with pytest.raises(ValueError, match="no tokens"):
                m.generate([torch.arange(3), torch.tensor([1, bad])], 8, temperature=0.5)
        assert m.cache.free_pages() == 4


def test_low_temperatures_and_another_default_type(model):  # noqa: F811
    """As the temperature goes to 0 what is drawn is the likeliest token; torch's default type changes nothing."""
    import bigsmall_amd
    from bigsmall_amd.paged_llama import PagedLlama
    path, config, _ = model
    prompts = [torch.arange(70) % config.vocab_size, torch.arange(3)]

    def draft(tokens, lengths, n):
        return tokens[torch.arange(2, device="cuda"), lengths.long() - 1][:, None].expand(2, n), None

    with bigsmall_amd.StreamingLoader(str(path), device="cuda") as loader:
        m = PagedLlama(loader, config, pages=8, sequences=2)
        greedy = [o.tolist() for o in m.generate(prompts, 10, draft=draft)]

        def drawn(temperature):
            g = torch.Generator(device="cuda").manual_seed(3)
            return [o.tolist() for o in m.generate(prompts, 10, draft=draft, temperature=temperature, generator=g)]

        for temperature in (1e-45, 1e-38, 1e-20):
            assert drawn(temperature) == greedy
        before = torch.get_default_dtype()
        try:
            torch.set_default_dtype(torch.bfloat16)
            assert [o.tolist() for o in m.generate(prompts, 10, draft=draft)] == greedy
            assert drawn(1e-20) == greedy
        finally:
            torch.set_default_dtype(before)


def test_example_runs(monkeypatch, capsys):
    monkeypatch.setattr(sys, "argv", ["draft_generate.py", "--layers", "2", "--tokens", "6", "--drafts", "3"])
    runpy.run_path(str(ROOT / "examples" / "draft_generate.py"), run_name="__main__")
    assert "prompt of 777 tokens" in capsys.readouterr().out

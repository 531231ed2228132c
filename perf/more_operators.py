"""Cases of a serving step with drafted tokens: products of e4m3 weights with a
scale for each block of 128 (fp8_quantise, fp8_linear), the drafts' verification
(draft_verify), and the paged KV cache's tables on the GPU (KVTables).

A case is a dict of plain values. `prepare` makes the tensors that a serving loop
has in hand before the call, `run` is one call (with `own`) or the same in
elementary torch operations, `exact` is the definition in 64 bits.

fp8: block j of a row x is x[128 j .. 128 j + 127] (the last may be shorter), a its
largest |x|, held to at least 2^-100; scale = a / 448, code = e4m3(448 x / a), to
nearest even. A weight has a scale for each 128 by 128 block.

Drafts: row r of p is the target's distribution after row r's token, q the draft
model's, draft[r] the token proposed to follow it. Sequence b has the rows cu[b] ..
cu[b + 1] - 1, one more than drafts. A draft is taken while accept * q < p; then one
token is drawn from max(p - q, 0), after the last draft from p: the first at which the
sum up to it exceeds pick times the whole.

Tables: pages of 64 tokens; a sequence holds a page for each 64 tokens that are
complete, the rest is in one of its two tails. Of a step's new tokens the first `sure`
are certain; the others may be taken back, so none of them may complete a page.
"""
import math

import torch

own = False

BLOCK, PAGE, E4M3 = 128, 64, 448.0
TINY = 2.0 ** -100
HALF = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # the hidden states of an 8,192-token prompt of an 8B-shaped model, before the q, k and v projections
        {"name": "quantise_prompt", "op": "quantise", "type": "bf16", "tokens": 8192, "inner": 4096},
        # a few rows of a width that is no multiple of a block, in f16
        {"name": "quantise_ragged", "op": "quantise", "type": "f16", "tokens": 77, "inner": 1000},
        # one token through the output projection: latency of a chat's decode step
        {"name": "linear_one", "op": "linear", "type": "bf16", "tokens": 1, "outer": 4096, "inner": 4096},
        # eight sequences of a token and four drafts each through the down projection
        {"name": "linear_drafts", "op": "linear", "type": "bf16", "tokens": 40, "outer": 4096, "inner": 14336},
        # a decode step of 64 sequences through the gate projection
        {"name": "linear_batch", "op": "linear", "type": "bf16", "tokens": 64, "outer": 14336, "inner": 4096},
        # a short prompt through a small layer whose sizes fit no tile
        {"name": "linear_ragged", "op": "linear", "type": "f16", "tokens": 777, "outer": 1000, "inner": 1400},
        # an 8,192-token prompt through the gate projection
        {"name": "linear_prompt", "op": "linear", "type": "bf16", "tokens": 8192, "outer": 14336, "inner": 4096},
        # five drafts of one conversation
        {"name": "verify_one", "op": "verify", "type": "f32", "seqs": 1, "drafts": 5, "vocab": 128256, "model": True},
        # a serving batch, up to four drafts a sequence
        {"name": "verify_batch", "op": "verify", "type": "f32", "seqs": 128, "drafts": 4, "vocab": 128256, "model": True},
        # drafts looked up in the text (no draft model), a GPT-2 vocabulary
        {"name": "verify_lookup", "op": "verify", "type": "f32", "seqs": 16, "drafts": 16, "vocab": 50257, "model": False},
        # the tables of a decode step: 128 sequences near 16,000 tokens, a token and up to four drafts each
        {"name": "tables_decode", "op": "tables", "form": "drafts", "seqs": 128, "places": 128, "hi": 16383, "new_hi": 5,
         "longest": 32768},
        # 32 finished requests leave and as many prompts take their places
        {"name": "tables_requests", "op": "tables", "form": "requests", "seqs": 32, "places": 64, "hi": 8192, "new_hi": 8192,
         "longest": 16384},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed ones' ranges."""
    op = rng.choice(["quantise", "linear", "linear", "linear", "verify", "verify", "tables", "tables"])
    if op == "quantise":
        k = _log(rng, 64, 14336)
        return {"op": op, "type": rng.choice(["bf16", "f16"]), "tokens": _log(rng, 1, 8192 * 4096 // k), "inner": k}
    if op == "linear":          # at most the operations of the listed prompt
        k, n = (rng.choice([128, 384, 1024, 1792, 4096, 14336]) if rng.random() < 0.6 else _log(rng, 64, 14336) for _ in "kn")
        most = min(8192, 8192 * 14336 * 4096 // (n * k))
        t = rng.choice([1, rng.randint(2, 16), _log(rng, 1, 128), _log(rng, 64, most)])
        return {"op": op, "type": rng.choice(["bf16", "bf16", "f16"]), "tokens": min(t, most), "outer": n, "inner": k}
    if op == "verify":          # at most the probabilities of the listed batch
        v, d = rng.choice([50257, 128256, _log(rng, 1000, 200000)]), rng.choice([1, 2, 4, 5, 8, 16])
        most = 128 * 5 * 128256 // (v * (d + 1))
        return {"op": op, "type": rng.choice(["f32", "f32", "bf16"]), "seqs": _log(rng, 1, max(1, min(256, most))), "drafts": d,
                "vocab": v, "model": rng.random() < 0.7}
    c = {"op": op, "form": rng.choice(["drafts", "requests"]), "seqs": _log(rng, 1, 512)}
    c["places"] = c["seqs"] + rng.choice([0, 0, rng.randint(1, 64)])
    c["longest"] = PAGE * rng.randint(8, max(9, min(2048, 200000 // c["seqs"])))
    c["new_hi"] = rng.randint(1, 17) if c["form"] == "drafts" else _log(rng, 1, max(1, min(c["longest"], 400000 // c["seqs"])))
    c["hi"] = _log(rng, 1, c["longest"] - c["new_hi"]) if c["form"] == "drafts" else c["longest"]
    return c


# ---- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rows(t, k, kind, g):
    """Activations: N(0, 1) with a factor for each row and a few strong channels, as a normed hidden state has."""
    x = torch.randn(t, k, generator=g, device="cuda")
    x *= 0.5 + torch.rand(t, 1, generator=g, device="cuda")
    x *= 1 + 15 * (torch.rand(k, generator=g, device="cuda") < 0.01)
    return x.to(HALF[kind])


def _weight(n, k, g):
    """A weight N(0, 0.02) as checkpoints hold it: e4m3 codes [n, k] and a scale for each block [n / 128, k / 128]."""
    rows, cols = -(-n // BLOCK), -(-k // BLOCK)
    w = torch.zeros(rows * BLOCK, cols * BLOCK, device="cuda")
    w[:n, :k] = 0.02 * torch.randn(n, k, generator=g, device="cuda")
    w = w.view(rows, BLOCK, cols, BLOCK)
    w *= 0.5 + torch.rand(rows, 1, cols, 1, generator=g, device="cuda")
    scale = w.abs().amax((1, 3)) / E4M3
    codes = (w / scale[:, None, :, None]).view(rows * BLOCK, cols * BLOCK)[:n, :k].to(torch.float8_e4m3fn)
    return codes.contiguous(), scale


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["op"] in ("quantise", "linear"):
        s["x"] = _rows(case["tokens"], case["inner"], case["type"], g)
    if case["op"] == "linear":
        s["codes"], s["scales"] = _weight(case["outer"], case["inner"], g)
        if own:                   # the handle a program keeps for each weight
            import bigsmall_amd as bs
            s["weight"] = bs.Fp8Weight(s["codes"], s["scales"])
    if case["op"] == "verify":
        _prepare_verify(s, case, g)
    if case["op"] == "tables":
        _prepare_tables(s, case, g, seed)
    return s


def _prepare_verify(s, case, g):
    b, d, v = case["seqs"], case["drafts"], case["vocab"]
    count = torch.randint(0, d + 1, (b,), generator=torch.Generator().manual_seed(21))      # part of the case, not of the seed
    count[0] = d
    s["cu"] = torch.cat([torch.zeros(1, dtype=torch.int64), (count + 1).cumsum(0)]).to(torch.int32).cuda()
    t = int((count + 1).sum())
    kind = torch.float32 if case["type"] == "f32" else torch.bfloat16
    # a language model's distributions: a few likely tokens over a long tail; the draft model's are near them
    logits = 2.5 * torch.randn(t, v, generator=g, device="cuda")
    logits.scatter_add_(1, torch.randint(v, (t, 8), generator=g, device="cuda"), 16 * torch.rand(t, 8, generator=g, device="cuda"))
    s["p"] = torch.softmax(logits, 1).to(kind)
    logits += 0.4 * torch.randn(t, v, generator=g, device="cuda")
    q = torch.softmax(logits, 1).to(kind)
    s["q"] = q if case["model"] else None
    # drafted from q: the largest of log q + Gumbel noise
    logits -= torch.log(-torch.log(torch.rand(t, v, generator=g, device="cuda").clamp_(1e-20, 1 - 2.0 ** -24)))
    s["draft"] = logits.argmax(1)
    s["accept"] = torch.rand(t, generator=g, device="cuda")
    s["pick"] = torch.rand(b, generator=g, device="cuda")


def _prepare_tables(s, case, g, seed):
    b, places, m = case["seqs"], case["places"], case["longest"] // PAGE
    host = torch.Generator().manual_seed(31)                     # lengths: part of the case
    hi = case["hi"] if case["form"] == "drafts" else min(case["hi"], case["longest"])
    length = torch.randint(0, hi + 1, (places,), generator=host)
    new = torch.randint(1, case["new_hi"] + 1, (b,), generator=host)
    seqs = torch.randperm(places, generator=torch.Generator().manual_seed(seed))[:b]       # which places: of the seed
    new[0] = case["new_hi"]
    used = length // PAGE
    pages = int(used.sum()) + int((new // PAGE + 1).sum()) + 16
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    col = torch.arange(m)
    table = torch.zeros(places, m, dtype=torch.int32, device="cuda")
    held = (col < used[:, None]).cuda()
    n = int(used.sum())
    table[held] = perm[:n]
    free = torch.zeros(pages, dtype=torch.int32, device="cuda")
    free[:pages - n] = perm[n:]
    s.update(seqs=seqs.to(torch.int32).cuda(), new=new.to(torch.int32).cuda(), sure=None, rows=int(new.sum()),
             max_new=int(new.max()), length=length.to(torch.int32).cuda(), table=table, free=free,
             n_free=torch.tensor([pages - n], dtype=torch.int32).cuda(),
             which=torch.randint(0, 2, (places,), generator=g, device="cuda").to(torch.int32),
             tails=2 * torch.randperm(places, generator=g, device="cuda").to(torch.int32))
    if case["form"] == "drafts":
        s["sure"] = torch.ones(b, dtype=torch.int32, device="cuda")
    if own:                       # the books a program keeps
        import bigsmall_amd as bs
        books = bs.KVTables(perm, s["tails"], case["longest"])
        for name in ("length", "table", "free", "n_free", "which"):
            getattr(books, name).copy_(s[name])
        s["books"] = books


# ---- one pass

def run(s):
    c = s["case"]
    if own:
        import bigsmall_amd as bs
        if c["op"] == "quantise":
            rows = bs.fp8_quantise(s["x"])
            return rows.codes, rows.scales
        if c["op"] == "linear":
            return bs.fp8_linear(s["x"], s["weight"])
        if c["op"] == "verify":
            return bs.draft_verify(s["p"], s["draft"], s["cu"], s["accept"], s["pick"], q=s["q"], max_drafts=c["drafts"])
        books = s["books"]
        if c["form"] == "requests":
            books.drop(s["seqs"])
        step, rows = books.step(s["seqs"], s["new"], sure=s["sure"], rows=s["rows"], max_new=s["max_new"])
        out = {"start": step.start, "cu": step.cu, "table": step.table, "tails": step.tails, "owner": rows.owner,
               "position": rows.position, "slot": rows.slot}
        if c["form"] == "requests":
            books.keep(step)
            out.update({"state_" + name: getattr(books, name) for name in ("length", "table", "free", "n_free", "which")})
        return out
    if c["op"] == "quantise":
        return _quantise(s["x"])
    if c["op"] == "linear":
        return _linear(s)
    if c["op"] == "verify":
        return _verify(s)
    if c["form"] == "requests":
        _drop(s)
    out, after = _step(s)
    if c["form"] == "requests":
        _keep(s, out, after)
        out.update({"state_" + name: s[name] for name in ("length", "table", "free", "n_free", "which")})
    return out


def _quantise(x):
    """Codes [T, K] and scales [T, K / 128]. The quotient is taken in 64 bits: codes next to a border hang on it."""
    t, k = x.shape
    cols = -(-k // BLOCK)
    y = torch.nn.functional.pad(x.double(), (0, cols * BLOCK - k)).view(t, cols, BLOCK)
    a = y.abs().amax(2)
    bad = ~torch.isfinite(a)
    a = a.clamp(min=TINY)
    codes = torch.where(bad[:, :, None], 0.0, y * E4M3 / a[:, :, None]).float().to(torch.float8_e4m3fn)
    scales = torch.where(bad, math.nan, a / E4M3).float()
    return codes.view(t, cols * BLOCK)[:, :k].contiguous(), scales


def _linear(s):
    x, n, k = s["x"], s["case"]["outer"], s["case"]["inner"]
    codes, scales = _quantise(x)
    x32 = codes.float() * scales.repeat_interleave(BLOCK, 1)[:, :k]
    w32 = s["codes"].float() * s["scales"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    return (x32 @ w32.T).to(x.dtype)


def _verify(s):
    c, p, q = s["case"], s["p"], s["q"]
    b, d, v = c["seqs"], c["drafts"], c["vocab"]
    cu = s["cu"].long()
    count = cu[1:] - cu[:-1] - 1
    seq = torch.arange(b, device="cuda")
    i = torch.arange(d, device="cuda")
    row = (cu[:-1, None] + i).clamp(max=p.shape[0] - 1)                       # [B, D]
    x = s["draft"][row]
    px = p[row, x].double()
    qx = q[row, x].double() if q is not None else torch.ones_like(px)
    taken = (s["accept"][row].double() * qx < px) & (i < count[:, None])
    a = taken.long().cumprod(1).sum(1)                                        # drafts taken
    at = cu[:-1] + a
    left = a < count                                                          # a draft was refused there
    w = p[at].double()
    if q is not None:
        r = (w - q[at].double()).clamp(min=0)
    else:
        r = w.clone()
        r[seq, s["draft"][at].clamp(0, v - 1)] = 0
    r = torch.where((r.sum(1) > 0)[:, None], r, w)
    total = torch.where(left[:, None], r, w).cumsum(1)
    token = (total <= (s["pick"].double() * total[:, -1])[:, None]).sum(1).clamp(max=v - 1)
    col = torch.arange(d + 1, device="cuda")
    drafts = torch.nn.functional.pad(x, (0, 1))
    tokens = torch.where(col < a[:, None], drafts, torch.where(col == a[:, None], token[:, None], -1))
    return tokens, (a + 1).to(torch.int32)


def _step(s):
    """The step's tables, and what `_keep` needs of it."""
    c, m = s["case"], s["table"].shape[1]
    seqs, new = s["seqs"].long(), s["new"].long()
    start = s["length"].long()[seqs]
    sure = torch.minimum(s["sure"].long(), new) if s["sure"] is not None else new
    end = torch.minimum(start + new, ((start + sure) // PAGE + 1) * PAGE - 1) if s["sure"] is not None else start + new
    need = end // PAGE - start // PAGE
    n_free = s["n_free"].long()
    # all or nothing
    fits = (start + sure <= c["longest"]).all() & (need.sum() <= n_free) & ((end - start).sum() <= s["rows"])
    end = torch.where(fits, end, start)
    need = torch.where(fits, need, torch.zeros_like(need))
    cu = torch.nn.functional.pad((end - start).cumsum(0), (1, 0))
    before = need.cumsum(0) - need
    col = torch.arange(m, device="cuda")
    first, last = (start // PAGE)[:, None], (end // PAGE)[:, None]
    taken = s["free"][(n_free - 1 - before[:, None] - (col - first)).clamp(0, s["free"].shape[0] - 1)]
    table = torch.where(col < first, s["table"][seqs], torch.where(col < last, taken, torch.zeros_like(taken)))
    which, tails = s["which"][seqs], s["tails"][seqs]
    moves = (need > 0).to(torch.int32)
    r = torch.arange(s["rows"], device="cuda")
    owner = torch.searchsorted(cu[1:], r, right=True).clamp(max=len(seqs) - 1)
    position = start[owner] + r - cu[owner]
    covered = r < cu[-1]
    none = torch.full_like(r, -1)
    out = {"start": start.to(torch.int32), "cu": cu.to(torch.int32), "table": table,
           "tails": torch.stack([tails + which, tails + (which ^ moves)], 1),
           "owner": torch.where(covered, owner, none).to(torch.int32),
           "position": torch.where(covered, position, none).to(torch.int32),
           "slot": torch.where(covered, seqs[owner] * c["longest"] + position, none)}
    return out, (seqs, end, need, moves)


def _keep(s, out, after):
    """Every new token stays."""
    seqs, end, need, moves = after
    s["length"][seqs] = end.to(torch.int32)
    s["which"][seqs] ^= moves
    col = torch.arange(s["table"].shape[1], device="cuda")
    fresh = (col >= (end // PAGE - need)[:, None]) & (col < (end // PAGE)[:, None])
    s["table"][seqs] = torch.where(fresh, out["table"], s["table"][seqs])
    s["n_free"] -= need.sum().to(torch.int32)


def _drop(s):
    seqs = s["seqs"].long()
    used = s["length"].long()[seqs] // PAGE
    before = used.cumsum(0) - used
    col = torch.arange(s["table"].shape[1], device="cuda")
    held = col < used[:, None]
    where = s["n_free"].long() + used.sum() - 1 - before[:, None] - col
    s["free"][where[held]] = s["table"][seqs][held]
    s["n_free"] += used.sum().to(torch.int32)
    s["length"][seqs] = 0
    s["which"][seqs] = 0


# ---- what a pass cannot do without

def work(case):
    if case["op"] == "quantise":
        t, k = case["tokens"], case["inner"]
        return {"bytes": 3 * t * k + 4 * t * -(-k // BLOCK), "flops": 3 * t * k}
    if case["op"] == "linear":
        t, n, k = case["tokens"], case["outer"], case["inner"]
        return {"bytes": n * k + 2 * t * k + 2 * t * n + 4 * -(-k // BLOCK) * -(-n // BLOCK), "flops": 2.0 * t * n * k}
    if case["op"] == "verify":
        # the row that each sequence draws from; of q where a draft was refused (about half of them)
        each = (4 if case["type"] == "f32" else 2) * case["vocab"]
        return {"bytes": case["seqs"] * each * (1.5 if case["model"] else 1.0), "flops": 3 * case["seqs"] * case["vocab"]}
    b, m = case["seqs"], case["longest"] // PAGE
    if case["form"] == "drafts":
        return {"bytes": b * (4 * 8 + 4 * m + 4 * min(m, case["hi"] // (2 * PAGE) + 1)) + 16 * b * (case["new_hi"] + 1) // 2,
                "flops": 10 * b}
    n = (case["new_hi"] + 1) // 2
    return {"bytes": b * (4 * 8 + 4 * m + 16 * n + 4 * 6 * (n // PAGE)), "flops": 10 * b}


# ---- the definition in 64 bits

def _exact_rows(x):
    """Codes and scales of x's blocks; rounding to e4m3 written out: 3 bits after the leading one, down to 2^-9."""
    t, k = x.shape
    cols = -(-k // BLOCK)
    codes = torch.zeros(t, k, dtype=torch.float64, device="cuda")
    scales = torch.zeros(t, cols, dtype=torch.float64, device="cuda")
    for j in range(cols):
        y = x[:, j * BLOCK:(j + 1) * BLOCK].double()
        top = torch.clamp(y.abs().max(1, keepdim=True).values, min=TINY)
        z = E4M3 * y / top
        step = torch.exp2(torch.floor(torch.log2(torch.clamp(z.abs(), min=2.0 ** -6))) - 3)
        codes[:, j * BLOCK:(j + 1) * BLOCK] = torch.round(z / step) * step
        scales[:, j] = top[:, 0] / E4M3
    return codes, scales


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantise":
        return _exact_rows(s["x"])
    if case["op"] == "linear":
        codes, scales = _exact_rows(s["x"])
        y = torch.zeros(case["tokens"], case["outer"], dtype=torch.float64, device="cuda")
        for j in range(scales.shape[1]):
            for i in range(s["scales"].shape[0]):
                part = s["codes"][i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK].float().double() * s["scales"][i, j].double()
                y[:, i * BLOCK:(i + 1) * BLOCK] += (codes[:, j * BLOCK:(j + 1) * BLOCK] * scales[:, j:j + 1]) @ part.T
        return y
    if case["op"] == "verify":
        return _exact_verify(s)
    return _exact_tables(s)


def _exact_verify(s):
    p, q, cu, d = s["p"], s["q"], s["cu"].tolist(), s["case"]["drafts"]
    draft, accept, pick = s["draft"].tolist(), s["accept"].tolist(), s["pick"].tolist()
    tokens = torch.full((len(pick), d + 1), -1, dtype=torch.int64)
    counts = torch.zeros(len(pick), dtype=torch.int32)
    for b in range(len(pick)):
        r, last = cu[b], cu[b + 1] - 1
        while r < last and accept[r] * (float(q[r, draft[r]]) if q is not None else 1.0) < float(p[r, draft[r]]):
            tokens[b, r - cu[b]] = draft[r]
            r += 1
        w = p[r].double()
        if r < last and q is not None:
            w = torch.relu(w - q[r].double())
        elif r < last:
            w[draft[r]] = 0
        if float(w.sum()) == 0:
            w = p[r].double()
        up = torch.cumsum(w, 0)
        tokens[b, r - cu[b]] = int(torch.searchsorted(up, up[-1] * pick[b], right=True).clamp(max=len(up) - 1))
        counts[b] = r - cu[b] + 1
    return tokens.cuda(), counts.cuda()


def _exact_tables(s):
    """The books kept on the host, sequence by sequence."""
    c, m = s["case"], s["table"].shape[1]
    turn = c["form"] == "requests"
    length, which, tails = s["length"].tolist(), s["which"].tolist(), s["tails"].tolist()
    seqs, new = s["seqs"].tolist(), s["new"].tolist()
    sure = s["sure"].tolist() if s["sure"] is not None else new
    n, old = int(s["n_free"]), s["free"].tolist()
    stack, table = old[:n], s["table"].tolist()
    if turn:
        back = [page for q in seqs for page in table[q][:length[q] // PAGE]]
        stack += back[::-1]
        for q in seqs:
            length[q] = which[q] = 0
        old[:len(stack)] = stack
    taken = list(stack)
    start, cu, rows, ends, place, slot, owner = [], [0], [], [], [], [], []
    for b, q in enumerate(seqs):
        at, end = length[q], length[q] + new[b]
        while s["sure"] is not None and end // PAGE * PAGE > at + min(sure[b], new[b]):
            end -= 1
        pages = table[q][:at // PAGE] + [taken.pop() for _ in range(end // PAGE - at // PAGE)]
        rows.append(pages + [0] * (m - len(pages)))
        moved = end // PAGE > at // PAGE
        ends.append((end, which[q] ^ moved, len(pages)))
        place.append([tails[q] + which[q], tails[q] + (which[q] ^ moved)])
        start.append(at)
        cu.append(cu[-1] + end - at)
        owner += [b] * (end - at)
        slot += [q * c["longest"] + i for i in range(at, end)]
    none = [-1] * (s["rows"] - cu[-1])
    position = [x % c["longest"] for x in slot]

    def put(x, kind=torch.int32):
        return torch.tensor(x, dtype=kind).cuda()

    out = {"start": put(start), "cu": put(cu), "table": put(rows), "tails": put(place), "owner": put(owner + none),
           "position": put(position + none), "slot": put(slot + none, torch.int64)}
    if turn:
        for b, q in enumerate(seqs):
            table[q][length[q] // PAGE:ends[b][2]] = rows[b][length[q] // PAGE:ends[b][2]]
            length[q], which[q] = ends[b][0], int(ends[b][1])
        out.update(state_length=put(length), state_table=put(table), state_free=put(old), state_n_free=put([len(taken)]),
                   state_which=put(which))
    return out

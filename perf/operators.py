"""Cases of the paged 8-bit KV cache: kv_append (position rotation and
quantising append), kv_attend (attention over the cache, from one new token to
whole prompts) and kv_read (a sequence back in bf16).

A case is a dict of plain values. `prepare` makes the tensors that a serving
loop has in hand before the call, `run` is one call (with `own`) or the same
in elementary torch operations, `exact` is the definition in 64 bits, written
as loops over sequences and heads.

Storage, as the operators define it: pages of 64 tokens; K pages
[pages, kv heads, 64, dim] and V pages [pages, kv heads, dim, 64] in int8 or
e4m3, one f32 scale per page and kv head; the tokens of a sequence's
unfinished page in bf16 in a tail of the same shape. A step (one call for every
sequence in it) is: start [B] cached tokens before it, cu [B + 1] where each
sequence's new tokens begin in the packed rows, table [B, M] page numbers,
tails [B, 2] the tail to read and the tail to write.
"""
import math

import torch

own = False

PAGE = 64
QMAX = {"int8": 127.0, "fp8": 448.0}
KIND = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
AMAX_LO, AMAX_HI = 2.0 ** -40, 2.0 ** 60


def listed():
    return [
        # the first decode step of a short chat: one sequence, one token, nothing but latency
        {"name": "append_one", "op": "append", "kind": "fp8", "seqs": 1, "lo": 200, "hi": 200, "new_lo": 1, "new_hi": 1,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False},
        # ragged chunks of a serving step (several short prompts with a head size that is no power of two), rotated by
        # neighbouring pairs over half the head; the step's first sequence is read back for the compressed store
        {"name": "append_ragged", "op": "append", "kind": "int8", "seqs": 7, "lo": 0, "hi": 900, "new_lo": 1, "new_hi": 1500,
         "q_heads": 8, "kv_heads": 8, "dim": 80, "rot": 40, "interleaved": True},
        # a 32,768-token prompt of an 8B-shaped model's layer going into the cache at once
        {"name": "append_prompt", "op": "append", "kind": "fp8", "seqs": 1, "lo": 0, "hi": 0, "new_lo": 32768,
         "new_hi": 32768, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False},
        # one token of one sequence over a 1,024-token cache: latency of a chat's decode step
        {"name": "attend_one", "op": "attend", "kind": "fp8", "seqs": 1, "lo": 1023, "hi": 1023, "new_lo": 1, "new_hi": 1,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "mask": "causal"},
        # a decode step of a serving batch, caches from one token to 8,192
        {"name": "attend_batch", "op": "attend", "kind": "int8", "seqs": 64, "lo": 0, "hi": 8191, "new_lo": 1, "new_hi": 1,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "mask": "causal"},
        # two very long caches: few rows, so the work is split over the cache's length
        {"name": "attend_long", "op": "attend", "kind": "fp8", "seqs": 2, "lo": 100001, "hi": 131071, "new_lo": 1, "new_hi": 1,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "mask": "causal"},
        # the largest decode step: 128 sequences of about 16,000 tokens, 4 GB of cache read
        {"name": "attend_wide", "op": "attend", "kind": "fp8", "seqs": 128, "lo": 15000, "hi": 16383, "new_lo": 1,
         "new_hi": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "mask": "causal"},
        # an 8,192-token prompt attending to itself (what follows its append)
        {"name": "attend_prompt", "op": "attend", "kind": "fp8", "seqs": 1, "lo": 0, "hi": 0, "new_lo": 8192,
         "new_hi": 8192, "q_heads": 32, "kv_heads": 8, "dim": 128, "mask": "causal"},
        # a chunk of a long prompt on 32,768 cached tokens, scores capped, half the layers' sliding window
        {"name": "attend_chunk", "op": "attend", "kind": "int8", "seqs": 1, "lo": 32768, "hi": 32768, "new_lo": 500,
         "new_hi": 500, "q_heads": 16, "kv_heads": 8, "dim": 256, "mask": "window", "window": 16384, "cap": 50.0},
        # prompts of a GPT-2-sized layer made of several documents each, a visible-to-all prefix, a distance bias
        {"name": "attend_documents", "op": "attend", "kind": "int8", "seqs": 5, "lo": 0, "hi": 300, "new_lo": 600,
         "new_hi": 2500, "q_heads": 12, "kv_heads": 12, "dim": 64, "mask": "documents", "bias": True},
        # a short conversation parked: its cache back in bf16 for the compressed store
        {"name": "read_short", "op": "read", "kind": "int8", "tokens": 777, "kv_heads": 8, "dim": 128},
        # a long one
        {"name": "read_long", "op": "read", "kind": "fp8", "tokens": 32768, "kv_heads": 8, "dim": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed ones' ranges."""
    op = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "read"])
    c = {"op": op, "kind": rng.choice(["int8", "fp8"]), "dim": rng.choice([64, 80, 96, 128, 128, 256])}
    kv = rng.choice([1, 2, 4, 8, 8, 12])
    if op == "read":
        return dict(c, kv_heads=kv, tokens=_log(rng, 1, (32768 * 1024) // (kv * c["dim"])))
    c.update(kv_heads=kv, q_heads=kv * rng.choice([1, 1, 2, 3, 4, 4, 6, 8]))
    width = c["q_heads"] * c["dim"]
    if op == "append":
        c.update(seqs=_log(rng, 1, 128), rot=rng.choice([c["dim"], c["dim"], c["dim"] // 2]),
                 interleaved=rng.random() < 0.4, lo=0, hi=_log(rng, 1, 8192))
        each = max(1, (32768 * 4096) // (width * c["seqs"]))
        c["new_hi"] = 1 if rng.random() < 0.4 else _log(rng, 1, min(each, 32768))
        c["new_lo"] = rng.randint(1, c["new_hi"])
        return c
    c.update(mask=rng.choice(["causal", "causal", "window", "documents"]), bias=rng.random() < 0.3,
             cap=rng.choice([0.0, 0.0, 20.0, 50.0]))
    form = rng.choice(["one", "one", "few", "prompt", "prompt"])
    if form == "prompt":          # at most the pairs of the listed prompt
        c["seqs"] = rng.choice([1, 1, 2, 5])
        c["new_hi"] = _log(rng, 17, max(18, int(math.sqrt(8192.0 * 8192 * 4096 / (width * c["seqs"])) * 0.7)))
        c["new_hi"] = min(c["new_hi"], 8192)
        c["new_lo"] = rng.randint(max(1, c["new_hi"] // 4), c["new_hi"])
        c.update(lo=0, hi=_log(rng, 1, c["new_hi"]))
    else:                         # at most the cache of the listed wide step
        c["new_hi"] = 1 if form == "one" else rng.randint(2, 16)
        c["new_lo"] = rng.randint(1, c["new_hi"])
        c["seqs"] = _log(rng, 1, 128)
        room = (128 * 16384 * 1024) // (c["seqs"] * kv * c["dim"] * c["new_hi"])
        c["hi"] = _log(rng, 1, max(2, min(131072, room)))
        c["lo"] = rng.randint(0, c["hi"])
    if c["mask"] == "window":
        c["window"] = _log(rng, 1, 20000)
    return c


# ---- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _whole(lo, hi, n, seed):
    """n whole numbers in [lo, hi], on the host; the last is hi, so that the largest does not hang on the seed."""
    g = torch.Generator().manual_seed(seed)
    v = torch.randint(lo, hi + 1, (n,), generator=g)
    v[-1] = hi
    return v


def _rows(shape, g):
    """q, k or v: N(0, 1) with a factor for each head and a few strong channels, as trained projections give."""
    x = torch.randn(shape, generator=g, device="cuda")
    x *= 0.6 + 0.8 * torch.rand(shape[1], 1, generator=g, device="cuda")
    x *= 1 + 2 * (torch.rand(shape[1], shape[2], generator=g, device="cuda") < 0.03)
    return x.to(torch.bfloat16)


def _codes(shape, kind, g):
    """Quantised pages of N(0, 1) values and their scales."""
    codes = torch.empty(shape, dtype=torch.int8 if kind == "int8" else torch.float8_e4m3fn, device="cuda")
    rows = max(1, (1 << 26) // (shape[1] * shape[2] * shape[3]))
    for at in range(0, shape[0], rows):
        x = torch.randn((min(rows, shape[0] - at),) + tuple(shape[1:]), generator=g, device="cuda")
        x *= QMAX[kind] / 4.5
        x.clamp_(-QMAX[kind], QMAX[kind])
        codes[at:at + rows] = (x.round_() if kind == "int8" else x).to(codes.dtype)
    head = 0.6 + 0.8 * torch.rand(1, shape[1], generator=g, device="cuda")
    scales = 4.5 / QMAX[kind] * head * (0.85 + 0.3 * torch.rand(shape[0], shape[1], generator=g, device="cuda"))
    return codes, scales


def _lengths(case):
    """Cached and new tokens of each sequence: part of the case, not of the seed."""
    b = case["seqs"]
    start, new = _whole(case["lo"], case["hi"], b, 11), _whole(case["new_lo"], case["new_hi"], b, 12)
    if b > 1 and case["lo"] == 0:
        start[0] = 0              # one that has just begun
    return start, new


def prepare(case, seed):
    g = _gen(seed)
    hk, d, kind = case["kv_heads"], case["dim"], case["kind"]
    s = {"case": case}
    if case["op"] == "read":
        start, new = torch.zeros(1, dtype=torch.int64), torch.tensor([case["tokens"]])
    else:
        start, new = _lengths(case)
    b = len(start)
    end = start + new
    m = int(((end + PAGE - 1) // PAGE).max())
    used = ((end + PAGE - 1) // PAGE).tolist()
    n_pages = sum(used) + 3
    perm = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(b, m, dtype=torch.int32, device="cuda")
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = perm[at:at + u]
        at += u
    s["k"], s["k_scale"] = _codes((n_pages, hk, PAGE, d), kind, g)
    s["v"], s["v_scale"] = _codes((n_pages, hk, d, PAGE), kind, g)
    s["k_tail"] = _rows((2 * b * PAGE, hk, d), g).view(2 * b, PAGE, hk, d).transpose(1, 2).contiguous()
    s["v_tail"] = _rows((2 * b * PAGE, hk, d), g).view(2 * b, PAGE, hk, d).permute(0, 2, 3, 1).contiguous()
    order = torch.randperm(2 * b, generator=g, device="cuda").to(torch.int32).view(b, 2)
    # a sequence whose last page is completed by this step goes on in its other tail
    moves = (end // PAGE > start // PAGE).cuda()
    s["tails"] = torch.stack([order[:, 0], torch.where(moves, order[:, 1], order[:, 0])], 1).contiguous()
    s["table"] = table
    s["start"] = start.to(torch.int32).cuda()
    s["cu"] = torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)]).to(torch.int32).cuda()
    s["max_new"], s["max_len"], s["total"] = int(new.max()), int(end.max()), int(new.sum())
    t = s["total"]
    if case["op"] != "read":
        s["q"] = _rows((t, case["q_heads"], d), g)
    if case["op"] == "append":
        s["new_k"], s["new_v"] = _rows((t, hk, d), g), _rows((t, hk, d), g)
        freq = 500000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64) / case["rot"])
        angle = torch.arange(s["max_len"], dtype=torch.float64)[:, None] * freq
        s["cos"], s["sin"] = angle.cos().float().cuda(), angle.sin().float().cuda()
    if case["op"] == "attend":
        s["scale"] = d ** -0.5
        s["cap"], s["window"] = case.get("cap", 0.0), case.get("window", 0)
        h = case["q_heads"]
        s["slopes"] = (2.0 ** (-8.0 * torch.arange(1, h + 1) / h)).cuda() if case.get("bias") else None
        s["prefix"] = s["first"] = None
        if case["mask"] == "documents":
            # documents of about 300 tokens: a token sees its own document, and the sequence's first 37 tokens see each other
            s["prefix"] = torch.full((b,), 37, dtype=torch.int32, device="cuda")
            seq, pos = _positions(s)
            length = torch.randint(200, 400, (b,), generator=g, device="cuda")
            s["first"] = (pos // length[seq] * length[seq]).to(torch.int32)
    if own:                       # the handles a program keeps: the pool's and the step's tensors, checked once
        import bigsmall_amd as bs
        s["pool"] = bs.KVPool(s["k"], s["v"], s["k_scale"], s["v_scale"], s["k_tail"], s["v_tail"])
        s["batch"] = bs.KVBatch(s["start"], s["cu"], s["table"], s["tails"], s["max_new"], s["max_len"])
        if case["op"] == "append":
            s["rope"] = bs.Rope(s["cos"], s["sin"], interleaved=case["interleaved"])
    return s


# ---- one pass

def run(s):
    c = s["case"]
    if own:
        import bigsmall_amd as bs
        if c["op"] == "append":
            q = bs.kv_append(s["pool"], s["batch"], s["q"], s["new_k"], s["new_v"], rope=s["rope"])
            first = bs.kv_read(s["pool"], s["table"][-1], c["hi"] + c["new_hi"], s["tails"][-1, 1:]) if c["kind"] == "int8" else None
            return _appended(s, q, first)
        if c["op"] == "read":
            return bs.kv_read(s["pool"], s["table"][0], c["tokens"], s["tails"][0, 1:])
        return bs.kv_attend(s["pool"], s["batch"], s["q"], scale=s["scale"], softcap=s["cap"], slopes=s["slopes"],
                            window=s["window"], prefix=s["prefix"], first=s["first"], return_lse=True)
    if c["op"] == "append":
        q = _append(s)
        first = _read(s, s["table"][-1], c["hi"] + c["new_hi"], s["tails"][-1, 1:]) if c["kind"] == "int8" else None
        return _appended(s, q, first)
    if c["op"] == "read":
        return _read(s, s["table"][0], c["tokens"], s["tails"][0, 1:])
    return _attend(s)


def _appended(s, q, read):
    """What an append leaves: rotated q, scales and tails, and the stored values: e4m3 pages as they are (their values
    are these times the scales), of int8 pages the longest sequence read back."""
    out = {"q": q, "k_scale": s["k_scale"], "v_scale": s["v_scale"], "k_tail": s["k_tail"], "v_tail": s["v_tail"]}
    if read is None:
        out.update(k=s["k"], v=s["v"])
    else:
        out.update(read_k=read[0], read_v=read[1])
    return out


def _positions(s):
    """Sequence and position of every new token."""
    cu, start = s["cu"].long(), s["start"].long()
    seq = torch.repeat_interleave(torch.arange(len(start), device="cuda"), cu[1:] - cu[:-1], output_size=s["total"])
    return seq, start[seq] + torch.arange(s["total"], device="cuda") - cu[seq]


def _rotate(x, cos, sin, interleaved):
    """x [T, heads, dim] bf16; the first 2 * cos.shape[1] channels turn in pairs, in 32 bits."""
    half = cos.shape[1]
    y = x.float()
    a, b = (y[..., 0:2 * half:2], y[..., 1:2 * half:2]) if interleaved else (y[..., :half], y[..., half:2 * half])
    c, n = cos[:, None, :], sin[:, None, :]
    u, w = a * c - b * n, b * c + a * n
    turned = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.cat([turned, y[..., 2 * half:]], -1).to(torch.bfloat16)


def _quantise(x, dims, kind):
    """Codes and scales of pages x; a page that holds a NaN has codes 0 and scale NaN."""
    x = x.float()
    amax = x.abs().amax(dims, keepdim=True)
    bad = torch.isnan(amax)
    amax = amax.clamp(AMAX_LO, AMAX_HI)
    y = (x * (QMAX[kind] / amax)).clamp(-QMAX[kind], QMAX[kind])
    y = torch.where(bad, torch.zeros_like(y), y)
    codes = y.round().to(torch.int8) if kind == "int8" else y.to(torch.float8_e4m3fn)
    return codes, torch.where(bad, amax * math.nan, amax / QMAX[kind]).flatten(1)


def _put(pages, index, codes):
    """pages[index] = codes, through bytes where the type has no indexed store."""
    if pages.dtype == torch.float8_e4m3fn:
        pages.view(torch.uint8)[index] = codes.view(torch.uint8)
    else:
        pages[index] = codes


def _append(s):
    c = s["case"]
    seq, pos = _positions(s)
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _rotate(s["q"], cos, sin, c["interleaved"])
    k, v = _rotate(s["new_k"], cos, sin, c["interleaved"]), s["new_v"]
    bad = ~(torch.isfinite(k).all(-1, keepdim=True) & torch.isfinite(v).all(-1, keepdim=True))
    k = torch.where(bad, torch.full_like(k, math.nan), k)
    v = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    # the pages that the step touches, and where each of their tokens comes from
    start, cu = s["start"].long(), s["cu"].long()
    end = start + cu[1:] - cu[:-1]
    first, last = start // PAGE, (end - 1) // PAGE
    count = last - first + 1
    b = torch.repeat_interleave(torch.arange(len(start), device="cuda"), count)
    page = first[b] + torch.arange(len(b), device="cuda") - (count.cumsum(0) - count)[b]
    at = page[:, None] * PAGE + torch.arange(PAGE, device="cuda")               # positions [units, 64]
    old, inside = at < start[b][:, None], at < end[b][:, None]
    src = (cu[b][:, None] + at - start[b][:, None]).clamp(0, s["total"] - 1)
    tail_in, tail_out = s["tails"][:, 0].long()[b], s["tails"][:, 1].long()[b]
    pk = torch.where(old[:, None, :, None], s["k_tail"][tail_in], k[src].transpose(1, 2))
    pv = torch.where(old[:, None, None, :], s["v_tail"][tail_in], v[src].permute(0, 2, 3, 1))
    full = inside[:, -1]
    where = s["table"].long()[b, page][full]
    for name, x in (("k", pk), ("v", pv)):
        codes, scales = _quantise(x[full], (2, 3), c["kind"])
        _put(s[name], where, codes)
        s[name + "_scale"][where] = scales
    rest = ~full
    keep = inside[rest]
    s["k_tail"][tail_out[rest]] = torch.where(keep[:, None, :, None], pk[rest], s["k_tail"][tail_out[rest]])
    s["v_tail"][tail_out[rest]] = torch.where(keep[:, None, None, :], pv[rest], s["v_tail"][tail_out[rest]])
    return q


def _take(pages, index):
    if pages.dtype == torch.float8_e4m3fn:
        return pages.view(torch.uint8)[index].view(pages.dtype).float()
    return pages[index].float()


def _read(s, row, n, tail):
    """K and V [kv heads, n, dim] of one sequence, in bf16."""
    m = (n + PAGE - 1) // PAGE
    ids = row[:m].long()
    k = _take(s["k"], ids) * s["k_scale"][ids][:, :, None, None]
    v = (_take(s["v"], ids) * s["v_scale"][ids][:, :, None, None]).transpose(2, 3)
    if n % PAGE:
        k[-1], v[-1] = s["k_tail"][tail.long()][0], s["v_tail"][tail.long()][0].transpose(1, 2)
    k, v = (x.transpose(0, 1).flatten(1, 2)[:, :n].to(torch.bfloat16).contiguous() for x in (k, v))
    return k, v


def _attend(s):
    c = s["case"]
    hq, hk, d = c["q_heads"], c["kv_heads"], c["dim"]
    start, cu = s["start"].long(), s["cu"].long()
    b, n = len(start), s["max_new"]
    count = cu[1:] - cu[:-1]
    end = start + count
    table = s["table"].long()
    m = table.shape[1]
    k = _take(s["k"], table) * s["k_scale"][table][..., None, None]             # [B, M, hk, 64, d]
    v = _take(s["v"], table) * s["v_scale"][table][..., None, None]
    has, at, row = end % PAGE > 0, (end // PAGE).clamp(max=m - 1), torch.arange(b, device="cuda")
    tail = s["tails"][:, 1].long()
    pick = has[:, None, None, None]
    k[row, at] = torch.where(pick, s["k_tail"][tail].float(), k[row, at])
    v[row, at] = torch.where(pick, s["v_tail"][tail].float(), v[row, at])
    length = m * PAGE
    k = k.permute(0, 2, 4, 1, 3).reshape(b, hk, d, length)
    v = v.permute(0, 2, 1, 4, 3).reshape(b, hk, length, d)
    step = torch.arange(n, device="cuda")
    new = step < count[:, None]                                                 # [B, n]
    src = (cu[:-1, None] + step).clamp(max=s["total"] - 1)
    q = s["q"].float()[src].view(b, n, hk, hq // hk, d).permute(0, 2, 3, 1, 4)  # [B, hk, G, n, d]
    x = (q.reshape(b, hk, -1, d) @ k).view(b, hk, hq // hk, n, length) * s["scale"]
    if s["cap"]:
        x = torch.tanh(x / s["cap"]) * s["cap"]
    pos = start[:, None] + step                                                 # [B, n]
    j = torch.arange(length, device="cuda")
    if s["slopes"] is not None:
        x = x - s["slopes"].view(1, hk, -1, 1, 1) * (pos[..., None] - j).abs()[:, None, None]
    seen = j <= pos[..., None]
    if s["prefix"] is not None:
        seen = seen | (j < s["prefix"].long()[:, None, None])
    if s["first"] is not None:
        seen = seen & (j >= s["first"].long()[src][..., None])
    if s["window"]:
        seen = seen & (j > pos[..., None] - s["window"])
    seen = seen & (j < end[:, None, None])
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    x = torch.exp(x - top)
    total = x.sum(-1, keepdim=True)
    y = (x.view(b, hk, -1, length) @ v).view(b, hk, hq // hk, n, d) / torch.where(total == 0, torch.ones_like(total), total)
    lse = (top + torch.log(total))[..., 0]
    y, lse = y.permute(0, 3, 1, 2, 4).reshape(b, n, hq, d), lse.permute(0, 3, 1, 2).reshape(b, n, hq)
    return y[new].to(torch.bfloat16), lse[new]


# ---- what a pass cannot do without

def _pairs(case):
    """Visible (query, key) pairs of one head, and keys that any query of its sequence sees, over all sequences
    (documents: as the mean length gives them)."""
    start, new = _lengths(case)
    pairs = keys = 0
    for a, n in zip(start.tolist(), new.tolist()):
        w = case.get("window", 0) if case["mask"] == "window" else 300 if case["mask"] == "documents" else 0
        w = w or a + n
        p = torch.arange(a, a + n, dtype=torch.float64) + 1
        pairs += float(torch.clamp(p, max=w).sum()) * (0.5 if case["mask"] == "documents" and a + n > 300 else 1.0)
        keys += min(a + n, n + w - 1)
    return pairs, keys


def work(case):
    hk, d = case["kv_heads"], case["dim"]
    if case["op"] == "read":
        return {"bytes": case["tokens"] * hk * d * 6 + case["tokens"] / PAGE * hk * 8, "flops": 2 * case["tokens"] * hk * d}
    start, new = _lengths(case)
    t, width = int(new.sum()), case["q_heads"] * d
    if case["op"] == "append":
        # q in and out, k and v in, 8-bit codes out (the few bf16 tail tokens among them), the rotation's rows
        b = t * (4 * width + 2 * hk * d * 3 + 4 * case["rot"])
        if case["kind"] == "int8":
            b += (case["hi"] + case["new_hi"]) * hk * d * 6
        return {"bytes": b, "flops": t * (3 * case["rot"] * (case["q_heads"] + hk) + 4 * hk * d)}
    pairs, keys = _pairs(case)
    return {"bytes": keys * hk * (2 * d + 8 / PAGE) + 4 * t * width + 4 * t * case["q_heads"],
            "flops": 4.0 * d * case["q_heads"] * pairs}


# ---- the definition in 64 bits

def _double_page(s, which, page, h):
    codes = s[which][page, h]
    codes = codes.double() if codes.dtype == torch.int8 else codes.float().double()
    codes = codes * s[which + "_scale"][page, h].double()
    return codes if which == "k" else codes.T


def _double_sequence(s, b, n, h):
    """K and V [n, dim] of head h of sequence b, as the cache holds them."""
    out = []
    for which in ("k", "v"):
        ids = s["table"][b, :n // PAGE].long()
        if which == "k":
            full = _take(s["k"][:, h], ids).double()
        else:
            full = _take(s["v"][:, h], ids).double().transpose(1, 2)
        full = (full * s[which + "_scale"][ids, h].double()[:, None, None]).reshape(-1, s["case"]["dim"])
        if n % PAGE:
            tail = s[which + "_tail"][int(s["tails"][b, 1]), h].double()
            full = torch.cat([full, (tail if which == "k" else tail.T)[:n % PAGE]])
        out.append(full)
    return out


def _exact_attend(s):
    c = s["case"]
    hq, hk, d = c["q_heads"], c["kv_heads"], c["dim"]
    group = hq // hk
    start, cu = s["start"].tolist(), s["cu"].tolist()
    out = torch.zeros(s["total"], hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((s["total"], hq), -math.inf, dtype=torch.float64, device="cuda")
    for b in range(len(start)):
        n = cu[b + 1] - cu[b]
        length = start[b] + n
        j = torch.arange(length, device="cuda")
        for h in range(hk):
            k, v = _double_sequence(s, b, length, h)
            rows = max(1, (1 << 27) // (length * group))
            for at in range(0, n, rows):
                t = torch.arange(at, min(n, at + rows), device="cuda")
                p = (start[b] + t)[:, None]
                hide = (j > p) & (j >= (int(s["prefix"][b]) if s["prefix"] is not None else 0)) if s["prefix"] is not None else j > p
                if s["first"] is not None:
                    hide = hide | (j < s["first"][cu[b] + t].long()[:, None])
                if s["window"]:
                    hide = hide | (p - j >= s["window"])
                for g in range(group):
                    head = h * group + g
                    w = s["scale"] * (s["q"][cu[b] + t, head].double() @ k.T)
                    if s["cap"]:
                        w = s["cap"] * torch.tanh(w / s["cap"])
                    if s["slopes"] is not None:
                        w = w - s["slopes"][head].double() * (p - j).abs()
                    w[hide] = -math.inf
                    z = torch.logsumexp(w, 1)
                    lse[cu[b] + t, head] = z
                    w = torch.exp(w - torch.where(z == -math.inf, torch.zeros_like(z), z)[:, None])
                    out[cu[b] + t, head] = w @ v
    return out, lse


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "read":
        n, hk = case["tokens"], case["kv_heads"]
        kv = [_double_sequence(s, 0, n, h) for h in range(hk)]
        return torch.stack([x[0] for x in kv]), torch.stack([x[1] for x in kv])
    if case["op"] == "attend":
        pairs, _ = _pairs(dict(case, mask="causal"))
        if 4.0 * case["dim"] * case["q_heads"] * pairs > 2e12 or case["seqs"] * case["kv_heads"] > 2000:
            return None
        return _exact_attend(s)
    # rotation in 64 bits; stored values go through bf16 and 8 bits, so only q has a value to compare with
    seq, pos = _positions(s)
    c, n = s["cos"].double()[pos][:, None], s["sin"].double()[pos][:, None]
    q = s["q"].double()
    half = s["cos"].shape[1]
    one = torch.arange(half, device="cuda")
    one, two = (2 * one, 2 * one + 1) if case["interleaved"] else (one, one + half)
    y = q.clone()
    y[..., one] = q[..., one] * c - q[..., two] * n
    y[..., two] = q[..., two] * c + q[..., one] * n
    names = ["q", "k_scale", "v_scale", "k_tail", "v_tail"] + (["read_k", "read_v"] if case["kind"] == "int8" else ["k", "v"])
    return {k: (y if k == "q" else None) for k in names}

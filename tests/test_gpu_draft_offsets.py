"""Offsets past 32 bits in fp8_quantise, fp8_linear, draft_verify and KVTables; calls side by side."""
from __future__ import annotations

import pytest
import torch

import fp8_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _free():
    yield
    torch.cuda.empty_cache()


def _weight(n, k, g):
    return ((torch.randn(n, k, generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn),
            (0.5 + torch.rand(-(-n // 128), -(-k // 128), generator=g)) * 1e-3)


def _check(y, rows, lo, hi, w, ws):
    codes, scales = rows.codes[lo:hi].cpu().float().double(), rows.scales[lo:hi].cpu().double()
    want, tol = ref.linear(codes, scales, w, ws, y.dtype)
    worst = float(((y[lo:hi].cpu().double() - want).abs() / tol).max())
    assert worst <= 1, worst


def test_codes_of_x():
    import bigsmall_amd as bs
    t, k = 1040000, 4224
    assert t * k > 1 << 32
    x = torch.empty(t, k, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    w, ws = _weight(17, k, torch.Generator().manual_seed(2))
    rows = bs.fp8_quantise(x)
    codes, scales = ref.quantise(x[-40:].cpu())
    assert torch.equal(rows.codes[-40:].cpu().float().double(), codes) and torch.equal(rows.scales[-40:].cpu(), scales.float())
    weight = bs.Fp8Weight(w.cuda(), ws.cuda())
    y = bs.fp8_linear(rows, weight)
    _check(y, rows, t - 40, t, w, ws)
    _check(y, rows, 0, 40, w, ws)
    assert torch.equal(bs.fp8_linear(x, weight), y)


def test_results():
    import bigsmall_amd as bs
    t, n, k = 65600, 66001, 100
    assert t * n > 1 << 32
    g = torch.Generator().manual_seed(3)
    w, ws = _weight(n, k, g)
    x = torch.randn(t, k, generator=g).to(torch.float16)
    rows = bs.fp8_quantise(x.cuda())
    y = bs.fp8_linear(rows, bs.Fp8Weight(w.cuda(), ws.cuda()))
    for lo in (0, 40000, t - 20):
        _check(y, rows, lo, lo + 20, w, ws)


@pytest.mark.parametrize("seqs", [3, 300])
def test_rows_of_probabilities(seqs):
    import bigsmall_amd as bs
    t, vocab, n = 33500, 128256, 2 * seqs
    assert (t - n) * vocab > 1 << 31 and t * vocab > 1 << 32
    g = torch.Generator(device="cuda").manual_seed(4)
    p, q = (torch.zeros(t, vocab, dtype=torch.bfloat16, device="cuda") for _ in "pq")
    for m in (p, q):
        m[t - n:] = torch.softmax(torch.randn(n, vocab, generator=g, device="cuda"), 1).bfloat16()
    draft = torch.multinomial(q[t - n:].float(), 1, generator=g)[:, 0]
    accept, pick = torch.rand(n, generator=g, device="cuda"), torch.rand(seqs, generator=g, device="cuda")
    cu = torch.arange(seqs + 1, dtype=torch.int32, device="cuda") * 2
    want = bs.draft_verify(p[t - n:], draft, cu, accept, pick, q=q[t - n:], max_drafts=1)
    wide = [torch.cat([torch.zeros(t - n, dtype=x.dtype, device="cuda"), x]) for x in (draft, accept)]
    got = bs.draft_verify(p, wide[0], cu + (t - n), wide[1], pick, q=q, max_drafts=1)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and int(want[0][:, 0].min()) >= 0


def test_slots():
    import bigsmall_amd as bs
    places, longest = 40000, 65536

    def i32(*x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    t = bs.KVTables(torch.arange(10, dtype=torch.int32, device="cuda"), torch.arange(0, 2 * places, 2, dtype=torch.int32, device="cuda"), longest)
    step, rows = t.step(i32(39999, 0, 32768), i32(70, 1, 2), rows=75)
    want = [39999 * longest + i for i in range(70)] + [0] + [32768 * longest, 32768 * longest + 1] + [-1, -1]
    assert rows.slot.tolist() == want and step.cu.tolist() == [0, 70, 71, 73]
    t.keep(step)
    assert t.length[[39999, 0, 32768]].tolist() == [70, 1, 2] and int(t.table[39999, 0]) == 9
    t.drop(i32(39999, 32768))
    assert t.length.any().item() and int(t.length.sum()) == 1 and int(t.n_free) == 10


def test_two_streams_at_once():
    """Products of more tiles than compute units, and verifications, on two streams side by side and in a graph beside eager ones."""
    import bigsmall_amd as bs
    g = torch.Generator().manual_seed(5)
    weights = [bs.Fp8Weight(*(z.cuda() for z in _weight(4400, k, g))) for k in (300, 700)]
    xs = [(torch.randn(4300, k, generator=g)).bfloat16().cuda() for k in (300, 700)]
    p = torch.softmax(torch.randn(40, 40000, generator=g), 1).cuda()
    rest = torch.randint(40000, (40,), generator=g).cuda(), (torch.arange(9, dtype=torch.int32) * 5).cuda(), torch.rand(40, generator=g).cuda()
    picks = [torch.rand(8, generator=g).cuda() for _ in range(2)]

    def both(i):
        return bs.fp8_linear(xs[i], weights[i]), *bs.draft_verify(p, *rest, picks[i], max_drafts=4)

    want = [both(i) for i in range(2)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = both(0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(both(i))
        graph.replay()
    torch.cuda.synchronize()
    for i in range(2):
        for one in got[i] + ([captured] if i == 0 else []):
            assert all(torch.equal(a, b) for a, b in zip(one, want[i]))

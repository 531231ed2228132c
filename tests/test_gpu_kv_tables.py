"""KVTables on the GPU against books kept in Python, and with the cache's append and attention."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE = 64
COUNT, BOUNDS = 2, 4


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Books:
    """The same in lists."""

    def __init__(self, pages, tails, longest):
        self.free, self.tails, self.cols = list(pages), list(tails), -(-longest // PAGE)
        self.length, self.which, self.pages = [0] * len(tails), [0] * len(tails), [[] for _ in tails]
        self.made = None

    def step(self, seqs, new, sure, rows):
        out, need, total = [], 0, 0
        ok = len(set(seqs)) == len(seqs)
        for i, (s, n) in enumerate(zip(seqs, new)):
            start = self.length[s] if 0 <= s < len(self.tails) else 0
            k = min(n, sure[i]) if sure is not None else n
            ok = ok and 0 <= s < len(self.tails) and n >= 0 and k >= 0 and start + k <= self.cols * PAGE
            end = start + n
            while sure is not None and end > start + k and (end // PAGE * PAGE > start + k or end > self.cols * PAGE):
                end -= 1
            out.append([s, start, end])
            need += end // PAGE - start // PAGE
            total += end - start
        ok = ok and need <= len(self.free) and total <= rows
        stack, cu = list(self.free), [0]
        start, tails, table, owner, position, slot = [], [], [], [], [], []
        for b, (s, lo, hi) in enumerate(out):
            hi = hi if ok else lo
            held = list(self.pages[s]) if 0 <= s < len(self.tails) else []
            held += [stack.pop() for _ in range(hi // PAGE - lo // PAGE)]
            start.append(lo)
            cu.append(cu[-1] + hi - lo)
            moved = hi // PAGE > lo // PAGE
            tail, which = (self.tails[s], self.which[s]) if 0 <= s < len(self.tails) else (0, 0)
            tails.append([tail + which, tail + (which ^ moved)])
            table.append(held + [0] * (self.cols - len(held)))
            owner += [b] * (hi - lo)
            position += range(lo, hi)
            slot += [s * self.cols * PAGE + p for p in range(lo, hi)]
            out[b] = [s, lo, hi]
        rest = [-1] * (rows - cu[-1])
        self.made = (out, table, stack, [min(n, k) for n, k in zip(new, sure)] if sure is not None else None)
        return ok, dict(start=start, cu=cu, tails=tails, table=table), dict(owner=owner + rest, position=position + rest, slot=slot + rest)

    def keep(self, kept=None):
        out, table, stack, sure = self.made
        self.free = stack
        for b, (s, lo, hi) in enumerate(out):
            if hi == lo:
                continue
            k = hi - lo if kept is None or sure is None else max(min(kept[b], hi - lo), min(sure[b], hi - lo))
            self.pages[s] = table[b][:hi // PAGE]
            self.which[s] ^= hi // PAGE > lo // PAGE
            self.length[s] = lo + k

    def drop(self, seqs):
        if len(set(seqs)) < len(seqs) or any(not 0 <= s < len(self.tails) for s in seqs):
            return
        self.free += [p for s in seqs for p in self.pages[s]][::-1]
        for s in seqs:
            self.length[s], self.which[s], self.pages[s] = 0, 0, []


def _same_state(t, b):
    assert t.length.tolist() == b.length and t.which.tolist() == [int(w) for w in b.which]
    assert int(t.n_free) == len(b.free) and t.free[:len(b.free)].tolist() == b.free
    for s, pages in enumerate(b.pages):
        assert t.table[s, :len(pages)].tolist() == pages


def _step(t, b, seqs, new, sure, rows):
    from bigsmall_amd.device import StatusWord
    status = StatusWord("cuda")
    step, r = t.step(_i32(seqs), _i32(new), _i32(sure) if sure is not None else None, rows=rows, status=status)
    ok, arrays, maps = b.step(seqs, new, sure, rows)
    assert bool(int(status.t)) != ok
    for name, want in arrays.items():
        assert getattr(step, name).tolist() == want, name
    for name, want in maps.items():
        assert getattr(r, name).tolist() == want, name
    return step


def _both(pages=200, places=8, longest=1000, seed=0):
    import bigsmall_amd as bs
    g = torch.Generator().manual_seed(seed)
    numbers = (torch.randperm(pages, generator=g) + 5).tolist()
    tails = (2 * torch.randperm(places, generator=g)).tolist()
    return bs.KVTables(_i32(numbers), _i32(tails), longest), Books(numbers, tails, longest)


def test_prompts_drafts_and_drops():
    t, b = _both()
    for seqs, new, sure, rows, kept in (([3, 0, 7], [1, 64, 500], None, 565, None),
                                        ([0, 3, 7, 1], [5, 5, 5, 200], [1, 1, 1, 200], 300, [2, 1, 5, 9]),
                                        ([7, 0], [200, 64], [3, 64], 1000, [1, 3]),
                                        ([0], [0], None, 4, None), ([0], [0], [0], 0, [0]),
                                        ([1, 7, 3, 0], [17, 17, 63, 70], [0, 1, 2, 3], 256, [4, 17, 0, 100]),
                                        ([2, 4, 5, 6], [1, 62, 63, 64], [1, 1, 1, 1], 256, None)):
        step = _step(t, b, seqs, new, sure, rows)
        t.keep(step, _i32(kept) if kept is not None else None)
        b.keep(kept)
        _same_state(t, b)
    for seqs in ([7, 2], [0], [1, 3, 4, 5, 6]):
        t.drop(_i32(seqs))
        b.drop(seqs)
        _same_state(t, b)
    assert int(t.n_free) == 200


@pytest.mark.parametrize("seed", range(8))
def test_random_walks(seed):
    import random
    rng = random.Random(seed)
    t, b = _both(pages=rng.choice([30, 60, 400]), places=rng.choice([1, 5, 70]), longest=rng.choice([64, 300, 2000, 100000]), seed=seed)
    places = len(b.tails)
    for _ in range(30):
        seqs = rng.sample(range(places), rng.randint(1, places))
        new = [rng.choice([0, 1, 2, 5, 17, 63, 64, 65, 130]) for _ in seqs]
        sure = None if rng.random() < 0.3 else [rng.choice([0, 1, 1, n]) for n in new]
        step = _step(t, b, seqs, new, sure, sum(new) + rng.choice([0, 0, 3, -1 if sum(new) else 0]))
        if rng.random() < 0.8:
            kept = None if rng.random() < 0.3 else [rng.randint(0, 130) for _ in seqs]
            t.keep(step, _i32(kept) if kept is not None else None)
            b.keep(kept)
        if rng.random() < 0.4:
            gone = rng.sample(range(places), rng.randint(1, places))
            t.drop(_i32(gone))
            b.drop(gone)
        _same_state(t, b)


def test_many_places_and_long_steps():
    t, b = _both(pages=9000, places=1500, longest=70000, seed=1)
    g = torch.Generator().manual_seed(2)
    new = torch.randint(0, 300, (1400,), generator=g).tolist()
    new[5] = 66000
    seqs = torch.randperm(1500, generator=g)[:1400].tolist()
    step = _step(t, b, seqs, new, None, sum(new) + 1000)
    t.keep(step)
    b.keep()
    _same_state(t, b)
    sure = [1] * 1400
    step = _step(t, b, seqs, [9] * 1400, sure, 9 * 1400)
    kept = torch.randint(0, 10, (1400,), generator=g).tolist()
    t.keep(step, _i32(kept))
    b.keep(kept)
    _same_state(t, b)
    t.drop(_i32(seqs[:900]))
    b.drop(seqs[:900])
    _same_state(t, b)


@pytest.mark.parametrize("seqs,new,sure,rows,bit", [
    ([0, 1, 0], [1, 1, 1], None, 9, BOUNDS), ([0, 8], [1, 1], None, 9, BOUNDS), ([-1], [1], None, 9, BOUNDS), ([0], [-2], None, 9, BOUNDS),
    ([0], [3], [-1], 9, BOUNDS), ([0, 1], [5, 5], None, 9, COUNT), ([0], [1025], None, 2000, COUNT), ([0], [2000], [1025], 3000, COUNT),
    ([2], [2147483647], None, 100, COUNT), ([0, 1, 2], [1000, 1000, 1000], None, 3000, COUNT)])
def test_all_or_nothing(seqs, new, sure, rows, bit):
    from bigsmall_amd.device import StatusWord
    t, b = _both(pages=40)
    first = _step(t, b, [0, 1], [70, 3], None, 73)
    t.keep(first)
    b.keep()
    if bit == COUNT and new[0] == 1025:          # (70 are there: more than 1,024 in all)
        new = [955]
    if sure == [1025]:
        sure = [955]
    status = StatusWord("cuda")
    step, rows_of = t.step(_i32(seqs), _i32(new), _i32(sure) if sure is not None else None, rows=rows, status=status)
    assert int(status.t) == bit
    assert step.cu.tolist() == [0] * (len(seqs) + 1) and rows_of.slot.tolist() == [-1] * rows
    t.keep(step)
    _same_state(t, b)
    _step(t, b, [1], [5], None, 5)


@pytest.mark.parametrize("longest", [1000, 200000])
def test_drop_all_or_nothing(longest):
    from bigsmall_amd.device import StatusWord
    t, b = _both(longest=longest)
    t.keep(_step(t, b, [0, 1], [700, 80], None, 780))
    b.keep()
    for seqs in ([0, 0], [0, 8], [-1], [1, 0, 1]):
        status = StatusWord("cuda")
        t.drop(_i32(seqs), status=status)
        assert int(status.t) == BOUNDS
        _same_state(t, b)
    t.drop(_i32([]))
    _same_state(t, b)
    t.drop(_i32([1, 5, 0]))
    b.drop([1, 5, 0])
    _same_state(t, b)


def test_keep_takes_the_last_step_once():
    t, b = _both()
    one, _ = t.step(_i32([0]), _i32([5]), rows=5)
    two, _ = t.step(_i32([0]), _i32([7]), rows=7)
    with pytest.raises(RuntimeError, match="last"):
        t.keep(one)
    t.keep(two)
    with pytest.raises(RuntimeError, match="last"):
        t.keep(two)
    assert t.length.tolist()[0] == 7
    step, _ = t.step(_i32([0]), _i32([7]), rows=7)
    t.drop(_i32([0]))
    with pytest.raises(RuntimeError, match="last"):
        t.keep(step)


def test_captured():
    """Step, keep and drop in a graph: each replay goes on from the books as they are."""
    t, b = _both()
    seqs, new, sure, kept = _i32([4, 2]), _i32([5, 5]), _i32([1, 1]), _i32([0, 0])
    t.keep(_step(t, b, [4, 2], [60, 600], None, 660))
    b.keep()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step, rows = t.step(seqs, new, sure, rows=10)
        t.keep(step, kept)
    _same_state(t, b)
    for i in range(8):
        k = [1 + i % 5, 1 + (3 * i) % 5]
        kept.copy_(_i32(k))
        graph.replay()
        _, arrays, maps = b.step([4, 2], [5, 5], [1, 1], 10)
        b.keep(k)
        assert step.table.tolist() == arrays["table"] and step.cu.tolist() == arrays["cu"] and rows.slot.tolist() == maps["slot"]
        _same_state(t, b)

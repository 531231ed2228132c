"""The paged KV cache's host side at the edges of what its calls take."""
from __future__ import annotations

import ctypes

import pytest
import torch

from bigsmall_amd.paged_kv import KVPool, _Books, kv_append, kv_attend
from test_paged_kv_cpu import _batch, _parts, on_gpu  # noqa: F401 (a fixture)


def test_calls_refuse_rows_that_are_not_the_steps(on_gpu):
    pool, batch = KVPool(*_parts()), _batch(total=2)
    for n in (0, 1, 3):
        x = torch.zeros(n, 2, 64, dtype=torch.bfloat16)
        with pytest.raises(ValueError, match="the step has 2"):
            kv_append(pool, batch, x, x, x)
        with pytest.raises(ValueError, match="the step has 2"):
            kv_append(pool, batch, None, x, x)
        with pytest.raises(ValueError, match="the step has 2"):
            kv_attend(pool, batch, x)


def _state(books):
    return books.free[:], books.free_tails[:], {s: [e[0], e[1][:], e[2], e[3]] for s, e in books.seqs.items()}


def test_books_take_a_step_back():
    books = _Books(10, 4)
    a, b, c = books.add(), books.add(), books.add()
    books.step({a: 70, b: 64, c: 1})
    for new in ({a: 1}, {b: 63, a: 58}, {c: 63, b: 130, a: 200}, {a: 57, c: 64}):
        was, before = _state(books), books.note(new)
        books.step(new)
        assert _state(books) != was
        books.undo(before)
        assert _state(books) == was
        with pytest.raises(RuntimeError, match="gone on"):
            books.undo(before)
        assert _state(books) == was
    # not after a later step, nor after a drop: nothing is touched
    first, _ = books.note({a: 3, b: 3}), books.step({a: 3, b: 3})
    second, _ = books.note({b: 1}), books.step({b: 1})
    was = _state(books)
    with pytest.raises(RuntimeError, match=f"sequence {b}"):
        books.undo(first)
    assert _state(books) == was
    books.undo(second)
    books.undo(first)
    before, _ = books.note({a: 3}), books.step({a: 3})
    books.drop(a)
    was = _state(books)
    with pytest.raises(RuntimeError, match="dropped"):
        books.undo(before)
    assert _state(books) == was
    with pytest.raises(KeyError):
        books.note({a: 1})


def test_forward_that_raises_takes_its_step_back():
    """With the cache's books and a layer that fails, on the host."""
    from bigsmall_amd.paged_llama import PagedLlama
    books = _Books(10, 2)

    class Cache:
        def step(self, new):
            self.before = books.note(new)
            books.step(new)
            return self

        def undo(self, step):
            books.undo(step.before)

    class Loader:
        def iter_layers(self, progress):
            raise MemoryError("layer 0")
    m = PagedLlama.__new__(PagedLlama)
    m.loader, m.cache, m.device, m.embed = Loader(), Cache(), torch.device("cpu"), torch.zeros(10, 4)
    a, b = books.add(), books.add()
    books.step({a: 60})
    was = _state(books)
    for new in ({a: [1] * 540, b: [2]}, {b: torch.tensor([3.5])}, {b: torch.zeros(1, 4, dtype=torch.int64)}):
        with pytest.raises((MemoryError, IndexError, RuntimeError)):
            m.forward(new)
        assert _state(books) == was


def test_generate_with_more_prompts_than_places_keeps_none():
    from types import SimpleNamespace

    from bigsmall_amd.paged_llama import PagedLlama
    books = _Books(4, 2)
    m = PagedLlama.__new__(PagedLlama)
    m.cache = SimpleNamespace(add=books.add, drop=books.drop)
    kept = books.add()
    for _ in range(3):
        with pytest.raises(RuntimeError, match="sequences"):
            m.generate([torch.zeros(1, dtype=torch.int64)] * 2, 1)
    assert list(books.seqs) == [kept] and len(books.free_tails) == 1


def test_park_refuses_a_sequence_without_tokens():
    """(The store has no entries of no elements: it could not be brought back.)"""
    from types import SimpleNamespace

    from bigsmall_amd.paged_llama import PagedLlama
    books, sets = _Books(4, 2), []
    m = PagedLlama.__new__(PagedLlama)
    m.cache = SimpleNamespace(length=books.length, drop=books.drop, pools=[None], read=lambda i, seq: (None, None))
    seq = books.add()
    with pytest.raises(ValueError, match="no tokens"):
        m.park(seq, SimpleNamespace(set=lambda *a: sets.append(a)))
    assert not sets and seq in books.seqs
    books.step({seq: 1})
    m.park(seq, SimpleNamespace(set=lambda *a: sets.append(a)))
    assert len(sets) == 1 and seq not in books.seqs


def test_rows_of_a_call_are_its_own(on_gpu, monkeypatch):
    """Two calls of different sizes on one batch, the second made while the first is on its way: each C structure names
    its own rows."""
    from bigsmall_amd import _native, paged_kv
    pool, batch = KVPool(*_parts()), _batch()
    seen = []


    class Lib:
        def bs_kv_attend_work_bytes(self, pool_ref, step, heads):
            return 0

    def call(name, p, step, *rest):
        if len(seen) < 2:                              # another thread's turn
            seen.append(None)
            kv_attend(pool, batch, torch.zeros(5, 2, 64, dtype=torch.bfloat16))
        c = _native.BsKvBatch.from_buffer_copy(step if isinstance(step, bytes) else step._obj)
        seen.append((name, c.n_rows, c.n_seqs, c.max_len, c.start))
    monkeypatch.setattr(paged_kv._native, "lib", lambda: Lib())
    monkeypatch.setattr(paged_kv, "_call", call)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    kv_attend(pool, batch, x)
    del seen[:]
    kv_append(pool, batch, None, x, x)
    calls = [s for s in seen if s]
    assert calls == [("bs_kv_attend", 5, 2, 6, batch.start.data_ptr()), ("bs_kv_attend", 5, 2, 6, batch.start.data_ptr()),
                     ("bs_kv_append", 3, 2, 6, batch.start.data_ptr())]


def test_strides_of_dimensions_of_one_are_not_looked_at():
    from bigsmall_amd.paged_kv import _rows
    pool = KVPool(*_parts())
    wide = torch.zeros(4, 2 * 64 + 3, dtype=torch.bfloat16)
    many = wide[:, :-3].unflatten(1, (2, 64))
    for i in range(4):
        one = many[i:i + 1]
        assert one.is_contiguous() and one.stride(0) % 8
        t, n, heads, p, s0, s1 = _rows("q", one, None, None, pool)
        assert (n, heads) == (1, 2) and p % 16 == 0 and s0 % 8 == 0 and s1 == 64 and t.data_ptr() == p
        assert (t is one) == (one.data_ptr() % 16 == 0)
    t, _, _, p, s0, s1 = _rows("q", many, None, None, pool)
    assert t is not many and (s0, s1) == (128, 64) and p % 16 == 0
    odd = torch.zeros(3, 1, 64, dtype=torch.bfloat16).as_strided((3, 1, 64), (64, 5, 1))
    t, _, _, _, s0, s1 = _rows("q", odd, None, None, pool)
    assert (s0, s1 % 8) == (64, 0)


class _Names:
    """A loader's names; nothing may be decoded."""

    def __init__(self, layers=2, extra=(), without=()):
        names = ["model.embed_tokens.weight", "model.norm.weight", "lm_head.weight"]
        for i in range(layers):
            names += [f"model.layers.{i}.{n}.weight" for n in
                      ("input_layernorm", "post_attention_layernorm", "self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj",
                       "self_attn.o_proj", "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj")]
        self.names, self.layers = [n for n in names + list(extra) if n not in without], layers

    def layer_count(self):
        return self.layers

    def layer_tensor_names(self, i):
        return [n for n in self.names if n.startswith(f"model.layers.{i}.")]

    def non_layer_tensor_names(self):
        return [n for n in self.names if not n.startswith("model.layers.")]

    def load_non_layer_tensors(self):
        raise AssertionError("decoding began")


def test_models_that_are_not_computed_are_refused():
    from transformers import LlamaConfig, MistralConfig

    from bigsmall_amd.paged_kv import Rope
    from bigsmall_amd.paged_llama import PagedLlama, check_model

    def config(kind=LlamaConfig, **change):
        args = dict(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                    max_position_embeddings=512)
        return kind(**{**args, **change})

    llama3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
              "original_max_position_embeddings": 128, "rope_theta": 10000.0}
    old = config()
    old.rope_parameters, old.rope_theta = None, 10000.0             # as earlier versions of the library have it
    old.rope_scaling = {"type": "dynamic", "factor": 2.0}
    other = config()
    other.model_type = "granite"
    for c, what in ((config(rope_parameters=llama3), "llama3"), (config(rope_parameters={"rope_type": "linear", "factor": 2.0, "rope_theta": 1e4}), "linear"),
                    (old, "dynamic"), (config(rope_parameters={"rope_type": "default", "rope_theta": 1e4, "partial_rotary_factor": 0.5}), "0.5"),
                    (config(attention_bias=True), "attention_bias"), (config(mlp_bias=True), "mlp_bias"),
                    (config(hidden_act="gelu"), "gelu"), (other, "granite"), (config(MistralConfig, sliding_window=128), "window of 128"),
                    (config(num_hidden_layers=3), "3 layers")):
        with pytest.raises(ValueError, match=what):
            PagedLlama(_Names(), c, pages=1, sequences=1)
    for names, what in ((_Names(extra=["model.layers.1.self_attn.q_proj.bias"]), "q_proj.bias"),
                        (_Names(extra=["model.layers.0.self_attn.q_norm.weight"]), "q_norm"), (_Names(extra=["lm_head.bias"]), "lm_head.bias"),
                        (_Names(without=["model.layers.1.mlp.up_proj.weight"]), "missing tensors: model.layers.1.mlp.up_proj")):
        with pytest.raises(ValueError, match=what):
            PagedLlama(names, config(), pages=1, sequences=1)
    # what it does compute
    rope = Rope.from_theta(64, 10, device="cpu")
    check_model(config(), _Names())
    check_model(config(rope_parameters=llama3), _Names(), rope)
    check_model(config(MistralConfig, sliding_window=None), _Names())
    check_model(config(MistralConfig, sliding_window=512), _Names())
    check_model(config(), _Names(extra=["model.layers.0.self_attn.rotary_emb.inv_freq"], without=["lm_head.weight"]))
    with pytest.raises(AssertionError, match="decoding began"):
        PagedLlama(_Names(), config(), pages=1, sequences=1)


def test_calls_that_would_lose_a_gradient_are_refused(on_gpu, monkeypatch):
    from bigsmall_amd import paged_kv
    pool, batch = KVPool(*_parts()), _batch()
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    g = x.clone().requires_grad_()
    for call in (lambda: kv_append(pool, batch, g, x, x), lambda: kv_append(pool, batch, x, g, x), lambda: kv_append(pool, batch, x, x, g),
                 lambda: kv_append(pool, batch, x, x, g * 2), lambda: kv_attend(pool, batch, g),
                 lambda: kv_attend(pool, batch, x, slopes=torch.zeros(2, requires_grad=True))):
        with pytest.raises(RuntimeError, match="backward"):
            call()
    calls = []

    class Lib:
        def bs_kv_attend_work_bytes(self, *a):
            return 0
    monkeypatch.setattr(paged_kv._native, "lib", lambda: Lib())
    monkeypatch.setattr(paged_kv, "_call", lambda name, *rest: calls.append(name))
    kv_append(pool, batch, g.detach(), x, x)
    with torch.no_grad():
        kv_append(pool, batch, g, g, g)
        kv_attend(pool, batch, g)
    assert calls == ["bs_kv_append", "bs_kv_append", "bs_kv_attend"]


def test_struct_layouts_match_the_kv_header(tmp_path):
    """Offsets and sizes of every field of include/bigsmall_kv.h's structures: of their ctypes copies, and of the two that
    are packed by hand."""
    import shutil
    import subprocess
    from pathlib import Path

    from bigsmall_amd import _native, paged_kv
    if shutil.which("gcc") is None:
        pytest.skip("needs gcc")
    structs = {"bs_kv_pool": _native.BsKvPool, "bs_kv_batch": _native.BsKvBatch, "bs_kv_rows": _native.BsKvRows,
               "bs_kv_query": _native.BsKvQuery}
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "bigsmall_kv.h"', "int main(void) {"]
    for name, c in structs.items():
        lines.append(f'  printf("{name} sizeof %zu 0\\n", sizeof({name}));')
        lines += [f'  printf("{name} {f[0]} %zu %zu\\n", offsetof({name}, {f[0]}), sizeof((({name}*)0)->{f[0]}));' for f in c._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    inc = Path(__file__).resolve().parents[1] / "include"
    subprocess.run(["gcc", "-I", str(inc), str(src), "-o", str(exe)], check=True, capture_output=True)
    got = {}
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, field, at, size = line.split()
        got[name, field] = (int(at), int(size))
    for name, c in structs.items():
        assert got[name, "sizeof"][0] == ctypes.sizeof(c), name
        for f in c._fields_:
            assert got[name, f[0]] == (getattr(c, f[0]).offset, getattr(c, f[0]).size), (name, f[0])
        # nothing between the fields: together they are the structure, the last one's padding aside
        end = max(at + size for (n, f), (at, size) in got.items() if n == name and f != "sizeof")
        assert sum(size for (n, f), (at, size) in got.items() if n == name and f != "sizeof") == end and ctypes.sizeof(c) - end < 8
    # packed by hand: each field's number, recognisable, where the C structure has it
    for packer, c in ((paged_kv._ROWS, _native.BsKvRows), (paged_kv._QUERY, _native.BsKvQuery)):
        assert packer.size == ctypes.sizeof(c)
        values = [float(i + 1) if f[1] is ctypes.c_float else i + 1 for i, f in enumerate(c._fields_)]
        back = c.from_buffer_copy(packer.pack(*values))
        assert [getattr(back, f[0]) for f in c._fields_] == values
    batch = _batch()
    a, b = _native.BsKvBatch.from_buffer_copy(batch.with_rows(12345)), batch.c
    assert a.n_rows == 12345 and all(getattr(a, f[0]) == getattr(b, f[0]) for f in b._fields_ if f[0] != "n_rows")

"""fp8 products, draft verification and the cache's tables on the GPU: argument checks, the C entry points' refusals, and
the C structures against their headers. Nothing is launched."""
from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

import fp8_reference as ref
from bigsmall_amd import _native, draft, fp8, kv_tables
from bigsmall_amd.draft import draft_verify
from bigsmall_amd.fp8 import Fp8Weight, fp8_linear, fp8_quantise
from bigsmall_amd.kv_tables import KVTables

E4M3 = torch.float8_e4m3fn


def _weight(n=200, k=300):
    return torch.zeros(n, k).to(E4M3), torch.ones(-(-n // 128), -(-k // 128))


def test_weight_refuses_what_does_not_fit():
    codes, scales = _weight()
    w = Fp8Weight(codes, scales)
    assert (w.outer, w.inner, w.c.stride, w.c.scale_stride) == (200, 300, 384, 3)
    assert w.codes.shape == (200, 300)
    for c, s in ((codes.float(), scales), (codes[0], scales), (codes[:0], scales[:0]), (codes[:, :0], scales[:, :0]), (codes, scales.double()),
                 (codes, scales[:1]), (codes, scales[:, :2]), (codes, scales.bfloat16()), (codes.view(torch.uint8), scales), (None, scales),
                 (codes, None), (codes.view(torch.uint8).view(torch.float8_e5m2), scales)):
        with pytest.raises(ValueError, match="Fp8Weight"):
            Fp8Weight(c, s)


def test_weight_is_used_in_place_or_padded():
    codes, scales = _weight(130, 256)
    assert Fp8Weight(codes, scales).codes.data_ptr() == codes.data_ptr()
    ragged = torch.randint(0, 120, (5, 130), dtype=torch.uint8).view(E4M3)
    w = Fp8Weight(ragged, torch.ones(1, 2))
    flat = torch.as_strided(w.codes.view(torch.uint8), (5, 256), (256, 1))
    assert torch.equal(flat[:, :130], ragged.view(torch.uint8)) and int(flat[:, 130:].sum()) == 0


def test_calls_refuse_what_does_not_fit():
    w = Fp8Weight(*_weight())
    x = torch.zeros(2, 300, dtype=torch.bfloat16)
    for bad in (x.float(), x[:, :299], torch.zeros((), dtype=torch.bfloat16), None, x.to(E4M3)):
        with pytest.raises(ValueError):
            fp8_linear(bad, w)
    for bad in (x.float(), torch.zeros((), dtype=torch.bfloat16), x[:, :0], None):
        with pytest.raises(ValueError):
            fp8_quantise(bad)
    with pytest.raises(ValueError, match="Fp8Weight"):
        fp8_linear(x, x)
    for call in (lambda: fp8_linear(x, w), lambda: fp8_quantise(x)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def _verify(**change):
    args = dict(p=torch.zeros(5, 10), draft=torch.zeros(5, dtype=torch.int64), cu=torch.tensor([0, 2, 5], dtype=torch.int32),
                accept=torch.zeros(5), pick=torch.zeros(2))
    args.update(change)
    return draft_verify(**args)


def test_verify_refuses_what_does_not_fit():
    with pytest.raises(RuntimeError, match="GPU"):
        _verify()
    for change in (dict(p=torch.zeros(5, 10, dtype=torch.float64)), dict(p=torch.zeros(10)), dict(p=torch.zeros(5, 0)), dict(p=None),
                   dict(draft=torch.zeros(4, dtype=torch.int64)), dict(draft=torch.zeros(5, dtype=torch.int32)), dict(accept=torch.zeros(6)),
                   dict(accept=torch.zeros(5).double()), dict(cu=torch.tensor([0, 2, 5])), dict(cu=torch.zeros(0, dtype=torch.int32)),
                   dict(pick=torch.zeros(3)), dict(q=torch.zeros(5, 9)), dict(q=torch.zeros(4, 10)), dict(q=torch.zeros(5, 10).bfloat16()),
                   dict(max_drafts=-1), dict(max_drafts=1025), dict(accept=torch.zeros(5, 1))):
        with pytest.raises(ValueError):
            _verify(**change)


def test_tables_refuse_what_does_not_fit():
    pages, tails = torch.arange(4, dtype=torch.int32), torch.arange(0, 4, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        KVTables(pages, tails, 100)
    for p, t, n in ((pages.long(), tails, 100), (pages, tails.long(), 100), (pages[:0], tails, 100), (pages, tails[:0], 100), (pages, tails, 0),
                    (pages, tails, -5), (pages.view(2, 2), tails, 100), (pages, tails, 1 << 31)):
        with pytest.raises(ValueError):
            KVTables(p, t, n)


@pytest.fixture
def tables(monkeypatch):
    """Books on the host, whose calls come to their checks; nothing may be launched."""
    t = KVTables.__new__(KVTables)
    t.places, t.longest, t.device, t.index, t._made = 3, 128, torch.device("cpu"), -1, None

    def nothing(self, name, *args):
        raise AssertionError(f"{name} was called")
    monkeypatch.setattr(KVTables, "_call", nothing)
    return t


def test_steps_refuse_what_does_not_fit(tables):
    a, b = torch.zeros(2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    for seqs, new, sure, rows in ((a.long(), a, None, 2), (a, a.long(), None, 2), (a, a, a.long(), 2), (a, a[:1], None, 2), (a, a, a[:1], 2),
                                  (b, b, None, 4), (a[:0], a[:0], None, 0), (a, a, None, -1), (a, a, None, 1 << 30), (a.view(1, 2), a, None, 2),
                                  ([0, 1], a, None, 2)):
        with pytest.raises(ValueError):
            tables.step(seqs, new, sure, rows=rows)
    for seqs in (b, a.long(), None):
        with pytest.raises(ValueError):
            tables.drop(seqs)
    with pytest.raises(RuntimeError, match="last"):
        tables.keep(None)


def _aligned(n):
    return (ctypes.c_uint8 * (n + 64))()


def _at(buf):
    return (ctypes.addressof(buf) + 63) // 64 * 64


def test_c_entries_refuse_bad_arguments():
    L, buf = _native.lib(), _aligned(4096)
    at = _at(buf)
    ARG, CAP = _native.BS_ERR_ARG, _native.BS_ERR_CAP

    def rows(**c):
        f = dict(codes=at, scales=at, rows=2, cols=200, code_stride=256, scale_stride=2)
        f.update(c)
        return _native.BsFp8Rows(**f)

    def weight(**c):
        f = dict(codes=at, scales=at, outer=8, inner=200, stride=256, scale_stride=2)
        f.update(c)
        return _native.BsFp8Weight(**f)

    p = ctypes.byref
    assert L.bs_fp8_quantise(at, 0, 200, p(rows(rows=0)), None) == 0
    for r, x, kind, stride in ((rows(codes=at + 8), at, 0, 200), (rows(codes=0), at, 0, 200), (rows(scales=0), at, 0, 200), (rows(cols=0), at, 0, 200),
                               (rows(code_stride=384), at, 0, 200), (rows(code_stride=128), at, 0, 200), (rows(code_stride=250), at, 0, 200),
                               (rows(scale_stride=1), at, 0, 200), (rows(), 0, 0, 200), (rows(), at + 1, 0, 200), (rows(), at, 2, 200),
                               (rows(), at, 0, -1), (rows(rows=1 << 30, scale_stride=1 << 30), at, 0, 200)):
        assert L.bs_fp8_quantise(x, kind, stride, p(r), None) == ARG
    assert L.bs_fp8_quantise(at, 0, 200, None, None) == ARG
    assert L.bs_fp8_linear(p(rows(rows=0)), p(weight()), at, 0, 8, None) == 0
    for r, w, y, kind, stride in ((rows(cols=201), weight(), at, 0, 8), (rows(), weight(stride=200), at, 0, 8), (rows(), weight(stride=128), at, 0, 8),
                                  (rows(), weight(codes=at + 4), at, 0, 8), (rows(), weight(scale_stride=1), at, 0, 8), (rows(), weight(outer=0), at, 0, 8),
                                  (rows(), weight(scales=0), at, 0, 8), (rows(), weight(), 0, 0, 8), (rows(), weight(), at, 0, 7), (rows(), weight(), at, 3, 8),
                                  (rows(), weight(), at + 1, 0, 8)):
        assert L.bs_fp8_linear(p(r), p(w), y, kind, stride, None) == ARG
    assert L.bs_fp8_linear_values(at, 0, 200, 0, p(weight()), at, 0, 8, None, 0, None) == 0
    for x, xk, xs, n, w, y, kind, stride in ((0, 0, 200, 2, weight(), at, 0, 8), (at + 1, 0, 200, 2, weight(), at, 0, 8), (at, 2, 200, 2, weight(), at, 0, 8),
                                             (at, 0, -1, 2, weight(), at, 0, 8), (at, 0, 200, 1 << 21, weight(), at, 0, 8), (at, 0, 200, 2, weight(inner=0), at, 0, 8),
                                             (at, 0, 200, 2, weight(), 0, 0, 8), (at, 0, 200, 2, weight(), at, 2, 8), (at, 0, 200, 2, weight(), at, 0, 7)):
        assert L.bs_fp8_linear_values(x, xk, xs, n, p(w), y, kind, stride, at, 1 << 40, None) == ARG
    big = weight(outer=4096, inner=100, stride=128, scale_stride=1)
    need = L.bs_fp8_linear_values_work_bytes(500, p(big))
    assert need >= 500 * 132 and L.bs_fp8_linear_values_work_bytes(1, p(big)) == 0
    assert L.bs_fp8_linear_values(at, 0, 100, 500, p(big), at, 0, 4096, at, need - 1, None) == CAP
    assert L.bs_fp8_linear_values(at, 0, 100, 500, p(big), at, 0, 4096, at + 8, need, None) == CAP

    def batch(**c):
        f = dict(p=at, q=at, draft=at, accept=at, cu=at, pick=at, tokens=at, counts=at, p_stride=10, q_stride=10, type=0, n_rows=3, vocab=10, n_seqs=1,
                 max_drafts=2)
        f.update(c)
        return _native.BsDraftBatch(**f)

    assert L.bs_draft_verify(p(batch(n_seqs=0)), None, 0, None, None) == 0
    for c in (dict(p=0), dict(draft=0), dict(accept=0), dict(cu=0), dict(pick=0), dict(tokens=0), dict(counts=0), dict(type=3), dict(vocab=0),
              dict(vocab=1 << 31), dict(max_drafts=1025), dict(n_seqs=1 << 21), dict(p=at + 2), dict(q=at + 1), dict(p_stride=-1), dict(n_rows=1 << 31)):
        assert L.bs_draft_verify(p(batch(**c)), at, 1 << 30, None, None) == ARG, c
    large = batch(vocab=100000, p_stride=100000, q_stride=100000)
    need = L.bs_draft_verify_work_bytes(1, 100000)
    assert need > 0 and L.bs_draft_verify(p(large), at, need - 1, None, None) == CAP
    assert L.bs_draft_verify(p(large), at + 4, need, None, None) == CAP and L.bs_draft_verify(p(large), None, need, None, None) == CAP

    def books(**c):
        f = dict(length=at, which=at, table=at, free=at, n_free=at, tails=at, n_places=4, cols=2, n_pages=8)
        f.update(c)
        return _native.BsKvBooks(**f)

    def tables(**c):
        f = dict(seqs=at, start=at, cu=at, tails=at, table=at, owner=at, position=at, slot=at, n_seqs=2, n_rows=3, max_new=3)
        f.update(c)
        return _native.BsKvTables(**f)

    assert L.bs_kv_books_step(p(books()), p(tables(n_seqs=0)), None, None, None, None) == 0
    bad_books = [dict([(n, 0)]) for n in ("length", "which", "table", "free", "n_free", "tails", "n_places", "cols", "n_pages")] + \
        [dict(n_places=65537), dict(cols=1 << 24), dict(n_pages=1 << 30)]
    bad_steps = [dict([(n, 0)]) for n in ("seqs", "start", "cu", "tails", "table", "owner", "position", "slot")] + \
        [dict(n_seqs=5), dict(n_rows=1 << 30), dict(slot=at + 4)]
    for c in bad_books:
        assert L.bs_kv_books_step(p(books(**c)), p(tables()), at, None, None, None) == ARG, c
        assert L.bs_kv_books_keep(p(books(**c)), p(tables()), None, None, None) == ARG, c
        assert L.bs_kv_books_drop(p(books(**c)), at, 1, None, None) == ARG, c
    for c in bad_steps:
        assert L.bs_kv_books_step(p(books()), p(tables(**c)), at, None, None, None) == ARG, c
        assert L.bs_kv_books_keep(p(books()), p(tables(**c)), None, None, None) == ARG, c
    assert L.bs_kv_books_step(p(books()), p(tables()), None, None, None, None) == ARG
    assert L.bs_kv_books_drop(p(books()), None, 1, None, None) == ARG and L.bs_kv_books_drop(p(books()), at, 5, None, None) == ARG
    assert L.bs_kv_books_drop(p(books()), None, 0, None, None) == 0


def test_c_structures_match_their_headers(tmp_path):
    mirrors = {"bs_kv_books": _native.BsKvBooks, "bs_kv_tables": _native.BsKvTables, "bs_fp8_rows": _native.BsFp8Rows,
               "bs_fp8_weight": _native.BsFp8Weight, "bs_draft_batch": _native.BsDraftBatch}
    lines = ["#include <stddef.h>", "#include <stdio.h>"] + [f'#include "bigsmall_{h}.h"' for h in ("kv", "fp8", "draft")] + ["int main(void) {"]
    for name, mirror in mirrors.items():
        lines.append(f'  printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name}.{f[0]} %zu %zu\\n", offsetof({name}, {f[0]}), sizeof((({name}*)0)->{f[0]}));' for f in mirror._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    inc = Path(__file__).resolve().parents[1] / "include"
    subprocess.run(["gcc", "-I", str(inc), str(src), "-o", str(exe)], check=True, capture_output=True)
    got = {l.split()[0]: tuple(map(int, l.split()[1:])) for l in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()}
    for name, mirror in mirrors.items():
        assert got[name] == (ctypes.sizeof(mirror),)
        for f in mirror._fields_:
            assert got[f"{name}.{f[0]}"] == (getattr(mirror, f[0]).offset, ctypes.sizeof(f[1])), (name, f[0])
    # packed by hand: each field's number where the C structure has it
    for packer, mirror in ((draft._BATCH, _native.BsDraftBatch), (fp8._ROWS, _native.BsFp8Rows), (kv_tables._TABLES, _native.BsKvTables)):
        values = [i + 1 for i in range(len(mirror._fields_))]
        back = mirror.from_buffer_copy(packer.pack(*values))
        assert packer.size == ctypes.sizeof(mirror) and [getattr(back, f[0]) for f in mirror._fields_] == values
    from bigsmall_amd import paged_kv
    b = _native.BsKvBatch.from_buffer_copy(paged_kv._BATCH_HEAD.pack(1, 2, 3, 4, 5, 6, 7) + (8).to_bytes(4, "little") + paged_kv._BATCH_REST.pack(9, 10))
    assert [getattr(b, f[0]) for f in _native.BsKvBatch._fields_] == list(range(1, 11))


def test_reference_quantiser_is_torchs_rounding():
    """The tests' own rounding to e4m3 against torch's conversion, on quotients that are exact in f32."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(20, 256, generator=g)
    x[:, ::128] = 7.0 * 2.0 ** torch.randint(-3, 3, (20, 1), generator=g)       # 448 / a is a power of two
    x[:, ::128] = x.abs().amax(1, keepdim=True).clamp(min=7.0 * 4)
    x[:, 0] = x[:, 128] = 7.0 * 4
    codes, scales = ref.quantise(x)
    assert torch.equal(codes, (x * 16).to(E4M3).double()) and torch.equal(scales, torch.full((20, 2), 28 / 448.0).double())


def test_exported():
    import bigsmall_amd as bs
    assert (bs.Fp8Weight, bs.fp8_quantise, bs.fp8_linear) == (fp8.Fp8Weight, fp8.fp8_quantise, fp8.fp8_linear)
    assert (bs.draft_verify, bs.KVTables, bs.StepRows) == (draft.draft_verify, kv_tables.KVTables, kv_tables.StepRows)


class _Names:
    """A loader's index."""

    dtype = None

    def __init__(self, layer=(), top=()):
        from bigsmall_amd.paged_llama import _LAYER, _TOP
        self.top, self.layer = list(_TOP) + list(top), [f"model.layers.0.{n}" for n in list(_LAYER) + list(layer)]

    def layer_count(self):
        return 1

    def non_layer_tensor_names(self):
        return self.top

    def layer_tensor_names(self, i):
        return self.layer


def test_models_with_fp8_weights():
    from types import SimpleNamespace

    from bigsmall_amd.paged_llama import _SCALES, check_model
    fp8_way = {"quant_method": "fp8", "weight_block_size": [128, 128], "activation_scheme": "dynamic"}

    def config(q=None):
        return SimpleNamespace(model_type="llama", num_hidden_layers=1, max_position_embeddings=64, quantization_config=q)

    check_model(config(), _Names())
    check_model(config(), _Names(_SCALES))
    check_model(config(), _Names(["mlp.up_proj.weight_scale_inv"]))            # some of them in bf16
    check_model(config(fp8_way), _Names(_SCALES))
    check_model(config(SimpleNamespace(to_dict=lambda: fp8_way)), _Names(_SCALES))
    for change in (dict(quant_method="awq"), dict(weight_block_size=[64, 128]), dict(weight_block_size=None), dict(activation_scheme="static")):
        with pytest.raises(ValueError, match="quantised otherwise"):
            check_model(config(dict(fp8_way, **change)), _Names(_SCALES))
    check_model(config(dict(quant_method="awq")), _Names())                    # weights as they are, whatever they were made from
    for names in (_Names(["input_layernorm.weight_scale_inv"]), _Names(["mlp.up_proj.input_scale"]), _Names(top=["lm_head.weight_scale_inv"])):
        with pytest.raises(ValueError, match="does not use"):
            check_model(config(), names)
    loader = _Names(_SCALES)
    loader.dtype = torch.bfloat16
    with pytest.raises(ValueError, match="casts"):
        check_model(config(), loader)
    with pytest.raises(ValueError, match="scale_inv"):
        from bigsmall_amd.paged_llama import PagedLlama
        PagedLlama._project(torch.zeros(1, 128), {"a.weight": torch.zeros(128, 128).to(E4M3)}, "a")

"""CPU-only checks of the C boundary of the rotary positions and the paged cache: symbols, struct layouts, and
what is refused on the host before a device is touched."""

import ctypes as C
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import superl8_b200 as s8
from superl8_b200 import _lib

HEADER = Path(__file__).resolve().parent.parent / "include" / "superl8_b200_paged.h"
STRUCTS = {"sl8_rope_params": _lib.RopeParams, "sl8_paged_cache": _lib.PagedCache, "sl8_append_params": _lib.AppendParams,
           "sl8_paged_attn_params": _lib.PagedAttnParams}


def test_symbols_and_struct_layouts(tmp_path):
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    names = sorted(set(re.findall(r"\b(sl8_[a-z0-9_]+)\s*\(", text)))
    assert len(names) >= 5
    for n in names:
        assert hasattr(_lib.load(), n) and n in _lib.SIGNATURES, n
    assert set(re.findall(r"typedef struct (sl8_[a-z0-9_]+)", text)) == set(STRUCTS)
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler")
    lines = ['#include <stdio.h>', f'#include "{HEADER.parent / "superl8_b200.h"}"', "int main(void) {"]
    for name, cls in STRUCTS.items():
        lines.append(f'  printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run([gcc, "-std=c99", "-Wall", "-Werror", str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    got = {(a, b): int(c) for a, b, c in (ln.split() for ln in out.splitlines())}
    for name, cls in STRUCTS.items():
        assert got[name, "size"] == C.sizeof(cls), name
        for f, _ in cls._fields_:
            assert got[name, f] == getattr(cls, f).offset, f"{name}.{f}"
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
        assert sum(len(d.split(",")) for d in body.split(";") if d.strip()) == len(cls._fields_), name


CACHE = dict(k=16, v=16, k_scale=16, v_scale=16, block_table=16, table_stride=4, context_lens=16, num_pages=8, Hkv=2, page_size=16,
             D=128, max_pages=4)


def test_rope_is_refused_on_the_host():
    f = _lib.load().sl8_rope
    ok = dict(q=16, q_out=16, positions=16, inv_freq=16, B=1, Hq=2, S=3, D=64, rot=64, n_axes=1)
    assert f(None, None) == _lib.ERR_NULL
    for bad in (dict(D=63), dict(rot=66), dict(rot=3), dict(B=-1), dict(n_axes=0), dict(S=-2), dict(rot=-2)):
        assert f(C.byref(_lib.RopeParams(**{**ok, **bad})), None) == _lib.ERR_BAD_SHAPE, bad
    assert f(C.byref(_lib.RopeParams(**{**ok, "dtype": 3})), None) == _lib.ERR_BAD_DTYPE
    for bad in ("q_out", "positions", "inv_freq"):
        assert f(C.byref(_lib.RopeParams(**{**ok, bad: None})), None) == _lib.ERR_NULL, bad
    for empty in (dict(B=0), dict(S=0), dict(Hq=0), dict(q=None)):
        assert f(C.byref(_lib.RopeParams(**{**ok, **empty})), None) == 0, empty


def test_paged_calls_are_refused_on_the_host():
    lib = _lib.load()
    cache = _lib.PagedCache(**CACHE)

    def c(**kw):
        return C.byref(_lib.PagedCache(**{**CACHE, **kw}))

    wrong = [(c(D=80), _lib.ERR_BAD_HEAD_DIM), (c(page_size=24), _lib.ERR_BAD_SHAPE), (c(page_size=512), _lib.ERR_BAD_SHAPE),
             (c(num_pages=-1), _lib.ERR_BAD_SHAPE), (c(block_table=None), _lib.ERR_NULL), (c(k_scale=None), _lib.ERR_NULL),
             (c(context_lens=None), _lib.ERR_NULL), (c(v=24), _lib.ERR_MISALIGNED), (None, _lib.ERR_NULL)]
    app = dict(k_new=16, v_new=16, B=1, Hq=4, M=2, n_axes=1)
    for w, rc in wrong:
        assert lib.sl8_kv_append_paged(w, C.byref(_lib.AppendParams(**app)), None) == rc
        assert lib.sl8_kv_read_paged(w, 1, None, 4, 0, 16, 16, None) == rc
    for bad, rc in ((dict(rot=24), _lib.ERR_BAD_SHAPE), (dict(rot=144), _lib.ERR_BAD_SHAPE), (dict(dtype=2), _lib.ERR_BAD_DTYPE),
                    (dict(k_new=None), _lib.ERR_NULL), (dict(rot=64), _lib.ERR_NULL), (dict(q=16), _lib.ERR_NULL),
                    (dict(k_stride_s=4), _lib.ERR_MISALIGNED), (dict(v_new=8), _lib.ERR_MISALIGNED),
                    (dict(q=16, q_out=16, q_stride_h=4), _lib.ERR_MISALIGNED), (dict(n_axes=0), _lib.ERR_BAD_SHAPE), (dict(M=0), 0), (dict(B=0), 0)):
        assert lib.sl8_kv_append_paged(C.byref(cache), C.byref(_lib.AppendParams(**{**app, **bad})), None) == rc, bad
    assert lib.sl8_kv_read_paged(C.byref(cache), 1, None, -1, 0, 16, 16, None) == _lib.ERR_BAD_SHAPE
    assert lib.sl8_kv_read_paged(C.byref(cache), 1, None, 4, 2, 16, 16, None) == _lib.ERR_BAD_DTYPE
    assert lib.sl8_kv_read_paged(C.byref(cache), 1, None, 4, 0, None, 16, None) == _lib.ERR_NULL
    assert lib.sl8_kv_read_paged(C.byref(cache), 1, None, 4, 0, 16, 24, None) == _lib.ERR_MISALIGNED
    assert lib.sl8_kv_read_paged(C.byref(cache), 0, None, 4, 0, None, None, None) == 0

    att = dict(q=16, out=16, B=1, Hq=4, M=1, causal=1, window_left=-1, softmax_scale=0.1)
    big = C.c_void_p(256)
    for w, rc in wrong:
        assert lib.sl8_attn_paged(w, C.byref(_lib.PagedAttnParams(**att)), big, 1 << 30, None) == rc
    for bad, rc in ((dict(Hq=3), _lib.ERR_BAD_SHAPE), (dict(dtype=2), _lib.ERR_BAD_DTYPE), (dict(q=None), _lib.ERR_NULL),
                    (dict(out=24), _lib.ERR_MISALIGNED), (dict(q_stride_b=4), _lib.ERR_MISALIGNED), (dict(M=0), 0), (dict(Hq=0), 0)):
        assert lib.sl8_attn_paged(C.byref(cache), C.byref(_lib.PagedAttnParams(**{**att, **bad})), big, 1 << 30, None) == rc, bad
    p = _lib.PagedAttnParams(**att)
    need = lib.sl8_attn_paged_workspace(C.byref(cache), C.byref(p))
    assert lib.sl8_attn_paged(C.byref(cache), C.byref(p), big, need - 1, None) == _lib.ERR_WORKSPACE
    assert lib.sl8_attn_paged(C.byref(cache), C.byref(p), None, need, None) == _lib.ERR_WORKSPACE
    assert lib.sl8_attn_paged(C.byref(cache), C.byref(p), C.c_void_p(8), need, None) == _lib.ERR_MISALIGNED


def test_python_layer_refuses_cpu_tensors_and_bad_sizes():
    x = torch.zeros(1, 2, 1, 64).half()
    cache = s8.empty_paged_cache(2, 2, 16, 64, "cpu")
    table, lens = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        s8.apply_rope(x, None, torch.zeros(1, dtype=torch.long), torch.ones(32))
    with pytest.raises(RuntimeError, match="CUDA"):
        s8.kv_append_paged(x, x, *cache, table, lens)
    with pytest.raises(RuntimeError, match="CUDA"):
        s8.kv_read_paged(*cache, table, lens, 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        s8.attn_paged_cached(x, *cache, table, lens)
    for page, d in ((8, 64), (48, 64), (16, 80)):
        with pytest.raises(ValueError):
            s8.empty_paged_cache(2, 2, page, d, "cpu")
    assert s8.rope_freq_axis((2, 1, 1)).tolist() == [0, 0, 1, 2]
    assert s8.rope_freq_axis((2, 1, 1), mixed=True).tolist() == [0, 1, 2, 0]

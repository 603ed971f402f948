"""Refusals of the serving operators that need no GPU: arguments are checked before the model or a device is touched."""
import ctypes
import os
import re

import numpy as np
import pytest

from conftest import ROOT
from q3asr import lib as q3lib


@pytest.fixture(scope="module")
def lib():
    return q3lib.load()


@pytest.fixture()
def handle():
    """Stands for a model: a call that is refused never looks into it."""
    held = ctypes.create_string_buffer(1 << 14)
    yield ctypes.addressof(held)


def _text(lib):
    return lib.q3asr_last_error().decode()


def _c_fields(name):
    header = open(os.path.join(ROOT, "include", "q3asr.h")).read()
    body = header[header.index(f"typedef struct {name} {{"):header.index(f"}} {name};")]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S).split("{", 1)[1]
    return [re.sub(r"[\s*]", "", n) for decl in body.split(";") if decl.strip() for n in re.sub(r"^\s*(const\s+)?\w+", "", decl).split(",")]


@pytest.mark.parametrize("name,cls", [("q3asr_kv_pages", q3lib.Q3Pages), ("q3asr_attn_batch", q3lib.AttentionBatch)])
def test_struct_images_match_the_header(name, cls):
    assert [n for n, _ in cls._fields_] == _c_fields(name)


def test_i8_refusals(lib, handle):
    P = 1 << 20     # an aligned address that is never read

    def linear(x=P, dt=1, ldx=64, w=P, ldw=64, sw=P, M=4, N=8, K=64, out=P, odt=1, ldo=8, ws=P, nb=1 << 20, m=handle):
        return lib.q3asr_i8_linear(m, x, dt, ldx, w, ldw, sw, None, M, N, K, out, odt, ldo, ws, nb, None)

    for kw, text in ((dict(m=None), "null"), (dict(x=None), "null"), (dict(w=None), "null"), (dict(sw=None), "null"), (dict(out=None), "null"),
                     (dict(ws=None), "null"), (dict(M=0), "empty"), (dict(N=-1), "empty"), (dict(K=0), "empty"), (dict(K=131057, ldx=200000, ldw=131072), "131056"),
                     (dict(ldx=63), "stride"), (dict(ldw=48), "stride"), (dict(ldw=65), "aligned"), (dict(w=P + 8), "aligned"), (dict(ldo=7), "stride"),
                     (dict(dt=2), "type"), (dict(odt=7), "type"), (dict(x=P + 1), "aligned"), (dict(dt=0, x=P + 2), "aligned"), (dict(nb=100), "too small"),
                     (dict(ws=P + 4), "workspace"), (dict(M=2 ** 31 - 1, N=2 ** 31 - 1, ldo=2 ** 31), "tiles"), (dict(M=2 ** 24), "2^24"),
                     (dict(N=2 ** 24, ldo=2 ** 25), "2^24")):
        assert linear(**kw) != 0, kw
        assert text in _text(lib), (kw, _text(lib))

    def matmul(a=P, lda=64, sa=P, K=64):
        return lib.q3asr_i8_matmul(handle, a, lda, sa, P, 64, P, None, 4, 8, K, P, 1, 8, None)

    for kw, text in ((dict(a=None), "null"), (dict(sa=None), "null"), (dict(K=60), "multiple of 16"), (dict(lda=48), "stride"), (dict(a=P + 1), "aligned")):
        assert matmul(**kw) != 0 and text in _text(lib), (kw, _text(lib))

    def quantize(x=P, dt=0, ldx=20, rows=3, cols=20, q=P, ldq=32, s=P):
        return lib.q3asr_i8_quantize(handle, x, dt, ldx, rows, cols, q, ldq, s, None)

    for kw, text in ((dict(x=None), "null"), (dict(q=None), "null"), (dict(s=None), "null"), (dict(rows=0), "empty"), (dict(ldx=19), "stride"),
                     (dict(ldq=16), "aligned"), (dict(ldq=40), "aligned"), (dict(rows=2 ** 24), "2^24"), (dict(q=P + 4), "aligned"), (dict(dt=3), "type")):
        assert quantize(**kw) != 0 and text in _text(lib), (kw, _text(lib))
    assert lib.q3asr_i8_workspace(handle, 0, 8, 8) == -1 and lib.q3asr_i8_workspace(handle, 8, 8, 131057) == -1
    assert lib.q3asr_i8_workspace(handle, 5, 8, 33) >= 5 * 48 + 20


def _cache(**over):
    P = 1 << 20
    kw = dict(k=P, v=P, table=P, lens=P, refs=P, status=P, layers=2, pages=10, kv_heads=2, head_dim=128, page_tokens=16, max_seqs=4,
              max_seq_pages=5, workspace=P, workspace_bytes=1 << 20)
    kw.update(over)
    return q3lib.Q3Pages(**kw)


def test_pages_refusals(lib, handle):
    P = 1 << 20
    bad = [(dict(k=None), "null"), (dict(status=None), "null"), (dict(head_dim=96), "head_dim"), (dict(page_tokens=24), "page_tokens"),
           (dict(page_tokens=8), "page_tokens"), (dict(page_tokens=512), "page_tokens"), (dict(layers=0), "non-positive"), (dict(pages=-1), "non-positive"),
           (dict(max_seq_pages=1 << 28), "2\\^31"), (dict(k=P + 2), "misaligned"), (dict(table=P + 2), "misaligned")]
    ws = [(dict(workspace=None), "workspace"), (dict(workspace_bytes=64), "workspace"), (dict(workspace=P + 8), "workspace")]
    for over, text in bad:
        c = ctypes.byref(_cache(**over))
        for rc in (lib.q3asr_pages_reset(handle, c, None), lib.q3asr_pages_fork(handle, c, P, P, 1, None), lib.q3asr_pages_compact(handle, c, None)):
            assert rc != 0 and re.search(text, _text(lib)), (over, _text(lib))
    for over, text in ws:
        c = ctypes.byref(_cache(**over))
        for rc in (lib.q3asr_pages_fork(handle, c, P, P, 1, None), lib.q3asr_pages_free(handle, c, P, 1, None),
                   lib.q3asr_pages_reserve(handle, c, P, P, 1, None), lib.q3asr_pages_compact(handle, c, None)):
            assert rc != 0 and text in _text(lib), (over, _text(lib))
    c = ctypes.byref(_cache())
    assert lib.q3asr_pages_fork(handle, c, P, P, 5, None) != 0 and "more entries" in _text(lib)
    assert lib.q3asr_pages_reserve(handle, c, P, P, -1, None) != 0
    assert lib.q3asr_pages_fork(handle, c, P, None, 1, None) != 0 and "null" in _text(lib)
    assert lib.q3asr_pages_free(handle, c, None, 1, None) != 0 and "null" in _text(lib)
    assert lib.q3asr_pages_reset(None, c, None) != 0 and lib.q3asr_pages_reset(handle, None, None) != 0
    assert lib.q3asr_pages_workspace(None) == -1 and lib.q3asr_pages_workspace(c) > 4 * 4 * 5
    assert lib.q3asr_pages_status(handle, c, None, 0, None) != 0


def test_attention_and_write_refusals(lib, handle):
    P = 1 << 20
    base = dict(seqs=P, cu_rows=P, cu_groups=P, shared=P, n=4, rows=6, n_groups=2, max_rows=2, max_group_rows=4, max_len=70, max_shared=32, max_own=40)

    def attention(cache=None, batch=None, layer=0, q=P, ld=512, heads=4, scale=0.1, out=P, old=512, lse=P, ws=P, nb=1 << 30):
        c, b = _cache(**(cache or {})), q3lib.AttentionBatch(**{**base, **(batch or {})})
        return lib.q3asr_paged_attention(handle, ctypes.byref(c), layer, q, ld, heads, scale, ctypes.byref(b), out, old, lse, ws, nb, None)

    long = dict(cache=dict(max_seq_pages=100), batch=dict(max_len=1500, max_own=1468))   # a small step needs no workspace
    for kw, text in ((dict(batch=dict(n=-1)), "bad batch"), (dict(batch=dict(seqs=None)), "null"), (dict(batch=dict(n=5)), "more entries"),
                     (dict(batch=dict(max_rows=0)), "max_rows"), (dict(batch=dict(max_rows=7)), "max_rows"), (dict(batch=dict(max_len=81)), "max_len"),
                     (dict(batch=dict(n_groups=5)), "groups"), (dict(batch=dict(cu_groups=None)), "groups"), (dict(batch=dict(max_group_rows=1)), "max_group_rows"),
                     (dict(batch=dict(max_shared=71)), "max_shared"), (dict(batch=dict(max_own=-1)), "max_own"), (dict(layer=2), "layer"), (dict(layer=-1), "layer"),
                     (dict(heads=3), "multiple"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(ld=511), "aligned"), (dict(ld=504), "hold all heads"),
                     (dict(old=516), "aligned"), (dict(q=P + 8), "aligned"), (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"), (dict(scale=-2e30), "finite"),
                     (dict(cache=dict(head_dim=32)), "head_dim"), (dict(batch=dict(rows=2 ** 24)), "2^24"),
                     (dict(cache=dict(max_seq_pages=(1 << 27) - 1), batch=dict(rows=100000, max_len=2 ** 31 - 16)), "too many rows"),
                     (dict(ws=None, **long), "workspace"), (dict(nb=16, **long), "workspace"), (dict(ws=P + 8, **long), "workspace")):
        assert attention(**kw) != 0, kw
        assert text in _text(lib), (kw, _text(lib))
    c, b = _cache(), q3lib.AttentionBatch(**base)
    for args in ((2, P, 256, P, 256), (0, None, 256, P, 256), (0, P, 255, P, 256), (0, P, 248, P, 256), (0, P + 2, 256, P, 256)):
        assert lib.q3asr_pages_write(handle, ctypes.byref(c), args[0], args[1], args[2], args[3], args[4], ctypes.byref(b), None) != 0, args
    assert lib.q3asr_paged_attention_workspace(handle, ctypes.byref(c), ctypes.byref(b), 3) == -1
    assert lib.q3asr_paged_attention_workspace(handle, ctypes.byref(c), ctypes.byref(b), 4) == 0
    c, b = _cache(max_seq_pages=100), q3lib.AttentionBatch(**{**base, **long["batch"]})
    assert lib.q3asr_paged_attention_workspace(handle, ctypes.byref(c), ctypes.byref(b), 4) > 6 * 4 * 128 * 4
    empty = q3lib.AttentionBatch(n=0, rows=0)
    assert lib.q3asr_paged_attention_workspace(handle, ctypes.byref(c), ctypes.byref(empty), 4) == 0


def test_python_side_refusals():
    from q3asr import serving
    with pytest.raises(ValueError, match="dtype"):
        serving._dtype("fp16")

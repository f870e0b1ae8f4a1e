"""CPU-side checks of the C entries of packed prompts and of the 4-bit cache: struct layouts, sizes, and the codes of what is refused
(which is decided before any device work)."""
import ctypes as C
import os
import subprocess

import pytest

from acctransformer_b200 import _lib, build as _build

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "acct_b200.h")
A = 0x10000      # some 16-byte aligned address: nothing that is refused looks at it
CODES = {"NULL": 1, "SHAPE": 2, "DTYPE": 3, "UNSUPPORTED_D": 4, "ALIGN": 5, "WORKSPACE": 6}

MIRRORS = {"acct_packed_args": "PackedArgs", "acct_kv4_cache": "Kv4CacheArgs", "acct_kv4_rows": "Kv4Rows", "acct_kv4_decode_args": "Kv4DecodeArgs",
           "acct_kv4_evict_args": "Kv4EvictArgs"}


@pytest.fixture(scope="module")
def lib():
    _build.build()
    return _lib.load()


def test_ctypes_mirrors_match_c_layout(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', 'int main(void){']
    for st, mirror in MIRRORS.items():
        lines.append(f'printf("{st} %zu\\n", sizeof({st}));')
        lines += [f'printf("{st}.{name} %zu\\n", offsetof({st}, {name}));' for name, _ in getattr(_lib, mirror)._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ['return 0;}']))
    subprocess.run(["gcc", "-std=c99", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")], check=True)
    said = dict(line.split() for line in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.splitlines())
    for st, mirror in MIRRORS.items():
        cls = getattr(_lib, mirror)
        assert int(said[st]) == C.sizeof(cls), st
        for name, _ in cls._fields_:
            assert int(said[f"{st}.{name}"]) == getattr(cls, name).offset, (st, name)


def test_sizes(lib):
    assert [lib.acct_kv4_record_bytes(D) for D in (8, 32, 40, 64, 96, 128)] == [640, 640, 1280, 1280, 1920, 2560]
    assert [lib.acct_kv4_record_bytes(D) for D in (0, -8, 12, 136)] == [0] * 4
    c = _cache()
    size = lambda N, splits, w: lib.acct_kv4_decode_workspace_bytes(c, N, splits, w)  # noqa: E731
    assert 0 < size(4, 1, 0) < size(4, 2, 0) < size(4, 64, 0) == size(4, 0, 0)
    assert size(4, 1, 1) - size(4, 1, 0) >= 2 * 2 * 100 * 2 * 4           # a score per slot and query head
    assert size(4, 65, 0) == size(1, 0, 0) == lib.acct_kv4_decode_workspace_bytes(None, 4, 0, 0) == 0


def _cache(**kw):
    c = _lib.Kv4CacheArgs()
    c.dtype, c.B, c.N_kv, c.S_max, c.D, c.records = _lib.ACCT_F16, 2, 2, 100, 64, A
    for k, v in kw.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [({"dtype": 7}, "DTYPE"), ({"B": 0}, "SHAPE"), ({"N_kv": -1}, "SHAPE"), ({"S_max": 0}, "SHAPE"), ({"D": 60}, "UNSUPPORTED_D"),
              ({"D": 136}, "UNSUPPORTED_D"), ({"D": 0}, "UNSUPPORTED_D"), ({"records": None}, "NULL"), ({"records": A + 8}, "ALIGN"),
              ({"block_table": A, "page_size": 24, "max_pages": 9, "num_pages": 9}, "SHAPE"),
              ({"block_table": A, "page_size": 8, "max_pages": 99, "num_pages": 9}, "SHAPE"),
              ({"block_table": A, "page_size": 16, "max_pages": 6, "num_pages": 9}, "SHAPE"),
              ({"block_table": A, "page_size": 16, "max_pages": 7, "num_pages": 0}, "SHAPE")]


@pytest.mark.parametrize("kw, code", BAD_CACHES, ids=str)
def test_caches_that_are_none(lib, kw, code):
    want = CODES[code]
    r, d, e = _rows(), _decode(), _evict()
    assert lib.acct_kv4_append(_cache(**kw), r, None) == want
    assert lib.acct_kv4_read(_cache(**kw), r, None) == want
    assert lib.acct_kv4_decode(_cache(**kw), d, None) == want
    assert lib.acct_kv4_evict(_cache(**kw), _cache(records=2 * A), e, None) == want
    assert lib.acct_kv4_evict(_cache(records=2 * A), _cache(**kw), e, None) == want


def _rows(**kw):
    r = _lib.Kv4Rows()
    r.k = r.v = r.start = A
    r.T = 2
    for k, v in kw.items():
        setattr(r, k, v)
    return r


@pytest.mark.parametrize("kw, code", [({"k": None}, "NULL"), ({"v": None}, "NULL"), ({"start": None}, "NULL"), ({"k": A + 2}, "ALIGN"), ({"T": 3}, "SHAPE"),
                                      ({"T": -1, "cu_seqlens": A}, "SHAPE"), ({"k_stride": (C.c_int64 * 2)(132, 64)}, "ALIGN"),
                                      ({"v_stride": (C.c_int64 * 2)(128, 56)}, "SHAPE")], ids=str)
def test_rows_that_are_none(lib, kw, code):
    want = CODES[code]
    assert lib.acct_kv4_append(_cache(), _rows(**kw), None) == want
    assert lib.acct_kv4_read(_cache(), _rows(**kw), None) == want


def _decode(**kw):
    a = _lib.Kv4DecodeArgs()
    a.N, a.q, a.y, a.workspace, a.workspace_bytes, a.scale = 4, A, A, A, 1 << 30, 0.1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw, code", [({"q": None}, "NULL"), ({"y": None}, "NULL"), ({"q": A + 4}, "ALIGN"), ({"N": 3}, "SHAPE"), ({"N": 0}, "SHAPE"),
                                      ({"N": 34}, "SHAPE"), ({"scale": 0.0}, "SHAPE"), ({"scale": float("nan")}, "SHAPE"), ({"num_splits": 65}, "SHAPE"),
                                      ({"num_splits": -1}, "SHAPE"), ({"workspace": None}, "WORKSPACE"), ({"workspace_bytes": 64}, "WORKSPACE"),
                                      ({"workspace": A + 8}, "ALIGN")], ids=str)
def test_decode_refusals(lib, kw, code):
    assert lib.acct_kv4_decode(_cache(), _decode(**kw), None) == CODES[code]


def test_decode_wants_room_for_the_scores(lib):
    need = lib.acct_kv4_decode_workspace_bytes(_cache(), 4, 1, 1)
    assert lib.acct_kv4_decode(_cache(), _decode(weights=A, num_splits=1, workspace_bytes=need - 1), None) == CODES["WORKSPACE"]


def _evict(**kw):
    a = _lib.Kv4EvictArgs()
    a.weights, a.seq_lens, a.keep, a.recent, a.weights_out, a.kept, a.seq_lens_out = A, A, 8, 2, 2 * A, A, 2 * A
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw, code", [({"weights": None}, "NULL"), ({"seq_lens": None}, "NULL"), ({"weights_out": None}, "NULL"), ({"kept": None}, "NULL"),
                                      ({"seq_lens_out": None}, "NULL"), ({"keep": 0}, "SHAPE"), ({"keep": 101}, "SHAPE"), ({"recent": 9}, "SHAPE"),
                                      ({"recent": -1}, "SHAPE"), ({"weights_out": A}, "SHAPE"), ({"seq_lens_out": A}, "SHAPE")], ids=str)
def test_evict_refusals(lib, kw, code):
    assert lib.acct_kv4_evict(_cache(), _cache(records=2 * A), _evict(**kw), None) == CODES[code]


@pytest.mark.parametrize("kw, code", [({"dtype": _lib.ACCT_BF16}, "DTYPE"), ({"B": 3}, "SHAPE"), ({"N_kv": 1}, "SHAPE"), ({"D": 128}, "SHAPE"),
                                      ({"records": A}, "SHAPE"), ({"S_max": 7}, "SHAPE")], ids=str)
def test_evict_into_another_kind_of_cache(lib, kw, code):
    kw = {"records": 2 * A, **kw}
    assert lib.acct_kv4_evict(_cache(), _cache(**kw), _evict(), None) == CODES[code]


def _packed(**kw):
    a = _lib.PackedArgs()
    a.dtype, a.B, a.N, a.N_kv, a.D, a.T_q, a.T_k, a.scale = _lib.ACCT_F16, 2, 4, 2, 64, 10, 10, 0.1
    a.q = a.k = a.v = a.y = a.cu_seqlens_q = A
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw, code", [({"dtype": 9}, "DTYPE"), ({"B": 0}, "SHAPE"), ({"N": 0}, "SHAPE"), ({"N_kv": 3}, "SHAPE"), ({"N_kv": -1}, "SHAPE"),
                                      ({"T_q": -1}, "SHAPE"), ({"T_k": 11}, "SHAPE"), ({"D": 60}, "UNSUPPORTED_D"), ({"D": 264}, "UNSUPPORTED_D"),
                                      ({"q": None}, "NULL"), ({"y": None}, "NULL"), ({"k": None}, "NULL"), ({"cu_seqlens_q": None}, "NULL"), ({"v": A + 2}, "ALIGN"),
                                      ({"scale": -1.0}, "SHAPE"), ({"scale": float("inf")}, "SHAPE"), ({"q_stride": (C.c_int64 * 2)(260, 64)}, "ALIGN"),
                                      ({"k_stride": (C.c_int64 * 2)(128, 32)}, "SHAPE")], ids=str)
def test_packed_refusals(lib, kw, code):
    assert lib.acct_infer_packed(_packed(**kw), None) == CODES[code]


def test_null_structs(lib):
    assert lib.acct_infer_packed(None, None) == CODES["NULL"]
    assert lib.acct_kv4_append(None, _rows(), None) == lib.acct_kv4_append(_cache(), None, None) == CODES["NULL"]
    assert lib.acct_kv4_read(None, _rows(), None) == lib.acct_kv4_read(_cache(), None, None) == CODES["NULL"]
    assert lib.acct_kv4_decode(None, _decode(), None) == lib.acct_kv4_decode(_cache(), None, None) == CODES["NULL"]
    assert lib.acct_kv4_evict(None, _cache(), _evict(), None) == lib.acct_kv4_evict(_cache(), None, _evict(), None) == CODES["NULL"]
    assert lib.acct_kv4_evict(_cache(), _cache(records=2 * A), None, None) == CODES["NULL"]

"""The entry points over a paged cache refuse bad arguments before anything is launched.  No GPU needed."""

import ctypes
import os
import subprocess

import pytest
import torch

import flash_colsum_b200 as fc
from flash_colsum_b200 import _cabi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_memory = (ctypes.c_char * 4096)()
ADDRESS = (ctypes.addressof(_memory) + 255) & ~255        # (never read: every call here is refused)


def cache(**changes):
    c = _cabi.PagedCache(key_pages=ADDRESS, value_pages=ADDRESS, key_stride=(2 * 64 * 128, 64 * 128, 128),
                         value_stride=(2 * 64 * 128, 64 * 128, 128), page_table=ADDRESS, table_stride=8, lens=ADDRESS, starts=ADDRESS,
                         pages=10, kv_heads=2, page_size=64, dim=128, dtype=1, sequences=3, table_width=8, tokens=5)
    for name, value in changes.items():
        setattr(c, name, value)
    return c


def rows(**changes):
    r = _cabi.PagedRows(key=ADDRESS, value=ADDRESS, query=ADDRESS, query_out=ADDRESS, key_stride=(256, 128), value_stride=(256, 128),
                        query_stride=(1024, 128), query_out_stride=(1024, 128), q_heads=8, cos=ADDRESS, sin=ADDRESS, table_rows=100,
                        rotary=128, interleaved=0, positions=None, bounds=ADDRESS, fill_tail=1)
    for name, value in changes.items():
        setattr(r, name, value)
    return r


def strides(*values):
    return (ctypes.c_int64 * len(values))(*values)


def append(c=None, r=None):
    return _cabi.load().fcs_append_paged(ctypes.byref(c or cache()), ctypes.byref(r or rows()), None, None)


def select(c=None, query=ADDRESS, st=(1024, 128), heads=8, bounds=ADDRESS, k=4, first=1, last=1, out=ADDRESS, ws=ADDRESS, size=1 << 40):
    return _cabi.load().fcs_select_pages(ctypes.byref(c or cache()), query, strides(*st), heads, bounds, k, first, last, out, 0, ws, size,
                                         None, None)


def attend(c=None, query=ADDRESS, st=(1024, 128), heads=8, pages=ADDRESS, k=4, scale=0.1, out=ADDRESS, out_st=(1024, 128)):
    return _cabi.load().fcs_attend_pages(ctypes.byref(c or cache()), query, strides(*st), heads, pages, k, scale, out, strides(*out_st),
                                         None, 0, None, None)


def test_structures_are_laid_out_as_the_header_has_them(tmp_path):
    source = tmp_path / "sizes.c"
    lines = []
    for name, struct in (("FcsPagedCache", _cabi.PagedCache), ("FcsPagedRows", _cabi.PagedRows)):
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {field[0]}));' for field in struct._fields_]
    source.write_text('#include <stdio.h>\n#include "flash_colsum_b200.h"\nint main(void) {' + "".join(lines) + "return 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(source), "-o", str(tmp_path / "sizes")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for struct in (_cabi.PagedCache, _cabi.PagedRows):
        want.append(ctypes.sizeof(struct))
        want += [getattr(struct, field[0]).offset for field in struct._fields_]
    assert got == want


@pytest.mark.parametrize("call", [append, select, attend])
@pytest.mark.parametrize("changes,word", [
    (dict(dim=100), "head dimension"), (dict(dim=136), "head dimension"), (dict(dim=0), "head dimension"),
    (dict(dtype=2), "dtype"), (dict(page_size=48), "page size"), (dict(page_size=256), "page size"),
    (dict(pages=0), "positive"), (dict(kv_heads=0), "positive"), (dict(sequences=0), "positive"), (dict(tokens=0), "positive"),
    (dict(table_width=0), "positive"), (dict(table_width=1 << 29, table_stride=1 << 29), "too many pages"),
    (dict(page_table=None), "page_table"), (dict(lens=None), "lens"), (dict(table_stride=7), "table_stride"),
    (dict(starts=None), "one token a sequence"),
])
def test_every_entry_point_checks_the_batch(call, changes, word):
    assert call(cache(**changes)) < 0
    assert word in _cabi.last_error()


@pytest.mark.parametrize("call", [append, attend])
@pytest.mark.parametrize("changes,word", [
    (dict(key_pages=None), "key_pages is NULL"), (dict(value_pages=ADDRESS + 8), "value_pages must be 16-byte aligned"),
    (dict(key_stride=(1, 1, 1)), "key_pages strides"), (dict(value_stride=(-8, 8, 8)), "value_pages strides"),
])
def test_pools_are_checked(call, changes, word):
    assert call(cache(**changes)) < 0
    assert word in _cabi.last_error()


@pytest.mark.parametrize("changes,word", [
    (dict(key=None), "key is NULL"), (dict(value=ADDRESS + 2), "value must be"), (dict(key_stride=(4, 128)), "key strides"),
    (dict(query_out=None), "query_out is NULL"), (dict(q_heads=7), "multiple"), (dict(q_heads=0), "multiple"),
    (dict(sin=None), "go together"), (dict(cos=ADDRESS + 4), "cos and sin must be"), (dict(rotary=24), "rotated features"),
    (dict(rotary=144), "rotated features"), (dict(rotary=0), "rotated features"), (dict(table_rows=0), "no rows"),
    (dict(bounds=ADDRESS + 2), "bounds must be"),
])
def test_append_refuses(changes, word):
    assert append(r=rows(**changes)) < 0
    assert word in _cabi.last_error()
    assert _cabi.load().fcs_append_paged(None, None, None, None) < 0


@pytest.mark.parametrize("kw,word", [
    (dict(query=None), "query is NULL"), (dict(st=(1024, 4)), "query strides"), (dict(heads=7), "multiple"), (dict(bounds=None), "bounds"),
    (dict(out=None), "chosen"), (dict(k=0), "k must hold"), (dict(first=-1), "k must hold"), (dict(last=0), "k must hold"),
    (dict(k=4, first=3, last=2), "k must hold"), (dict(first=2 ** 31 - 1, last=2 ** 31 - 1), "k must hold"),
    (dict(ws=None), "workspace"), (dict(ws=ADDRESS + 8), "workspace"), (dict(size=5 * 2 * 12 * 8 - 1), "workspace"),
])
def test_select_refuses(kw, word):
    assert select(**kw) < 0
    assert word in _cabi.last_error()


@pytest.mark.parametrize("kw,word", [
    (dict(query=None), "query is NULL"), (dict(heads=7), "multiple"), (dict(pages=None), "chosen"), (dict(k=0), "chosen"),
    (dict(out=None), "out is NULL"), (dict(out_st=(1024, 4)), "out strides"), (dict(scale=float("nan")), "scale"),
    (dict(c=cache(key_stride=(0, 64 * 128, 128))), "positive"),
])
def test_attend_refuses(kw, word):
    assert attend(**kw) < 0
    assert word in _cabi.last_error()


def test_workspace_of_a_selection_is_bounded():
    """Eight bytes of a 64-bit sum per page, and with many tokens a sequence four of a 32-bit one and the error; at most 256 MiB
    of them unless one token alone needs more."""
    size = lambda **kw: _cabi.load().fcs_select_pages_workspace_bytes(ctypes.byref(cache(**kw)))  # noqa: E731
    assert size(sequences=5, starts=None) == 5 * 2 * 12 * 8
    assert size(tokens=5) == 5 * 2 * 12 * 8
    assert size(tokens=24) >= 24 * 2 * 12 * 12
    assert size(tokens=1 << 20, table_width=4096, table_stride=4096) <= (256 << 20) + (1 << 20)
    assert size(tokens=1 << 20, kv_heads=16, table_width=1 << 24, table_stride=1 << 24) >= 16 * (1 << 24) * 12
    assert size(tokens=0) == 0


def test_python_entry_points_refuse_tensors_that_are_not_on_a_gpu():
    half = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    pool = torch.zeros(3, 4, 16, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    pages = torch.zeros(2, 4, 1, dtype=torch.int32)
    bounds = torch.zeros(3, 4, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: fc.append_paged(half, half, pool, pool, table, lens),
                 lambda: fc.select_pages(half, bounds, table, lens, 2, page_size=16),
                 lambda: fc.attend_pages(half, pool, pool, table, lens, pages)):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call()
    with pytest.raises(ValueError, match="tokens, heads, head_dim"):
        fc.append_paged(half[0], half[0], pool, pool, table, lens)

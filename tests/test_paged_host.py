"""The cache in pages and beam selection without a device: refusals, the page
arithmetic, the drafted trees' masks."""
import ctypes as C
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

from llm_core_amd import _ffi, hip

ROOT = Path(__file__).resolve().parent.parent

# A context whose fields are all zero: argument checks come before any device call, so a
# refusal must be seen with it.  The addresses are never read by the host.
_blank = (C.c_char * 256)()
CTX = C.cast(_blank, C.c_void_p)
D = 1 << 20  # an aligned address


def pool(**kw):
    f = dict(k=D, v=D, type=0, n_layers=2, n_pages=8, page_rows=16, n_kv_heads=2, head_dim=128)
    f.update(kw)
    return _ffi.KvPages(*[f[n] for n, _ in _ffi.KvPages._fields_])


def refused(name, args, code=_ffi.AXF_ERR_INVALID_ARG):
    rc = getattr(_ffi.lib, name)(CTX, *args)
    assert rc == code, (name, args, rc, _ffi.last_error())
    assert name in _ffi.last_error()


FORK = dict(kv=None, table_out=D, refs_out=D, info=D, table=2 * D, refs=D, n_in=2, parent=D, len=D,
            n_out=2, table_ld=4, extra=1)
STORE = dict(kv=None, layer=0, table=D, table_ld=4, len=D, n_tok=D, n_seq=2, max_tok=3, k=D,
             k_ld=256, bk=D, v=D, v_ld=256, bv=D, pos=D, cos=D, sin=D, n_pos=9)
ATTN = dict(out=D, outq8=D, q=3 * D, q_ld=512, bq=D, kv=None, layer=0, table=D, table_ld=4, len=D,
            n_tok=D, mask=D, pos=D, cos=D, sin=D, n_pos=9, n_seq=2, max_tok=3, max_len=40,
            n_heads=4)
COMPACT = dict(kv=None, len_out=D, table=D, table_ld=4, len=D, path=D, n_path=D, n_seq=2,
               max_path=3)
SELECT = dict(token=D, parent=D, score=D, logits=D, ld=100, cum=2 * D, done=D, eos=2, n_seq=2,
              n_beams=4, n_vocab=100, n_out=8)
CALLS = {"axf_hip_kv_fork": FORK, "axf_hip_kv_store": STORE, "axf_hip_attn_paged": ATTN,
         "axf_hip_kv_compact": COMPACT, "axf_hip_beam_select": SELECT}


def call_args(base, **kw):
    f = dict(base)
    f.update(kw)
    if "kv" in f and f["kv"] is None:
        f["kv"] = C.byref(pool())
    return list(f.values())


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(type=8), dict(n_layers=0),
                                 dict(n_pages=0), dict(n_pages=-1), dict(page_rows=0),
                                 dict(page_rows=24), dict(page_rows=2048), dict(n_kv_heads=0),
                                 dict(n_kv_heads=257), dict(head_dim=96), dict(k=D + 8),
                                 dict(v=D + 4), dict(n_layers=20000),
                                 dict(n_pages=1 << 28, page_rows=16)])
@pytest.mark.parametrize("name", [n for n in CALLS if "kv" in CALLS[n]])
def test_bad_pools_are_refused(name, bad):
    refused(name, call_args(CALLS[name], kv=C.byref(pool(**bad))))


@pytest.mark.parametrize("name,bad", [
    (n, b) for n, bads in {
        "axf_hip_kv_fork": [dict(table_out=None), dict(refs_out=None), dict(info=None),
                            dict(table=None), dict(refs=None), dict(n_in=-1), dict(parent=None),
                            dict(len=None), dict(n_out=-1), dict(n_out=70000), dict(table_ld=0),
                            dict(table_ld=1 << 27), dict(extra=-1), dict(table_out=2 * D),
                            dict(table_out=2 * D + 16), dict(table_out=2 * D - 16),
                            dict(refs_out=D + 16), dict(table=2 * D + 2), dict(info=D + 1)],
        "axf_hip_kv_store": [dict(layer=-1), dict(layer=2), dict(table=None), dict(table_ld=0),
                             dict(len=None), dict(n_seq=-1), dict(max_tok=-1),
                             dict(n_seq=1 << 20, max_tok=64), dict(k=None), dict(v=None),
                             dict(k_ld=255), dict(v_ld=255), dict(cos=None), dict(sin=None),
                             dict(n_pos=0), dict(k=D + 2), dict(pos=D + 2), dict(n_tok=D + 1)],
        "axf_hip_attn_paged": [dict(out=None), dict(q=None), dict(q_ld=511), dict(layer=2),
                               dict(table=None), dict(table_ld=0), dict(len=None), dict(cos=None),
                               dict(n_pos=0), dict(n_seq=-1), dict(max_tok=65), dict(max_tok=-1),
                               dict(max_len=-1), dict(n_seq=65536, max_tok=64, n_heads=32, q_ld=1 << 14),
                               dict(n_heads=0), dict(n_heads=3),
                               dict(n_heads=2048), dict(mask=D + 4), dict(out=D + 2),
                               dict(outq8=D + 2), dict(q=D + 1), dict(q=D),
                               dict(q=D + 6 * 2048 - 4), dict(q=D - 4)],
        "axf_hip_kv_compact": [dict(len_out=None), dict(table=None), dict(len=None),
                               dict(path=None), dict(n_path=None), dict(n_seq=-1),
                               dict(n_seq=70000), dict(max_path=65), dict(max_path=-1),
                               dict(table_ld=-1), dict(path=D + 2), dict(len_out=D + 4)],
        "axf_hip_beam_select": [dict(token=None), dict(parent=None), dict(score=None),
                                dict(logits=None), dict(cum=None), dict(ld=99), dict(n_beams=0),
                                dict(n_beams=65), dict(n_out=0), dict(n_out=65), dict(n_vocab=0),
                                dict(n_vocab=(1 << 26) + 1, ld=1 << 27), dict(n_seq=-1),
                                dict(eos=-1), dict(eos=100), dict(logits=D + 2), dict(done=D + 2),
                                dict(score=2 * D), dict(score=2 * D + 4), dict(cum=D)],
    }.items() for b in bads])
def test_bad_arguments_are_refused(name, bad):
    refused(name, call_args(CALLS[name], **bad))


@pytest.mark.parametrize("name,nothing", [("axf_hip_kv_store", dict(n_seq=0)),
                                          ("axf_hip_kv_store", dict(max_tok=0)),
                                          ("axf_hip_attn_paged", dict(n_seq=0)),
                                          ("axf_hip_attn_paged", dict(max_tok=0)),
                                          ("axf_hip_kv_compact", dict(n_seq=0)),
                                          ("axf_hip_beam_select", dict(n_seq=0))])
def test_nothing_to_do_is_ok(name, nothing):
    assert getattr(_ffi.lib, name)(CTX, *call_args(CALLS[name], **nothing)) == 0


def test_tree_masks():
    parent = [-1, 0, 0, 1, -1, 4, 3]
    mask, depth = hip.tree_masks(parent)
    assert depth.tolist() == [0, 1, 1, 2, 0, 1, 3]
    assert [bin(m) for m in mask.tolist()] == ["0b1", "0b11", "0b101", "0b1011", "0b10000",
                                               "0b110000", "0b1001011"]
    mask, depth = hip.tree_masks(np.arange(64) - 1)
    assert mask.tolist() == [(1 << (i + 1)) - 1 for i in range(64)]
    assert depth.tolist() == list(range(64))
    for bad in ([0], [-2], [-1, 1], [-1, 2, 0], list(range(-1, 64))):
        with pytest.raises(_ffi.AxfError):
            hip.tree_masks(bad)


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_page_arithmetic(tmp_path):
    """kv_row / kv_len, the kernels' own, over bad pages, short tables and offsets past
    32 bits."""
    src = tmp_path / "t.cpp"
    src.write_text("""
#include "paged_index.hpp"
#include <cstdio>
using namespace axf;
int main() {
    const int t[4] = {3, -1, 9, 0};
    const int pos[] = {-1, 0, 15, 16, 31, 32, 47, 48, 63, 64, 1 << 30, 2147483647};
    for (int p : pos) std::printf("%ld ", kv_row(p, t, 4, 9, 4));
    const int big[1] = {2000000000};
    std::printf("%ld ", kv_row(1023, big, 1, 2147483647, 10));
    std::printf("| %d %d %d %d %d\\n", kv_len(-5, 4, 4), kv_len(0, 4, 4), kv_len(64, 4, 4),
                kv_len(65, 4, 4), kv_len(2147483647, 1 << 20, 10));
}
""")
    exe = tmp_path / "t"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror",
                    f"-I{ROOT / 'llm_core_amd/csrc/kernels'}", str(src), "-o", str(exe)], check=True)
    rows, lens = subprocess.run([str(exe)], capture_output=True, text=True,
                                check=True).stdout.split("|")
    assert [int(x) for x in rows.split()] == [-1, 48, 63, -1, -1, -1, -1, 0, 15, -1, -1, -1,
                                              2000000000 * 1024 + 1023]
    assert [int(x) for x in lens.split()] == [0, 0, 64, 64, 1 << 30]

"""Refusals of the calls for several continuations, each by its own message, with arrays that
are apart.  What is not refused goes on to the device, so these run only where there is none."""
import ctypes as C

import pytest

from llm_core_amd import _ffi, hip

pytestmark = pytest.mark.skipif(hip.device_count() > 0, reason="calls that pass their checks are "
                                "launched, with addresses that hold nothing")

_blank = (C.c_char * 256)()  # a context: checks come before any use of it
CTX = C.cast(_blank, C.c_void_p)


def at(n):
    """The n-th of some far-apart addresses."""
    return (n + 1) << 44


def pool(**kw):
    f = dict(k=at(40), v=at(41), type=0, n_layers=2, n_pages=8, page_rows=16, n_kv_heads=2,
             head_dim=128)
    f.update(kw)
    return _ffi.KvPages(*[f[n] for n, _ in _ffi.KvPages._fields_])


POOL_BYTES = 2 * 8 * 16 * 256 * 4
CALLS = {
    "axf_hip_kv_fork": dict(kv=None, table_out=at(0), refs_out=at(1), info=at(2), table=at(3),
                            refs=at(4), n_in=2, parent=at(5), len=at(6), n_out=2, table_ld=4,
                            extra=1),
    "axf_hip_kv_store": dict(kv=None, layer=1, table=at(3), table_ld=4, len=at(4), n_tok=at(5),
                             n_seq=2, max_tok=3, k=at(6), k_ld=300, bk=at(7), v=at(8), v_ld=256,
                             bv=at(9), pos=at(10), cos=at(11), sin=at(12), n_pos=9),
    "axf_hip_attn_paged": dict(out=at(0), outq8=at(1), q=at(2), q_ld=600, bq=at(3), kv=None, layer=1,
                               table=at(4), table_ld=4, len=at(5), n_tok=at(6), mask=at(7),
                               pos=at(8), cos=at(9), sin=at(10), n_pos=9, n_seq=2, max_tok=3,
                               max_len=40, n_heads=4),
    "axf_hip_kv_compact": dict(kv=None, len_out=at(0), table=at(1), table_ld=4, len=at(2),
                               path=at(3), n_path=at(4), n_seq=2, max_path=3),
    "axf_hip_beam_select": dict(token=at(0), parent=at(1), score=at(2), logits=at(3), ld=104,
                                cum=at(4), done=at(5), eos=2, n_seq=2, n_beams=4, n_vocab=100,
                                n_out=8),
}
# Bytes of what each call writes and reads; kv_k / kv_v: a layer's, from the layer's start, where
# the call has a layer
LAYER = POOL_BYTES // 2
WRITES = {
    "axf_hip_kv_fork": dict(table_out=32, refs_out=32, info=12, kv_k=POOL_BYTES, kv_v=POOL_BYTES),
    "axf_hip_kv_store": dict(kv_k=LAYER, kv_v=LAYER),
    "axf_hip_attn_paged": dict(out=6 * 512 * 4, outq8=6 * 16 * 36),
    "axf_hip_kv_compact": dict(len_out=8, kv_k=POOL_BYTES, kv_v=POOL_BYTES),
    "axf_hip_beam_select": dict(token=64, parent=64, score=64),
}
READS = {
    "axf_hip_kv_fork": dict(table=32, refs=32, parent=8, len=8),
    "axf_hip_kv_store": dict(table=32, len=8, n_tok=8, k=(5 * 300 + 256) * 4, bk=1024, v=6 * 1024,
                             bv=1024, pos=24, cos=9 * 256, sin=9 * 256),
    "axf_hip_attn_paged": dict(q=(5 * 600 + 512) * 4, bq=2048, kv_k=LAYER, kv_v=LAYER, table=32,
                               len=8, n_tok=8, mask=48, pos=24, cos=9 * 256, sin=9 * 256),
    "axf_hip_kv_compact": dict(table=32, path=24, n_path=8, len=8),
    "axf_hip_beam_select": dict(logits=(7 * 104 + 100) * 4, cum=32, done=32),
}


def call(name, **kw):
    f = dict(CALLS[name])
    pages = {k: kw.pop(k) for k in list(kw) if k.startswith("kv_")}
    f.update(kw)
    if "kv" in f:
        f["kv"] = C.byref(pool(**{k[3:]: v for k, v in pages.items()}))
    rc = getattr(_ffi.lib, name)(CTX, *f.values())
    return rc, _ffi.last_error()


def refused(name, why, **kw):
    rc, said = call(name, **kw)
    assert rc == _ffi.AXF_ERR_INVALID_ARG and name in said and why in said, (rc, said)


@pytest.mark.parametrize("name", CALLS)
def test_apart_is_not_refused(name):
    """The calls that the refusals below differ from pass every check."""
    rc, said = call(name)
    assert rc == _ffi.AXF_ERR_HIP, (rc, said)


def pairs():
    for name, outs in WRITES.items():
        names = list(outs)
        for i, w in enumerate(names):
            for x in names[i + 1:] + list(READS[name]):
                yield name, w, x


def start(name, arg):
    """Where the call's bytes of an argument begin."""
    if not arg.startswith("kv_"):
        return CALLS[name][arg]
    return getattr(pool(), arg[3:]) + (LAYER if "layer" in CALLS[name] else 0)


@pytest.mark.parametrize("name,w,x", pairs())
def test_outputs_are_apart(name, w, x):
    """No byte of what a call writes is another output's or is read; the next byte may be."""
    unit = 16 if "kv_" in w + x else 8 if x == "mask" else 4
    wb = WRITES[name][w]
    xb = WRITES[name].get(x) or READS[name][x]
    base = start(name, x)
    move = CALLS[name].get(w) if not w.startswith("kv_") else getattr(pool(), w[3:])
    off = start(name, w) - move  # of the call's bytes in the argument
    up = -(-xb // unit) * unit  # the first address behind x that w may have
    down = -(-wb // unit) * unit
    for shift, apart in ((up - unit, False), (-(down - unit), wb <= down - unit), (up, True),
                         (-down, True)):
        moved = {w: base + shift - off}
        if apart:
            rc, said = call(name, **moved)
            assert rc == _ffi.AXF_ERR_HIP, (shift, rc, said)
        else:
            refused(name, "overlap", **moved)


@pytest.mark.parametrize("name,same,fine", [
    ("axf_hip_kv_fork", dict(refs_out=at(4)), True),
    ("axf_hip_kv_fork", dict(kv_v=at(40), extra=0), True),  # the pool is not touched
    ("axf_hip_kv_fork", dict(kv_v=at(40)), False),
    ("axf_hip_attn_paged", dict(kv_v=at(40)), True),  # read alone
    ("axf_hip_attn_paged", dict(outq8=None), True),
    ("axf_hip_attn_paged", dict(out=at(9), pos=None), True),  # tables that are not read
    ("axf_hip_kv_compact", dict(len_out=at(2)), True),
    ("axf_hip_beam_select", dict(score=at(4), n_out=4), True),
    ("axf_hip_beam_select", dict(score=at(4), n_out=8), False),
    ("axf_hip_beam_select", dict(score=at(4), n_out=3), False)])
def test_what_may_be_one_array(name, same, fine):
    if fine:
        rc, said = call(name, **same)
        assert rc == _ffi.AXF_ERR_HIP, (rc, said)
    else:
        refused(name, "overlap", **same)


@pytest.mark.parametrize("n_out,table_ld", [(65536, 1 << 15), (65536, 1 << 26), (2, 1 << 30)])
def test_fork_counts_its_entries_in_32_bits(n_out, table_ld):
    page = (1 << 30) // table_ld if table_ld > 1 << 26 else 16
    refused("axf_hip_kv_fork", "2^31", n_out=n_out, table_ld=table_ld, extra=1 << 19,
            kv_page_rows=page)


def test_fork_just_below():
    rc, said = call("axf_hip_kv_fork", n_out=65536, table_ld=(1 << 15) - 1, extra=1 << 19)
    assert rc == _ffi.AXF_ERR_HIP, (rc, said)


def test_fork_walks_its_pool_in_32_bits():
    big = dict(kv_page_rows=1, kv_n_kv_heads=1, kv_head_dim=64, kv_type=1, kv_n_layers=1)
    refused("axf_hip_kv_fork", "2^30 pages", kv_n_pages=(1 << 30) + 1, **big)
    refused("axf_hip_kv_fork", "2^30 pages", kv_n_pages=(1 << 31) - 1, **big)
    rc, said = call("axf_hip_kv_fork", kv_n_pages=1 << 20, **big)
    assert rc == _ffi.AXF_ERR_HIP, (rc, said)


def test_tree_masks_over_the_parents():
    """One array for a tree's parents and what is made of them."""
    both = (C.c_uint64 * 64)()
    parent = C.cast(both, C.POINTER(C.c_int32))
    for i, p in enumerate([-1, -1, 1, -1]):
        parent[i] = p
    depth = (C.c_int32 * 4)()
    assert _ffi.lib.axf_tree_masks(both, depth, both, 4) == 0
    assert list(both[:4]) == [1, 2, 6, 8] and list(depth) == [0, 0, 1, 0]
    tree = (C.c_int32 * 4)(-1, 0, 1, 0)
    mask = (C.c_uint64 * 4)()
    assert _ffi.lib.axf_tree_masks(mask, tree, tree, 4) == 0
    assert list(mask) == [1, 3, 7, 9] and list(tree) == [0, 1, 2, 1]

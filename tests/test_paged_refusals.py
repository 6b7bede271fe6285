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

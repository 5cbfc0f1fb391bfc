"""CPU checks of the sparse-attention C ABI: refusals before anything is launched, workspace queries,
empty calls (no GPU needed)."""
import ctypes
import os

import pytest

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sglang0.5.18-opt_b200", "hcu_ops",
                   "libhcu_indexer.so")
OK, ARG, UNSUPPORTED = 0, 1, 4
i64, i32, vp, f32 = ctypes.c_int64, ctypes.c_int32, ctypes.c_void_p, ctypes.c_float
P = 256  # an aligned address that is never dereferenced


@pytest.fixture(scope="module")
def lib():
    return ctypes.CDLL(LIB)


def _tables(lib, n_req=4, max_pages=8, stride=8, batch=2, n_free=8, rows=2, width=256, head=P, out=P, pt=P):
    f = lib.hcu_step_tables
    f.restype = ctypes.c_int
    return f(vp(P), i64(n_req), i64(max_pages), i64(stride), vp(P), vp(P), vp(P), i64(batch), vp(P), i64(n_free),
             vp(head), i64(rows), i64(width), vp(P), vp(pt), vp(P), vp(P), vp(P), vp(P), vp(out), None)


def test_step_tables_refusals(lib):
    assert _tables(lib, width=100) == ARG and _tables(lib, width=0) == ARG
    assert _tables(lib, stride=4) == ARG and _tables(lib, batch=-1) == ARG and _tables(lib, rows=-1) == ARG
    assert _tables(lib, head=None) == ARG and _tables(lib, out=None) == ARG and _tables(lib, pt=P + 4) == ARG
    assert _tables(lib, rows=2 ** 30, width=2 ** 20) == UNSUPPORTED


def _blocks(lib, rows=2, width=4096, stride=4096, mstride=256, n=8, sink=1, local=1, score=P):
    f = lib.hcu_select_blocks
    f.restype = ctypes.c_int
    return f(vp(score), i64(rows), i64(width), i64(stride), vp(P), i64(mstride), vp(P), i64(n), i64(sink), i64(local),
             vp(P), None)


def test_select_blocks_refusals(lib):
    assert _blocks(lib, rows=0) == OK
    assert _blocks(lib, stride=4095) == ARG and _blocks(lib, stride=4098) == ARG and _blocks(lib, mstride=10) == ARG
    assert _blocks(lib, n=0) == ARG and _blocks(lib, n=3, sink=2, local=2) == ARG and _blocks(lib, sink=-1) == ARG
    assert _blocks(lib, score=P + 4) == ARG and _blocks(lib, score=None) == ARG
    assert _blocks(lib, width=2 ** 22, stride=2 ** 22, mstride=2 ** 18) == UNSUPPORTED


def test_kv4_refusals(lib):
    f = lib.hcu_store_mla_kv4
    f.restype = ctypes.c_int

    def store(kv=P, tok=512, n=1, stride=432, buf=P):
        return f(vp(kv), i64(tok), vp(P), i64(64), vp(P), i64(n), vp(buf), i64(4), i64(stride), None)

    assert store(n=0) == OK
    assert store(kv=P + 2) == ARG and store(tok=513) == ARG and store(stride=416) == ARG and store(stride=440) == ARG
    assert store(buf=None) == ARG and store(n=-1) == ARG
    g = lib.hcu_dequant_mla_kv4_paged
    g.restype = ctypes.c_int
    assert g(vp(P), i64(4), i64(432), vp(P), i64(0), vp(P), None) == OK
    assert g(vp(P), i64(4), i64(400), vp(P), i64(1), vp(P), None) == ARG
    assert g(vp(P), i64(4), i64(432), vp(P), i64(1), vp(P + 8), None) == ARG


def test_attention_refusals_and_workspace(lib):
    w = lib.hcu_sparse_mla_attention_workspace_bytes
    w.restype = i64
    assert w(i64(-1), i64(64), i64(2048)) < 0
    one, many = w(i64(1), i64(64), i64(2048)), w(i64(4096), i64(64), i64(2048))
    assert 0 < one < many <= 256 * 2 * (64 * 512 + 64) * 4
    f = lib.hcu_sparse_mla_attention
    f.restype = ctypes.c_int

    def call(q=P, rows=1, heads=64, qr=64 * 576, qh=576, slots=100, stride=656, fmt=0, idx=P, n=64, bt=None, nbt=0,
             lens=None, ws=P, wsb=None, out=P):
        return f(vp(q), i64(rows), i64(heads), i64(qr), i64(qh), vp(P), i64(slots), i64(stride), i32(fmt), vp(idx),
                 i64(n), i64(n), vp(bt), i64(nbt), i64(nbt), vp(lens), f32(1.0), vp(ws),
                 i64(one * 4 if wsb is None else wsb), vp(out), vp(P), None)

    assert call(rows=0) == OK
    assert call(fmt=2) == ARG and call(heads=0) == ARG and call(qr=577) == ARG and call(qh=580) == ARG
    assert call(stride=640) == ARG and call(stride=660) == ARG and call(fmt=1, stride=416) == ARG
    assert call(q=P + 8) == ARG and call(ws=None) == ARG and call(wsb=16) == ARG and call(out=None) == ARG
    assert call(bt=P, nbt=4) == ARG  # block form without lengths
    assert call(idx=None) == ARG and call(n=-1) == ARG
    assert call(heads=2048) == UNSUPPORTED

"""The C ABI library without a GPU: it loads, exports every symbol the header
declares, and rejects bad arguments before touching the device."""

import ctypes
import re

import pytest

from qgemv_roofline_b200 import _lib


def declared_symbols():
    text = open(_lib.HEADER).read()
    return re.findall(r"QGEMV_API\s+[\w\s\*]+?\b(qgemv_\w+)\s*\(", text)


def test_library_loads_and_exports_every_declared_symbol():
    lib = _lib.lib()
    names = declared_symbols()
    assert len(names) >= 15
    for n in names:
        assert hasattr(lib, n), n
    # the ctypes signature table covers the whole header
    assert set(names) == set(_lib.SIGNATURES)


def test_version_and_status_strings():
    lib = _lib.lib()
    assert lib.qgemv_version() == 100
    for code, name in _lib.STATUS_NAMES.items():
        assert lib.qgemv_status_string(code).decode() == name


FAKE = 0x100000  # 16-byte aligned, never dereferenced: validation fails first


def rc(name, *args):
    return getattr(_lib.lib(), name)(*args)


@pytest.mark.parametrize("fn", ["qgemv_q8_0_soa", "qgemv_q4_0_soa"])
def test_soa_validation(fn):
    E = _lib
    assert rc(fn, FAKE, FAKE, FAKE, FAKE, 64, 100, 1, 100, 64, None) == 2  # K % 32
    assert "multiple of 32" in E.last_error()
    assert rc(fn, FAKE, FAKE, FAKE, FAKE, -1, 64, 1, 64, 1, None) == 2
    assert rc(fn, FAKE, FAKE, FAKE, FAKE, 64, 64, -1, 64, 64, None) == 2
    assert rc(fn, None, FAKE, FAKE, FAKE, 64, 64, 1, 64, 64, None) == 1
    assert rc(fn, FAKE, FAKE, None, FAKE, 64, 64, 1, 64, 64, None) == 1
    assert rc(fn, FAKE + 8, FAKE, FAKE, FAKE, 64, 64, 1, 64, 64, None) == 3  # q not 16-B
    assert rc(fn, FAKE, FAKE + 1, FAKE, FAKE, 64, 64, 1, 64, 64, None) == 3  # d not 2-B
    assert rc(fn, FAKE, FAKE, FAKE + 2, FAKE, 64, 64, 1, 64, 64, None) == 3  # x not 4-B
    assert rc(fn, FAKE, FAKE, FAKE, FAKE, 64, 64, 2, 32, 64, None) == 2  # ldx < K
    assert rc(fn, FAKE, FAKE, FAKE, FAKE, 64, 64, 2, 64, 32, None) == 2  # ldy < M
    assert rc(fn, FAKE, FAKE, FAKE, FAKE, 1 << 31, 64, 1, 64, 1, None) == 5
    # empty work is a no-op that needs no device
    assert rc(fn, None, None, None, None, 0, 64, 1, 64, 0, None) == 0
    assert rc(fn, None, None, None, None, 64, 64, 0, 64, 64, None) == 0


@pytest.mark.parametrize("fn", ["qgemv_q8_0_aos", "qgemv_q4_0_aos"])
def test_aos_validation(fn):
    assert rc(fn, FAKE, FAKE, FAKE, 64, 48, 1, 48, 64, None) == 2
    assert rc(fn, None, FAKE, FAKE, 64, 64, 1, 64, 64, None) == 1
    assert rc(fn, FAKE + 2, FAKE, FAKE, 64, 64, 1, 64, 64, None) == 3


def test_quantize_repack_roof_validation():
    assert rc("qgemv_quantize_soa", 5, FAKE, 4, 64, 64, FAKE, FAKE, None) == 7  # format
    assert rc("qgemv_quantize_soa", 8, FAKE, 4, 40, 40, FAKE, FAKE, None) == 2
    assert rc("qgemv_quantize_soa", 4, FAKE, 4, 64, 32, FAKE, FAKE, None) == 2  # ldw < K
    assert rc("qgemv_quantize_soa", 4, None, 4, 64, 64, FAKE, FAKE, None) == 1
    assert rc("qgemv_quantize_aos", 8, FAKE + 1, 4, 64, 64, FAKE, None) == 3
    assert rc("qgemv_dequant_soa", 4, FAKE, FAKE + 1, FAKE, 4, 64, None) == 3
    assert rc("qgemv_repack", 8, 2, FAKE, FAKE, FAKE, 4, 64, None) == 7
    assert rc("qgemv_repack", 8, 1, None, FAKE, FAKE, 4, 64, None) == 1
    assert rc("qgemv_roof_stream_read", FAKE, 100, FAKE, 4, None) == 2
    assert rc("qgemv_roof_stream_read", FAKE + 4, 128, FAKE, 4, None) == 3
    assert rc("qgemv_roof_stream_read", FAKE, 128, FAKE, 0, None) == 7
    assert rc("qgemv_roof_bulk_read", FAKE, 128, FAKE, None, None) == 1
    assert rc("qgemv_roof_d2d", None, FAKE, 16, None) == 1
    assert rc("qgemv_device_info_get", 0, None) == 1


def test_errors_are_per_thread_messages():
    import threading
    rc("qgemv_q8_0_soa", FAKE, FAKE, FAKE, FAKE, 64, 100, 1, 100, 64, None)
    seen = {}

    def other():
        seen["msg"] = _lib.last_error()

    t = threading.Thread(target=other)
    t.start()
    t.join()
    assert seen["msg"] == ""
    assert "multiple of 32" in _lib.last_error()


def test_python_raises_typed_error():
    with pytest.raises(_lib.QGemvError) as ei:
        _lib.call("qgemv_q8_0_soa", FAKE, FAKE, FAKE, FAKE, 64, 100, 1, 100, 64, None)
    assert ei.value.status == 2 and "QGEMV_ERR_SHAPE" in str(ei.value)


def test_workspace_and_tile_sizes_are_host_computations():
    lib = _lib.lib()
    # batched SoA calls with no device: the mma.sync kernel's 128 + 2064 * ceil(K / 512) *
    # min(N, 16) bytes, 0 when no workspace (on a B200 the tcgen05 kernel's need, larger)
    assert lib.qgemv_soa_workspace_bytes(8, 1000, 4096, 4) == 128 + 2064 * 8 * 4
    assert lib.qgemv_soa_workspace_bytes(4, 1000, 4096, 40) == 128 + 2064 * 8 * 16
    assert lib.qgemv_soa_workspace_bytes(8, 1000, 4096, 1) == 0
    assert lib.qgemv_soa_workspace_bytes(8, 1000, 4000, 4) == 0     # K % 256 != 0
    assert lib.qgemv_soa_workspace_bytes(3, 1000, 4096, 4) == 0     # bad format
    assert lib.qgemv_tiled_workspace_bytes(800, 3) == 128 + 2064 * 2 * 3
    assert lib.qgemv_tiled_workspace_bytes(800, 0) == 0
    # batch tiles: ceil(M/16) * ceil(K/512) blocks of 16 x 512 quants + 512 scale bytes
    assert lib.qgemv_tiled_bytes(8, 17, 800) == 2 * 2 * (16 * 512 + 512)
    assert lib.qgemv_tiled_bytes(4, 16, 512) == 1 * 1 * (16 * 256 + 512)
    assert lib.qgemv_tiled_bytes(8, 16, 33) == 0                    # K % 32 != 0


def test_fused_and_tiled_validation():
    from qgemv_roofline_b200._lib import FuseDesc
    f = FuseDesc()
    f.nranks = 0
    assert rc("qgemv_soa_fused", 8, FAKE, FAKE, FAKE, FAKE, 64, 4096, ctypes.byref(f), None) == 7
    f.nranks, f.npeer = 2, 1
    assert rc("qgemv_soa_fused", 8, FAKE, FAKE, FAKE, FAKE, 64, 4096, ctypes.byref(f), None) == 1
    assert rc("qgemv_soa_fused", 8, FAKE, FAKE, FAKE, FAKE, 64, 4096, None, None) == 1
    assert rc("qgemv_token_fence", None, 0, FAKE, FAKE, None) == 7
    assert rc("qgemv_token_fence", None, 2, FAKE, FAKE, None) == 1
    assert rc("qgemv_tile_weights", 8, 2, FAKE, FAKE, 16, 512, FAKE, None) == 7   # bad layout
    assert rc("qgemv_tile_weights", 8, 0, FAKE, FAKE, 16, 512, FAKE + 8, None) == 3
    assert rc("qgemv_tiled_gemv", 8, FAKE, 16, 100, FAKE, FAKE, 1, 100, 16, None, 0, None) == 2
    assert rc("qgemv_tiled_gemv", 8, FAKE, 16, 1 << 21, FAKE, FAKE, 1, 1 << 21, 16, None, 0,
              None) == 5
    assert rc("qgemv_tiled_gemv", 8, FAKE + 4, 16, 512, FAKE, FAKE, 1, 512, 16, None, 0,
              None) == 3


def test_multi_gpu_handle_validation():
    lib = _lib.lib()
    h = ctypes.c_void_p()
    devs = (ctypes.c_int32 * 2)(0, 1)
    assert lib.qgemv_mg_init(2, None, ctypes.byref(h)) == 1
    assert lib.qgemv_mg_init(2, devs, None) == 1
    assert lib.qgemv_mg_init(0, devs, ctypes.byref(h)) == 7
    assert lib.qgemv_mg_init(9, devs, ctypes.byref(h)) == 7
    assert not h.value
    # a NULL handle is refused by every entry point; destroying it is a no-op
    r0, rows = ctypes.c_int64(), ctypes.c_int64()
    assert lib.qgemv_mg_shard(None, 8, 0, FAKE, FAKE, 64, 64) == 1
    assert lib.qgemv_mg_rows(None, 0, ctypes.byref(r0), ctypes.byref(rows)) == 1
    assert lib.qgemv_mg_gemv(None, None, None, 1, 1, None) == 1
    assert lib.qgemv_mg_synchronize(None) == 1
    assert lib.qgemv_mg_destroy(None) == 0


def test_moe_validation():
    L = _lib
    r = L.MoeRouter(FAKE, 0, 8, 64, None, 2, 0, 1, 1.0)
    e = L.ExpertSet(8, 4, 9, 1, 64, 32, FAKE, FAKE)
    R, S = ctypes.byref(r), ctypes.byref(e)

    def layer(x=FAKE, dt=0, ldx=64, n=2, y=FAKE, ldy=64, ws=FAKE, nb=1 << 30):
        return rc("qgemv_moe_layer", S, R, x, dt, ldx, n, y, ldy, ws, nb, None)

    assert rc("qgemv_moe_layer", None, R, FAKE, 0, 64, 2, FAKE, 64, FAKE, 1 << 30, None) == 1
    assert rc("qgemv_moe_layer", S, None, FAKE, 0, 64, 2, FAKE, 64, FAKE, 1 << 30, None) == 1
    assert layer(n=0) == 0
    assert layer(x=None) == 1 and layer(y=None) == 1
    assert layer(dt=3) == 7 and layer(n=-1) == 2
    assert layer(ldx=63) == 2 and layer(ldy=63) == 2
    assert layer(x=FAKE + 2) == 3 and layer(y=FAKE + 2) == 3 and layer(ws=FAKE + 8) == 3
    assert layer(nb=16) == 7 and "workspace" in L.last_error()

    def with_(s, **kw):
        old = {k: getattr(s, k) for k in kw}
        for k, v in kw.items():
            setattr(s, k, v)
        got = layer()
        for k, v in old.items():
            setattr(s, k, v)
        return got

    assert with_(r, top_k=0) == 7 and with_(r, top_k=9) == 7 and with_(r, scoring=2) == 7
    assert with_(r, w=None) == 1 and with_(r, w=FAKE + 2) == 3 and with_(r, bias=FAKE + 1) == 3
    assert with_(r, n_experts=7) == 2          # not the routed experts
    assert with_(r, n_experts=1025) == 7 and with_(r, ldw=63) == 2 and with_(r, w_dtype=5) == 7
    assert with_(e, format=5) == 7 and with_(e, format_down=3) == 7
    assert with_(e, n_experts=0) == 7 and with_(e, n_shared=-1) == 7 and with_(e, n_experts=1025) == 7
    assert with_(e, hidden=48) == 2 and with_(e, ffn=0) == 2 and with_(e, ffn=(1 << 20) + 32) == 5
    assert with_(e, gate_up=None) == 1 and with_(e, down=FAKE + 4) == 3

    def experts(ids=FAKE, w=FAKE, slots=2):
        return rc("qgemv_moe_experts", S, FAKE, 0, 64, ids, w, slots, 2, FAKE, 64, FAKE, 1 << 30, None)

    assert experts(ids=None) == 1 and experts(w=None) == 1 and experts(ids=FAKE + 2) == 3
    assert experts(slots=0) == 7 and experts(slots=33) == 7
    assert rc("qgemv_moe_route", R, FAKE, 0, 64, 2, 64, None, FAKE, None) == 1
    assert rc("qgemv_moe_route", R, FAKE, 0, 64, 2, 64, FAKE, FAKE + 2, None) == 3
    assert rc("qgemv_moe_route", R, FAKE, 0, 64, 2, 0, FAKE, FAKE, None) == 2
    assert rc("qgemv_moe_route", R, FAKE, 0, 64, 0, 64, None, None, None) == 0
    assert rc("qgemv_moe_tile", 8, FAKE, FAKE, None, None, 2, 48, 64, FAKE, None) == 2
    assert rc("qgemv_moe_tile", 8, FAKE, FAKE, FAKE, None, 2, 64, 64, FAKE, None) == 1
    assert rc("qgemv_moe_tile", 8, FAKE + 8, FAKE, None, None, 2, 64, 64, FAKE, None) == 3
    assert rc("qgemv_moe_tile", 4, FAKE, FAKE, None, None, 1025, 64, 64, FAKE, None) == 7
    assert rc("qgemv_moe_tile", 4, None, None, None, None, 0, 64, 64, None, None) == 0
    # 16 rows x 128 columns: quants and 64 scales; rows padded to 64, columns to 128
    assert _lib.lib().qgemv_moe_tiles_bytes(8, 3, 96, 160) == 3 * 8 * 2 * (2048 + 128)
    assert _lib.lib().qgemv_moe_tiles_bytes(4, 3, 64, 160) == 3 * 4 * 2 * (1024 + 128)
    assert _lib.lib().qgemv_moe_tiles_bytes(4, 3, 40, 160) == 0
    assert _lib.lib().qgemv_moe_workspace_bytes(1, 33, 64, 64) == 0


def test_int8_validation():
    E = _lib

    def mm(xq=FAKE, xs=FAKE, ldx=64, wq=FAKE, ws=FAKE, ldw=64, b=None, n=2, m=8, k=64, y=FAKE, dt=0, ldy=8):
        return rc("qgemv_int8_matmul", xq, xs, ldx, wq, ws, ldw, b, n, m, k, y, dt, ldy, None)

    assert mm(n=0) == 0 and mm(m=0, ldy=0) == 0
    assert mm(n=-1) == 2 and mm(m=-1) == 2 and mm(k=0) == 2 and mm(k=40) == 2
    assert mm(k=1 << 17, ldx=1 << 17, ldw=1 << 17) == 5 and "int32" in E.last_error()
    assert mm(n=1 << 31) == 5 and mm(m=1 << 31) == 5
    assert mm(xq=None) == 1 and mm(xs=None) == 1 and mm(wq=None) == 1 and mm(ws=None) == 1 and mm(y=None) == 1
    assert mm(xq=FAKE + 8) == 3 and mm(wq=FAKE + 4) == 3 and mm(ldx=72) == 3 and mm(ldw=65) == 3
    assert mm(xs=FAKE + 2) == 3 and mm(b=FAKE + 1) == 3 and mm(y=FAKE + 2) == 3
    assert mm(ldx=48) == 2 and mm(ldw=32) == 2 and mm(ldy=7) == 2 and mm(dt=3) == 7

    def lin(x=FAKE, dt=0, ldx=64, wq=FAKE, n=2, k=64, y=FAKE, ydt=0, ws=FAKE, nb=1 << 20):
        return rc("qgemv_int8_linear", x, dt, ldx, wq, FAKE, 64, None, n, 8, k, y, ydt, 8, ws, nb, None)

    assert lin(n=0) == 0 and lin(x=None) == 1 and lin(dt=-1) == 7 and lin(ydt=9) == 7
    assert lin(x=FAKE + 2) == 3 and lin(ldx=63) == 2 and lin(k=72) == 2 and lin(y=None) == 1
    assert lin(ws=FAKE + 4) == 3 and lin(nb=100) == 7 and "workspace" in E.last_error()
    assert _lib.lib().qgemv_int8_linear_workspace_bytes(33, 64) == 64 * 4 + 33 * 64
    assert _lib.lib().qgemv_int8_linear_workspace_bytes(33, 65) == 0

    def quant(x=FAKE, dt=0, ldx=64, n=2, k=64, q=FAKE, ldq=64, s=FAKE):
        return rc("qgemv_int8_quantize", x, dt, ldx, n, k, q, ldq, s, None)

    assert quant(n=0) == 0 and quant(n=-1) == 2 and quant(k=0) == 2 and quant(dt=4) == 7
    assert quant(x=None) == 1 and quant(q=None) == 1 and quant(s=None) == 1
    assert quant(ldx=63) == 2 and quant(ldq=63) == 2 and quant(s=FAKE + 2) == 3 and quant(x=FAKE + 1, dt=1) == 3

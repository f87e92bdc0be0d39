"""What the calls of gated blocks refuse, on the CPU: they look at their arguments before the handle's contents, and launch
nothing.  And what their Python forms pass on, natively (csrc/call.cpp) and through ctypes."""
import ctypes
import subprocess

import numpy as np
import pytest

import cumpsgemm_amd as cg
from cumpsgemm_amd import _lib

P = 0x1000  # an address that nothing is read from


@pytest.fixture(scope="module")
def memory():
    return ctypes.create_string_buffer(4096)


@pytest.fixture
def handle(memory):
    """A handle that no call gets as far as using."""
    h = cg.Handle.__new__(cg.Handle)
    h._L, h._h, h._addr = _lib.lib(), ctypes.c_void_p(ctypes.addressof(memory)), ctypes.addressof(memory)
    h.close = lambda: None
    return h


GATED = dict(op_a=cg.OP_T, activation=cg.SILU, m=8, n=4, k=16, gate=P, up=P, lda=16, stridea=128, b=P, ldb=16, c=P, ldc=8, z_gate=P, z_up=2 * P,
             ldz=8, offsets=P, groups=2, mode=cg.FP16TCEC, type=cg.R_32F)
BACKWARD = dict(op_a=cg.OP_N, activation=cg.SILU, m=8, n=4, k=16, a=P, lda=8, stridea=128, b=P, ldb=16, z_gate=P, z_up=2 * P, ldz=8, d_gate=3 * P,
                d_up=4 * P, ldd=8, c=5 * P, ldc=8, offsets=P, groups=2, mode=cg.TF32TCEC, type=cg.R_32F)
COMMON = [dict(op_a=110), dict(activation=-1), dict(activation=4), dict(m=1 << 31), dict(n=1 << 31), dict(k=1 << 31), dict(groups=1 << 31),
          dict(mode=cg.AUTO), dict(mode=cg.CUBLAS), dict(mode=cg.FP16TCEC_SCALING), dict(type=cg.R_8I), dict(type=cg.R_8F_E4M3), dict(offsets=None),
          dict(b=None), dict(ldb=15)]


@pytest.mark.parametrize("bad", COMMON + [dict(gate=None), dict(up=None), dict(lda=15), dict(op_a=cg.OP_N, lda=7), dict(c=None), dict(ldc=7),
                                          dict(z_gate=None), dict(z_up=None), dict(ldz=7)], ids=str)
def test_gated_refuses(handle, bad):
    assert handle.gemm_gated(**{**GATED, **bad}) == cg.STATUS_INVALID_VALUE


@pytest.mark.parametrize("bad", COMMON + [dict(a=None), dict(lda=7), dict(op_a=cg.OP_T, lda=15), dict(z_gate=None), dict(z_up=None), dict(ldz=7),
                                          dict(d_gate=None), dict(d_up=None), dict(ldd=7), dict(ldc=7), dict(d_gate=P, ldd=9),
                                          dict(d_up=2 * P, ldd=9), dict(d_gate=2 * P), dict(d_up=P)], ids=str)
def test_backward_refuses(handle, bad):
    assert handle.gemm_gated_backward(**{**BACKWARD, **bad}) == cg.STATUS_INVALID_VALUE


F8 = dict(op_a=cg.OP_T, m=8, n=4, k=160, a=P, lda=160, stridea=1280, type_a=cg.R_8F_E4M3, scale_a=P, stridescale=2, b=P, ldb=160,
          type_b=cg.R_8F_E5M2, scale_b=P, c=P, ldc=8, type_c=cg.R_16BF, offsets=P, groups=2)
GATED_F8 = dict(activation=cg.GELU, m=8, n=4, k=160, gate=P, up=P, lda=160, stridea=1280, type_a=cg.R_8F_E4M3, scale_gate=P, scale_up=P,
                stridescale=2, b=P, ldb=160, type_b=cg.R_8F_E4M3, scale_b=P, c=P, ldc=8, type_c=cg.R_16F, offsets=P, groups=2)
QUANTIZE = dict(k=160, n=4, x=P, ldx=160, stridex=640, type_x=cg.R_16BF, block_n=1, q=P, ldq=160, strideq=640, type_q=cg.R_8F_E4M3, scale=P,
                batch=2)
COMMON_F8 = [dict(m=1 << 31), dict(n=1 << 31), dict(k=1 << 31), dict(groups=1 << 31), dict(type_a=cg.R_8F_E5M2), dict(type_a=cg.R_8I),
             dict(type_a=1000), dict(type_b=cg.R_8I), dict(type_b=cg.R_16F), dict(type_c=cg.R_8F_E4M3), dict(type_c=cg.R_8I), dict(offsets=None),
             dict(lda=159), dict(b=None), dict(ldb=159), dict(scale_b=None), dict(c=None), dict(ldc=7)]


@pytest.mark.parametrize("bad", COMMON_F8 + [dict(op_a=110), dict(a=None), dict(scale_a=None), dict(op_a=cg.OP_N, lda=7)], ids=str)
def test_f8_refuses(handle, bad):
    assert handle.gemm_f8(**{**F8, **bad}) == cg.STATUS_INVALID_VALUE


@pytest.mark.parametrize("bad", COMMON_F8 + [dict(activation=4), dict(activation=-1), dict(gate=None), dict(up=None), dict(scale_gate=None),
                                             dict(scale_up=None)], ids=str)
def test_gated_f8_refuses(handle, bad):
    assert handle.gemm_gated_f8(**{**GATED_F8, **bad}) == cg.STATUS_INVALID_VALUE


@pytest.mark.parametrize("bad", [dict(k=1 << 31), dict(n=1 << 31), dict(batch=1 << 31), dict(type_x=cg.R_8I), dict(type_x=cg.R_8F_E4M3),
                                 dict(type_q=cg.R_8I), dict(type_q=1000), dict(block_n=0), dict(block_n=64), dict(block_n=256), dict(x=None),
                                 dict(q=None), dict(scale=None), dict(ldx=159), dict(ldq=159), dict(strideq=639)], ids=str)
def test_quantize_refuses(handle, bad):
    assert handle.quantize_f8(**{**QUANTIZE, **bad}) == cg.STATUS_INVALID_VALUE


def test_no_handle():
    h = cg.Handle.__new__(cg.Handle)
    h._L, h._h, h._addr, h.close = _lib.lib(), None, None, lambda: None
    for call, args in ((h.gemm_gated, GATED), (h.gemm_gated_backward, BACKWARD), (h.gemm_f8, F8), (h.gemm_gated_f8, GATED_F8), (h.quantize_f8, QUANTIZE)):
        assert call(**args) == cg.STATUS_INVALID_VALUE


@pytest.mark.parametrize("empty", [dict(m=0), dict(n=0), dict(groups=0)], ids=str)
def test_nothing_to_do(handle, empty):
    none = dict(a=None, gate=None, up=None, b=None, c=None, z_gate=None, z_up=None, d_gate=None, d_up=None, offsets=None, groups=1,
                scale_a=None, scale_b=None, scale_gate=None, scale_up=None)
    for call, args in ((handle.gemm_gated, GATED), (handle.gemm_gated_backward, BACKWARD), (handle.gemm_f8, F8), (handle.gemm_gated_f8, GATED_F8)):
        assert call(**{**args, **{k: v for k, v in none.items() if k in args}, **empty}) == 0


@pytest.mark.parametrize("empty", [dict(k=0), dict(n=0), dict(batch=0)], ids=str)
def test_nothing_to_quantize(handle, empty):
    assert handle.quantize_f8(**{**QUANTIZE, **dict(x=None, q=None, scale=None), **empty}) == 0


STUB = """
#include <stdint.h>
extern "C" {
double got[32];
#define P(x) (double)(uintptr_t)(x)
static int put(int n, const double *v) { for (int i = 0; i < n; i++) got[i] = v[i]; return n; }
int cuMpSGEMM_gemm_gated(void *h, int op, int act, uint64_t m, uint64_t n, uint64_t k, void *gate, void *up, uint64_t lda, uint64_t sa, void *b,
    uint64_t ldb, void *c, uint64_t ldc, void *zg, void *zu, uint64_t ldz, void *off, uint64_t g, int mode, int t) {
  const double v[] = {P(h), (double)op, (double)act, (double)m, (double)n, (double)k, P(gate), P(up), (double)lda, (double)sa, P(b), (double)ldb,
                      P(c), (double)ldc, P(zg), P(zu), (double)ldz, P(off), (double)g, (double)mode, (double)t};
  return put(21, v); }
int cuMpSGEMM_gemm_gated_backward(void *h, int op, int act, uint64_t m, uint64_t n, uint64_t k, void *a, uint64_t lda, uint64_t sa, void *b,
    uint64_t ldb, void *zg, void *zu, uint64_t ldz, void *dg, void *du, uint64_t ldd, void *c, uint64_t ldc, void *off, uint64_t g, int mode, int t) {
  const double v[] = {P(h), (double)op, (double)act, (double)m, (double)n, (double)k, P(a), (double)lda, (double)sa, P(b), (double)ldb, P(zg), P(zu),
                      (double)ldz, P(dg), P(du), (double)ldd, P(c), (double)ldc, P(off), (double)g, (double)mode, (double)t};
  return put(23, v); }
int cuMpSGEMM_gemm_f8(void *h, int op, uint64_t m, uint64_t n, uint64_t k, void *a, uint64_t lda, uint64_t sa, int ta, void *xa, uint64_t ss, void *b,
    uint64_t ldb, int tb, void *xb, void *c, uint64_t ldc, int tc, void *off, uint64_t g) {
  const double v[] = {P(h), (double)op, (double)m, (double)n, (double)k, P(a), (double)lda, (double)sa, (double)ta, P(xa), (double)ss, P(b),
                      (double)ldb, (double)tb, P(xb), P(c), (double)ldc, (double)tc, P(off), (double)g};
  return put(20, v); }
int cuMpSGEMM_gemm_gated_f8(void *h, int act, uint64_t m, uint64_t n, uint64_t k, void *ga, void *up, uint64_t lda, uint64_t sa, int ta, void *xg,
    void *xu, uint64_t ss, void *b, uint64_t ldb, int tb, void *xb, void *c, uint64_t ldc, int tc, void *off, uint64_t g) {
  const double v[] = {P(h), (double)act, (double)m, (double)n, (double)k, P(ga), P(up), (double)lda, (double)sa, (double)ta, P(xg), P(xu),
                      (double)ss, P(b), (double)ldb, (double)tb, P(xb), P(c), (double)ldc, (double)tc, P(off), (double)g};
  return put(22, v); }
int cuMpSGEMM_quantize_f8(void *h, uint64_t k, uint64_t n, void *x, uint64_t ldx, uint64_t sx, int tx, uint64_t bn, void *q, uint64_t ldq,
    uint64_t sq, int tq, void *s, uint64_t batch) {
  const double v[] = {P(h), (double)k, (double)n, P(x), (double)ldx, (double)sx, (double)tx, (double)bn, P(q), (double)ldq, (double)sq, (double)tq,
                      P(s), (double)batch};
  return put(14, v); }
"""
CALLS = {
    "gemm_gated": [112, 1, 3, 4, 5, 0x100, 0x200, 6, 60, 0x300, 7, 0x400, 8, 0x500, 0x600, 9, 0x700, 10, 1, 14],
    "gemm_f8": [111, 3, 4, 5, 0x100, 6, 60, 28, 0x200, 7, 0x300, 8, 29, 0x400, 0x500, 9, 14, 0x600, 10],
    "gemm_gated_f8": [2, 3, 4, 5, 0x100, 0x200, 6, 60, 28, 0x300, 0x400, 7, 0x500, 8, 28, 0x600, 0x700, 9, 2, 0x800, 10],
    "quantize_f8": [3, 4, 0x100, 5, 50, 14, 128, 0x200, 6, 60, 29, 0x300, 7],
    "gemm_gated_backward": [111, 2, 3, 4, 5, 0x100, 6, 60, 0x200, 7, 0x300, 0x400, 8, 0x500, 0x600, 9, 0x700, 10, 0x800, 11, 2, 0],
}


@pytest.fixture
def stubbed(tmp_path):
    """(handle, what the last call passed): natively and through ctypes the stub is called"""
    assert _lib.lib() is not None and _lib._native is not None, "csrc/call.cpp is not built"
    (tmp_path / "stub.cpp").write_text(STUB + "}\n")
    subprocess.check_call(["g++", "-shared", "-fPIC", "-o", str(tmp_path / "stub.so"), str(tmp_path / "stub.cpp")])
    stub = ctypes.CDLL(str(tmp_path / "stub.so"))
    for name in _lib._GATED_FUNCTIONS:
        getattr(stub, name).argtypes = getattr(_lib.lib(), name).argtypes
    _lib._native.bind_gated(*(ctypes.cast(getattr(stub, n), ctypes.c_void_p).value for n in _lib._GATED_FUNCTIONS))
    h = cg.Handle.__new__(cg.Handle)
    h._L, h._h, h._addr = stub, ctypes.c_void_p(0x1230), 0x1230
    h.close = lambda: None
    yield h, (ctypes.c_double * 32).in_dll(stub, "got")
    _lib._native.bind_gated(*(ctypes.cast(getattr(_lib.lib(), n), ctypes.c_void_p).value for n in _lib._GATED_FUNCTIONS))


@pytest.mark.parametrize("name", CALLS)
def test_every_argument_arrives_in_its_place(stubbed, monkeypatch, name):
    h, got = stubbed
    for native in (True, False):
        if not native:
            monkeypatch.setattr(_lib, "_native", None)
        n = getattr(h, name)(*CALLS[name])
        assert list(got)[:n] == [0x1230, *CALLS[name]]


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("value", [np.int64(3), 3, 3.0, None, -1, 1 << 70, "3", 1j, True])
def test_other_types_are_what_ctypes_makes_of_them(stubbed, monkeypatch, name, value):
    h, got = stubbed

    def outcomes():
        out = []
        for where in range(len(CALLS[name])):
            args = list(CALLS[name])
            args[where] = value
            got[:] = [77.0] * 32
            try:
                out.append((getattr(h, name)(*args), list(got)))
            except Exception as e:  # noqa: BLE001
                out.append((type(e), list(got)))
        return out
    native = outcomes()
    monkeypatch.setattr(_lib, "_native", None)
    assert native == outcomes()

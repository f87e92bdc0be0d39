"""The experts' products' calls of the Python binding: natively (csrc/call.cpp) and through ctypes the same arguments arrive."""
import ctypes
import subprocess

import numpy as np
import pytest
import torch

import cumpsgemm_amd as cg
from cumpsgemm_amd import _lib

STUB = """
#include <stdint.h>
extern "C" {
double got[32];
#define P(x) (double)(uintptr_t)(x)
static int put(int n, const double *v) { for (int i = 0; i < n; i++) got[i] = v[i]; return n; }
int cuMpSGEMM_gemm_grouped(void *h, int op, uint64_t m, uint64_t n, uint64_t k, const float *al, void *a, uint64_t lda,
    uint64_t sa, void *b, uint64_t ldb, const float *be, void *c, uint64_t ldc, void *off, uint64_t g, int mode, int tab, int tc) {
  const double v[] = {P(h), (double)op, (double)m, (double)n, (double)k, *al, P(a), (double)lda, (double)sa, P(b), (double)ldb, *be,
                      P(c), (double)ldc, P(off), (double)g, (double)mode, (double)tab, (double)tc};
  return put(19, v); }
int cuMpSGEMM_gemm_grouped_k(void *h, uint64_t m, uint64_t n, uint64_t k, const float *al, void *a, uint64_t lda, void *b,
    uint64_t ldb, const float *be, void *c, uint64_t ldc, uint64_t sc, void *off, uint64_t g, int mode, int tab, int tc) {
  const double v[] = {P(h), (double)m, (double)n, (double)k, *al, P(a), (double)lda, P(b), (double)ldb, *be, P(c), (double)ldc,
                      (double)sc, P(off), (double)g, (double)mode, (double)tab, (double)tc};
  return put(18, v); }
int cuMpSGEMM_gemm_i8(void *h, uint64_t m, uint64_t n, uint64_t k, void *a, uint64_t lda, uint64_t sa, void *xa, void *b,
    uint64_t ldb, void *xb, void *c, uint64_t ldc, int tc, void *off, uint64_t g) {
  const double v[] = {P(h), (double)m, (double)n, (double)k, P(a), (double)lda, (double)sa, P(xa), P(b), (double)ldb, P(xb), P(c),
                      (double)ldc, (double)tc, P(off), (double)g};
  return put(16, v); }
int cuMpSGEMM_quantize_i8(void *h, uint64_t k, uint64_t n, void *x, uint64_t ldx, int t, void *q, uint64_t ldq, void *s) {
  const double v[] = {P(h), (double)k, (double)n, P(x), (double)ldx, (double)t, P(q), (double)ldq, P(s)};
  return put(9, v); }
}
"""
CALLS = {
    "gemm_grouped": [112, 3, 4, 5, 2.5, 0x100, 6, 60, 0x200, 7, 0.5, 0x300, 8, 0x400, 9, 1, 0, 14],
    "gemm_grouped_k": [3, 4, 5, 2.5, 0x100, 6, 0x200, 7, 0.5, 0x300, 8, 80, 0x400, 9, 2, 2, 0],
    "gemm_i8": [3, 4, 5, 0x100, 6, 60, 0x500, 0x200, 7, 0x600, 0x300, 8, 14, 0x400, 9],
    "quantize_i8": [3, 4, 0x100, 5, 2, 0x200, 6, 0x300],
}


@pytest.fixture
def stubbed(tmp_path):
    """(handle, what the last call passed): natively and through ctypes the stub is called"""
    assert _lib.lib() is not None and _lib._native is not None, "csrc/call.cpp is not built"
    (tmp_path / "stub.cpp").write_text(STUB)
    subprocess.check_call(["g++", "-shared", "-fPIC", "-o", str(tmp_path / "stub.so"), str(tmp_path / "stub.cpp")])
    stub = ctypes.CDLL(str(tmp_path / "stub.so"))
    for name in _lib._GROUPED_FUNCTIONS:
        getattr(stub, name).argtypes = getattr(_lib.lib(), name).argtypes
    _lib._native.bind_grouped(*(ctypes.cast(getattr(stub, n), ctypes.c_void_p).value for n in _lib._GROUPED_FUNCTIONS))
    h = cg.Handle.__new__(cg.Handle)
    h._L, h._h, h._addr = stub, ctypes.c_void_p(0x1230), 0x1230
    h.close = lambda: None
    yield h, (ctypes.c_double * 32).in_dll(stub, "got")
    _lib._native.bind_grouped(*(ctypes.cast(getattr(_lib.lib(), n), ctypes.c_void_p).value for n in _lib._GROUPED_FUNCTIONS))


@pytest.mark.parametrize("name", CALLS)
def test_every_argument_arrives_in_its_place(stubbed, monkeypatch, name):
    h, got = stubbed
    for native in (True, False):
        if not native:
            monkeypatch.setattr(_lib, "_native", None)
        n = getattr(h, name)(*CALLS[name])
        assert list(got)[:n] == [0x1230, *CALLS[name]]


def test_defaults_and_tensors(stubbed):
    h, got = stubbed
    t = torch.zeros(4)
    n = h.gemm_grouped(112, 3, 4, 5, 1.0, t, 6, 60, None, 7, 0.0, t, 8, t, 9, cg.FP16TCEC)
    assert list(got)[6] == t.data_ptr() and list(got)[9] == 0 and list(got)[16:n] == [1, cg.R_32F, cg.R_32F]
    n = h.gemm_i8(3, 4, 5, t, 6, 60, t, t, 7, t, t, 8)
    assert list(got)[13:n] == [cg.R_32F, 0, 1]


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

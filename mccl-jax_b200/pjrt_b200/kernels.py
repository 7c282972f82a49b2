"""ctypes binding of the 8-bit linear layer's kernels exported by libpjrt_b200.so (include/b200_kernels.h).

Arguments are those of the C entry points, in their order: device addresses as integers (None: no array),
sizes and row pitches in elements, PJRT_Buffer_Type codes, and the stream's handle.  A call that the library
refuses or cannot launch raises KernelError."""
from __future__ import annotations

import ctypes as C

from .pjrt import DEFAULT_LIB

REASONS = {-1: "bad arguments", -2: "no tensor map", -3: "launch failure", -4: "scratch too small or misaligned"}
ACT_NONE, ACT_GELU = 0, 1


class KernelError(RuntimeError):
    def __init__(self, name: str, code: int):
        super().__init__(f"{name}: {REASONS.get(code, 'error')} ({code})")
        self.code = code


class Kernels:
    def __init__(self, lib_path: str = DEFAULT_LIB):
        lib = C.CDLL(lib_path)
        p, n, i = C.c_void_p, C.c_int64, C.c_int
        self._quantize = lib.b200_quantize_i8
        self._quantize.argtypes = [p, n, p, n, p, n, n, i, p]
        self._rms_norm = lib.b200_rms_norm_i8
        self._rms_norm.argtypes = [p, n, p, n, p, p, n, p, n, p, n, n, i, i, C.c_float, p]
        self._gemm = lib.b200_gemm_i8
        self._gemm.argtypes = [p, n, p, n, p, p, p, p, n, n, n, n, i, i, p, C.c_size_t, p]
        self._scratch = lib.b200_gemm_i8_scratch_bytes
        self._scratch.argtypes = [p, n, p, n, n, n, n]
        self._scratch.restype = C.c_size_t

    def quantize_i8(self, x, ldx, q, ldq, scale, rows, cols, dtype, stream=None):
        rc = self._quantize(x, ldx, q, ldq, scale, rows, cols, dtype, stream)
        if rc:
            raise KernelError("quantize_i8", rc)

    def rms_norm_i8(self, x, ldx, residual, ldr, weight, h, ldh, q, ldq, scale, rows, cols, dtype, weight_dtype, eps,
                    stream=None):
        rc = self._rms_norm(x, ldx, residual, ldr, weight, h, ldh, q, ldq, scale, rows, cols, dtype, weight_dtype, eps,
                            stream)
        if rc:
            raise KernelError("rms_norm_i8", rc)

    def gemm_i8_scratch_bytes(self, a, lda, b, ldb, m, n, k) -> int:
        return self._scratch(a, lda, b, ldb, m, n, k)

    def gemm_i8(self, a, lda, b, ldb, a_scale, b_scale, bias, c, ldc, m, n, k, out_type, act=ACT_NONE, scratch=None,
                scratch_bytes=0, stream=None):
        rc = self._gemm(a, lda, b, ldb, a_scale, b_scale, bias, c, ldc, m, n, k, out_type, act, scratch, scratch_bytes,
                        stream)
        if rc:
            raise KernelError("gemm_i8", rc)

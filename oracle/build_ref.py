"""Builds oracle/_ref/libref_tile_scale.so from the reference's own scale computation (TEST INFRASTRUCTURE).

    python oracle/build_ref.py [reference_root]

The reference's MX quantizers compute their ue8m0 scale in `compute_tile_scale`, a plain integer C++ function
(csrc/kernels/quantization/quantization_mxfp8.cu:68-105 for e4m3 / e5m2 and quantization_mxfp4.cu:149-181 for e2m1)
inside HIP translation units that cannot be compiled here as a whole.  This recipe reads the two function bodies, the
constants they use (csrc/include/primus_turbo/quantization.h:82-104) and `e8m0_to_scale`
(csrc/include/primus_turbo/device/utils.cuh:124-126) from the reference tree WHERE THEY LIE, wraps them in a host
shim (the device qualifiers become empty, float_as_uint / uint_as_float become memcpy) and compiles the result with
g++.  The generated translation unit and the library are written to oracle/_ref/ only (git-ignored); no reference
source is kept in this repository.  tests/golden/make_golden.py calls the library to produce the committed scale
vectors, and tests/test_oracle_golden.py compares the oracle with the library directly when it is present.
"""
import os
import re
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
OUT = os.path.join(HERE, "_ref")
LIB = os.path.join(OUT, "libref_tile_scale.so")
# the files of the reference tree that are read
SOURCES = ("csrc/include/primus_turbo/quantization.h", "csrc/kernels/quantization/quantization_mxfp8.cu",
           "csrc/kernels/quantization/quantization_mxfp4.cu", "csrc/include/primus_turbo/device/utils.cuh")

SHIM_HEAD = r'''
#include <cstdint>
#include <cstring>
#include <type_traits>
#define __device__
#define __forceinline__ inline
#define PRIMUS_TURBO_DEVICE static inline
static inline uint32_t float_as_uint(float f) { uint32_t u; std::memcpy(&u, &f, 4); return u; }
static inline float uint_as_float(uint32_t u) { float f; std::memcpy(&f, &u, 4); return f; }
namespace primus_turbo {
namespace dtype { struct float8_e4m3 {}; struct float8_e5m2 {}; }
namespace detail {
'''

SHIM_TAIL = r'''
extern "C" {
// fmt: 0 = e4m3, 1 = e5m2, 2 = e2m1.  byte[i], native[i] = compute_tile_scale(amax[i]).
void ref_tile_scale(int fmt, const float *amax, int n, uint8_t *byte, float *native) {
    for (int i = 0; i < n; ++i) {
        if (fmt == 0) primus_turbo::fp8::compute_tile_scale<primus_turbo::dtype::float8_e4m3>(amax[i], native[i], byte[i]);
        else if (fmt == 1) primus_turbo::fp8::compute_tile_scale<primus_turbo::dtype::float8_e5m2>(amax[i], native[i], byte[i]);
        else primus_turbo::fp4::compute_tile_scale(amax[i], native[i], byte[i]);
    }
}
void ref_e8m0_to_scale(const uint8_t *byte, int n, float *scale) {
    for (int i = 0; i < n; ++i) scale[i] = primus_turbo::shared::e8m0_to_scale(byte[i]);
}
}
'''


def _slice(text, start_pat, end_pat, what):
    m = re.search(start_pat, text)
    if not m:
        raise RuntimeError(f"reference layout changed: start of {what} not found")
    e = re.search(end_pat, text[m.start():])
    if not e:
        raise RuntimeError(f"reference layout changed: end of {what} not found")
    return text[m.start(): m.start() + e.end()]


def build(ref_root="/root/reference"):
    """Returns the library path, or None when the reference tree is absent (no directory, or one without the sources; prebuilt
    files travel)."""
    if not os.path.isfile(os.path.join(ref_root, SOURCES[0])):
        return LIB if os.path.exists(LIB) else None
    rd = lambda rel: open(os.path.join(ref_root, rel)).read()
    consts = _slice(rd(SOURCES[0]), r"constexpr int FP32_MANTISSA_BITS", r"constexpr int E8M0_EXPONENT_BIAS = 127;",
                    "the format constants")
    fn8 = _slice(rd(SOURCES[1]), r"template <typename DType>\s*__device__ __forceinline__ void compute_tile_scale",
                 r"\n}\n", "compute_tile_scale (fp8)")
    fn4 = _slice(rd(SOURCES[2]), r"__device__ __forceinline__ void compute_tile_scale", r"\n}\n",
                 "compute_tile_scale (fp4)")
    e8 = _slice(rd(SOURCES[3]), r"PRIMUS_TURBO_DEVICE float e8m0_to_scale", r"\n}\n", "e8m0_to_scale")
    os.makedirs(OUT, exist_ok=True)
    src = os.path.join(OUT, "ref_tile_scale.cpp")
    with open(src, "w") as f:
        f.write("// GENERATED by oracle/build_ref.py from the reference tree; not kept in version control.\n")
        f.write(SHIM_HEAD + consts + "\n} }  // namespace detail, primus_turbo\n")
        f.write("namespace primus_turbo { namespace fp8 {\n" + fn8 + "\n} }\n")
        f.write("namespace primus_turbo { namespace fp4 {\n" + fn4 + "\n} }\n")
        f.write("namespace primus_turbo { namespace shared {\n" + e8 + "\n} }\n")
        f.write(SHIM_TAIL)
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-o", LIB, src], check=True)
    return LIB


def load():
    """ctypes handle of the library, or None when it has not been built."""
    import ctypes
    if not os.path.exists(LIB):
        return None
    lib = ctypes.CDLL(LIB)
    lib.ref_tile_scale.argtypes = [ctypes.c_int, ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p]
    lib.ref_e8m0_to_scale.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p]
    return lib


def tile_scale(lib, fmt: str, amax):
    """(byte uint8[n], native float32[n]) of the reference's compute_tile_scale for float32 amax values."""
    import numpy as np
    a = np.ascontiguousarray(amax, dtype=np.float32).reshape(-1)
    byte = np.empty(a.size, dtype=np.uint8)
    native = np.empty(a.size, dtype=np.float32)
    lib.ref_tile_scale({"e4m3": 0, "e5m2": 1, "e2m1": 2}[fmt], a.ctypes.data, a.size, byte.ctypes.data, native.ctypes.data)
    return byte, native


if __name__ == "__main__":
    print(build(*sys.argv[1:2]))

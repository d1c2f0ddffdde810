"""The division-free quotient of the 8-bit codes, x r + r (x - (x r) s) with r the rounded reciprocal of s: the bits of the fp32 division for every
value x of 8 significant bits and every fp32 significand of the scale s.  Powers of two pass through all its operations, signs too, so the pairs of significands
stand for all values whose quotient, product and remainder stay in range."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

SOURCE = r"""
#include <math.h>
#include <stdint.h>
#include <string.h>
static float number(uint32_t bits) { float f; memcpy(&f, &bits, 4); return f; }
/* significands first .. last of s: the pairs whose corrected quotient is not the division's, and (*plain) those whose x r is not */
int64_t differing(uint32_t first, uint32_t last, int64_t *plain) {
    int64_t bad = 0, off = 0;
    for (uint32_t i = first; i < last; ++i) {
        const float s = number(0x3f800000u + i), r = 1.0f / s;
        int32_t b = 0, o = 0;
        for (uint32_t j = 0; j < 128; ++j) {
            const float x = number(0x3f800000u + (j << 16)), q = x / s, q0 = x * r;
            o += q0 != q;
            b += __builtin_fmaf(__builtin_fmaf(-q0, s, x), r, q0) != q;
        }
        bad += b;
        off += o;
    }
    *plain = off;
    return bad;
}
"""


@pytest.mark.skipif(not shutil.which("gcc") or " fma " not in open("/proc/cpuinfo").read(), reason="needs gcc and a CPU with fused multiply-adds")
def test_every_pair_of_significands(tmp_path):
    from concurrent.futures import ThreadPoolExecutor
    src, lib = tmp_path / "q.c", tmp_path / "q.so"
    src.write_text(SOURCE)
    subprocess.check_call(["gcc", "-O3", "-mavx2", "-mfma", "-ffp-contract=off", "-shared", "-fPIC", "-o", lib, src])
    f = C.CDLL(os.fspath(lib)).differing
    f.argtypes, f.restype = [C.c_uint32, C.c_uint32, C.POINTER(C.c_int64)], C.c_int64
    parts, each = 64, (1 << 23) // 64

    def part(i):
        off = C.c_int64()
        return f(i * each, (i + 1) * each, C.byref(off)), off.value
    with ThreadPoolExecutor(8) as pool:
        results = list(pool.map(part, range(parts)))
    assert sum(b for b, _ in results) == 0
    assert sum(o for _, o in results) > (1 << 30) // 8           # without the correction a good part of them is off

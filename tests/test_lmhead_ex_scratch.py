"""The scratch that lcs_lmhead_ex's adapters take of a context (ad_low_floats) and
lm_low's grid on it (low_grid), compiled for the CPU from the sources: a state's
parts stay inside the scratch, and a row of a context costs 1 KB of it."""
import ctypes
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUS = 256


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    def source(name):
        with open(os.path.join(ROOT, "locus_amd", "csrc", name)) as f:
            return f.read()

    ex, internal = source("lcs_lmhead_ex.hip"), source("lcs_internal.hpp")
    consts = re.findall(r"^constexpr uint32_t (?:kAdWideMax|kAdParts) = .*$", internal, re.M)
    floats = internal[internal.index("constexpr uint64_t ad_low_floats("):]
    floats = floats[:floats.index("\n}\n") + 3]
    low = re.findall(r"^constexpr (?:int kLowWaves|uint32_t kLowRows) = .*$", ex, re.M)
    grid = ex[ex.index("struct LowGrid {"):]
    grid = grid[:grid.index("\n}\n") + 3]
    d = tmp_path_factory.mktemp("scratch")
    (d / "s.cpp").write_text("#include <cstdint>\n" + "\n".join(consts + low) + "\n" + floats + grid + """
extern "C" uint64_t floats(uint32_t max_rows) { return ad_low_floats(max_rows); }
extern "C" void grid(uint32_t rows, uint32_t n, uint32_t wide, uint32_t hidden, uint64_t floats, uint32_t cus, uint32_t* o) {
    const LowGrid g = low_grid(rows, n, wide, hidden, floats, cus);
    o[0] = g.x, o[1] = g.y, o[2] = g.z, o[3] = g.s;
}
""")
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-o", str(d / "s.so"), str(d / "s.cpp")], check=True, timeout=120)
    so = ctypes.CDLL(str(d / "s.so"))
    so.floats.restype = ctypes.c_uint64
    so.grid.argtypes = [ctypes.c_uint32] * 4 + [ctypes.c_uint64, ctypes.c_uint32, ctypes.c_void_p]
    return so


def test_a_row_of_a_context_costs_1_kb(lib):
    for rows in (1, 16, 64, 256, 257, 1024, 4096, 65536, 1 << 22):
        assert rows * 256 <= lib.floats(rows) <= rows * 256 + 256 * 768, rows
        assert 4 * lib.floats(rows) <= 1024 * rows + 3 * 1024 * min(rows, 256)


def test_states_fit_the_scratch(lib):
    o = (ctypes.c_uint32 * 4)()
    seen = set()
    for max_rows in (1, 5, 64, 256, 300, 512, 2048, 65536):
        for rows in {1, 5, 16, 63, 64, 65, 200, 256, 300, 511, 512, 1024, 2048, 40000, max_rows}:
            if rows > max_rows:
                continue
            for n in (1, 3, 8, 64, 1024):
                for wide in (8, 16, 64, 72, 128, 256):
                    for hidden in (64, 1024, 1088, 2048, 4096, 8192, 65536):
                        lib.grid(rows, n, wide, hidden, lib.floats(max_rows), CUS, o)
                        x, y, z, s = o
                        at = (max_rows, rows, n, wide, hidden, tuple(o))
                        assert rows * wide << s <= lib.floats(max_rows), at
                        assert x == min(n, rows) and y == -(-wide // 16) and z >= 1 and 0 <= s <= 2, at
                        assert z <= -(-rows // 16) and (s == 0 or x * y * z << s <= 2 * CUS), at
                        lib.grid(rows, n, wide, hidden, 1 << 60, CUS, o)   # (with all the scratch there is)
                        if rows <= 256 or rows * wide * 4 <= lib.floats(max_rows):
                            assert tuple(o) == (x, y, z, s), at
                        seen.add((o[3], s))
    assert seen == {(0, 0), (1, 1), (2, 2), (1, 0), (2, 1), (2, 0)}

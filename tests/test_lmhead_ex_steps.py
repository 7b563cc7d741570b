"""The adapters' steps of lcs_lmhead_ex's tiles (last_step, lcs_lmtile.hpp), compiled
for the CPU from the kernel's source: with any number of ranks that a tile's LDS
takes at a time, an adapter's accumulator is added to its rows once for each
window of ranks that it reaches, and the steps past the last one, which the
tiles take to keep their loads in flight, add nothing: rows without an adapter
carry the mark of such a step."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def last_step(tmp_path_factory):
    with open(os.path.join(ROOT, "locus_amd", "csrc", "lcs_lmtile.hpp")) as f:
        text = f.read()
    body = text[text.index("constexpr bool last_step("):]
    body = body[:body.index("\n}\n") + 3]
    d = tmp_path_factory.mktemp("steps")
    (d / "s.cpp").write_text("#include <cstdint>\n" + body +
                             'extern "C" int f(int32_t who, uint32_t k, uint32_t end) { return last_step(who, k, end); }\n')
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-o", str(d / "s.so"), str(d / "s.cpp")], check=True, timeout=120)
    fn = ctypes.CDLL(str(d / "s.so")).f
    fn.argtypes = [ctypes.c_int32, ctypes.c_uint32, ctypes.c_uint32]
    return fn


@pytest.mark.parametrize("fits", [16, 32, 48, 64, 112, 256])
def test_each_window_of_an_adapter_ends_once(last_step, fits):
    for wide in (8, 16, 24, 64, 256):
        for rank in {1, 7, 8, 15, 16, 17, 33, wide} & set(range(1, wide + 1)):
            for ad in (0, 5, 1023):
                who, ends = rank << 16 | ad, []
                for kw in range(0, wide, fits):   # the windows, and the tile's walk of one
                    k, n = kw, 0
                    while k < min(rank, kw + fits):
                        n += last_step(who, k, kw + fits)
                        assert (k + 16 >= min(rank, kw + fits)) == bool(last_step(who, k, kw + fits))
                        k += 16
                    ends.append(n)
                assert ends == [int(kw < rank) for kw in range(0, wide, fits)]


@pytest.mark.parametrize("fits", [16, 32, 48, 64, 112, 256])
def test_a_step_past_the_last_one_adds_nothing(last_step, fits):
    for kw in range(0, 256, fits):
        assert not last_step(-1, kw, kw + fits)

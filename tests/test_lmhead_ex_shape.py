"""lcs_lmhead_ex's choice of a tile (lmhead_ex_shape, and lmhead_shape's under it),
compiled for the CPU from the kernels' sources: the GPU tests' list names the tile
that each case runs on, and every tile has one."""
import ctypes
import os
import re
import subprocess

from tests.test_gpu_lmhead_ex import TILES

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUS = 256


def source(name):
    with open(os.path.join(ROOT, "locus_amd", "csrc", name)) as f:
        return f.read()


def test_cases_cover_every_tile(tmp_path):
    ex, plain = source("lcs_lmhead_ex.hip"), source("lcs_lmhead.hip")
    above = ex[ex.index("struct LmExShape {"):ex.index("template <bool F8, bool AD>\nvoid tiles(")]
    below = plain[plain.index("struct LmShape {"):plain.index("hipError_t launch_lmhead(")]
    consts = re.findall(r"^constexpr uint32_t (?:kMaxVocab|kLmMaxBlocks) = .*$", source("lcs_internal.hpp"), re.M)
    big = re.search(r"^constexpr uint32_t kBigHidden = .*$", plain, re.M).group(0)
    (tmp_path / "shape.cpp").write_text(
        "#include <cstdint>\n" + "\n".join(consts) + "\n" + big + "\n" + below +
        """static void lmhead_shape_of(uint32_t rows, uint32_t vocab, uint32_t hidden, uint32_t cus, uint32_t* vt, uint32_t* br) {
    const LmShape s = lmhead_shape(rows, vocab, hidden, cus);
    *vt = s.vt, *br = s.br;
}
""" + above + """extern "C" void shape(uint32_t rows, uint32_t vocab, int f8, uint32_t cus, uint32_t* o) {
    const LmExShape s = lmhead_ex_shape(rows, vocab, 448, f8 != 0, cus);
    o[0] = s.vt, o[1] = s.br;
}
""")
    so = str(tmp_path / "shape.so")
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-o", so, str(tmp_path / "shape.cpp")], check=True, timeout=120)
    fn = ctypes.CDLL(so).shape
    out = (ctypes.c_uint32 * 2)()
    for rows, vocab, vt, br in TILES:
        for f8 in (0, 1):
            fn(rows, vocab, f8, CUS, out)
            assert tuple(out) == (vt, br), (rows, vocab, f8, tuple(out))
    launched = {(int(v), int(b)) for v, b in re.findall(r"tile<(\d+), (\d+), [^>]*F8, AD(?:, 1)?>\(", ex)}
    assert launched == {(4, 256), (4, 192), (4, 128), (2, 128), (5, 64), (4, 64), (2, 64), (1, 64), (4, 32), (2, 32)} == {c[2:] for c in TILES}
    # with several row tiles too
    assert {c[2:] for c in TILES if c[0] > c[3]} == {(4, 256), (4, 192), (4, 128), (2, 128), (2, 64), (1, 64)}
    # every shape fits the context's records (lmhead_max_blocks, by the vocabulary alone)
    for vocab in list(range(1, 262145, 997)) + [262144]:
        most = max(min(-(-vocab // 64), 2 * CUS), min(-(-vocab // 128), 4 * CUS))
        most = max(min(most, 1024), -(-vocab // 256))
        for rows in (1, 33, 64, 65, 128, 200, 300, 1024):
            for f8 in (0, 1):
                fn(rows, vocab, f8, CUS, out)
                assert -(-vocab // (64 * out[0])) <= most, (rows, vocab, tuple(out))

"""What lcs_add_rmsnorm and lcs_lmhead_ex refuse (lcs_check.hpp, compiled here for
the CPU), and what the Python binding refuses before that."""
import ctypes as C
import os
import subprocess

import pytest

from locus_amd import sampler as S

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("check")
    (d / "check.cpp").write_text('''#include "lcs_check.hpp"
extern "C" int norm(const lcs_norm_batch* b, const lcs_norm_out* o, const char** why) {
    return lcs::check_add_rmsnorm(b, o, 32768, why);
}
extern "C" int head(const lcs_lmhead_ex_batch* b, const lcs_lmhead_out* o, const char** why) {
    return lcs::check_lmhead_ex(b, o, 512, 262144, why);
}
''')
    so = str(d / "check.so")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROOT, "locus_amd", "csrc"), "-o", so, str(d / "check.cpp")], check=True, timeout=120)
    return C.CDLL(so)


def call(fn, b, o):
    why = C.c_char_p(b"")
    rc = fn(None if b is None else C.byref(b), None if o is None else C.byref(o), C.byref(why))
    return rc, why.value.decode()


A = 0x10000   # (an address: nothing reads it)


def norm_args(**kw):
    b = dict(rows=3, hidden=100, x_dtype=S.LCS_BF16, y_dtype=S.LCS_E4M3, eps=1e-6, x=A, residual=A, weight=A,
             x_stride=100, residual_stride=100)
    o = dict(y=A, y_scale=A, sum=A, y_stride=100, sum_stride=100)
    for k, v in kw.items():
        (b if k in b else o)[k] = v
    return S._NBatch(**b), S._NOut(**o)


def test_norm_arguments(lib):
    assert call(lib.norm, *norm_args()) == (0, "")
    assert call(lib.norm, *norm_args(rows=0, x=None)) == (0, "")
    assert call(lib.norm, *norm_args(residual=None, sum=None, residual_stride=0, sum_stride=0)) == (0, "")
    assert call(lib.norm, *norm_args(sum=None, sum_stride=0)) == (0, "")
    assert call(lib.norm, *norm_args(x=A + 2, y=A + 1, y_dtype=S.LCS_E4M3)) == (0, "")
    assert call(lib.norm, *norm_args(hidden=32768, x_stride=40000, residual_stride=32768, y_stride=32769,
                                     sum_stride=32768)) == (0, "")
    assert call(lib.norm, *norm_args(y_dtype=S.LCS_F32, y_scale=None)) == (0, "")
    for kw, text in [(dict(x_dtype=S.LCS_E4M3), "x_dtype"), (dict(x_dtype=7), "x_dtype"), (dict(y_dtype=3), "y_dtype"),
                     (dict(hidden=0), "hidden"), (dict(hidden=32769), "hidden"), (dict(eps=0.0), "eps"),
                     (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
                     (dict(x=None), "null"), (dict(weight=None), "null"), (dict(y=None), "null"),
                     (dict(y_scale=None), "y_scale"), (dict(residual=None), "residual"), (dict(x=A + 1), "aligned"),
                     (dict(weight=A + 1), "aligned"), (dict(residual=A + 1), "aligned"), (dict(sum=A + 1), "aligned"),
                     (dict(y_scale=A + 2), "aligned"), (dict(y=A + 2, y_dtype=S.LCS_F32), "aligned"),
                     (dict(x_stride=99), "strides"), (dict(residual_stride=99), "strides"),
                     (dict(y_stride=99), "strides"), (dict(sum_stride=0), "strides")]:
        rc, why = call(lib.norm, *norm_args(**kw))
        assert rc == S.LCS_ERR_INVALID_ARG and text in why, (kw, rc, why)
    b, o = norm_args()
    assert call(lib.norm, None, o)[0] == S.LCS_ERR_INVALID_ARG and call(lib.norm, b, None)[0] == S.LCS_ERR_INVALID_ARG


def head_args(ad=None, **kw):
    b = dict(rows=6, vocab=1000, hidden=128, rows_per_seq=3, dtype=S.LCS_E4M3, x=A, w=A, x_scale=A, w_scale=A, draft=A,
             slot=A)
    o = dict(logits=A, ld_logits=1000, argmax_ids=A, log_z=A, draft_lp=A, accept_len=A, stats=A)
    for k, v in kw.items():
        (b if k in b else o)[k] = v
    if ad is not None:
        b["adapters"] = C.pointer(S._Adapters(**{**dict(n=4, wide=16, a=A, b=A, rank=A, scale=A), **ad}))
    return S._LExBatch(**b), S._LOut(**o)


def test_lmhead_ex_arguments(lib):
    ok = (0, "")
    assert call(lib.head, *head_args({})) == ok
    assert call(lib.head, *head_args(slot=None)) == ok
    assert call(lib.head, *head_args({"rank": None, "scale": None}, dtype=S.LCS_BF16, x_scale=None, w_scale=None)) == ok
    assert call(lib.head, *head_args(slot=None, x_scale=None, w_scale=None, draft=None, draft_lp=None, accept_len=None,
                                     logits=None, ld_logits=0)) == ok
    assert call(lib.head, *head_args({}, rows=0, x=None)) == ok
    assert call(lib.head, *head_args({"n": 1024, "wide": 256})) == ok
    for ad, kw, text in [
            ({}, dict(dtype=S.LCS_F32), "dtype"), ({}, dict(x=None), "null"), ({}, dict(argmax_ids=None), "null"),
            ({}, dict(x=A + 8), "16-byte"), ({}, dict(w=A + 8), "16-byte"), ({}, dict(hidden=0), "hidden"),
            ({}, dict(hidden=96), "hidden"), ({}, dict(hidden=65600), "hidden"), ({}, dict(vocab=0), "vocab"),
            ({}, dict(ld_logits=999), "ld_logits"), ({}, dict(rows_per_seq=4), "rows_per_seq"),
            ({}, dict(rows=130, rows_per_seq=65), "rows_per_seq"), ({}, dict(draft_lp=None), "draft_lp"),
            ({}, dict(draft=None), "accept_len"), ({}, dict(rows_per_seq=0), "accept_len"),
            ({}, dict(dtype=S.LCS_BF16), "scales"), ({}, dict(x_scale=A + 2), "aligned"),
            ({"n": 0}, {}, "1 to 1024"), ({"n": 1025}, {}, "1 to 1024"), ({"wide": 0}, {}, "wide"),
            ({"wide": 12}, {}, "wide"), ({"wide": 264}, {}, "wide"), ({"a": None}, {}, "null"), ({"b": None}, {}, "null"),
            ({}, dict(slot=None), "null"), ({"a": A + 8}, {}, "16-byte"), ({"b": A + 8}, {}, "16-byte"),
            ({"rank": A + 1}, {}, "aligned"), ({"scale": A + 1}, {}, "aligned"), (None, {}, "slot given")]:
        rc, why = call(lib.head, *head_args(ad, **kw))
        assert rc == S.LCS_ERR_INVALID_ARG and text in why, (ad, kw, rc, why)
    for kw in (dict(rows=513, rows_per_seq=0, accept_len=None), dict(vocab=262145, ld_logits=262145)):
        rc, why = call(lib.head, *head_args({}, **kw))
        assert rc == S.LCS_ERR_CAPACITY and "limits" in why, (kw, rc, why)


def test_x_of_4_gib_is_refused_with_adapters(tmp_path, lib):
    # (the check's own limits here: 512 rows x 65536 stay far below)
    (tmp_path / "c.cpp").write_text('''#include "lcs_check.hpp"
extern "C" int head(const lcs_lmhead_ex_batch* b, const lcs_lmhead_out* o, const char** why) {
    return lcs::check_lmhead_ex(b, o, 1u << 20, 262144, why);
}
''')
    so = str(tmp_path / "c.so")
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROOT, "locus_amd", "csrc"), "-o", so, str(tmp_path / "c.cpp")], check=True, timeout=120)
    fn = C.CDLL(so).head
    kw = dict(hidden=65536, rows_per_seq=0, accept_len=None)
    assert call(fn, *head_args({}, rows=65535, **kw)) == (0, "")
    rc, why = call(fn, *head_args({}, rows=65536, **kw))
    assert rc == S.LCS_ERR_CAPACITY and "4 GiB" in why
    assert call(fn, *head_args(None, rows=65536, slot=None, **kw)) == (0, "")


def test_adapters_of_the_binding():
    torch = pytest.importorskip("torch")
    a = torch.zeros((3, 16, 64), dtype=torch.bfloat16)
    b = torch.zeros((3, 50, 16), dtype=torch.bfloat16)
    rank, scale = torch.zeros(3, dtype=torch.int32), torch.zeros(3)
    ad = S.Adapters(a, b, rank=rank, scale=scale)
    assert (ad.n, ad.wide, ad.hidden, ad.vocab) == (3, 16, 64, 50)
    S.Adapters(a, b)
    for args, kw, text in [((a.float(), b), {}, "bfloat16"), ((a, b[:2]), {}, "must be"), ((a, b[:, :, :8]), {}, "must be"),
                           ((a[0], b), {}, "must be"), ((a[:, :, ::2], b), {}, "contiguous"),
                           ((a, b), {"rank": rank.long()}, "rank"), ((a, b), {"rank": rank[:2]}, "rank"),
                           ((a, b), {"scale": scale.double()}, "scale")]:
        with pytest.raises(S.SamplerError, match=text):
            S.Adapters(*args, **kw)

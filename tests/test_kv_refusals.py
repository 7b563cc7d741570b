"""What the paged cache's calls, lcs_tree_attn and lcs_tree_verify refuse
(lcs_kv_check.hpp, compiled here for the CPU), and what the Python binding refuses
before that."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from locus_amd import sampler as S

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 0x10000   # (an address: nothing reads it)


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("check")
    (d / "check.cpp").write_text('''#include "lcs_kv_check.hpp"
using namespace lcs;
extern "C" int cache(const lcs_kv_cache* c, const char** why) { return check_kv_cache(c, why); }
extern "C" int requests(const lcs_kv_cache* c, uint32_t n, const int32_t* s, const int32_t* a, const int32_t* b,
                        const int32_t* r, const char** why) { return check_kv_requests(c, n, s, a, b, r, 1024, why); }
extern "C" int compact(const lcs_kv_cache* c, uint32_t n, uint32_t m, const int32_t* s, const int32_t* a, const int32_t* b,
                       const int32_t* r, const char** why) { return check_kv_compact(c, n, m, s, a, b, r, 1024, why); }
extern "C" int append(const lcs_kv_cache* c, const lcs_kv_append_batch* b, const char** why) { return check_kv_append(c, b, 1024, why); }
extern "C" int attn(const lcs_tree_attn_batch* b, const lcs_tree_attn_out* o, const char** why) { return check_tree_attn(b, o, 1024, 65536, why); }
extern "C" int verify(const lcs_tree_verify_batch* b, const lcs_tree_verify_out* o, const char** why) { return check_tree_verify(b, o, why); }
''')
    so = str(d / "check.so")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROOT, "locus_amd", "csrc"), "-o", so, str(d / "check.cpp")], check=True, timeout=120)
    L = C.CDLL(so)
    p, u = C.c_void_p, C.c_uint32
    L.requests.argtypes = [p, u, p, p, p, p, p]
    L.compact.argtypes = [p, u, u, p, p, p, p, p]
    return L


def call(fn, *args):
    why = C.c_char_p(b"")
    return fn(*(C.byref(a) if isinstance(a, C.Structure) else a for a in args), C.byref(why)), why.value.decode()


def cache(**kw):
    c = dict(layers=2, pages=10, page_tokens=16, kv_heads=3, head_dim=64, dtype=S.LCS_BF16, seqs=4, max_pages=5, k=A, v=A,
             layer_stride=10 * 3 * 16 * 64, page_stride=3 * 16 * 64, head_stride=16 * 64, token_stride=64, table=A, refs=A)
    c.update(kw)
    return S._KvCache(**c)


F8 = dict(dtype=S.LCS_E4M3, k_scale=A, v_scale=A)


def test_cache(lib):
    for kw in [{}, F8, dict(head_dim=16, token_stride=64), dict(page_tokens=1024, head_stride=1024 * 64, page_stride=3 * 1024 * 64, layer_stride=30 * 1024 * 64),
               # tokens ahead of heads, k and v in one buffer, heads ahead of pages
               dict(head_stride=64, token_stride=3 * 64), dict(page_stride=2 * 3 * 16 * 64, layer_stride=20 * 3 * 16 * 64),
               dict(head_stride=10 * 16 * 64, page_stride=16 * 64), dict(layers=1, layer_stride=7), dict(kv_heads=1, head_stride=0),
               dict(head_dim=256, token_stride=256, head_stride=16 * 256, page_stride=48 * 256, layer_stride=480 * 256)]:
        assert call(lib.cache, cache(**kw)) == (0, ""), kw
    bad = [(dict(dtype=S.LCS_F32), "dtype"), (dict(layers=0), "layers"), (dict(layers=4097), "layers"), (dict(pages=0), "pages"),
           (dict(pages=1 << 31), "pages"), (dict(page_tokens=8), "page_tokens"), (dict(page_tokens=24), "page_tokens"),
           (dict(page_tokens=2048), "page_tokens"), (dict(kv_heads=0), "kv_heads"), (dict(head_dim=8), "head_dim"),
           (dict(head_dim=0), "head_dim"), (dict(head_dim=272), "head_dim"), (dict(head_dim=72), "head_dim"),
           (dict(seqs=0), "table"), (dict(max_pages=0), "table"), (dict(seqs=1 << 20, max_pages=1 << 11), "table"),
           (dict(k=None), "null"), (dict(v=None), "null"), (dict(table=None), "null"), (dict(refs=None), "null"),
           (dict(k=A + 8), "aligned"), (dict(refs=A + 4), "aligned"), (dict(table=A + 2), "aligned"),
           (dict(k_scale=A), "scale"), (dict(dtype=S.LCS_E4M3), "scale"), (dict(F8, v_scale=None), "scale"),
           (dict(F8, k_scale=A + 2), "aligned"), (dict(token_stride=68), "16 bytes"), (dict(F8, token_stride=72), "16 bytes"),
           (dict(token_stride=0), "overlap"), (dict(head_stride=16 * 64 - 8), "overlap"), (dict(page_stride=2 * 16 * 64), "overlap"),
           (dict(layer_stride=9 * 3 * 16 * 64), "overlap"), (dict(head_stride=0), "overlap"),
           (dict(layer_stride=1 << 61, layers=4), "overlap"),
           (dict(token_stride=1 << 26, head_stride=64, page_stride=1 << 31, layer_stride=1 << 40), "2 GiB")]
    for kw, text in bad:
        rc, why = call(lib.cache, cache(**kw))
        assert rc == -1 and text in why, (kw, rc, why)
    assert call(lib.cache, None)[0] == -1


def test_requests(lib):
    c = cache()
    assert call(lib.requests, c, 3, A, A, A, A) == (0, "")
    assert call(lib.requests, c, 0, None, None, None, None) == (0, "")
    assert call(lib.requests, c, 1024, A, A, A, A) == (0, "")
    assert call(lib.requests, c, 1025, A, A, A, A)[0] == -4
    for i in range(4):
        ptr = [A] * 4
        ptr[i] = None
        assert call(lib.requests, c, 3, *ptr)[0] == -1
        ptr[i] = A + 2
        assert call(lib.requests, c, 3, *ptr)[0] == -1
    assert call(lib.requests, cache(pages=0), 3, A, A, A, A)[0] == -1
    assert call(lib.compact, c, 3, 7, A, A, A, A) == (0, "")
    assert call(lib.compact, c, 3, 1 << 31, A, A, A, A)[0] == -1
    assert call(lib.compact, c, 3, 0, A, A, None, A) == (0, "")
    assert call(lib.compact, c, 3, 1, A, A, None, A)[0] == -1
    big = dict(layers=4096, kv_heads=1024, pages=1, head_stride=16 * 64, page_stride=0, layer_stride=1024 * 16 * 64)
    assert call(lib.compact, cache(**big), 200, 7, A, A, A, A) == (0, "")
    assert call(lib.compact, cache(**big), 300, 7, A, A, A, A)[0] == -4


def append(c=None, **kw):
    b = dict(n_seq=3, rows_per_seq=5, layer=0, n_layers=2, k=A, v=A, layer_stride=15 * 192, k_stride=192, v_stride=192, pos=A)
    b.update(kw)
    return S._AppendBatch(**b)


def test_append(lib):
    for kw in [{}, dict(n_seq=0, k=None), dict(n_layers=0, pos=None), dict(seq=A, count=A, index=A), dict(layer=1, n_layers=1, layer_stride=3),
               dict(k_stride=200, v_stride=1024), dict(rows_per_seq=1 << 20)]:
        assert call(lib.append, cache(), append(**kw)) == (0, ""), kw
    for kw, rc in [(dict(n_seq=1025), -4), (dict(rows_per_seq=0), -1), (dict(rows_per_seq=(1 << 20) + 1), -1), (dict(layer=2), -1),
                   (dict(layer=1), -1), (dict(n_layers=0xffffffff, layer=1), -1), (dict(k=None), -1), (dict(v=None), -1),
                   (dict(pos=None), -1), (dict(k=A + 2), -1), (dict(pos=A + 1), -1), (dict(index=A + 2), -1), (dict(k_stride=184), -1),
                   (dict(v_stride=196), -1), (dict(layer_stride=4), -1)]:
        assert call(lib.append, cache(), append(**kw))[0] == rc, kw
    assert call(lib.append, cache(), None)[0] == -1
    assert call(lib.append, None, append())[0] == -1


def attn(**kw):
    c = kw.pop("cache", cache())
    b = dict(n_seq=3, rows_per_seq=5, heads=6, layer=0, scale=0.125, mask_words=0, cache=C.pointer(c) if c else None, q=A, k=A, v=A,
             q_stride=6 * 64, k_stride=3 * 64, v_stride=3 * 64, length=A)
    o = dict(o=A, o_stride=6 * 64, lse=A)
    for k, v in kw.items():
        (o if k in o else b)[k] = v
    return S._TreeBatch(**b), S._TreeOut(**o)


def test_attention(lib):
    for kw in [{}, dict(n_seq=0, q=None), dict(lse=None), dict(seq=A, mask=A, mask_words=1), dict(rows_per_seq=256, mask=A, mask_words=8),
               dict(scale=-1.0), dict(scale=0.0), dict(scale=-9e29), dict(layer=1), dict(q_stride=1000, o_stride=392, k_stride=1000), dict(heads=3)]:
        assert call(lib.attn, *attn(**kw)) == (0, ""), kw
    for kw, rc in [(dict(n_seq=1025), -4), (dict(rows_per_seq=0), -1), (dict(rows_per_seq=257), -1), (dict(heads=0), -1), (dict(heads=7), -1),
                   (dict(heads=3 << 20), -1), (dict(layer=2), -1), (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(scale=1.1e30), -1), (dict(scale=-1.1e30), -1), (dict(q=None), -1),
                   (dict(k=None), -1), (dict(v=None), -1), (dict(length=None), -1), (dict(o=None), -1), (dict(q=A + 8), -1), (dict(o=A + 2), -1),
                   (dict(seq=A + 2), -1), (dict(lse=A + 1), -1), (dict(mask=A), -1), (dict(rows_per_seq=33, mask=A, mask_words=1), -1),
                   (dict(q_stride=6 * 64 - 8), -1), (dict(o_stride=6 * 64 - 8), -1), (dict(k_stride=184), -1), (dict(v_stride=196), -1),
                   (dict(q_stride=6 * 64 + 4), -1), (dict(o_stride=6 * 64 + 2), -1), (dict(cache=None), -1), (dict(cache=cache(pages=0)), -1),
                   (dict(n_seq=1024, rows_per_seq=256, heads=3 * 4096, q_stride=1 << 20, o_stride=1 << 20), -4)]:
        assert call(lib.attn, *attn(**kw))[0] == rc, kw
    wide = cache(kv_heads=128, head_stride=16 * 64, page_stride=128 * 16 * 64, layer_stride=1280 * 16 * 64)
    many = dict(cache=wide, heads=128, q_stride=128 * 64, k_stride=128 * 64, v_stride=128 * 64, o_stride=128 * 64)
    assert call(lib.attn, *attn(n_seq=512, **many)) == (0, "")
    assert call(lib.attn, *attn(n_seq=513, **many))[0] == -4
    assert call(lib.attn, *attn(k_stride=(1 << 25) + 8))[0] == -1
    long = cache(seqs=1024, max_pages=2 ** 21 - 1, page_tokens=1024, kv_heads=64, head_dim=16, token_stride=16, head_stride=16 * 1024,
                 page_stride=64 * 16 * 1024, layer_stride=640 * 16 * 1024)
    few = dict(cache=long, heads=64, q_stride=1024, k_stride=1024, v_stride=1024, o_stride=1024)
    assert call(lib.attn, *attn(n_seq=1, **few)) == (0, "")
    assert call(lib.attn, *attn(n_seq=2, **few))[0] == -4
    b, o = attn()
    assert call(lib.attn, None, o)[0] == -1 and call(lib.attn, b, None)[0] == -1


def verify(**kw):
    b = dict(n_seq=3, rows_per_seq=5, vocab=100, dtype=S.LCS_BF16, row_stride=104, logits=A, tokens=A, parent=A, length=A)
    o = dict(argmax_ids=A, node_lp=A, path=A, n_path=A, next_id=A)
    olen = kw.pop("new_length", A)
    for k, v in kw.items():
        (o if k in o else b)[k] = v
    return S._TreeVBatch(**b), S._TreeVOut(**o, length=olen)


def test_verdict(lib):
    for kw in [{}, dict(n_seq=0, tokens=None), dict(logits=None, node_lp=None, vocab=0, dtype=9, row_stride=0), dict(new_length=None),
               dict(length=None, new_length=None), dict(dtype=S.LCS_F32, row_stride=100), dict(rows_per_seq=256)]:
        assert call(lib.verify, *verify(**kw)) == (0, ""), kw
    for kw, rc in [(dict(rows_per_seq=0), -1), (dict(rows_per_seq=257), -1), (dict(n_seq=1 << 30), -4), (dict(tokens=None), -1), (dict(parent=None), -1),
                   (dict(argmax_ids=None), -1), (dict(path=None), -1), (dict(n_path=None), -1), (dict(next_id=None), -1), (dict(length=None), -1),
                   (dict(logits=None), -1), (dict(dtype=S.LCS_E4M3), -1), (dict(vocab=0), -1), (dict(vocab=105), -1), (dict(row_stride=108), -1),
                   (dict(logits=A + 8), -1), (dict(tokens=A + 2), -1), (dict(path=A + 1), -1)]:
        assert call(lib.verify, *verify(**kw))[0] == rc, kw


def test_cache_tensors():
    """What KvCache itself refuses (the tensors' device is the CPU's here)."""
    k = torch.zeros(2, 10, 3, 16, 64, dtype=torch.bfloat16)
    table, refs = torch.zeros(4, 5, dtype=torch.int32), torch.zeros(10, dtype=torch.int32)
    good = S.KvCache(k, k.clone(), table, refs)
    assert good.shape == (2, 10, 3, 16, 64)
    both = torch.zeros(2, 10, 2, 3, 16, 64, dtype=torch.bfloat16)
    S.KvCache(both[:, :, 0], both[:, :, 1], table, refs)
    k8, sc = k.to(torch.float8_e4m3fn), torch.zeros(2, 10, 3, 16)
    S.KvCache(k8, k8.clone(), table, refs, k_scale=sc, v_scale=sc.clone())
    for bad in [lambda: S.KvCache(k.float(), k.float(), table, refs), lambda: S.KvCache(k, k8, table, refs),
                lambda: S.KvCache(k[0], k[0], table, refs), lambda: S.KvCache(k, k.transpose(2, 3).contiguous().transpose(2, 3), table, refs),
                lambda: S.KvCache(k[..., ::2], k[..., ::2], table, refs), lambda: S.KvCache(k, k, table.long(), refs),
                lambda: S.KvCache(k, k, table[:, ::2], refs), lambda: S.KvCache(k, k, table[0], refs), lambda: S.KvCache(k, k, table, refs[:9]),
                lambda: S.KvCache(k, k, table, refs.float()), lambda: S.KvCache(k, k, table, refs, k_scale=sc), lambda: S.KvCache(k8, k8, table, refs),
                lambda: S.KvCache(k8, k8, table, refs, k_scale=sc, v_scale=sc.double()),
                lambda: S.KvCache(k8, k8, table, refs, k_scale=sc, v_scale=sc[:1])]:
        with pytest.raises(S.SamplerError):
            bad()


def test_append_workgroups(lib):
    """A workgroup for four tokens of a sequence and layer: 2^32 of them are too many."""
    c = cache(layers=4096, pages=1, kv_heads=1, head_stride=0, page_stride=0, layer_stride=16 * 64)
    for n, rows, layers, rc in [(1024, 1 << 20, 15, 0), (1024, 1 << 20, 16, -4), (1024, 4097, 4096, -4), (1023, 4096, 4096, 0), (1024, 4092, 4096, 0),
                                (1024, 1 << 20, 4096, -4), (1, 1 << 20, 4096, 0)]:
        assert call(lib.append, c, append(n_seq=n, rows_per_seq=rows, n_layers=layers))[0] == rc, (n, rows, layers)

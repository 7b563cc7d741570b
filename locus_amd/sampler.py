"""Python binding of the C ABI in include/locus_sampler.h (ctypes).

The product path is liblocus_sampler.so (HIP kernels for gfx950); this module
only marshals device pointers. PyTorch supplies device memory and the HIP
stream. There is no CPU fallback: a missing library or device raises.
"""
from __future__ import annotations

import ctypes as C
import os

import numpy as np

from .workloads import PARAMS_DTYPE

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "liblocus_sampler.so")

LCS_OK, LCS_ERR_INVALID_ARG, LCS_ERR_NO_DEVICE, LCS_ERR_HIP, LCS_ERR_CAPACITY = 0, -1, -2, -3, -4
LCS_F32, LCS_BF16, LCS_E4M3 = 0, 1, 2
LCS_WANT_LOGPROBS, LCS_WRITE_PENALIZED = 1, 2
PATH_GREEDY, PATH_WINDOW, PATH_WINDOW_EXACT, PATH_GENERAL = 1, 2, 3, 4

DIAG_DTYPE = np.dtype([
    ("n_cand", "<u4"), ("keep", "<u4"), ("maxl", "<f4"), ("boundary", "<f4"),
    ("path", "<u4"), ("reserved", "<u4"), ("sum", "<f8"), ("kept_sum", "<f8"),
])

_P = C.c_void_p


class _Batch(C.Structure):
    _fields_ = [("rows", C.c_uint32), ("vocab", C.c_uint32), ("dtype", C.c_uint32),
                ("flags", C.c_uint32), ("row_stride", C.c_uint64), ("logits", _P),
                ("params", _P), ("params_host", _P), ("hist_off", _P), ("hist_ids", _P),
                ("u", _P), ("mask", _P), ("has_mask", _P), ("mask_words", C.c_uint32),
                ("n_top", C.c_uint32), ("lp_ids", _P), ("win_slot", _P), ("win_push", _P),
                ("win_len", _P), ("raw_stats", _P)]


class _Out(C.Structure):
    _fields_ = [("ids", _P), ("chosen_lp", _P), ("top_ids", _P), ("top_lp", _P), ("diag", _P)]


class _VBatch(C.Structure):
    _fields_ = [("n_seq", C.c_uint32), ("rows_per_seq", C.c_uint32), ("vocab", C.c_uint32),
                ("dtype", C.c_uint32), ("row_stride", C.c_uint64), ("logits", _P), ("draft", _P)]


class _VOut(C.Structure):
    _fields_ = [("argmax_ids", _P), ("draft_lp", _P), ("accept_len", _P)]


class _DBatch(C.Structure):
    _fields_ = [("n_seq", C.c_uint32), ("ngram", C.c_uint32), ("max_draft", C.c_uint32),
                ("ctx_off", _P), ("ctx_ids", _P)]


class _DOut(C.Structure):
    _fields_ = [("draft", _P), ("draft_len", _P)]


class _LBatch(C.Structure):
    _fields_ = [("rows", C.c_uint32), ("vocab", C.c_uint32), ("hidden", C.c_uint32),
                ("rows_per_seq", C.c_uint32), ("x", _P), ("w", _P), ("draft", _P)]


class _LOut(C.Structure):
    _fields_ = [("logits", _P), ("ld_logits", C.c_uint64), ("argmax_ids", _P), ("log_z", _P),
                ("draft_lp", _P), ("accept_len", _P), ("stats", _P)]


class _Adapters(C.Structure):
    _fields_ = [("n", C.c_uint32), ("wide", C.c_uint32), ("a", _P), ("b", _P), ("rank", _P), ("scale", _P)]


class _LExBatch(C.Structure):
    _fields_ = [("rows", C.c_uint32), ("vocab", C.c_uint32), ("hidden", C.c_uint32),
                ("rows_per_seq", C.c_uint32), ("dtype", C.c_uint32), ("x", _P), ("w", _P), ("x_scale", _P),
                ("w_scale", _P), ("draft", _P), ("adapters", C.POINTER(_Adapters)), ("slot", _P)]


class _NBatch(C.Structure):
    _fields_ = [("rows", C.c_uint32), ("hidden", C.c_uint32), ("x_dtype", C.c_uint32), ("y_dtype", C.c_uint32),
                ("eps", C.c_float), ("x", _P), ("residual", _P), ("weight", _P), ("x_stride", C.c_uint64),
                ("residual_stride", C.c_uint64)]


class _NOut(C.Structure):
    _fields_ = [("y", _P), ("y_scale", _P), ("sum", _P), ("y_stride", C.c_uint64), ("sum_stride", C.c_uint64)]


class _KvCache(C.Structure):
    _fields_ = [("layers", C.c_uint32), ("pages", C.c_uint32), ("page_tokens", C.c_uint32), ("kv_heads", C.c_uint32),
                ("head_dim", C.c_uint32), ("dtype", C.c_uint32), ("seqs", C.c_uint32), ("max_pages", C.c_uint32),
                ("k", _P), ("v", _P), ("k_scale", _P), ("v_scale", _P), ("layer_stride", C.c_uint64),
                ("page_stride", C.c_uint64), ("head_stride", C.c_uint64), ("token_stride", C.c_uint64),
                ("table", _P), ("refs", _P)]


class _TreeBatch(C.Structure):
    _fields_ = [("n_seq", C.c_uint32), ("rows_per_seq", C.c_uint32), ("heads", C.c_uint32), ("layer", C.c_uint32),
                ("scale", C.c_float), ("mask_words", C.c_uint32), ("cache", C.POINTER(_KvCache)), ("q", _P), ("k", _P),
                ("v", _P), ("q_stride", C.c_uint64), ("k_stride", C.c_uint64), ("v_stride", C.c_uint64), ("seq", _P),
                ("length", _P), ("mask", _P)]


class _TreeOut(C.Structure):
    _fields_ = [("o", _P), ("o_stride", C.c_uint64), ("lse", _P)]


class _TreeVBatch(C.Structure):
    _fields_ = [("n_seq", C.c_uint32), ("rows_per_seq", C.c_uint32), ("vocab", C.c_uint32), ("dtype", C.c_uint32),
                ("row_stride", C.c_uint64), ("logits", _P), ("tokens", _P), ("parent", _P), ("length", _P)]


class _TreeVOut(C.Structure):
    _fields_ = [("argmax_ids", _P), ("node_lp", _P), ("path", _P), ("n_path", _P), ("next_id", _P), ("length", _P)]


class _AppendBatch(C.Structure):
    _fields_ = [("n_seq", C.c_uint32), ("rows_per_seq", C.c_uint32), ("layer", C.c_uint32), ("n_layers", C.c_uint32),
                ("k", _P), ("v", _P), ("layer_stride", C.c_uint64), ("k_stride", C.c_uint64), ("v_stride", C.c_uint64),
                ("seq", _P), ("pos", _P), ("count", _P), ("index", _P)]


class SamplerError(RuntimeError):
    pass


def _addr(t):
    return None if t is None else t.data_ptr()


class Adapters:
    """A pool of n low-rank adapters for lmhead_ex_dev: `a` (n, wide, hidden)
    and `b` (n, vocab, wide) bf16, contiguous, wide a multiple of 8; `rank`
    (n,) int32 and `scale` (n,) f32, or None (wide, and 1). Device tensors;
    nothing is copied."""

    def __init__(self, a, b, rank=None, scale=None):
        import torch
        if a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16:
            raise SamplerError("adapters: a and b must be bfloat16")
        if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
            raise SamplerError("adapters: a must be (n, wide, hidden) and b (n, vocab, wide)")
        if not (a.is_contiguous() and b.is_contiguous()):
            raise SamplerError("adapters: a and b must be contiguous")
        n, self.wide, self.hidden = a.shape
        self.n, self.vocab, self.device = n, b.shape[1], a.get_device()
        if b.get_device() != self.device:
            raise SamplerError("adapters: tensors on different devices")
        for t, dtype, name in ((rank, torch.int32, "rank"), (scale, torch.float32, "scale")):
            if t is not None and (t.dtype != dtype or t.dim() != 1 or t.numel() != n or not t.is_contiguous() or
                                  t.get_device() != self.device):
                raise SamplerError(f"adapters: {name} must be ({n},) {dtype}, contiguous, on the adapters' device")
        self._keep = (a, b, rank, scale)
        self._c = _Adapters(n, self.wide, a.data_ptr(), b.data_ptr(), _addr(rank), _addr(scale))


class KvCache:
    """A paged cache for kv_*_dev and tree_attn_dev: `k` and `v` (layers, pages,
    kv_heads, page_tokens, head_dim), bf16 or float8_e4m3fn, of the same strides (any,
    with a head's elements together); `table` (seqs, max_pages) int32, -1 where a slot
    has no page; `refs` (pages,) int32; for 8 bits `k_scale` and `v_scale` (layers,
    pages, kv_heads, page_tokens) f32. Device tensors; nothing is copied."""

    def __init__(self, k, v, table, refs, k_scale=None, v_scale=None):
        import torch
        types = {torch.bfloat16: LCS_BF16, torch.float8_e4m3fn: LCS_E4M3}
        if k.dtype not in types or v.dtype != k.dtype:
            raise SamplerError("cache: k and v must both be bfloat16 or both float8_e4m3fn")
        if k.dim() != 5 or v.shape != k.shape:
            raise SamplerError("cache: k and v must be (layers, pages, kv_heads, page_tokens, head_dim)")
        ks, vs = k.stride(), v.stride()
        if ks[4] != 1 or any(a != b and n > 1 for a, b, n in zip(ks, vs, k.shape)):
            raise SamplerError("cache: k and v must have the same strides, a head's elements together")
        layers, pages, heads, tokens, dim = k.shape
        self.device, self.shape = k.get_device(), tuple(k.shape)
        if table.dim() != 2 or table.dtype != torch.int32 or not table.is_contiguous():
            raise SamplerError("cache: table must be (seqs, max_pages) int32, contiguous")
        if refs.dim() != 1 or refs.dtype != torch.int32 or refs.numel() != pages or not refs.is_contiguous():
            raise SamplerError(f"cache: refs must be ({pages},) int32, contiguous")
        for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            if (t is not None) != (k.dtype == torch.float8_e4m3fn):
                raise SamplerError(f"cache: {name} goes with float8_e4m3fn")
            if t is not None and (t.dtype != torch.float32 or t.shape != k.shape[:4] or not t.is_contiguous()):
                raise SamplerError(f"cache: {name} must be (layers, pages, kv_heads, page_tokens) f32, contiguous")
        if any(t is not None and t.get_device() != self.device for t in (v, table, refs, k_scale, v_scale)):
            raise SamplerError("cache: tensors on different devices")
        self._keep = (k, v, table, refs, k_scale, v_scale)
        self._c = _KvCache(layers, pages, tokens, heads, dim, types[k.dtype], table.shape[0], table.shape[1], k.data_ptr(),
                           v.data_ptr(), _addr(k_scale), _addr(v_scale), ks[0], ks[1], ks[2], ks[3], table.data_ptr(),
                           refs.data_ptr())
        self._p = C.pointer(self._c)


_lib = None


def lib():
    """Loads liblocus_sampler.so; raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise SamplerError(f"{LIB_PATH} is missing: run __graft_entry__.build()")
        L = C.CDLL(LIB_PATH)
        L.lcs_probe.restype = C.c_int
        L.lcs_probe.argtypes = [C.POINTER(C.c_int)]
        L.lcs_create.restype = _P
        L.lcs_create.argtypes = [C.c_int, C.c_uint32, C.c_uint32, C.c_uint32, C.c_uint32]
        L.lcs_destroy.restype = None
        L.lcs_destroy.argtypes = [_P]
        L.lcs_sample.restype = C.c_int
        L.lcs_sample.argtypes = [_P, C.POINTER(_Batch), C.POINTER(_Out), _P]
        L.lcs_sample_noalloc.restype = C.c_int
        L.lcs_sample_noalloc.argtypes = [C.POINTER(_Batch), C.POINTER(_Out), _P]
        L.lcs_verify.restype = C.c_int
        L.lcs_verify.argtypes = [_P, C.POINTER(_VBatch), C.POINTER(_VOut), _P]
        L.lcs_ngram_draft.restype = C.c_int
        L.lcs_ngram_draft.argtypes = [_P, C.POINTER(_DBatch), C.POINTER(_DOut), _P]
        L.lcs_lmhead.restype = C.c_int
        L.lcs_lmhead.argtypes = [_P, C.POINTER(_LBatch), C.POINTER(_LOut), _P]
        L.lcs_lmhead_ex.restype = C.c_int
        L.lcs_lmhead_ex.argtypes = [_P, C.POINTER(_LExBatch), C.POINTER(_LOut), _P]
        L.lcs_add_rmsnorm.restype = C.c_int
        L.lcs_add_rmsnorm.argtypes = [_P, C.POINTER(_NBatch), C.POINTER(_NOut), _P]
        cache, i32 = C.POINTER(_KvCache), C.c_uint32
        L.lcs_kv_reserve.restype = C.c_int
        L.lcs_kv_reserve.argtypes = [_P, i32]
        for name in ("lcs_kv_grow", "lcs_kv_fork"):
            getattr(L, name).restype = C.c_int
            getattr(L, name).argtypes = [_P, cache, i32, _P, _P, _P, _P, _P]
        L.lcs_kv_free.restype = C.c_int
        L.lcs_kv_free.argtypes = [_P, cache, i32, _P, _P, _P, _P]
        L.lcs_kv_compact.restype = C.c_int
        L.lcs_kv_compact.argtypes = [_P, cache, i32, i32, _P, _P, _P, _P, _P]
        L.lcs_kv_append.restype = C.c_int
        L.lcs_kv_append.argtypes = [_P, cache, C.POINTER(_AppendBatch), _P]
        L.lcs_tree_attn.restype = C.c_int
        L.lcs_tree_attn.argtypes = [_P, C.POINTER(_TreeBatch), C.POINTER(_TreeOut), _P]
        L.lcs_tree_verify.restype = C.c_int
        L.lcs_tree_verify.argtypes = [_P, C.POINTER(_TreeVBatch), C.POINTER(_TreeVOut), _P]
        L.lcs_last_error.restype = C.c_char_p
        L.lcs_last_error.argtypes = [_P]
        L.lcs_logprobs.restype = C.c_int
        L.lcs_logprobs.argtypes = [_P, C.POINTER(_Batch), _P, C.POINTER(_Out), _P]
        L.lcs_windows_reserve.restype = C.c_int
        L.lcs_windows_reserve.argtypes = [_P, C.c_uint32, C.c_uint32]
        L.lcs_windows_load.restype = C.c_int
        L.lcs_windows_load.argtypes = [_P, C.c_uint32, _P, C.c_uint32, C.c_uint32, C.c_uint32, _P]
        L.lcs_get_status.restype = C.c_int
        L.lcs_get_status.argtypes = [_P, C.POINTER(C.c_uint32), C.c_int]
        _lib = L
    return _lib


def probe() -> int:
    n = C.c_int(0)
    lib().lcs_probe(C.byref(n))
    return n.value


def _dptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _stream_handle(torch, stream):
    s = stream if stream is not None else torch.cuda.current_stream()
    return C.c_void_p(s.cuda_stream)


class Sampler:
    """One lcs_ctx on one device; workspace is allocated here, once."""

    def __init__(self, device: int = 0, max_rows: int = 256, max_vocab: int = 262144,
                 max_hist: int = 4096, max_top: int = 20):
        import torch  # plumbing: device memory and streams
        self.torch = torch
        self.device = device
        self._types = {torch.float32: LCS_F32, torch.bfloat16: LCS_BF16, torch.float8_e4m3fn: LCS_E4M3}
        self._bf16, self._i32, self._f32 = torch.bfloat16, torch.int32, torch.float32
        self._current = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        L = lib()
        self.ctx = L.lcs_create(device, max_rows, max_vocab, max_hist, max_top)
        if not self.ctx:
            raise SamplerError(L.lcs_last_error(None).decode())
        self.max_rows, self.max_vocab, self.max_top = max_rows, max_vocab, max_top

    def close(self):
        if getattr(self, "ctx", None):
            lib().lcs_destroy(self.ctx)
            self.ctx = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, rc: int):
        if rc != LCS_OK:
            raise SamplerError(f"lcs error {rc}: {lib().lcs_last_error(self.ctx).decode()}")

    def status(self, reset: bool = True) -> int:
        s = C.c_uint32(0)
        self._check(lib().lcs_get_status(self.ctx, C.byref(s), int(reset)))
        return s.value

    # ------------------------------------------------- device-resident windows
    def windows_reserve(self, slots: int, max_window: int):
        self._check(lib().lcs_windows_reserve(self.ctx, slots, max_window))

    def windows_load(self, slot: int, ids, window: int, vocab: int, stream=None):
        """Starts `slot` from a history (a device int32 tensor, or None for an
        empty one)."""
        n = 0 if ids is None else int(ids.numel())
        self._check(lib().lcs_windows_load(self.ctx, slot, _dptr(ids) if n else None, n, window, vocab,
                                           _stream_handle(self.torch, stream)))

    # ---------------------------------------------------------------- inputs
    def upload(self, w, stride: int | None = None):
        """Device copies of a workloads.Workload (sampling configs)."""
        torch = self.torch
        dev = torch.device("cuda", self.device)
        V = w.vocab
        G = 8 if w.dtype == "bf16" else 4
        stride = stride or ((V + G - 1) // G * G)
        if w.dtype == "bf16":
            host = np.zeros((w.rows, stride), dtype=np.uint16)
            host[:, :V] = w.logits
            logits = torch.from_numpy(host.view(np.int16)).to(dev).view(torch.bfloat16)
        else:
            host = np.zeros((w.rows, stride), dtype=np.float32)
            host[:, :V] = w.logits
            logits = torch.from_numpy(host).to(dev)
        d = {"logits": logits, "stride": stride, "w": w}
        if w.params is not None:
            d["params"] = torch.from_numpy(np.ascontiguousarray(w.params).view(np.uint8).copy()).to(dev)
            d["params_host"] = np.ascontiguousarray(w.params)
        if w.u is not None:
            d["u"] = torch.from_numpy(np.ascontiguousarray(w.u, dtype=np.float64)).to(dev)
        if w.hist_off is not None:
            d["hist_off"] = torch.from_numpy(w.hist_off.astype(np.int32).view(np.int32)).to(dev)
            ids = np.ascontiguousarray(w.hist_ids, dtype=np.int32)
            if ids.size == 0:  # an empty tensor has no data pointer
                ids = np.zeros(1, dtype=np.int32)
            d["hist_ids"] = torch.from_numpy(ids).to(dev)
        if w.mask is not None:
            d["mask"] = torch.from_numpy(np.ascontiguousarray(w.mask).view(np.int32)).to(dev)
        if w.draft is not None:
            d["draft"] = torch.from_numpy(np.ascontiguousarray(w.draft, dtype=np.int32)).to(dev)
        return d

    def alloc_out(self, rows: int, n_top: int, want_lp: bool, diag: bool = True):
        torch = self.torch
        dev = torch.device("cuda", self.device)
        o = {"ids": torch.full((rows,), -7, dtype=torch.int32, device=dev)}
        if want_lp:
            o["chosen_lp"] = torch.zeros(rows, dtype=torch.float32, device=dev)
            o["top_ids"] = torch.zeros((rows, max(n_top, 1)), dtype=torch.int32, device=dev)
            o["top_lp"] = torch.zeros((rows, max(n_top, 1)), dtype=torch.float32, device=dev)
        if diag:
            o["diag"] = torch.zeros(rows * DIAG_DTYPE.itemsize, dtype=torch.uint8, device=dev)
        return o

    # ---------------------------------------------------------------- calls
    def prepare(self, d, out, n_top: int | None = None, want_lp: bool | None = None,
                has_mask=None, flags_extra: int = 0, use_host_params: bool = True, win=None, raw_stats=None):
        """Builds the C structs of one lcs_sample call once; returns a
        zero-argument launcher (for tight benchmark loops)."""
        w = d["w"]
        want_lp = w.want_logprobs if want_lp is None else want_lp
        n_top = w.n_top if n_top is None else n_top
        b = _Batch()
        b.rows, b.vocab = w.rows, w.vocab
        b.dtype = LCS_BF16 if w.dtype == "bf16" else LCS_F32
        b.flags = (LCS_WANT_LOGPROBS if want_lp else 0) | flags_extra
        b.row_stride = d["stride"]
        b.logits = _dptr(d["logits"])
        b.params = _dptr(d["params"])
        ph = d["params_host"] if use_host_params else None
        b.params_host = None if ph is None else ph.ctypes.data_as(C.c_void_p)
        b.hist_off = _dptr(d.get("hist_off"))
        b.hist_ids = _dptr(d.get("hist_ids"))
        b.u = _dptr(d.get("u"))
        b.mask = _dptr(d.get("mask"))
        b.has_mask = _dptr(has_mask)
        b.mask_words = w.mask_words
        b.n_top = n_top if want_lp else 0
        if win is not None:
            b.win_slot, b.win_push, b.win_len = _dptr(win["slot"]), _dptr(win["push"]), _dptr(win["len"])
            b.hist_off = b.hist_ids = None
        b.raw_stats = _dptr(raw_stats)
        o = _Out()
        o.ids = _dptr(out["ids"])
        o.chosen_lp = _dptr(out.get("chosen_lp"))
        o.top_ids = _dptr(out.get("top_ids"))
        o.top_lp = _dptr(out.get("top_lp"))
        o.diag = _dptr(out.get("diag"))
        fn, ctx, bp, op = lib().lcs_sample, self.ctx, C.byref(b), C.byref(o)
        keep = (ph, b, o, d, out, win, raw_stats)

        def launch(stream_handle):
            _ = keep
            rc = fn(ctx, bp, op, stream_handle)
            if rc != LCS_OK:
                self._check(rc)
        return launch

    def prepare_verify(self, d, out):
        w = d["w"]
        b = _VBatch()
        b.n_seq, b.rows_per_seq, b.vocab = w.n_seq, w.rows_per_seq, w.vocab
        b.dtype = LCS_BF16 if w.dtype == "bf16" else LCS_F32
        b.row_stride = d["stride"]
        b.logits = _dptr(d["logits"])
        b.draft = _dptr(d["draft"])
        o = _VOut()
        o.argmax_ids = _dptr(out["argmax_ids"])
        o.draft_lp = _dptr(out["draft_lp"])
        o.accept_len = _dptr(out["accept_len"])
        fn, ctx, bp, op = lib().lcs_verify, self.ctx, C.byref(b), C.byref(o)
        keep = (b, o, d, out)

        def launch(stream_handle):
            _ = keep
            rc = fn(ctx, bp, op, stream_handle)
            if rc != LCS_OK:
                self._check(rc)
        return launch

    def stream_handle(self, stream=None):
        return _stream_handle(self.torch, stream)

    def sample_dev(self, d, out, n_top: int | None = None, want_lp: bool | None = None,
                   has_mask=None, flags_extra: int = 0, use_host_params: bool = True, stream=None,
                   lp_ids=None, noalloc: bool = False, win=None, raw_stats=None):
        """Enqueues lcs_sample on device buffers from upload()/alloc_out();
        `lp_ids` (device int32 per row) makes chosen_lp report those ids;
        `noalloc` calls lcs_sample_noalloc (no context) instead; `win`
        ({"slot", "push", "len"}: device int32 / int32 / uint32 per row) takes
        the rows' penalty windows from device-resident slots instead of the
        workload's history; `raw_stats` (the "stats" output of lmhead_dev on
        the same logits) gives the rows' raw log-normalisers."""
        w = d["w"]
        want_lp = w.want_logprobs if want_lp is None else want_lp
        n_top = w.n_top if n_top is None else n_top
        b = _Batch()
        b.rows, b.vocab = w.rows, w.vocab
        b.dtype = LCS_BF16 if w.dtype == "bf16" else LCS_F32
        b.flags = (LCS_WANT_LOGPROBS if want_lp else 0) | flags_extra
        b.row_stride = d["stride"]
        b.logits = _dptr(d["logits"])
        b.params = _dptr(d["params"])
        ph = d["params_host"] if use_host_params else None
        b.params_host = None if ph is None else ph.ctypes.data_as(C.c_void_p)
        b.hist_off = _dptr(d.get("hist_off"))
        b.hist_ids = _dptr(d.get("hist_ids"))
        b.u = _dptr(d.get("u"))
        b.mask = _dptr(d.get("mask"))
        b.has_mask = _dptr(has_mask)
        b.mask_words = w.mask_words
        b.n_top = n_top if want_lp else 0
        b.lp_ids = _dptr(lp_ids)
        if win is not None:
            b.win_slot, b.win_push, b.win_len = _dptr(win["slot"]), _dptr(win["push"]), _dptr(win["len"])
            b.hist_off = b.hist_ids = None
        b.raw_stats = _dptr(raw_stats)
        o = _Out()
        o.ids = _dptr(out["ids"])
        o.chosen_lp = _dptr(out.get("chosen_lp"))
        o.top_ids = _dptr(out.get("top_ids"))
        o.top_lp = _dptr(out.get("top_lp"))
        o.diag = _dptr(out.get("diag"))
        self._keep = (ph, b, o, lp_ids, win, raw_stats)
        sh = _stream_handle(self.torch, stream)
        if noalloc:
            rc = lib().lcs_sample_noalloc(C.byref(b), C.byref(o), sh)
            if rc != LCS_OK:
                raise SamplerError(f"lcs error {rc}: {lib().lcs_last_error(None).decode()}")
            return
        self._check(lib().lcs_sample(self.ctx, C.byref(b), C.byref(o), sh))

    def sample(self, w, **kw):
        """Uploads a Workload, samples it, and returns host numpy results."""
        d = self.upload(w)
        out = self.alloc_out(w.rows, w.n_top, w.want_logprobs)
        self.sample_dev(d, out, **kw)
        self.torch.cuda.synchronize()
        return self.fetch(out, w.n_top)

    def logprobs_dev(self, d, out, chosen=None, n_top: int | None = None, raw_stats=None, stream=None):
        """Enqueues lcs_logprobs (logprobs_from over the batch, no draw) on
        device buffers from upload()/alloc_out(): `chosen` (device int32 per
        row, or None for each row's argmax)."""
        w = d["w"]
        b = _Batch()
        b.rows, b.vocab = w.rows, w.vocab
        b.dtype = LCS_BF16 if w.dtype == "bf16" else LCS_F32
        b.row_stride = d["stride"]
        b.logits = _dptr(d["logits"])
        b.n_top = w.n_top if n_top is None else n_top
        b.raw_stats = _dptr(raw_stats)
        o = _Out()
        o.ids = _dptr(out.get("ids"))
        o.chosen_lp = _dptr(out.get("chosen_lp"))
        o.top_ids = _dptr(out.get("top_ids"))
        o.top_lp = _dptr(out.get("top_lp"))
        self._keep = (b, o, chosen, raw_stats)
        self._check(lib().lcs_logprobs(self.ctx, C.byref(b), _dptr(chosen), C.byref(o),
                                       _stream_handle(self.torch, stream)))

    @staticmethod
    def fetch(out, n_top: int):
        r = {"ids": out["ids"].cpu().numpy()}
        if "chosen_lp" in out:
            r["chosen_lp"] = out["chosen_lp"].cpu().numpy()
            r["top_ids"] = out["top_ids"].cpu().numpy()[:, :n_top]
            r["top_lp"] = out["top_lp"].cpu().numpy()[:, :n_top]
        if "diag" in out:
            r["diag"] = out["diag"].cpu().numpy().view(DIAG_DTYPE)
        return r

    def verify_dev(self, d, out, stream=None):
        w = d["w"]
        b = _VBatch()
        b.n_seq, b.rows_per_seq, b.vocab = w.n_seq, w.rows_per_seq, w.vocab
        b.dtype = LCS_BF16 if w.dtype == "bf16" else LCS_F32
        b.row_stride = d["stride"]
        b.logits = _dptr(d["logits"])
        b.draft = _dptr(d["draft"])
        o = _VOut()
        o.argmax_ids = _dptr(out["argmax_ids"])
        o.draft_lp = _dptr(out["draft_lp"])
        o.accept_len = _dptr(out["accept_len"])
        self._keep = (b, o)
        self._check(lib().lcs_verify(self.ctx, C.byref(b), C.byref(o),
                                     _stream_handle(self.torch, stream)))

    def alloc_verify_out(self, w):
        torch = self.torch
        dev = torch.device("cuda", self.device)
        return {"argmax_ids": torch.full((w.rows,), -7, dtype=torch.int32, device=dev),
                "draft_lp": torch.zeros(w.rows, dtype=torch.float32, device=dev),
                "accept_len": torch.full((w.n_seq,), 99, dtype=torch.int32, device=dev)}

    def ngram_draft(self, contexts, ngram: int, max_draft: int):
        """Batched prompt-lookup drafts (lcs_ngram_draft) for a list of token
        sequences; returns (drafts: list of lists, raw (n_seq, max_draft) array)."""
        torch = self.torch
        dev = torch.device("cuda", self.device)
        n = len(contexts)
        off = np.zeros(n + 1, dtype=np.uint32)
        off[1:] = np.cumsum([len(c) for c in contexts])
        ids = np.concatenate([np.asarray(c, dtype=np.int32) for c in contexts]) if off[-1] else np.zeros(1, np.int32)
        off_d = torch.from_numpy(off.view(np.int32)).to(dev)
        ids_d = torch.from_numpy(ids).to(dev)
        dr = torch.full((n, max(max_draft, 1)), -7, dtype=torch.int32, device=dev)
        ln = torch.full((n,), 999, dtype=torch.int32, device=dev)
        b = _DBatch()
        b.n_seq, b.ngram, b.max_draft = n, ngram, max_draft
        b.ctx_off, b.ctx_ids = _dptr(off_d), _dptr(ids_d)
        o = _DOut()
        o.draft, o.draft_len = _dptr(dr), _dptr(ln)
        self._check(lib().lcs_ngram_draft(self.ctx, C.byref(b), C.byref(o), None))
        torch.cuda.synchronize()
        raw = dr.cpu().numpy()[:, :max_draft]
        lens = ln.cpu().numpy()
        return [raw[i, :lens[i]].tolist() for i in range(n)], raw

    def lmhead_dev(self, x, w, out, draft=None, rows_per_seq: int = 0, stream=None):
        """The fused lm-head product (lcs_lmhead) on device tensors: x (rows,
        hidden) and w (vocab, hidden) bf16, contiguous; `out` holds any of
        "logits" (rows, >= vocab) f32, "argmax_ids", "log_z", "draft_lp",
        "accept_len", "stats" (rows x 16 bytes, lcs_row_stats: pass it as
        sample_dev's raw_stats) (missing keys are not written; argmax_ids is
        required)."""
        torch = self.torch
        if x.dtype != torch.bfloat16 or w.dtype != torch.bfloat16:
            raise SamplerError("x and w must be bfloat16")
        if not (x.is_contiguous() and w.is_contiguous()):
            raise SamplerError("x and w must be contiguous")
        b = _LBatch()
        b.rows, b.hidden = x.shape
        b.vocab = w.shape[0]
        if w.shape[1] != b.hidden:
            raise SamplerError("x and w disagree on hidden")
        b.rows_per_seq = rows_per_seq
        b.x, b.w, b.draft = _dptr(x), _dptr(w), _dptr(draft)
        o = _LOut()
        lg = out.get("logits")
        if lg is not None:
            if lg.dtype != torch.float32 or lg.stride(1) != 1:
                raise SamplerError("logits must be f32 with unit column stride")
            o.logits, o.ld_logits = _dptr(lg), lg.stride(0)
        for k in ("argmax_ids", "log_z", "draft_lp", "accept_len", "stats"):
            setattr(o, k, _dptr(out.get(k)))
        self._keep = (b, o)
        self._check(lib().lcs_lmhead(self.ctx, C.byref(b), C.byref(o),
                                     _stream_handle(torch, stream)))

    def alloc_lmhead_out(self, rows: int, vocab: int, logits: bool = True, draft: bool = False,
                         n_seq: int = 0, stats: bool = False):
        torch = self.torch
        dev = torch.device("cuda", self.device)
        out = {"argmax_ids": torch.full((rows,), -7, dtype=torch.int32, device=dev),
               "log_z": torch.full((rows,), -7.0, dtype=torch.float32, device=dev)}
        if logits:
            out["logits"] = torch.full((rows, vocab), -7.0, dtype=torch.float32, device=dev)
        if draft:
            out["draft_lp"] = torch.full((rows,), -7.0, dtype=torch.float32, device=dev)
        if n_seq:
            out["accept_len"] = torch.full((n_seq,), 99, dtype=torch.int32, device=dev)
        if stats:   # lcs_row_stats: (f64 log_z, f32 max, i32 argmax) per row
            out["stats"] = torch.full((rows, 2), -7.0, dtype=torch.float64, device=dev)
        return out

    # (a serving step makes these calls once a token: their checks read each
    # tensor's attributes once, and messages are put together where one is raised)
    def _vec(self, t, n: int, dtype, name: str):
        """The address of an optional (n,) device vector."""
        if t is None:
            return None
        if t.dtype != dtype or t.dim() != 1 or t.numel() != n or not t.is_contiguous() or t.get_device() != self.device:
            raise SamplerError(f"{name} must be ({n},) {dtype}, contiguous, on the sampler's device")
        return t.data_ptr()

    def _raw_stream(self, stream):
        if stream is not None:
            return stream.cuda_stream
        if self._current is not None:   # the handle alone, without a Stream object (1.2 us a call)
            return self._current(self.device)
        return self.torch.cuda.current_stream(self.device).cuda_stream

    def lmhead_ex_dev(self, x, w, out, x_scale=None, w_scale=None, adapters: Adapters | None = None, slot=None,
                      draft=None, rows_per_seq: int = 0, stream=None):
        """The fused lm-head product in bf16 or 8 bits, with the rows' adapters
        (lcs_lmhead_ex): x (rows, hidden) and w (vocab, hidden), contiguous,
        both bf16 or both float8_e4m3fn (then `x_scale` (rows,) and `w_scale`
        (vocab,) f32, or None for 1); `adapters` with `slot` (rows,) int32, the
        row's adapter or -1. `out` as for lmhead_dev."""
        torch = self.torch
        dtype = self._types.get(x.dtype)
        if dtype not in (LCS_BF16, LCS_E4M3) or w.dtype != x.dtype:
            raise SamplerError("x and w must both be bfloat16 or both float8_e4m3fn")
        if x.dim() != 2 or w.dim() != 2 or not (x.is_contiguous() and w.is_contiguous()):
            raise SamplerError("x and w must be 2-d and contiguous")
        if x.get_device() != self.device or w.get_device() != self.device:
            raise SamplerError("x and w must be on the sampler's device")
        (rows, hidden), (vocab, wh) = x.shape, w.shape
        if wh != hidden:
            raise SamplerError("x and w disagree on hidden")
        ad = None
        if adapters is not None:
            if adapters.hidden != hidden or adapters.vocab != vocab or adapters.device != self.device:
                raise SamplerError("the adapters' hidden, vocab or device are not those of x and w")
            if slot is None:
                raise SamplerError("adapters need slot")
            ad = C.pointer(adapters._c)
        i32, f32, vec = torch.int32, torch.float32, self._vec
        b = _LExBatch(rows, vocab, hidden, rows_per_seq, dtype, x.data_ptr(), w.data_ptr(),
                      vec(x_scale, rows, f32, "x_scale"), vec(w_scale, vocab, f32, "w_scale"),
                      vec(draft, rows, i32, "draft"), ad, vec(slot, rows, i32, "slot"))
        lg, lp, ld = out.get("logits"), None, 0
        if lg is not None:
            if (lg.dtype != f32 or lg.dim() != 2 or lg.shape[0] != rows or lg.shape[1] < vocab or
                    (lg.stride(1) != 1 and vocab > 1) or lg.get_device() != self.device):
                raise SamplerError("logits must be (rows, >= vocab) f32 with unit column stride, on the sampler's device")
            lp, ld = lg.data_ptr(), lg.stride(0) if rows > 1 else vocab
        acc, st = out.get("accept_len"), out.get("stats")
        if acc is not None and rows_per_seq > 0:
            acc = vec(acc, rows // rows_per_seq, i32, "accept_len")
        elif acc is not None:
            raise SamplerError("accept_len needs rows_per_seq")
        if st is not None:
            if not st.is_contiguous() or st.numel() * st.element_size() < 16 * rows or st.get_device() != self.device:
                raise SamplerError("stats must hold 16 contiguous bytes a row, on the sampler's device")
            st = st.data_ptr()
        o = _LOut(lp, ld, vec(out.get("argmax_ids"), rows, i32, "argmax_ids"), vec(out.get("log_z"), rows, f32, "log_z"),
                  vec(out.get("draft_lp"), rows, f32, "draft_lp"), acc, st)
        rc = _lib.lcs_lmhead_ex(self.ctx, b, o, self._raw_stream(stream))
        if rc != LCS_OK:
            self._check(rc)

    def add_rmsnorm_dev(self, x, weight, out, residual=None, eps: float = 1e-6, stream=None):
        """Residual addition and root-mean-square norm (lcs_add_rmsnorm): x and
        `residual` (rows, hidden), bf16 or f32, any row stride; `weight`
        (hidden,) of their type. `out` holds "y" (rows, hidden) in bf16, f32 or
        float8_e4m3fn (then "y_scale" (rows,) f32 too) and, with a residual,
        optionally "sum" of x's type; missing keys are not written (y is
        required)."""
        y, total, dtype, dev = out["y"], out.get("sum"), x.dtype, self.device
        ytype = y.dtype
        xt, yt = self._types.get(dtype), self._types.get(ytype)
        if xt not in (LCS_F32, LCS_BF16):
            raise SamplerError("x must be float32 or bfloat16")
        if yt is None:
            raise SamplerError("y must be float32, bfloat16 or float8_e4m3fn")
        shape = x.shape
        if len(shape) != 2:
            raise SamplerError("x must be (rows, hidden)")
        rows, hidden = shape
        at = []   # address and row stride of each
        for t, want in ((x, dtype), (residual, dtype), (y, ytype), (total, dtype)):
            if t is None:
                at += (None, 0)
                continue
            if t.dtype != want or t.shape != shape or t.get_device() != dev:
                name = "x" if t is x else "residual" if t is residual else "y" if t is y else "sum"
                raise SamplerError(f"{name} must be ({rows}, {hidden}) {want} on the sampler's device")
            per, one = t.stride()
            if one != 1 and hidden > 1:
                raise SamplerError("rows must have unit column stride")
            at += (t.data_ptr(), per if rows > 1 else hidden)
        xp, xs, rp, rs, yp, ys, sp, ss = at
        b = _NBatch(rows, hidden, xt, yt, eps, xp, rp, self._vec(weight, hidden, dtype, "weight"), xs, rs)
        o = _NOut(yp, self._vec(out.get("y_scale"), rows, self.torch.float32, "y_scale"), sp, ys, ss)
        rc = _lib.lcs_add_rmsnorm(self.ctx, b, o, self._raw_stream(stream))
        if rc != LCS_OK:
            self._check(rc)

    # ------------------------------------------- a paged cache and trees of drafts
    def kv_reserve(self, new_pages: int):
        """The workspace of the calls below (lcs_kv_reserve), once, ahead of the loop:
        new_pages bounds what one kv_grow_dev call may allocate."""
        self._check(lib().lcs_kv_reserve(self.ctx, new_pages))

    def _cache(self, cache):
        if not isinstance(cache, KvCache) or cache.device != self.device:
            raise SamplerError("cache must be a KvCache on the sampler's device")
        return cache._c

    def _requests(self, *named):
        """The number of requests and the addresses of their (n,) int32 vectors."""
        n, i32, vec = named[0][0].numel(), self._i32, self._vec
        return n, *[vec(t, n, i32, name) for t, name in named]

    def kv_grow_dev(self, cache, seq, start, end, result, stream=None):
        """Pages of their own for slots seq[i] at tokens [start[i], end[i])
        (lcs_kv_grow): missing ones allocated, shared ones replaced by copies.
        All (n,) int32; result[i] is 0, or -1 where a request was refused: from the
        first that there are not enough pages for on, every one."""
        n, q, s, e, r = self._requests((seq, "seq"), (start, "start"), (end, "end"), (result, "result"))
        rc = _lib.lcs_kv_grow(self.ctx, self._cache(cache), n, q, s, e, r, self._raw_stream(stream))
        if rc != LCS_OK:
            self._check(rc)

    def kv_fork_dev(self, cache, src, dst, tokens, result, stream=None):
        """Slots dst[i], which hold nothing, share the first tokens[i] tokens of
        slots src[i] (lcs_kv_fork). All (n,) int32; result as kv_grow_dev."""
        n, s, d, t, r = self._requests((src, "src"), (dst, "dst"), (tokens, "tokens"), (result, "result"))
        rc = _lib.lcs_kv_fork(self.ctx, self._cache(cache), n, s, d, t, r, self._raw_stream(stream))
        if rc != LCS_OK:
            self._check(rc)

    def kv_free_dev(self, cache, seq, keep, result, stream=None):
        """Slots seq[i] give up their pages past their first keep[i] tokens (keep
        None: all) (lcs_kv_free). All (n,) int32; result as kv_grow_dev."""
        n, s, k, r = self._requests((seq, "seq"), (keep, "keep"), (result, "result"))
        rc = _lib.lcs_kv_free(self.ctx, self._cache(cache), n, s, k, r, self._raw_stream(stream))
        if rc != LCS_OK:
            self._check(rc)

    def kv_compact_dev(self, cache, seq, count, keep, result, stream=None):
        """Slots seq[i] keep the count[i] tokens that keep[i] names, ascending, moved
        to their front in all layers (lcs_kv_compact). seq, count, result (n,)
        and keep (n, max_keep) int32, contiguous; result as kv_grow_dev."""
        n, s, c, r = self._requests((seq, "seq"), (count, "count"), (result, "result"))
        if (keep.dtype != self.torch.int32 or keep.dim() != 2 or keep.shape[0] != n or not keep.is_contiguous() or
                keep.get_device() != self.device):
            raise SamplerError(f"keep must be ({n}, max_keep) int32, contiguous, on the sampler's device")
        rc = _lib.lcs_kv_compact(self.ctx, self._cache(cache), n, keep.shape[1], s, c, keep.data_ptr(), r,
                                 self._raw_stream(stream))
        if rc != LCS_OK:
            self._check(rc)

    def _heads(self, t, shape, name: str):
        """Address and row stride of bf16 rows (..., rows, heads, dim), a row's heads together."""
        if t.dtype != self._bf16 or t.shape != shape or t.get_device() != self.device:
            raise SamplerError(f"{name} must be {shape} bfloat16 on the sampler's device")
        at = t.stride()
        heads, dim = shape[-2], shape[-1]
        if (at[-1] != 1 and dim > 1) or (at[-2] != dim and heads > 1):
            raise SamplerError(f"{name}: a row's heads must be contiguous")
        return t.data_ptr(), at[-3] if shape[-3] > 1 else heads * dim

    def kv_append_dev(self, cache, k, v, seq, pos, count=None, rows_per_seq: int = 1, index=None, layer: int = 0,
                      stream=None):
        """New rows of a cache (lcs_kv_append): token j < count[i] (None:
        rows_per_seq) of slot seq[i] to position pos[i] + j, from row index[i, j]
        (None: j) of sequence i's rows_per_seq ones. k and v (layers, n *
        rows_per_seq, kv_heads, head_dim) bf16 for the layers from `layer` on, or of
        one layer without the first dimension."""
        c, i32, vec = self._cache(cache), self._i32, self._vec
        n = seq.numel()
        rows = n * rows_per_seq
        shape, layers, apart = (rows, cache.shape[2], cache.shape[4]), 1, 0
        if k.dim() == 4:
            layers, apart = k.shape[0], k.stride(0)
            if layers == 0:
                raise SamplerError("k and v must have a layer at least")
            shape = (layers, *shape)
            if layers > 1 and (v.dim() != 4 or v.stride(0) != apart):
                raise SamplerError("k and v must have the same layer stride")
        kp, ks = self._heads(k, shape, "k")
        vp, vs = self._heads(v, shape, "v")
        if index is not None and (index.dtype != i32 or index.numel() != rows or not index.is_contiguous() or
                                  index.get_device() != self.device):
            raise SamplerError(f"index must be ({n}, {rows_per_seq}) int32, contiguous, on the sampler's device")
        b = _AppendBatch(n, rows_per_seq, layer, layers, kp, vp, apart, ks, vs, vec(seq, n, i32, "seq"),
                         vec(pos, n, i32, "pos"), vec(count, n, i32, "count"), _addr(index))
        rc = _lib.lcs_kv_append(self.ctx, c, b, self._raw_stream(stream))
        if rc != LCS_OK:
            self._check(rc)

    def tree_attn_dev(self, q, k, v, cache, out, length, seq=None, rows_per_seq: int = 1, mask=None, layer: int = 0,
                      scale: float | None = None, stream=None):
        """Attention of a step's new tokens over their cached context and over each
        other (lcs_tree_attn): q (rows, heads, head_dim), k and v (rows, kv_heads,
        head_dim) bf16, any row stride, rows_per_seq rows for each sequence;
        `length` and `seq` (n,) int32: cached tokens and slots (None: 0, 1, ..);
        `mask` (rows, words) int32, or None for chains; scale None: head_dim ** -0.5.
        `out` holds "o" as q, and "lse" (rows, heads) f32 if wanted."""
        c, i32, vec = self._cache(cache), self._i32, self._vec
        n, kv_heads, dim = length.numel(), cache.shape[2], cache.shape[4]
        rows = n * rows_per_seq
        if q.dim() != 3:
            raise SamplerError("q must be (rows, heads, head_dim)")
        heads = q.shape[1]
        shape, new = (rows, heads, dim), (rows, kv_heads, dim)
        qp, qs = self._heads(q, shape, "q")
        kp, ks = self._heads(k, new, "k")
        vp, vs = self._heads(v, new, "v")
        op, os_ = self._heads(out["o"], shape, "o")
        lse, words = out.get("lse"), 0
        if lse is not None and (lse.dtype != self.torch.float32 or lse.shape != (rows, heads) or not lse.is_contiguous() or
                                lse.get_device() != self.device):
            raise SamplerError(f"lse must be ({rows}, {heads}) f32, contiguous, on the sampler's device")
        if mask is not None:
            mask = mask.view(rows, -1) if mask.is_contiguous() and rows and mask.numel() % rows == 0 else mask
            if (mask.dtype != i32 or mask.dim() != 2 or mask.shape[0] != rows or not mask.is_contiguous() or
                    mask.get_device() != self.device):
                raise SamplerError(f"mask must be ({rows}, words) int32, contiguous, on the sampler's device")
            words = mask.shape[1]
        b = _TreeBatch(n, rows_per_seq, heads, layer, dim ** -0.5 if scale is None else scale, words, cache._p, qp, kp,
                       vp, qs, ks, vs, vec(seq, n, i32, "seq"), vec(length, n, i32, "length"), _addr(mask))
        rc = _lib.lcs_tree_attn(self.ctx, b, _TreeOut(op, os_, _addr(lse)), self._raw_stream(stream))
        if rc != LCS_OK:
            self._check(rc)

    def tree_verify_dev(self, tokens, parent, out, rows_per_seq: int, logits=None, length=None, stream=None):
        """The greedy verdict on trees of drafts (lcs_tree_verify): `tokens` and
        `parent` (n * rows_per_seq,) int32; `logits` (rows, vocab) f32 or bf16, any
        16-byte row stride, or None where out["argmax_ids"] already holds the rows'
        argmax. `out` holds "argmax_ids" (rows,), "path" (n, rows_per_seq),
        "n_path" and "next_id" (n,) int32, and if wanted "node_lp" (rows,) f32 and
        "length" (n,) int32: `length` + n_path."""
        i32, f32, vec = self._i32, self._f32, self._vec
        rows = tokens.numel()
        if rows_per_seq < 1 or rows % rows_per_seq:
            raise SamplerError("rows_per_seq must divide the rows")
        n = rows // rows_per_seq
        vocab = dtype = stride = 0
        if logits is not None:
            dtype = self._types.get(logits.dtype)
            if dtype not in (LCS_F32, LCS_BF16) or logits.dim() != 2 or logits.shape[0] != rows or logits.get_device() != self.device:
                raise SamplerError(f"logits must be ({rows}, vocab) float32 or bfloat16 on the sampler's device")
            vocab = logits.shape[1]
            if logits.stride(1) != 1 and vocab > 1:
                raise SamplerError("logits must have unit column stride")
            per = 4 if dtype == LCS_F32 else 8
            stride = logits.stride(0) if rows > 1 else (vocab + per - 1) // per * per
        path = out["path"]
        if path.dtype != i32 or path.numel() != rows or not path.is_contiguous() or path.get_device() != self.device:
            raise SamplerError(f"path must be ({n}, {rows_per_seq}) int32, contiguous, on the sampler's device")
        b = _TreeVBatch(n, rows_per_seq, vocab, dtype, stride, _addr(logits), vec(tokens, rows, i32, "tokens"),
                        vec(parent, rows, i32, "parent"), vec(length, n, i32, "length"))
        o = _TreeVOut(vec(out["argmax_ids"], rows, i32, "argmax_ids"), vec(out.get("node_lp"), rows, f32, "node_lp"),
                      path.data_ptr(), vec(out["n_path"], n, i32, "n_path"), vec(out["next_id"], n, i32, "next_id"),
                      vec(out.get("length"), n, i32, "length"))
        rc = _lib.lcs_tree_verify(self.ctx, b, o, self._raw_stream(stream))
        if rc != LCS_OK:
            self._check(rc)

    def verify(self, w):
        d = self.upload(w)
        out = self.alloc_verify_out(w)
        self.verify_dev(d, out)
        self.torch.cuda.synchronize()
        return {k: v.cpu().numpy() for k, v in out.items()}

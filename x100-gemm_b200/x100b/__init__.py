"""Python binding of libx100gemm_b200.so (ctypes over the C ABI).

The library is the product: hand-written sm_100a kernels behind the C ABI
declared in include/x100_gemm.h and include/x100q.h.  This module only loads
it, declares the signatures and offers numpy / torch conveniences for the
tests and bench.py.  There is no fallback: if the shared library is missing
or a call fails, an exception is raised.
"""
from __future__ import annotations

import ctypes as C
import os
import re
import struct

import numpy as np

PKG_DIR = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
REPO = os.path.dirname(PKG_DIR)
LIB_PATH = os.path.join(PKG_DIR, "libx100gemm_b200.so")
HEADERS = [os.path.join(REPO, "include", "x100_gemm.h"), os.path.join(REPO, "include", "x100q.h")]

X100_OK, X100_E_ARG, X100_E_NODEV, X100_E_ARCH, X100_E_ALLOC, X100_E_COPY, X100_E_LAUNCH, \
    X100_E_TIMEOUT, X100_E_COMM, X100_E_INJECTED, X100_E_UNSUPPORTED, X100_E_TOO_LARGE, X100_E_FORMAT = range(13)

Q_F32, Q4_0, Q8_0, Q3_K, Q4_K = 0, 2, 8, 11, 12
Q_F16 = 1


class X100Error(RuntimeError):
    def __init__(self, code: int, what: str = ""):
        self.code = code
        super().__init__(f"{what}: x100 error {code} ({strerror(code)})")


class Caps(C.Structure):
    _fields_ = [("vlen_bits", C.c_int), ("vlenb", C.c_int), ("has_v", C.c_int), ("has_zvfh", C.c_int),
                ("has_zvbb", C.c_int), ("has_ime", C.c_int), ("mvendorid", C.c_ulong), ("isa", C.c_char * 1024)]


_lib = None
vp, i32, i64 = C.c_void_p, C.c_int, C.c_long

_SIGS = {
    # reference signatures (void)
    "gemm_ref_f32": ([i32, i32, i32, vp, vp, vp], None),
    "gemm_rvv_f32": ([i32, i32, i32, vp, vp, vp], None),
    "gemm_rvv_f16": ([i32, i32, i32, vp, vp, vp], None),
    "gemm_f16_f32acc": ([i32, i32, i32, vp, vp, vp], None),
    "gemm_ref_i8": ([i32, i32, i32, vp, vp, vp], None),
    "gemm_ime_i8": ([i32, i32, i32, vp, vp, vp], None),
    "gemm_ime2_pack_a": ([i32, i32, vp, vp], None),
    "gemm_ime2_pack_b": ([i32, i32, vp, vp], None),
    "gemm_ime2_i8_st": ([i32, i32, i32, vp, vp, vp], None),
    "gemm_ime2_i8_mt": ([i32, i32, i32, vp, vp, vp, i32], None),
    "x100_detect": ([vp], None),
    "x100_caps_print": ([vp], None),
    # device variants
    "gemm_ime_i8_dev": ([i32, i32, i32, vp, vp, vp, vp], i32),
    "gemm_ref_i8_dev": ([i32, i32, i32, vp, vp, vp, vp], i32),
    "gemm_f16_f32acc_dev": ([i32, i32, i32, vp, vp, vp, vp], i32),
    "gemm_f16_dev": ([i32, i32, i32, vp, vp, vp, vp], i32),
    "gemm_f32_dev": ([i32, i32, i32, vp, vp, vp, vp], i32),
    "gemm_ref_f32_dev": ([i32, i32, i32, vp, vp, vp, vp], i32),
    "gemm_ime_i8_dev_ld": ([i32, i32, i32, vp, i64, vp, i64, vp, i64, vp], i32),
    "x100_sync": ([vp], i32),
    "x100_last_error": ([], i32),
    "x100_strerror": ([i32], C.c_char_p),
    "x100_set_device": ([i32], i32),
    # quantised path
    "x100q_row_bytes": ([i32, i32], C.c_size_t),
    "x100q_lin_create": ([i32, i32, i32, vp], vp),
    "x100q_lin_destroy": ([vp], None),
    "x100q_lin_info": ([vp, vp, vp, vp, vp], i32),
    "x100q_lin_gemv": ([vp, vp, vp, i32], i32),
    "x100q_lin_gemv_dev": ([vp, vp, vp, i32, vp], i32),
    "x100q_lin_gemv_dev_flags": ([vp, vp, vp, i32, i32, vp], i32),
    "x100q_moe_create": ([i32, i32, i32, i32, i32, vp, vp, vp, vp, i32, i32], vp),
    "x100q_moe_destroy": ([vp], None),
    "x100q_moe_ffn": ([vp, vp, vp, i32, vp, vp], i32),
    "x100q_moe_ffn_dev": ([vp, vp, vp, i32, vp, vp, vp], i32),
    "x100q_router_topk_noalloc": ([vp, vp, i32, i32, i32, i32, vp, vp, vp], i32),
    # decode step
    "x100q_model_create": ([vp], vp),
    "x100q_model_create_kv4": ([vp, vp, vp, i32], vp),
    "x100q_model_destroy": ([vp], None),
    "x100q_model_set_layer": ([vp, i32] + [vp] * 12, i32),
    "x100q_model_set_output": ([vp, vp, vp, vp], i32),
    "x100q_model_kv_copy": ([vp, i32, i32, i32, i32, vp, vp, i32], i32),
    "x100q_model_embed_dev": ([vp, vp, vp, i32, vp], i32),
    "x100q_model_layer_dev": ([vp, i32, vp, vp, i32, vp, vp, vp, vp], i32),
    "x100q_model_head_dev": ([vp, vp, vp, i32, vp], i32),
    "x100q_model_forward_dev": ([vp, vp, vp, vp, vp, i32, vp], i32),
    "x100q_model_forward": ([vp, vp, vp, vp, i32], i32),
    "x100q_model_forward_slots_dev": ([vp, vp, vp, vp, vp, vp, i32, vp], i32),
    "x100q_model_prefill": ([vp, i32, vp, i32, i32, vp], i32),
    "x100q_model_timing": ([vp, i32], i32),
    "x100q_model_timing_read": ([vp, vp, vp], i32),
    "x100q_timing_bucket_name": ([i32], C.c_char_p),
    # expert-parallel combine
    "x100q_ep_create": ([i32, i32, i32], vp),
    "x100q_ep_handle": ([vp, vp], i32),
    "x100q_ep_open": ([vp, vp], i32),
    "x100q_ep_allreduce_dev": ([vp, vp, vp, i32, i32, vp], i32),
    "x100q_ep_destroy": ([vp], None),
    # GGUF ingest
    "x100q_gguf_open": ([C.c_char_p], vp),
    "x100q_gguf_close": ([vp], None),
    "x100q_gguf_n_tensors": ([vp], i32),
    "x100q_gguf_tensor_at": ([vp, i32, vp], i32),
    "x100q_gguf_find": ([vp, C.c_char_p, vp], i32),
    "x100q_gguf_data_offset": ([vp], C.c_uint64),
    "x100q_gguf_n_tokens": ([vp], i32),
    "x100q_gguf_token": ([vp, i32], C.c_char_p),
    "x100q_gguf_get_int": ([vp, C.c_char_p, vp], i32),
    "x100q_gguf_get_f32": ([vp, C.c_char_p, vp], i32),
    "x100q_gguf_get_str": ([vp, C.c_char_p, vp], i32),
    "x100q_gguf_model_cfg": ([vp, vp], i32),
    "x100q_model_load_gguf": ([vp, vp], vp),
    "x100q_model_load_gguf_kv4": ([vp, vp, vp, vp, i32], vp),
    "x100q_gguf_dequant_dev": ([i32, vp, C.c_long, vp, vp], i32),
    "x100q_quantize_q8_0_dev": ([vp, C.c_long, vp, vp], i32),
    "x100q_pack_act_dev": ([i32, vp, i32, i32, vp, vp], i32),
    # paged 4-bit KV cache, residual RMS norm with 8-bit output
    "x100q_kv4_bytes": ([vp], C.c_size_t),
    "x100q_kv4_append_dev": ([vp, vp, vp], i32),
    "x100q_kv4_read_dev": ([vp, vp, vp, i32, vp, i32, i32, vp, vp, vp], i32),
    "x100q_rope_table_dev": ([vp, i32, i32, C.c_float, vp], i32),
    "x100q_kv4_attn_work": ([vp, i32, i32, i32], C.c_size_t),
    "x100q_kv4_attn_dev": ([vp, vp, vp], i32),
    "x100q_add_rmsnorm_q8_dev": ([vp, vp], i32),
}


class GgufTensor(C.Structure):
    """x100q_gguf_tensor (include/x100q.h)."""
    _fields_ = [("name", C.c_char_p), ("type", C.c_int), ("n_dims", C.c_int), ("dims", C.c_uint64 * 4),
                ("n_elems", C.c_uint64), ("bytes", C.c_uint64), ("data", C.c_void_p)]


class ModelCfg(C.Structure):
    """x100q_model_cfg (include/x100q.h)."""
    _fields_ = [(n, C.c_int) for n in ("n_layers", "d", "n_heads", "n_kv_heads", "head_dim", "vocab", "n_exp",
                                       "n_act", "moe_ffn", "attn_qtype", "expert_qtype", "lm_qtype", "ctx",
                                       "max_batch", "expert_lo", "expert_hi")] + \
               [("rope_base", C.c_float), ("eps", C.c_float)]


class Kv4(C.Structure):
    """x100q_kv4 (include/x100q.h)."""
    _fields_ = [("pages", vp)] + [(n, i32) for n in ("n_pages", "page_size", "n_kv_heads", "head_dim")]


class Kv4AppendArgs(C.Structure):
    """x100q_kv4_append_args (include/x100q.h)."""
    _fields_ = [(n, i32) for n in ("dtype", "n_tokens", "n_heads")] + [(n, vp) for n in ("q", "k", "v", "q_out")] + \
               [(n, i64) for n in ("q_stride", "k_stride", "v_stride", "q_out_stride")] + \
               [("q_norm", vp), ("k_norm", vp), ("eps", C.c_float), ("rope", vp), ("rope_len", i32), ("pos", vp),
                ("seq", vp), ("page_table", vp), ("table_stride", i32), ("n_seqs", i32)]


class Kv4AttnArgs(C.Structure):
    """x100q_kv4_attn_args (include/x100q.h)."""
    _fields_ = [("dtype", i32), ("n_heads", i32), ("q", vp), ("out", vp), ("q_stride", i64), ("out_stride", i64),
                ("q_start", vp), ("n_tokens", i32), ("max_q", i32), ("kv_len", vp), ("page_table", vp),
                ("table_stride", i32), ("n_seqs", i32), ("scale", C.c_float), ("work", vp), ("work_bytes", C.c_size_t)]


class NormQ8Args(C.Structure):
    """x100q_norm_q8_args (include/x100q.h)."""
    _fields_ = [(n, i32) for n in ("dtype", "rows", "d", "group")] + [(n, vp) for n in ("x", "residual", "residual_out")] + \
               [(n, i64) for n in ("ldx", "ldr", "ldo", "ldq")] + [("w", vp), ("eps", C.c_float), ("q", vp), ("scales", vp)]


def lib():
    """Load libx100gemm_b200.so; raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise FileNotFoundError(f"{LIB_PATH} missing: run __graft_entry__.build() (make -C x100-gemm_b200)")
        L = C.CDLL(LIB_PATH)
        for name, (args, res) in _SIGS.items():
            fn = getattr(L, name, None)
            if fn is None:
                continue
            fn.argtypes = args
            fn.restype = res
        _lib = L
    return _lib


TIMING_BUCKETS = 8   # X100Q_NBUCKETS


def timing_bucket_name(i: int) -> str | None:
    """Name of step-timing bucket i (x100q_timing_bucket_name)."""
    n = lib().x100q_timing_bucket_name(i)
    return n.decode() if n else None


def header_functions() -> list[str]:
    """Names of every function declared in include/*.h."""
    names = []
    for h in HEADERS:
        src = open(h).read()
        src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
        for m in re.finditer(r"^[A-Za-z_][\w \*]*?\b([a-z_][a-z0-9_]*)\s*\(", src, flags=re.M):
            if m.group(1) not in ("defined",):
                names.append(m.group(1))
    return sorted(set(names))


def strerror(code: int) -> str:
    return lib().x100_strerror(code).decode()


def last_error() -> int:
    return lib().x100_last_error()


def check(code: int, what: str = "x100") -> None:
    if code != X100_OK:
        raise X100Error(code, what)


def check_last(what: str) -> None:
    check(last_error(), what)


def detect() -> Caps:
    caps = Caps()
    lib().x100_detect(C.byref(caps))
    return caps


def _p(a):
    """Raw pointer of a numpy array or torch tensor."""
    if a is None:
        return None
    if isinstance(a, np.ndarray):
        return a.ctypes.data
    return a.data_ptr()


def _stream(stream):
    if stream is None:
        import torch
        return torch.cuda.current_stream().cuda_stream
    return stream if isinstance(stream, int) else stream.cuda_stream


# ---- host-pointer (reference-signature) calls ------------------------------------
def gemm_host(fn: str, A, B, Cm) -> None:
    """Call a void reference-signature GEMM (gemm_ime_i8, gemm_ref_f32, ...)
    on numpy arrays (or torch tensors); C += A @ B in place."""
    M, K = A.shape
    N = B.shape[1]
    getattr(lib(), fn)(M, N, K, _p(A), _p(B), _p(Cm))
    check_last(fn)


# ---- device-pointer calls (torch tensors) ----------------------------------------------
def gemm_dev(fn: str, A, B, Cm, stream=None) -> None:
    M, K = A.shape
    N = B.shape[1]
    check(getattr(lib(), fn)(M, N, K, _p(A), _p(B), _p(Cm), _stream(stream)), fn)


def sync(stream=None) -> None:
    check(lib().x100_sync(_stream(stream)), "x100_sync")


# ---- quantised linear / MoE -----------------------------------------------------------
class Lin:
    """x100q_lin handle: an N x K block-quantised linear resident in HBM."""

    def __init__(self, qtype: int, N: int, K: int, blocks: np.ndarray):
        blocks = np.ascontiguousarray(blocks, np.uint8)
        self.qtype, self.N, self.K = qtype, N, K
        self.h = lib().x100q_lin_create(qtype, N, K, blocks.ctypes.data)
        if not self.h:
            check_last("x100q_lin_create")

    def gemv(self, x, y, batch: int) -> None:
        check(lib().x100q_lin_gemv(self.h, _p(x), _p(y), batch), "x100q_lin_gemv")

    def gemv_dev(self, x, y, batch: int, stream=None, independent: bool = False, a8: bool = False) -> None:
        flags = (1 if independent else 0) | (2 if a8 else 0)
        check(lib().x100q_lin_gemv_dev_flags(self.h, _p(x), _p(y), batch, flags, _stream(stream)),
              "x100q_lin_gemv_dev_flags")

    def device_bytes(self) -> int:
        b = C.c_size_t()
        check(lib().x100q_lin_info(self.h, None, None, None, C.byref(b)), "x100q_lin_info")
        return b.value

    def close(self):
        if getattr(self, "h", None) and _lib is not None:
            _lib.x100q_lin_destroy(self.h)
            self.h = None

    __del__ = close


class Moe:
    """x100q_moe handle: router + top-k + SwiGLU experts [lo, hi) in HBM."""

    def __init__(self, d, n_exp, n_act, ffn, qtype, router, gate, up, down, expert_lo=0, expert_hi=None):
        expert_hi = n_exp if expert_hi is None else expert_hi
        self.d, self.n_exp, self.n_act, self.ffn = d, n_exp, n_act, ffn
        router = np.ascontiguousarray(router, np.float32)
        self.h = lib().x100q_moe_create(d, n_exp, n_act, ffn, qtype, router.ctypes.data, _p(gate), _p(up),
                                        _p(down), expert_lo, expert_hi)
        if not self.h:
            check_last("x100q_moe_create")

    def ffn_host(self, hn: np.ndarray):
        hn = np.ascontiguousarray(hn, np.float32).reshape(-1, self.d)
        B = hn.shape[0]
        eout = np.empty_like(hn)
        sel = np.empty((B, self.n_act), np.int32)
        w = np.empty((B, self.n_act), np.float32)
        check(lib().x100q_moe_ffn(self.h, hn.ctypes.data, eout.ctypes.data, B, sel.ctypes.data, w.ctypes.data),
              "x100q_moe_ffn")
        return eout, sel, w

    def ffn_dev(self, hn, eout, batch, sel=None, w=None, stream=None):
        check(lib().x100q_moe_ffn_dev(self.h, _p(hn), _p(eout), batch, _p(sel), _p(w), _stream(stream)),
              "x100q_moe_ffn_dev")

    def close(self):
        if getattr(self, "h", None) and _lib is not None:
            _lib.x100q_moe_destroy(self.h)
            self.h = None

    __del__ = close


class Model:
    """x100q_model handle: a Qwen3-MoE-shaped decode model (weights, KV cache,
    scratch) resident on the current device.  The cache is fp16, or, with
    kv4 = (n_pages, page_size, table), pages of 4-bit codes: table int32
    [max_batch, entries] on the GPU names each slot's pages, for all layers."""

    def __init__(self, kv4=None, **cfg):
        self.cfg = ModelCfg(**cfg)
        self._open("x100q_model_create", (), kv4)

    def _open(self, fn, args, kv4):
        """Call fn(*args, cfg), or with a paged cache fn_kv4(*args, cfg, pool, table, entries)."""
        self.h, self._kv4, args = None, None, (*args, C.byref(self.cfg))
        if kv4 is not None:
            torch, c, fn = _torch()[0], self.cfg, fn + "_kv4"
            n_pages, page_size, table = kv4
            if not (table.dtype is torch.int32 and table.is_cuda and table.get_device() == torch.cuda.current_device()
                    and table.is_contiguous() and table.dim() == 2 and table.shape[0] >= c.max_batch):
                _refuse(fn, f"the page table has to be contiguous int32 [{c.max_batch}, entries] on the current device")
            kv = Kv4(None, n_pages, page_size, c.n_kv_heads, c.head_dim)
            n = lib().x100q_kv4_bytes(C.byref(kv))
            if n == 0 or c.n_layers < 1:
                _refuse(fn, f"no pool of {n_pages} pages of {page_size} x {c.n_kv_heads} x {c.head_dim}")
            self._pages = torch.zeros(c.n_layers, n, dtype=torch.uint8, device="cuda")
            torch.cuda.current_stream().synchronize()   # zeroed before a step on another stream
            kv.pages, self.kv4_table, self._kv4 = self._pages.data_ptr(), table, kv
            args += (C.byref(kv), table.data_ptr(), table.shape[1])
        self.h = getattr(lib(), fn)(*args)
        if not self.h:
            check_last(fn)

    def kv4_cache(self, layer: int) -> "Kv4Cache":
        """The pool of a layer of a model made with kv4, on the model's own pages."""
        kv = self._kv4
        if kv is None or not 0 <= layer < self.cfg.n_layers:
            _refuse("Model.kv4_cache", "a layer of a model made with kv4 has one")
        return Kv4Cache(kv.n_pages, kv.page_size, kv.n_kv_heads, kv.head_dim, pages=self._pages[layer])

    def set_layer(self, layer, attn_norm, wq, wk, wv, q_norm, k_norm, wo, ffn_norm, router, gate, up, down):
        check(lib().x100q_model_set_layer(self.h, layer, *(_p(a) for a in (attn_norm, wq, wk, wv, q_norm, k_norm,
                                                                            wo, ffn_norm, router, gate, up, down))),
              "x100q_model_set_layer")

    def set_output(self, tok_embd, out_norm, lm):
        check(lib().x100q_model_set_output(self.h, _p(tok_embd), _p(out_norm), _p(lm)), "x100q_model_set_output")

    def kv_write(self, layer, slot, pos0, k, v):
        npos = k.shape[1]
        check(lib().x100q_model_kv_copy(self.h, layer, slot, pos0, npos, _p(k), _p(v), 1), "x100q_model_kv_copy")

    def kv_read(self, layer, slot, pos0, npos):
        c = self.cfg
        k = np.empty((c.n_kv_heads, npos, c.head_dim), np.uint16)
        v = np.empty_like(k)
        check(lib().x100q_model_kv_copy(self.h, layer, slot, pos0, npos, _p(k), _p(v), 0), "x100q_model_kv_copy")
        return k, v

    def layer_dev(self, layer, h, pos, batch, eout=None, sel=None, w=None, stream=None):
        check(lib().x100q_model_layer_dev(self.h, layer, _p(h), _p(pos), batch, _p(eout), _p(sel), _p(w),
                                          _stream(stream)), "x100q_model_layer_dev")

    def head_dev(self, h, logits, batch, stream=None):
        check(lib().x100q_model_head_dev(self.h, _p(h), _p(logits), batch, _stream(stream)), "x100q_model_head_dev")

    def embed_dev(self, tokens, h, batch, stream=None):
        check(lib().x100q_model_embed_dev(self.h, _p(tokens), _p(h), batch, _stream(stream)),
              "x100q_model_embed_dev")

    def forward_dev(self, tokens, h, pos, logits, batch, stream=None):
        check(lib().x100q_model_forward_dev(self.h, _p(tokens), _p(h), _p(pos), _p(logits), batch,
                                            _stream(stream)), "x100q_model_forward_dev")

    def forward_slots_dev(self, tokens, h, pos, slot, logits, batch, stream=None):
        check(lib().x100q_model_forward_slots_dev(self.h, _p(tokens), _p(h), _p(pos), _p(slot), _p(logits), batch,
                                                  _stream(stream)), "x100q_model_forward_slots_dev")

    def _ordered(self):
        """The host calls run on the library's own stream and read a paged cache's table and pages, which the
        caller writes on the current one: wait for that (the call itself waits for the default stream)."""
        if self._kv4 is not None:
            s = _torch()[0].cuda.current_stream(self._pages.device)
            if s.cuda_stream:
                s.synchronize()

    def prefill(self, slot: int, tokens, pos0: int, logits: bool = True):
        """n tokens of the sequence in `slot` at positions pos0 .. pos0+n-1 in
        one step; returns their logits [n][vocab] (or None)."""
        tokens = np.ascontiguousarray(tokens, np.int32)
        n = tokens.shape[0]
        out = np.empty((n, self.cfg.vocab), np.float32) if logits else None
        self._ordered()
        check(lib().x100q_model_prefill(self.h, slot, _p(tokens), n, pos0, _p(out)), "x100q_model_prefill")
        return out

    def forward(self, tokens, pos):
        tokens = np.ascontiguousarray(tokens, np.int32)
        pos = np.ascontiguousarray(pos, np.int32)
        B = tokens.shape[0]
        logits = np.empty((B, self.cfg.vocab), np.float32)
        self._ordered()
        check(lib().x100q_model_forward(self.h, _p(tokens), _p(pos), _p(logits), B), "x100q_model_forward")
        return logits

    def timing(self, on: bool):
        """Start (clearing the totals) or stop per-bucket step timing."""
        check(lib().x100q_model_timing(self.h, 1 if on else 0), "x100q_model_timing")

    def timing_read(self) -> tuple[dict, int]:
        """({bucket name: total ms}, timed calls) since timing started."""
        ms = np.zeros(TIMING_BUCKETS, np.float64)
        steps = C.c_long(0)
        check(lib().x100q_model_timing_read(self.h, _p(ms), C.byref(steps)), "x100q_model_timing_read")
        return {timing_bucket_name(i): float(ms[i]) for i in range(TIMING_BUCKETS)}, steps.value

    def close(self):
        if getattr(self, "h", None) and _lib is not None:
            _lib.x100q_model_destroy(self.h)
            self.h = None

    __del__ = close


class Gguf:
    """x100q_gguf handle: a GGUF file mapped and parsed (no GPU needed)."""

    def __init__(self, path: str):
        self.h = lib().x100q_gguf_open(os.fsencode(path))
        if not self.h:
            check_last("x100q_gguf_open")

    def _info(self, t: GgufTensor) -> dict:
        return {"name": t.name.decode(), "type": t.type, "n_dims": t.n_dims, "dims": list(t.dims[: t.n_dims]),
                "n_elems": t.n_elems, "bytes": t.bytes, "data": t.data}

    def tensors(self) -> list[dict]:
        out = []
        for i in range(lib().x100q_gguf_n_tensors(self.h)):
            t = GgufTensor()
            check(lib().x100q_gguf_tensor_at(self.h, i, C.byref(t)), "x100q_gguf_tensor_at")
            out.append(self._info(t))
        return out

    def find(self, name: str) -> dict:
        t = GgufTensor()
        check(lib().x100q_gguf_find(self.h, name.encode(), C.byref(t)), "x100q_gguf_find")
        return self._info(t)

    def tensor_bytes(self, name: str) -> np.ndarray:
        """The tensor's raw data (a copy out of the mapping)."""
        t = self.find(name)
        return np.ctypeslib.as_array((C.c_uint8 * t["bytes"]).from_address(t["data"])).copy()

    @property
    def data_offset(self) -> int:
        return int(lib().x100q_gguf_data_offset(self.h))

    def tokens(self) -> list[str]:
        L = lib()
        return [L.x100q_gguf_token(self.h, i).decode() for i in range(L.x100q_gguf_n_tokens(self.h))]

    def get_int(self, key: str) -> int:
        v = C.c_int64()
        check(lib().x100q_gguf_get_int(self.h, key.encode(), C.byref(v)), key)
        return v.value

    def get_f32(self, key: str) -> float:
        v = C.c_float()
        check(lib().x100q_gguf_get_f32(self.h, key.encode(), C.byref(v)), key)
        return v.value

    def get_str(self, key: str) -> str:
        v = C.c_char_p()
        check(lib().x100q_gguf_get_str(self.h, key.encode(), C.byref(v)), key)
        return v.value.decode()

    def model_cfg(self) -> dict:
        c = ModelCfg()
        check(lib().x100q_gguf_model_cfg(self.h, C.byref(c)), "x100q_gguf_model_cfg")
        return {n: getattr(c, n) for n, _ in ModelCfg._fields_}

    def load_model(self, kv4=None, **overrides) -> "Model":
        """x100q_model_load_gguf with the file's configuration, fields such as
        ctx, max_batch or expert_lo / expert_hi replaced by `overrides`; kv4
        as of Model."""
        cfg = dict(self.model_cfg(), **overrides)
        m = Model.__new__(Model)
        m.cfg = ModelCfg(**cfg)
        m._open("x100q_model_load_gguf", (self.h,), kv4)
        return m

    def close(self):
        if getattr(self, "h", None) and _lib is not None:
            _lib.x100q_gguf_close(self.h)
            self.h = None

    __del__ = close


def gguf_dequant_dev(gtype: int, data, n: int, out, stream=None) -> None:
    check(lib().x100q_gguf_dequant_dev(gtype, _p(data), n, _p(out), _stream(stream)), "x100q_gguf_dequant_dev")


PACK_I8, PACK_Q3K, PACK_HP = 1, 2, 3
GEMV_INDEPENDENT, GEMV_A8 = 1, 2


def pack_act_dev(mode: int, x, K: int, batch: int, out, stream=None) -> None:
    """The reference's pack_act_i8 (mode PACK_I8) / pack_act_q3k (PACK_Q3K) /
    pack_act_hp (PACK_HP)."""
    check(lib().x100q_pack_act_dev(mode, _p(x), K, batch, _p(out), _stream(stream)), "x100q_pack_act_dev")


def quantize_q8_0_dev(x, n: int, blocks, stream=None) -> None:
    check(lib().x100q_quantize_q8_0_dev(_p(x), n, _p(blocks), _stream(stream)), "x100q_quantize_q8_0_dev")


# ---- paged 4-bit KV cache, residual RMS norm with 8-bit output (torch tensors) ---------------
# A decode step calls these for every layer, so the checks are plain expressions
# on the way through and only a failed one goes looking for its reason, and the
# argument structs go as packed bytes, in native alignment as the ctypes ones
# (1 us a call less than filling those).
_APPEND, _ATTN, _NORM = (struct.Struct(f).pack for f in ("@3i4P4q2PfPi3P2i", "@2i2P2qP2i2P2if4xPN", "@4i3P4qPf4x2P"))
_TORCH = None   # (torch, {dtype: Q_F32 / Q_F16}, float16, float32, int32, int8, uint8, current device, its current stream)


# a tensor made here belongs to the current stream, and the allocator may hand its memory on while another one writes it
_OWN_STREAM = "outputs and scratch have to be given together with a stream"


def _torch():
    global _TORCH
    if _TORCH is None:
        import torch
        torch.cuda.current_device()   # initialises CUDA
        _TORCH = (torch, {torch.float32: Q_F32, torch.float16: Q_F16}, torch.float16, torch.float32, torch.int32, torch.int8, torch.uint8,
                  torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream)
    return _TORCH


def _refuse(what: str, why: str, code: int = X100_E_ARG):
    raise X100Error(code, f"{what}: {why}")


def _placed(what: str, dev: int, **named) -> None:
    """Raise for the first of name = (tensor or None, dtype) of another type or device; integers have to be contiguous too."""
    torch = _torch()[0]
    for name, (t, dt) in named.items():
        if t is not None and (t.dtype is not dt or t.get_device() != dev):
            _refuse(what, f"{name} has to be {dt} on the current device (cuda:{dev}), not {t.dtype} on {t.device}")
        if t is not None and dt is torch.int32 and not t.is_contiguous():
            _refuse(what, f"{name} has to be contiguous")


def _token_stride(t, name: str, what: str, dim: int) -> int:
    """Token stride of [tokens, heads, dim] that is not contiguous: the heads of a token have to lie side by side."""
    if t.dim() != 3 or t.shape[2] != dim or t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != dim):
        _refuse(what, f"{name} has to be [tokens, heads, {dim}], a token's heads side by side")
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1] * dim)


class Kv4Cache:
    """A pool of 4-bit KV pages (x100q_kv4): `pages` is a uint8 tensor of the pool's bytes, allocated on
    the current device unless given.  Page tables are int32 [sequences, entries]; see include/x100q.h for the
    layout, the masks and what is out of range.  Methods allocate nothing unless an output or the scratch is left out."""

    def __init__(self, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, pages=None):
        torch = _torch()[0]
        self.kv = Kv4(None, n_pages, page_size, n_kv_heads, head_dim)
        self._ref = C.byref(self.kv)
        n = lib().x100q_kv4_bytes(self._ref)
        if n == 0:
            _refuse("Kv4Cache", f"no pool of {n_pages} pages of {page_size} x {n_kv_heads} x {head_dim}")
        if pages is None:
            pages = torch.zeros(n, dtype=torch.uint8, device="cuda")
            torch.cuda.current_stream().synchronize()   # zeroed before an append on another stream
        if pages.dtype is not torch.uint8 or not pages.is_cuda or not pages.is_contiguous() or pages.numel() < n:
            _refuse("Kv4Cache", f"pages has to be {n} contiguous uint8 on a GPU")
        self.pages, self.kv.pages, self.device = pages, pages.data_ptr(), pages.get_device()
        self.head_dim, self.n_kv_heads = head_dim, n_kv_heads
        self._append, self._read, self._attn = lib().x100q_kv4_append_dev, lib().x100q_kv4_read_dev, lib().x100q_kv4_attn_dev

    def _elsewhere(self, what, dev):
        _refuse(what, f"the pool is on cuda:{self.device}, the current device is cuda:{dev}")

    def append(self, k, v, pos, table, seq=None, q=None, q_out=None, q_norm=None, k_norm=None, eps=1e-6, rope=None, stream=None):
        """x100q_kv4_append_dev: k, v [tokens, kv heads, dim] into the pages; returns q_out, the normed and rotated q."""
        torch, kinds, _, f32, i32_, _, _, device, current = _torch()
        what, dev, D, KV, dt = "Kv4Cache.append", device(), self.head_dim, self.n_kv_heads, k.dtype
        if dev != self.device:
            self._elsewhere(what, dev)
        kind = kinds.get(dt)
        if kind is None:
            _refuse(what, f"float32 or float16 is taken, not {dt}", X100_E_UNSUPPORTED)
        if q is not None and q_out is None:
            if stream is not None:
                _refuse(what, _OWN_STREAM)
            q_out = torch.empty(q.shape, dtype=dt, device=q.device)
        if not (k.get_device() == dev and v.get_device() == dev and v.dtype is dt and pos.dtype is i32_ and pos.get_device() == dev and pos.is_contiguous()
                and table.dtype is i32_ and table.get_device() == dev and table.is_contiguous()
                and (seq is None or (seq.dtype is i32_ and seq.get_device() == dev and seq.is_contiguous()))
                and (q is None or (q.dtype is dt and q.get_device() == dev and q_out.dtype is dt and q_out.get_device() == dev))
                and (q_norm is None or (q_norm.dtype is f32 and q_norm.get_device() == dev)) and (k_norm is None or (k_norm.dtype is f32 and k_norm.get_device() == dev))
                and (rope is None or (rope.dtype is f32 and rope.get_device() == dev))):
            _placed(what, dev, k=(k, dt), v=(v, dt), q=(q, dt), q_out=(q_out, dt), q_norm=(q_norm, f32), k_norm=(k_norm, f32), rope=(rope, f32), pos=(pos, i32_),
                    seq=(seq, i32_), table=(table, i32_))
        n, want = pos.numel(), (pos.numel(), KV, D)
        if not (k.shape == want and v.shape == want and table.dim() == 2 and (seq is None or seq.numel() == n)):
            _refuse(what, f"k and v have to be {want}, the page table [sequences, entries], and seq as long as pos")
        ks = KV * D if k.is_contiguous() else _token_stride(k, "k", what, D)
        vs = KV * D if v.is_contiguous() else _token_stride(v, "v", what, D)
        qp = op = qs = os_ = heads = 0
        if q is not None:
            if q.dim() != 3 or q.shape[0] != n or q.shape[2] != D or q_out.shape != q.shape:
                _refuse(what, f"q and q_out have to be [{n}, heads, {D}]")
            heads = q.shape[1]
            qs = heads * D if q.is_contiguous() else _token_stride(q, "q", what, D)
            os_ = heads * D if q_out.is_contiguous() else _token_stride(q_out, "q_out", what, D)
            qp, op = q.data_ptr(), q_out.data_ptr()
        if not ((q_norm is None or (q_norm.numel() == D and q_norm.is_contiguous())) and (k_norm is None or (k_norm.numel() == D and k_norm.is_contiguous()))
                and (rope is None or (rope.numel() % D == 0 and rope.is_contiguous()))):
            _refuse(what, f"q_norm and k_norm have to be {D} contiguous values and rope [positions, {D // 2}, 2]")
        tn, ts = table.shape
        a = _APPEND(kind, n, heads, qp, k.data_ptr(), v.data_ptr(), op, qs, ks, vs, os_, 0 if q_norm is None else q_norm.data_ptr(),
                          0 if k_norm is None else k_norm.data_ptr(), eps, 0 if rope is None else rope.data_ptr(), 0 if rope is None else rope.numel() // D,
                          pos.data_ptr(), 0 if seq is None else seq.data_ptr(), table.data_ptr(), ts, tn)
        rc = self._append(self._ref, a, current(dev) if stream is None else _stream(stream))
        if rc:
            check(rc, "x100q_kv4_append_dev")
        return q_out

    def read(self, pos, table, seq=None, k_out=None, v_out=None, stream=None):
        """x100q_kv4_read_dev: the values (k, v) of the positions, fp16 [tokens, kv heads, dim]; both are made when neither is given."""
        torch, _, f16, _, i32_, _, _, device, current = _torch()
        what, dev, n = "Kv4Cache.read", device(), pos.numel()
        if dev != self.device:
            self._elsewhere(what, dev)
        if k_out is None and v_out is None:
            if stream is not None:
                _refuse(what, _OWN_STREAM)
            k_out, v_out = (torch.zeros(n, self.n_kv_heads, self.head_dim, dtype=f16, device=pos.device) for _ in range(2))
        if not (pos.dtype is i32_ and pos.get_device() == dev and pos.is_contiguous() and table.dtype is i32_ and table.get_device() == dev and table.is_contiguous()
                and (seq is None or (seq.dtype is i32_ and seq.get_device() == dev and seq.is_contiguous()))
                and (k_out is None or (k_out.dtype is f16 and k_out.get_device() == dev)) and (v_out is None or (v_out.dtype is f16 and v_out.get_device() == dev))):
            _placed(what, dev, k_out=(k_out, f16), v_out=(v_out, f16), pos=(pos, i32_), seq=(seq, i32_), table=(table, i32_))
        size = n * self.n_kv_heads * self.head_dim
        if not (table.dim() == 2 and (seq is None or seq.numel() == n) and (k_out is None or (k_out.numel() == size and k_out.is_contiguous()))
                and (v_out is None or (v_out.numel() == size and v_out.is_contiguous()))):
            _refuse(what, f"k_out and v_out have to be {size} contiguous values, the page table [sequences, entries], and seq as long as pos")
        tn, ts = table.shape
        rc = self._read(self._ref, pos.data_ptr(), 0 if seq is None else seq.data_ptr(), n, table.data_ptr(), ts, tn, 0 if k_out is None else k_out.data_ptr(),
                        0 if v_out is None else v_out.data_ptr(), current(dev) if stream is None else _stream(stream))
        if rc:
            check(rc, "x100q_kv4_read_dev")
        return k_out, v_out

    def attend_work(self, n_tokens: int, n_heads: int, n_seqs: int):
        """Scratch for attend(); calls that overlap on the GPU need one each."""
        torch = _torch()[0]
        return torch.empty(lib().x100q_kv4_attn_work(self._ref, n_tokens, n_heads, n_seqs), dtype=torch.uint8, device=self.pages.device)

    def attend(self, q, out, table, kv_len, q_start=None, max_q=1, scale=None, work=None, stream=None):
        """x100q_kv4_attn_dev: q [tokens, heads, dim] over the pages into out (made when None); q_start None: one token per sequence."""
        torch, kinds, _, _, i32_, _, u8, device, current = _torch()
        what, dev, D, dt, n = "Kv4Cache.attend", device(), self.head_dim, q.dtype, kv_len.numel()
        if dev != self.device:
            self._elsewhere(what, dev)
        kind = kinds.get(dt)
        if kind is None:
            _refuse(what, f"float32 or float16 is taken, not {dt}", X100_E_UNSUPPORTED)
        if q.dim() != 3 or q.shape[2] != D:
            _refuse(what, f"q has to be [tokens, heads, {D}]")
        rows, heads, _ = q.shape
        if stream is not None and (out is None or work is None):
            _refuse(what, _OWN_STREAM)
        if out is None:
            out = torch.empty(q.shape, dtype=dt, device=q.device)
        if work is None:
            work = self.attend_work(rows, heads, n)
        if not (q.get_device() == dev and out.dtype is dt and out.get_device() == dev and work.dtype is u8 and work.get_device() == dev and work.is_contiguous()
                and kv_len.dtype is i32_ and kv_len.get_device() == dev and kv_len.is_contiguous() and table.dtype is i32_ and table.get_device() == dev
                and table.is_contiguous() and (q_start is None or (q_start.dtype is i32_ and q_start.get_device() == dev and q_start.is_contiguous()))):
            _placed(what, dev, q=(q, dt), out=(out, dt), work=(work, u8), kv_len=(kv_len, i32_), table=(table, i32_), q_start=(q_start, i32_))
            _refuse(what, "work has to be contiguous")
        if not (out.shape == q.shape and table.dim() == 2 and table.shape[0] == n and (q_start is None or q_start.numel() == n + 1)):
            _refuse(what, "out has to be as q, the page table [sequences, entries] and q_start as long as kv_len, and one more")
        qs = heads * D if q.is_contiguous() else _token_stride(q, "q", what, D)
        os_ = heads * D if out.is_contiguous() else _token_stride(out, "out", what, D)
        a = _ATTN(kind, heads, q.data_ptr(), out.data_ptr(), qs, os_, 0 if q_start is None else q_start.data_ptr(), rows, max_q, kv_len.data_ptr(),
                        table.data_ptr(), table.shape[1], n, D ** -0.5 if scale is None else scale, work.data_ptr(), work.numel())
        rc = self._attn(self._ref, a, current(dev) if stream is None else _stream(stream))
        if rc:
            check(rc, "x100q_kv4_attn_dev")
        return out


def rope_table(n_pos: int, head_dim: int, base: float, stream=None, out=None):
    """x100q_rope_table_dev: (cos, sin) [n_pos, head_dim / 2, 2] for Kv4Cache.append, into out (made when None)."""
    torch, _, _, f32, _, _, _, device, _ = _torch()
    if out is None:
        if stream is not None:
            _refuse("rope_table", _OWN_STREAM)
        out = torch.empty(n_pos, head_dim // 2, 2, dtype=f32, device="cuda")
    _placed("rope_table", device(), out=(out, f32))
    if out.shape != (n_pos, head_dim // 2, 2) or not out.is_contiguous():
        _refuse("rope_table", f"out has to be [{n_pos}, {head_dim // 2}, 2] contiguous values")
    check(lib().x100q_rope_table_dev(out.data_ptr(), n_pos, head_dim, base, _stream(stream)), "x100q_rope_table_dev")
    return out


def add_rmsnorm_q8(x, w, q, scales, residual=None, residual_out=None, eps=1e-6, group=0, stream=None):
    """x100q_add_rmsnorm_q8_dev: rows of x (+ residual, the sum to residual_out) RMS-normed with w into int8 q and its scales."""
    torch, kinds, _, f32, _, i8, _, device, current = _torch()
    what, dev, dt = "add_rmsnorm_q8", device(), x.dtype
    kind = kinds.get(dt)
    if kind is None:
        _refuse(what, f"float32 or float16 is taken, not {dt}", X100_E_UNSUPPORTED)
    if x.dim() != 2:
        _refuse(what, "x has to be [rows, elements]")
    if not (x.get_device() == dev and w.dtype is f32 and w.get_device() == dev and q.dtype is i8 and q.get_device() == dev and scales.dtype is f32
            and scales.get_device() == dev and (residual is None or (residual.dtype is dt and residual.get_device() == dev))
            and (residual_out is None or (residual_out.dtype is dt and residual_out.get_device() == dev))):
        _placed(what, dev, x=(x, dt), residual=(residual, dt), residual_out=(residual_out, dt), w=(w, f32), q=(q, i8), scales=(scales, f32))
    shape = x.shape
    rows, d = shape
    if not (w.numel() == d and w.is_contiguous() and scales.is_contiguous() and scales.numel() == rows * (d // group if group > 0 else 1)):
        _refuse(what, f"w has to be {d} and scales [{rows}, groups] contiguous values")

    def pitch(t, name):
        if t is None:
            return 0
        if t.shape != shape or (d > 1 and t.stride(1) != 1):
            _refuse(what, f"{name} has to be [{rows}, {d}] with contiguous rows")
        return d if rows <= 1 or t.is_contiguous() else t.stride(0)

    a = _NORM(kind, rows, d, group, x.data_ptr(), 0 if residual is None else residual.data_ptr(), 0 if residual_out is None else residual_out.data_ptr(),
                   pitch(x, "x"), pitch(residual, "residual"), pitch(residual_out, "residual_out"), pitch(q, "q"), w.data_ptr(), eps, q.data_ptr(),
                   scales.data_ptr())
    rc = lib().x100q_add_rmsnorm_q8_dev(a, current(dev) if stream is None else _stream(stream))
    if rc:
        check(rc, "x100q_add_rmsnorm_q8_dev")


EP_HANDLE_BYTES = 64


class EpGroup:
    """x100q_ep handle: the peer-memory combine of expert-parallel partials.
    `exchange(bytes) -> list[bytes]` must return every process's handle in
    rank order (e.g. torch.distributed.all_gather_object)."""

    def __init__(self, world: int, rank: int, max_floats: int, exchange):
        self.h = lib().x100q_ep_create(world, rank, max_floats)
        if not self.h:
            check_last("x100q_ep_create")
        mine = C.create_string_buffer(EP_HANDLE_BYTES)
        check(lib().x100q_ep_handle(self.h, mine), "x100q_ep_handle")
        allh = b"".join(exchange(mine.raw))
        assert len(allh) == world * EP_HANDLE_BYTES
        buf = C.create_string_buffer(allh, len(allh))
        check(lib().x100q_ep_open(self.h, buf), "x100q_ep_open")

    def allreduce_dev(self, src, dst, n: int, accum: bool = False, stream=None):
        check(lib().x100q_ep_allreduce_dev(self.h, _p(src), _p(dst), n, 1 if accum else 0, _stream(stream)),
              "x100q_ep_allreduce_dev")

    def close(self):
        if getattr(self, "h", None) and _lib is not None:
            _lib.x100q_ep_destroy(self.h)
            self.h = None

    __del__ = close

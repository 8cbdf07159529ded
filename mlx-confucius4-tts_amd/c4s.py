"""Python binding of libc4s_sampling.so (C ABI in include/c4s_sampling.h and,
for the decoder layer's operators, include/c4s_layers.h).

ctypes only; torch supplies device memory and streams, nothing else. Loading
fails loudly when the library has not been built or no gfx950 device is
present: there is no CPU fallback in this package.
"""
from __future__ import annotations

import atexit
import ctypes as C
import os
import re
import struct
import weakref

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
LIB_PATH = os.path.join(HERE, "lib", "libc4s_sampling.so")
HEADER = os.path.join(REPO, "include", "c4s_sampling.h")
LAYERS_HEADER = os.path.join(REPO, "include", "c4s_layers.h")

OK, EINVAL, EHIP, ENOMEM, ETIMEOUT = 0, 1, 2, 3, 4
F32, BF16 = 0, 1
MODE_CHAIN = 0
P_PENALTY, P_TEMPERATURE, P_TOP_K, P_TOP_P = 1, 2, 4, 8
T_ARGMAX, T_DRAW = 16, 32
MODE_CUSTOM = 256
STAT_PATH, STAT_TOPP_EXACT, STAT_DRAW_EXACT, STAT_KEPT = 0, 1, 2, 3
STREAM_SEQUENTIAL = 1
STREAM_NO_SPECULATION = 2
W_BF16, W_F32, W_Q8 = 0, 1, 2   # c4s_head.wdtype, c4s_linear_desc.wdtype
NORM_LAYER, NORM_RMS = 0, 1
ACTS = {"none": 0, "gelu": 1, "silu": 2, "relu": 3}   # c4s_linear_desc.act
KV_BF16, KV_Q8 = 0, 1

_vp = C.c_void_p


class Rows(C.Structure):
    _fields_ = [("logits", _vp), ("ld", C.c_int64), ("dtype", C.c_int32), ("n_rows", C.c_int32),
                ("vocab", C.c_int32), ("hist_ids", _vp), ("hist_offsets", _vp),
                ("temperature", _vp), ("top_k", _vp), ("top_p", _vp), ("rep_penalty", _vp),
                ("min_keep", _vp), ("do_sample", _vp), ("row_active", _vp), ("rng_state", _vp),
                ("out_token", _vp), ("out_masked", _vp), ("out_stats", _vp), ("mode", C.c_uint32),
                ("hist_bits", _vp), ("stop_token", C.c_int32)]


class Stream(C.Structure):
    _fields_ = [("logits", _vp), ("ld", C.c_int64), ("step_stride", C.c_int64),
                ("n_steps", C.c_int32), ("n_rows", C.c_int32), ("vocab", C.c_int32),
                ("stop_token", C.c_int32), ("hist_ids", _vp), ("hist_offsets", _vp),
                ("temperature", _vp), ("top_k", _vp), ("top_p", _vp), ("rep_penalty", _vp),
                ("do_sample", _vp), ("rng_state", _vp), ("out_tokens", _vp), ("out_stats", _vp),
                ("flags", C.c_uint32)]


class Head(C.Structure):
    _fields_ = [("hidden", _vp), ("gamma", _vp), ("beta", _vp), ("eps", C.c_float),
                ("weight", _vp), ("bias", _vp), ("M", C.c_int32), ("D", C.c_int32),
                ("V", C.c_int32), ("logits", _vp), ("ld_out", C.c_int64), ("wdtype", C.c_int32),
                ("group", C.c_int32), ("wscale", _vp), ("wbias", _vp)]


class HeadWeights(C.Structure):
    """c4s_head_weights: the LM head's tensors on the device (c4s_head_weights_load)."""
    _fields_ = [("gamma", _vp), ("beta", _vp), ("weight", _vp), ("bias", _vp), ("wscale", _vp),
                ("wbias", _vp), ("D", C.c_int32), ("V", C.c_int32), ("wdtype", C.c_int32), ("group", C.c_int32)]


class Norm(C.Structure):
    _fields_ = [("M", C.c_int32), ("D", C.c_int32), ("kind", C.c_int32), ("eps", C.c_float),
                ("x", _vp), ("ldx", C.c_int64), ("x_dtype", C.c_int32), ("y_dtype", C.c_int32),
                ("y", _vp), ("ldy", C.c_int64), ("post", C.c_int32), ("gate_rows", C.c_int32),
                ("post_gamma", _vp), ("post_beta", _vp), ("gate", _vp), ("ld_gate", C.c_int64),
                ("res_scale", C.c_float), ("out_dtype", C.c_int32), ("gamma", _vp), ("beta", _vp),
                ("x_out", _vp), ("ld_x_out", C.c_int64), ("out", _vp), ("ld_out", C.c_int64)]


class Linear(C.Structure):
    _fields_ = [("M", C.c_int32), ("N", C.c_int32), ("K", C.c_int32), ("act", C.c_int32),
                ("x", _vp), ("ldx", C.c_int64), ("weight", _vp), ("wdtype", C.c_int32), ("group", C.c_int32),
                ("wscale", _vp), ("wbias", _vp), ("bias", _vp), ("residual", _vp), ("ld_res", C.c_int64),
                ("res_dtype", C.c_int32), ("out_dtype", C.c_int32), ("out", _vp), ("ld_out", C.c_int64)]


class KvCacheDesc(C.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("k_scale", _vp), ("v_scale", _vp), ("block_table", _vp),
                ("table_ld", C.c_int64), ("n_seqs", C.c_int32), ("max_pages", C.c_int32), ("n_pages", C.c_int32),
                ("page_size", C.c_int32), ("n_kv_heads", C.c_int32), ("head_dim", C.c_int32), ("store", C.c_int32)]


class KvRows(C.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("ldk", C.c_int64), ("ldv", C.c_int64), ("lens", _vp), ("rows_off", _vp),
                ("n_rows", C.c_int32), ("dtype", C.c_int32)]


class Attn(C.Structure):
    _fields_ = [("q", _vp), ("ldq", C.c_int64), ("out", _vp), ("ld_out", C.c_int64), ("lse", _vp), ("lens", _vp),
                ("rows_off", _vp), ("first", _vp), ("n_rows", C.c_int32), ("max_new", C.c_int32),
                ("n_heads", C.c_int32), ("scale", C.c_float)]


def header_functions(header: str = HEADER) -> list[str]:
    """Names of every function a public header declares."""
    txt = open(header).read()
    txt = re.sub(r"/\*.*?\*/", "", txt, flags=re.S)
    return sorted(set(re.findall(r"\b(c4s_[a-z0-9_]+)\s*\(", txt)))


_lib = None


def _share_torch_runtime() -> None:
    """torch ships its own HIP runtime library. When torch is present its runtime
    is started before this library loads, so that the library binds to the same
    runtime: a second HIP runtime in the process could not open the device."""
    try:
        import torch
    except ImportError:
        return
    if torch.cuda.device_count() > 0:
        torch.cuda.init()


def lib() -> C.CDLL:
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(f"{LIB_PATH} is not built; run __graft_entry__.build()")
    _share_torch_runtime()
    L = C.CDLL(LIB_PATH)
    L.c4s_create.argtypes = [C.c_int, C.POINTER(_vp)]
    L.c4s_destroy.argtypes = [_vp]
    L.c4s_last_error.argtypes = [_vp]
    L.c4s_last_error.restype = C.c_char_p
    L.c4s_version.restype = C.c_char_p
    L.c4s_sample_rows.argtypes = [_vp, C.POINTER(Rows), _vp]
    L.c4s_sample_stream.argtypes = [_vp, C.POINTER(Stream), _vp]
    L.c4s_stream_status.argtypes = [_vp, _vp]
    L.c4s_set_wait_limit.argtypes = [_vp, C.c_int32]
    L.c4s_hist_bits_init.argtypes = [_vp, _vp, _vp, C.c_int32, C.c_int32, _vp, _vp]
    L.c4s_lmhead.argtypes = [_vp, C.POINTER(Head), _vp]
    L.c4s_lmhead_sample.argtypes = [_vp, C.POINTER(Head), C.POINTER(Rows), _vp]
    L.c4s_lmhead_sample_noalloc.argtypes = [_vp, C.POINTER(Head), C.POINTER(Rows), _vp]
    L.c4s_seed_single.argtypes = [C.c_uint64]
    L.c4s_seed_single.restype = C.c_uint64
    L.c4s_seed_batch.argtypes = [C.c_uint64, C.c_int32, _vp]
    L.c4s_host_temperature.argtypes = [_vp, _vp, C.c_int32, C.c_float]
    L.c4s_host_repetition_penalty.argtypes = [_vp, _vp, C.c_int32, _vp, C.c_int64, C.c_float]
    L.c4s_host_top_k.argtypes = [_vp, _vp, C.c_int32, C.c_int32]
    L.c4s_host_top_p.argtypes = [_vp, _vp, C.c_int32, C.c_float, C.c_int32]
    L.c4s_host_argmax.argtypes = [_vp, _vp, C.c_int32, _vp]
    L.c4s_host_draw.argtypes = [_vp, _vp, C.c_int32, _vp, _vp]
    L.c4s_hbm_probe.argtypes = [_vp, _vp, _vp, C.c_int64, C.c_int32, _vp]
    L.c4s_tensor_read_f32.argtypes = [C.c_char_p, C.c_char_p, _vp, C.c_int64, _vp, _vp]
    L.c4s_head_weights_load.argtypes = [C.c_char_p, C.c_int32, C.c_int32, C.POINTER(HeadWeights)]
    L.c4s_head_weights_free.argtypes = [C.POINTER(HeadWeights)]
    L.c4s_weights_last_error.restype = C.c_char_p
    for f in (L.c4s_block_norm, L.c4s_linear):   # descriptors as bytes (_packer)
        f.argtypes = [_vp, C.c_char_p, _vp]
    for f in (L.c4s_kv_append, L.c4s_kv_read, L.c4s_attn):
        f.argtypes = [_vp, C.c_char_p, C.c_char_p, _vp]
    _lib = L
    return L


def _p(t):
    """Device (or host numpy) pointer of a tensor/array, or None."""
    if t is None:
        return None
    if hasattr(t, "data_ptr"):
        return t.data_ptr()
    return t.ctypes.data


def _stream_handle(stream):
    if stream is None:
        import torch
        return torch.cuda.current_stream().cuda_stream
    if hasattr(stream, "cuda_stream"):
        return stream.cuda_stream
    return stream


class C4SError(RuntimeError):
    pass


# Contexts still open when the interpreter exits are closed by an atexit hook:
# Python runs atexit hooks before it tears down modules and before the C
# runtime's exit handlers unload the HIP runtime (and, under a profiler, the
# profiler's tool library), so c4s_destroy's stream syncs and frees still find
# a live runtime. Leaving them to __del__ during module teardown would run
# those HIP calls in whatever order the garbage collector picks.
_live_contexts: "weakref.WeakSet[Context]" = weakref.WeakSet()


@atexit.register
def _close_live_contexts() -> None:
    for ctx in list(_live_contexts):
        try:
            ctx.close()
        except Exception:
            pass


def read_tensor(root: str, name: str):
    """One tensor of the reference's weight store (<root>.safetensors, else
    <root>/<name>.npy) as float32 numpy, read by the library on the host."""
    import numpy as np
    shape = np.zeros(8, np.int64)
    nd = C.c_int32(0)
    rc = lib().c4s_tensor_read_f32(root.encode(), name.encode(), None, 0, shape.ctypes.data, C.byref(nd))
    if rc:
        raise C4SError(f"tensor_read: code {rc}: {lib().c4s_weights_last_error().decode()}")
    out = np.empty(tuple(shape[: nd.value]), np.float32)
    rc = lib().c4s_tensor_read_f32(root.encode(), name.encode(), out.ctypes.data, out.size, shape.ctypes.data,
                                   C.byref(nd))
    if rc:
        raise C4SError(f"tensor_read: code {rc}: {lib().c4s_weights_last_error().decode()}")
    return out


def load_head_weights(root: str, wdtype: int = W_BF16, group: int = 64) -> HeadWeights:
    """final_norm.* and semantic_head.* of the store at `root` on the current
    device, in storage `wdtype`; free with free_head_weights."""
    hw = HeadWeights()
    rc = lib().c4s_head_weights_load(root.encode(), wdtype, group, C.byref(hw))
    if rc:
        raise C4SError(f"head_weights_load: code {rc}: {lib().c4s_weights_last_error().decode()}")
    return hw


def free_head_weights(hw: HeadWeights) -> None:
    lib().c4s_head_weights_free(C.byref(hw))


# The layer calls come once a layer and AR step, so their host time counts: what
# they check is checked in few Python operations (an attribute of a tensor costs
# about 0.1 us), messages are constants, and descriptors are packed as bytes,
# which takes half the time of filling a ctypes structure.

def _packer(cls):
    """pack(*fields) -> the bytes of a ctypes structure; pointers as integers (0: NULL)."""
    s = struct.Struct("@" + "".join({C.c_int32: "i", C.c_float: "f", C.c_int64: "q", _vp: "P"}[t]
                                    for _, t in cls._fields_) + "0P")
    assert s.size == C.sizeof(cls)
    return s.pack


_pack_norm, _pack_linear, _pack_rows, _pack_attn = (_packer(c) for c in (Norm, Linear, KvRows, Attn))


class _Torch:
    """torch's dtypes and its current stream, from the first context on."""
    kinds, bf16, f32, i32, u8, raw_stream = {}, None, None, None, None, None

    @classmethod
    def load(cls):
        import torch
        cls.kinds = {torch.float32: F32, torch.bfloat16: BF16}
        cls.bf16, cls.f32, cls.i32, cls.u8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8
        cls.raw_stream = torch._C._cuda_getCurrentRawStream


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _refuse(t, what, device):
    """Raises what is wrong with tensor t. (A kernel that is given an address of the host's, or of another GPU,
    faults and takes the process with it, so every helper below looks where its tensor lives.)"""
    raise ValueError(what if t.get_device() == device else f"{what}; it must be on the context's device, cuda:{device}")


def _vector(t, n, what, device):
    """The address of a contiguous float32 vector of n values on this device; 0 of None."""
    if t is None:
        return 0
    if t.dtype is _Torch.f32 and t.numel() == n and t.is_contiguous() and t.get_device() == device:
        return t.data_ptr()
    _refuse(t, what, device)


def _i32(t, n, what, device):
    """The address of a contiguous int32 vector of n values on this device; 0 of None."""
    if t is None:
        return 0
    if t.dtype is _Torch.i32 and t.numel() == n and t.is_contiguous() and t.get_device() == device:
        return t.data_ptr()
    _refuse(t, what, device)


def _rows(t, shape, what, device, own=False):
    """(address, row stride, C4S_DTYPE_*) of a [rows][width] tensor of this shape (own: which is its own) on this
    device, bfloat16 or float32, whose rows are contiguous; (0, 0, F32) of None."""
    if t is None:
        return 0, 0, F32
    kind = _Torch.kinds.get(t.dtype)
    if kind is not None and t.get_device() == device and (own or t.shape == shape):
        ld, one = t.stride()
        if one == 1 or shape[1] <= 1:
            return t.data_ptr(), (ld if shape[0] > 1 else shape[1]), kind
    _refuse(t, what, device)


def _heads(t, shape, what, device, own=False):
    """As _rows, of a [rows][heads][dim] tensor."""
    kind = _Torch.kinds.get(t.dtype)
    if kind is not None and t.get_device() == device and (own or t.shape == shape):
        ld, dim, one = t.stride()
        if one == 1 and (dim == shape[2] or shape[1] == 1):
            return t.data_ptr(), (ld if shape[0] > 1 else shape[1] * shape[2]), kind
    _refuse(t, what, device)


class KvCache:
    """The tensors of one layer's paged cache (c4s_kv_cache in include/c4s_layers.h):

    k            [n_pages][n_kv_heads][page_size][head_dim]  bfloat16, or int8 codes
    v            [n_pages][n_kv_heads][head_dim][page_size]  as k
    k_scale, v_scale  [n_pages][n_kv_heads][page_size]       float32, with int8 codes
    block_table  [n_seqs][max_pages]                         int32, shared by the layers

    The object keeps the tensors and their addresses; their contents may change
    at any time."""

    def __init__(self, k, v, block_table, k_scale=None, v_scale=None):
        import torch
        _need(k.dim() == 4 and k.is_contiguous() and v.is_contiguous(), "KvCache: k and v must be contiguous, 4-d")
        pages, heads, size, dim = k.shape
        _need(tuple(v.shape) == (pages, heads, dim, size), "KvCache: v must be [n_pages][n_kv_heads][head_dim][page_size]")
        _need(k.dtype == v.dtype and k.dtype in (torch.bfloat16, torch.int8), "KvCache: k and v must be bfloat16 or int8")
        q8 = k.dtype == torch.int8
        _need(q8 == (k_scale is not None) and q8 == (v_scale is not None), "KvCache: scales go with int8 codes")
        for s in (k_scale, v_scale):
            _need(s is None or (s.dtype == torch.float32 and s.is_contiguous() and tuple(s.shape) == (pages, heads, size)),
                  "KvCache: scales must be contiguous float32 [n_pages][n_kv_heads][page_size]")
        _need(block_table.dtype == torch.int32 and block_table.dim() == 2 and
              (block_table.shape[1] <= 1 or block_table.stride(1) == 1), "KvCache: block_table must be int32 rows")
        self.device = k.get_device()
        _need(self.device >= 0 and all(t is None or t.get_device() == self.device for t in (v, block_table, k_scale, v_scale)),
              "KvCache: all tensors must be on one GPU")
        n_seqs, max_pages = block_table.shape
        self.k, self.v, self.k_scale, self.v_scale, self.block_table = k, v, k_scale, v_scale, block_table
        self.n_seqs, self.n_kv_heads, self.head_dim, self.page_size = n_seqs, heads, dim, size
        self.desc = KvCacheDesc(_p(k), _p(v), _p(k_scale), _p(v_scale), _p(block_table),
                                block_table.stride(0) if n_seqs > 1 else max_pages, n_seqs, max_pages, pages, size,
                                heads, dim, KV_Q8 if q8 else KV_BF16)
        self.packed = bytes(self.desc)

    @classmethod
    def empty(cls, n_pages, n_kv_heads, page_size, head_dim, block_table, q8=False):
        """A cache of its own on block_table's device; nothing in it is set."""
        import torch
        t, d = torch.int8 if q8 else torch.bfloat16, block_table.device
        k = torch.empty((n_pages, n_kv_heads, page_size, head_dim), dtype=t, device=d)
        v = torch.empty((n_pages, n_kv_heads, head_dim, page_size), dtype=t, device=d)
        scales = [torch.empty((n_pages, n_kv_heads, page_size), device=d) for _ in range(2)] if q8 else [None, None]
        return cls(k, v, block_table, *scales)


class Context:
    """One library context on one device (not thread-safe)."""

    def __init__(self, device: int = 0):
        self._h = _vp()
        _Torch.load()
        rc = lib().c4s_create(device, C.byref(self._h))
        if rc != OK:
            raise C4SError(f"c4s_create(device={device}) failed with code {rc} "
                           "(no gfx950 device visible?)")
        self.device = device
        _live_contexts.add(self)

    def close(self):
        if self._h:
            h, self._h = self._h, _vp()
            lib().c4s_destroy(h)
        _live_contexts.discard(self)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, rc, what):
        if rc != OK:
            msg = lib().c4s_last_error(self._h).decode()
            raise C4SError(f"{what}: code {rc}: {msg}")

    # ---- device entry points (torch tensors on the GPU) ------------------------
    def sample_rows(self, logits, hist_ids, hist_off, temp, top_k, top_p, pen, rng, out_token,
                    do_sample=None, min_keep=None, row_active=None, out_masked=None,
                    out_stats=None, mode=MODE_CHAIN, vocab=None, stream=None, hist_bits=None,
                    stop_token=-1):
        import torch
        n_rows, ld = logits.shape
        r = Rows(logits=_p(logits), ld=ld, dtype=BF16 if logits.dtype == torch.bfloat16 else F32,
                 n_rows=n_rows, vocab=vocab or ld, hist_ids=_p(hist_ids), hist_offsets=_p(hist_off),
                 temperature=_p(temp), top_k=_p(top_k), top_p=_p(top_p), rep_penalty=_p(pen),
                 min_keep=_p(min_keep), do_sample=_p(do_sample), row_active=_p(row_active),
                 rng_state=_p(rng), out_token=_p(out_token), out_masked=_p(out_masked),
                 out_stats=_p(out_stats), mode=mode, hist_bits=_p(hist_bits), stop_token=stop_token)
        self._check(lib().c4s_sample_rows(self._h, C.byref(r), _stream_handle(stream)), "sample_rows")

    def hist_bits_init(self, hist_ids, hist_off, n_rows, vocab, hist_bits, stream=None):
        """hist_bits[b] (int32 words, [n_rows][(vocab+31)//32]) = the set of row b's CSR history."""
        self._check(lib().c4s_hist_bits_init(self._h, _p(hist_ids), _p(hist_off), n_rows, vocab, _p(hist_bits),
                                             _stream_handle(stream)), "hist_bits_init")

    def sample_stream(self, logits, hist_ids, hist_off, temp, top_k, top_p, pen, rng, out_tokens,
                      do_sample=None, stop_token=-1, out_stats=None, stream=None, sequential=False,
                      speculate=True):
        n_steps, n_rows, ld = logits.shape
        s = Stream(logits=_p(logits), ld=ld, step_stride=n_rows * ld, n_steps=n_steps,
                   n_rows=n_rows, vocab=ld, stop_token=stop_token, hist_ids=_p(hist_ids),
                   hist_offsets=_p(hist_off), temperature=_p(temp), top_k=_p(top_k),
                   top_p=_p(top_p), rep_penalty=_p(pen), do_sample=_p(do_sample),
                   rng_state=_p(rng), out_tokens=_p(out_tokens), out_stats=_p(out_stats),
                   flags=(STREAM_SEQUENTIAL if sequential else 0) | (0 if speculate else STREAM_NO_SPECULATION))
        self._check(lib().c4s_sample_stream(self._h, C.byref(s), _stream_handle(stream)),
                    "sample_stream")

    def stream_status(self, stream=None):
        """C4S_OK, or C4S_ETIMEOUT when a sample_stream call gave up a row (the
        record is cleared); synchronizes `stream` first."""
        return lib().c4s_stream_status(self._h, _stream_handle(stream))

    def set_wait_limit(self, polls):
        """Polls of the speculative chains' bounded waits before they give up (<= 0: default)."""
        self._check(lib().c4s_set_wait_limit(self._h, int(polls)), "set_wait_limit")

    @staticmethod
    def _head(hidden, gamma, beta, weight, bias, logits, eps, quant=None):
        """quant: None for bf16 or fp32 weights (from weight's dtype), else
        (scales, biases, group) of 8-bit codes (uint8 weight)."""
        M, D = hidden.shape
        V = weight.shape[0]
        kind = {"torch.bfloat16": W_BF16, "torch.int16": W_BF16, "torch.float32": W_F32,
                "torch.uint8": W_Q8}.get(str(weight.dtype))
        if kind is None:
            raise ValueError(f"lmhead: unsupported weight dtype {weight.dtype}")
        if (kind == W_Q8) != (quant is not None):
            raise ValueError("lmhead: 8-bit weights need quant=(scales, biases, group), others none")
        ws, wb, group = quant if quant is not None else (None, None, 0)
        return Head(hidden=_p(hidden), gamma=_p(gamma), beta=_p(beta), eps=eps, weight=_p(weight),
                    bias=_p(bias), M=M, D=D, V=V, logits=_p(logits),
                    ld_out=(logits.shape[1] if logits is not None else V), wdtype=kind, group=group,
                    wscale=_p(ws), wbias=_p(wb))

    def lmhead_loaded(self, hw: HeadWeights, hidden, logits, eps=1e-5, stream=None):
        """c4s_lmhead with the tensors of load_head_weights."""
        M, D = hidden.shape
        if D != hw.D:
            raise ValueError(f"hidden has D={D}, the head D={hw.D}")
        h = Head(hidden=_p(hidden), gamma=hw.gamma, beta=hw.beta, eps=eps, weight=hw.weight, bias=hw.bias,
                 M=M, D=D, V=hw.V, logits=_p(logits), ld_out=logits.shape[1], wdtype=hw.wdtype, group=hw.group,
                 wscale=hw.wscale, wbias=hw.wbias)
        self._check(lib().c4s_lmhead(self._h, C.byref(h), _stream_handle(stream)), "lmhead")

    def lmhead_sample_loaded(self, hw: HeadWeights, hidden, temp, top_k, top_p, pen, rng, out_token, logits=None,
                             hist_ids=None, hist_off=None, hist_bits=None, do_sample=None, stop_token=-1, eps=1e-5,
                             stream=None):
        """c4s_lmhead_sample with the tensors of load_head_weights: one AR step
        from the hidden rows to the tokens (text2semantic.cpp:297-337)."""
        M, D = hidden.shape
        if D != hw.D:
            raise ValueError(f"hidden has D={D}, the head D={hw.D}")
        h = Head(hidden=_p(hidden), gamma=hw.gamma, beta=hw.beta, eps=eps, weight=hw.weight, bias=hw.bias,
                 M=M, D=D, V=hw.V, logits=_p(logits), ld_out=hw.V if logits is None else logits.shape[1],
                 wdtype=hw.wdtype, group=hw.group, wscale=hw.wscale, wbias=hw.wbias)
        r = Rows(hist_ids=_p(hist_ids), hist_offsets=_p(hist_off), temperature=_p(temp), top_k=_p(top_k),
                 top_p=_p(top_p), rep_penalty=_p(pen), do_sample=_p(do_sample), rng_state=_p(rng),
                 out_token=_p(out_token), mode=MODE_CHAIN, hist_bits=_p(hist_bits), stop_token=stop_token)
        self._check(lib().c4s_lmhead_sample(self._h, C.byref(h), C.byref(r), _stream_handle(stream)),
                    "lmhead_sample")

    def lmhead(self, hidden, gamma, beta, weight, bias, logits, eps=1e-5, stream=None, quant=None):
        h = self._head(hidden, gamma, beta, weight, bias, logits, eps, quant)
        self._check(lib().c4s_lmhead(self._h, C.byref(h), _stream_handle(stream)), "lmhead")

    def lmhead_sample(self, hidden, gamma, beta, weight, bias, hist_ids, hist_off, temp, top_k,
                      top_p, pen, rng, out_token, logits=None, do_sample=None, out_masked=None,
                      out_stats=None, eps=1e-5, stream=None, hist_bits=None, stop_token=-1, quant=None):
        h = self._head(hidden, gamma, beta, weight, bias, logits, eps, quant)
        r = Rows(hist_ids=_p(hist_ids), hist_offsets=_p(hist_off), temperature=_p(temp),
                 top_k=_p(top_k), top_p=_p(top_p), rep_penalty=_p(pen), do_sample=_p(do_sample),
                 rng_state=_p(rng), out_token=_p(out_token), out_masked=_p(out_masked),
                 out_stats=_p(out_stats), mode=MODE_CHAIN, hist_bits=_p(hist_bits), stop_token=stop_token)
        self._check(lib().c4s_lmhead_sample(self._h, C.byref(h), C.byref(r), _stream_handle(stream)),
                    "lmhead_sample")

    def lmhead_sample_noalloc(self, hidden, gamma, beta, weight, bias, hist_ids, hist_off, temp, top_k,
                              top_p, pen, rng, out_token, logits=None, do_sample=None, out_masked=None,
                              out_stats=None, eps=1e-5, stream=None, hist_bits=None, stop_token=-1, quant=None):
        """c4s_lmhead_sample with its workspace in the library's static device scratch."""
        h = self._head(hidden, gamma, beta, weight, bias, logits, eps, quant)
        r = Rows(hist_ids=_p(hist_ids), hist_offsets=_p(hist_off), temperature=_p(temp),
                 top_k=_p(top_k), top_p=_p(top_p), rep_penalty=_p(pen), do_sample=_p(do_sample),
                 rng_state=_p(rng), out_token=_p(out_token), out_masked=_p(out_masked),
                 out_stats=_p(out_stats), mode=MODE_CHAIN, hist_bits=_p(hist_bits), stop_token=stop_token)
        self._check(lib().c4s_lmhead_sample_noalloc(self._h, C.byref(h), C.byref(r), _stream_handle(stream)),
                    "lmhead_sample_noalloc")

    # ---- the decoder layer's operators (include/c4s_layers.h) ---------------------------
    def _queue(self, stream):
        """The HIP stream of a call: the given one, or this device's current one."""
        return _Torch.raw_stream(self.device) if stream is None else _stream_handle(stream)

    def block_norm(self, x, gamma, beta, out, y=None, x_out=None, post=False, post_gamma=None, post_beta=None,
                   gate=None, gate_rows=1, scale=1.0, eps=1e-5, rms=False, stream=None):
        """r = x + scale * gate (.) u with u = y, or norm(y) when post; x_out = r;
        out = norm(r). x, y, x_out, out: [rows][D], bfloat16 or float32; gate:
        float32 [ceil(rows / gate_rows)][D]; without y, r = x."""
        shape, dev = x.shape, self.device
        M, D = shape
        xp, ldx, xt = _rows(x, shape, "block_norm: x must be bfloat16 or float32, its rows contiguous", dev, True)
        yp, ldy, yt = _rows(y, shape, "block_norm: y must be bfloat16 or float32 of x's shape, its rows contiguous", dev)
        op, ldo, ot = _rows(out, shape, "block_norm: out must be bfloat16 or float32 of x's shape, its rows contiguous", dev)
        xo = ldxo = g = ldg = 0
        if x_out is not None:
            xo, ldxo, t = _rows(x_out, shape, "block_norm: x_out must have x's shape and dtype, its rows contiguous", dev)
            _need(t == xt, "block_norm: x_out must have x's dtype")
        if gate is not None:
            g, ldg, t = _rows(gate, (gate.shape[0], D), "block_norm: gate must be float32 [ceil(rows / gate_rows)][D]", dev)
            _need(t == F32 and gate_rows >= 1 and gate.shape[0] * gate_rows >= M,
                  "block_norm: gate must be float32 [ceil(rows / gate_rows)][D]")
        if post_gamma is not None or post_beta is not None:
            post_gamma = _vector(post_gamma, D, "block_norm: post_gamma must be a float32 vector of D", dev)
            post_beta = _vector(post_beta, D, "block_norm: post_beta must be a float32 vector of D", dev)
        rc = _lib.c4s_block_norm(
            self._h, _pack_norm(M, D, NORM_RMS if rms else NORM_LAYER, eps, xp, ldx, xt, yt, yp, ldy, 1 if post else 0,
                                gate_rows, post_gamma or 0, post_beta or 0, g, ldg, scale, ot,
                                _vector(gamma, D, "block_norm: gamma must be a float32 vector of D", dev),
                                _vector(beta, D, "block_norm: beta must be a float32 vector of D", dev), xo, ldxo, op, ldo),
            _Torch.raw_stream(self.device) if stream is None else _stream_handle(stream))
        if rc:
            self._check(rc, "block_norm")

    def linear(self, x, weight, out, bias=None, residual=None, act="none", quant=None, stream=None):
        """out = residual + act(x @ weight^T + bias). x: bfloat16 [M][K]; weight:
        [N][K], bfloat16, or uint8 codes with quant=(scales, offsets, group);
        residual, out: [M][N], bfloat16 or float32; act: none, gelu, silu, relu."""
        xs, ws, dev = x.shape, weight.shape, self.device
        M, K = xs
        N = ws[0]
        xp, ldx, t = _rows(x, xs, "linear: x must be bfloat16 [M][K], its rows contiguous", dev, True)
        if not (t == BF16 and ws == (N, K) and weight.is_contiguous() and weight.get_device() == dev):
            _refuse(weight, "linear: x must be bfloat16 [M][K], weight contiguous [N][K]", dev)
        sp = bp = group = 0
        wt = W_BF16
        if quant is not None:
            scales, offsets, group = quant
            wt = W_Q8
            if not (group > 0 and scales.shape == offsets.shape == (N, K // group)):
                raise ValueError("linear: scales and offsets must be contiguous float32 [N][K / group]")
            sp = _vector(scales, N * (K // group), "linear: scales must be contiguous float32 [N][K / group]", dev)
            bp = _vector(offsets, N * (K // group), "linear: offsets must be contiguous float32 [N][K / group]", dev)
        if weight.dtype is not (_Torch.bf16 if quant is None else _Torch.u8):
            raise ValueError("linear: weights are bfloat16, or uint8 with quant=(scales, offsets, group)")
        kind = ACTS.get(act)
        if kind is None:
            raise ValueError("linear: act must be none, gelu, silu or relu")
        shape = (M, N)
        op, ldo, ot = _rows(out, shape, "linear: out must be bfloat16 or float32 [M][N], its rows contiguous", dev)
        rp, ldr, rt = _rows(residual, shape, "linear: residual must be bfloat16 or float32 [M][N], its rows contiguous", dev)
        rc = _lib.c4s_linear(
            self._h, _pack_linear(M, N, K, kind, xp, ldx, weight.data_ptr(), wt, group, sp, bp,
                                  _vector(bias, N, "linear: bias must be a float32 vector of N", dev), rp, ldr, rt, ot, op, ldo),
            _Torch.raw_stream(self.device) if stream is None else _stream_handle(stream))
        if rc:
            self._check(rc, "linear")

    def _kv_rows(self, cache, k, v, lens, rows_off):
        shape, dev = k.shape, self.device
        rows, heads, dim = shape
        if not (heads == cache.n_kv_heads and dim == cache.head_dim and cache.device == dev):
            raise ValueError(f"kv rows: k must be [rows][n_kv_heads][head_dim], the cache on the context's device, cuda:{dev}")
        kp, ldk, t = _heads(k, shape, "kv rows: k must be bfloat16 or float32, a row contiguous", dev, True)
        vp, ldv, vt = _heads(v, shape, "kv rows: v must have k's shape and dtype, a row contiguous", dev)
        _need(vt == t, "kv rows: k and v must have one dtype")
        n = cache.n_seqs
        return _pack_rows(kp, vp, ldk, ldv, _i32(lens, n, "kv rows: lens must be an int32 vector of n_seqs", dev),
                          _i32(rows_off, n + 1, "kv rows: rows_off must be an int32 vector of n_seqs + 1", dev), rows, t)

    def kv_append(self, cache, k, v, lens, rows_off=None, stream=None):
        """The rows k, v (bfloat16 [rows][n_kv_heads][head_dim]) into the cache, as
        the last positions of lens[b]; rows_off as in include/c4s_layers.h."""
        rc = _lib.c4s_kv_append(self._h, cache.packed, self._kv_rows(cache, k, v, lens, rows_off), self._queue(stream))
        if rc:
            self._check(rc, "kv_append")

    def kv_read(self, cache, k, v, lens, rows_off=None, stream=None):
        """The cache's values at the last positions of lens[b] into the rows k, v
        (bfloat16 or float32)."""
        rc = _lib.c4s_kv_read(self._h, cache.packed, self._kv_rows(cache, k, v, lens, rows_off), self._queue(stream))
        if rc:
            self._check(rc, "kv_read")

    def attn(self, q, cache, lens, out, rows_off=None, max_new=None, scale=None, first=None, lse=None, stream=None):
        """Attention of the rows q (bfloat16 [rows][n_heads][head_dim], the last
        positions of lens[b]) over the cache, into out. max_new: with rows_off the most
        rows a sequence has, by which the kernel is chosen (default: all rows); scale:
        1 / sqrt(head_dim) by default."""
        shape, dev = q.shape, self.device
        rows, heads, dim = shape
        qp, ldq, qt = _heads(q, shape, "attn: q must be bfloat16 [rows][n_heads][head_dim], a row contiguous", dev, True)
        op, ldo, ot = _heads(out, shape, "attn: out must be bfloat16 of q's shape, a row contiguous", dev)
        if not (qt == BF16 and ot == BF16 and dim == cache.head_dim and cache.device == dev):
            raise ValueError("attn: q and out must be bfloat16 [rows][n_heads][head_dim], head_dim as the cache's, "
                             f"the cache on the context's device, cuda:{dev}")
        n = cache.n_seqs
        rc = _lib.c4s_attn(
            self._h, cache.packed,
            _pack_attn(qp, ldq, op, ldo, _vector(lse, rows * heads, "attn: lse must be contiguous float32 [rows][n_heads]", dev),
                       _i32(lens, n, "attn: lens must be an int32 vector of n_seqs", dev),
                       _i32(rows_off, n + 1, "attn: rows_off must be an int32 vector of n_seqs + 1", dev),
                       _i32(first, n, "attn: first must be an int32 vector of n_seqs", dev), rows,
                       rows if max_new is None or max_new > rows else max_new, heads,
                       dim ** -0.5 if scale is None else scale),
            self._queue(stream))
        if rc:
            self._check(rc, "attn")

    def hbm_probe(self, src, dst, nbytes, mode=0, stream=None):
        self._check(lib().c4s_hbm_probe(self._h, _p(src), _p(dst), nbytes, mode,
                                        _stream_handle(stream)), "hbm_probe")

    # ---- host-buffer single-row helpers (numpy, synchronous) ---------------------
    def host_temperature(self, row, temp):
        import numpy as np
        v = np.array(row, dtype=np.float32, copy=True)
        self._check(lib().c4s_host_temperature(self._h, v.ctypes.data, v.size, temp), "temperature")
        return v

    def host_repetition_penalty(self, row, ids, pen):
        import numpy as np
        v = np.array(row, dtype=np.float32, copy=True)
        ids = np.ascontiguousarray(ids, dtype=np.int32)
        self._check(lib().c4s_host_repetition_penalty(self._h, v.ctypes.data, v.size,
                                                      ids.ctypes.data if ids.size else None,
                                                      ids.size, pen), "repetition_penalty")
        return v

    def host_top_k(self, row, k):
        import numpy as np
        v = np.array(row, dtype=np.float32, copy=True)
        self._check(lib().c4s_host_top_k(self._h, v.ctypes.data, v.size, k), "top_k")
        return v

    def host_top_p(self, row, p, min_keep=1):
        import numpy as np
        v = np.array(row, dtype=np.float32, copy=True)
        self._check(lib().c4s_host_top_p(self._h, v.ctypes.data, v.size, p, min_keep), "top_p")
        return v

    def host_argmax(self, row):
        import numpy as np
        v = np.ascontiguousarray(row, dtype=np.float32)
        out = C.c_int32(0)
        self._check(lib().c4s_host_argmax(self._h, v.ctypes.data, v.size, C.addressof(out)), "argmax")
        return out.value

    def host_draw(self, row, state):
        import numpy as np
        v = np.ascontiguousarray(row, dtype=np.float32)
        s = C.c_uint64(state)
        out = C.c_int32(0)
        self._check(lib().c4s_host_draw(self._h, v.ctypes.data, v.size, C.addressof(s),
                                        C.addressof(out)), "draw")
        return out.value, s.value


def seed_single(seed: int) -> int:
    return int(lib().c4s_seed_single(seed))


def seed_batch(seed: int, n: int):
    import numpy as np
    out = np.zeros(n, dtype=np.uint64)
    lib().c4s_seed_batch(seed, n, out.ctypes.data)
    return out

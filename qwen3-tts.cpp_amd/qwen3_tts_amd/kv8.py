"""ctypes binding of the 8-bit attention cache's operators (include/q3t_kv8.h)
over torch tensors on the GPU.

A cache is the caller's tensors: codes k, v int8 [S, H, C, D], scales ks, vs
float32 [S, H, C / 16] and, where slots are to be evicted, acc float32
[S, H, C], the attention weight each slot has drawn; S sequences, H key/value
heads, C slots (a multiple of 16), D 64 or 128.  Calls run on the tensors'
device and torch's current stream there, and return without waiting; lengths
and positions are int32 tensors on that device.
"""
import ctypes
import struct

import numpy as np
import torch

from .device import load_library

KV8_EXPORTS = [
    "q3t_kv8_last_error", "q3t_kv8_rope_freqs", "q3t_kv8_rope", "q3t_kv8_append", "q3t_kv8_attend_ws",
    "q3t_kv8_attend", "q3t_kv8_evict", "q3t_kv8_read",
]

BLOCK = 16
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_SCALINGS = {"none": 0, "linear": 1, "base": 2, "turns": 3}

_vp, _i32, _i64, _f32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float


class CCache(ctypes.Structure):
    """q3t_kv8"""
    _fields_ = [("k", _vp), ("v", _vp), ("ks", _vp), ("vs", _vp), ("acc", _vp), ("seq", _i64), ("head", _i64),
                ("scale_seq", _i64), ("scale_head", _i64), ("acc_seq", _i64), ("acc_head", _i64), ("n_seq", _i32),
                ("n_kv_head", _i32), ("n_slots", _i32), ("head_dim", _i32)]


class CRopeRows(ctypes.Structure):
    """q3t_kv8_rope_rows"""
    _fields_ = [("x", _vp), ("y", _vp), ("x_token", _i64), ("x_head", _i64), ("y_token", _i64), ("y_head", _i64),
                ("gain", _vp), ("n_head", _i32), ("x_type", _i32), ("y_type", _i32)]


class CAttendArgs(ctypes.Structure):
    """q3t_kv8_attend_args"""
    _fields_ = [("q", _vp), ("out", _vp), ("q_seq", _i64), ("q_row", _i64), ("q_head", _i64), ("o_seq", _i64),
                ("o_row", _i64), ("o_head", _i64), ("q_type", _i32), ("o_type", _i32), ("n_rows", _i32),
                ("n_head", _i32), ("lens", _vp), ("len0", _i32), ("n_new", _vp), ("max_len", _i32), ("causal", _i32),
                ("scale", _f32), ("weights", _i32)]


def _packer(cls):
    """A struct.Struct with the fields of a ctypes structure at their places (filling one of these is a call's
    largest host cost otherwise)."""
    code, at = "", 0
    for name, kind in cls._fields_:
        f = getattr(cls, name)
        code += "%dx" % (f.offset - at) if f.offset > at else ""
        code += {_vp: "Q", _i64: "q", _i32: "i", _f32: "f"}[kind]
        at = f.offset + f.size
    return struct.Struct("=" + code + ("%dx" % (ctypes.sizeof(cls) - at) if ctypes.sizeof(cls) > at else ""))


_pack_rope, _pack_attend = _packer(CRopeRows).pack, _packer(CAttendArgs).pack

_lib = None


def load_kv8_library():
    """the device library (lib/libq3t_hip.so) with the cache operators' entry points typed"""
    global _lib
    if _lib is None:
        lib = load_library()
        cc = ctypes.POINTER(CCache)
        lib.q3t_kv8_last_error.argtypes = []
        lib.q3t_kv8_last_error.restype = ctypes.c_char_p
        lib.q3t_kv8_rope_freqs.argtypes = [_i32, ctypes.c_double, _i32, ctypes.c_double, _i32, _vp]
        lib.q3t_kv8_rope.argtypes = [_i32, _vp, _i32, _i64, _i32, _i32, _i32, _vp, _i32, _vp,
                                     _f32, _f32, _vp]
        lib.q3t_kv8_append.argtypes = [_i32, cc, _vp, _vp, _i32, _i64, _i64, _i64, _i32, _vp, _i32, _vp, _vp]
        lib.q3t_kv8_attend_ws.argtypes = [cc, _vp]
        lib.q3t_kv8_attend_ws.restype = _i64
        lib.q3t_kv8_attend.argtypes = [_i32, cc, _vp, _vp, _i64, _vp]
        lib.q3t_kv8_evict.argtypes = [_i32, cc, cc, _vp, _i32, _i32, _i32, _i32, _vp, _vp, _vp]
        lib.q3t_kv8_read.argtypes = [_i32, cc, _vp, _i32, _i32, _i32, _vp, _vp, _vp]
        _lib = lib
    return _lib


class Kv8Error(RuntimeError):
    pass


def _check(rc, what):
    if rc < 0:
        raise Kv8Error(f"{what}: {load_kv8_library().q3t_kv8_last_error().decode()}")
    return rc


def _need(ok, message):
    if not ok:
        raise Kv8Error(message)


def _ints(t, n, index, what):
    """Address of an int32 tensor of n values on GPU `index` (0 for None)."""
    if t is None:
        return 0
    if t.dtype is not torch.int32 or t.get_device() != index or t.shape != (n,) or not t.is_contiguous():
        raise Kv8Error(f"{what} must be {n} contiguous int32 on the same GPU")
    return t.data_ptr()


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(index):
    """torch's current stream on GPU `index`"""
    return _raw_stream(index) if _raw_stream else torch.cuda.current_stream(index).cuda_stream


class Cache:
    """The caller's tensors as one cache (a view: it holds no memory of its own)."""

    def __init__(self, k, v, ks, vs, acc=None):
        _need(k.dim() == 4 and k.is_cuda, "codes must be [S, H, C, D] on a GPU")
        s, h, c, d = k.shape
        both = (k, v)
        _need(all(t.dtype == torch.int8 and t.shape == k.shape and t.device == k.device for t in both),
              "k and v must be int8 of one shape and device")
        _need(k.stride() == v.stride() and k.stride(3) == 1 and k.stride(2) == d, "codes' slots must be dense, k and v alike")
        _need(all(t.dtype == torch.float32 and t.shape == (s, h, c // BLOCK) and t.device == k.device for t in (ks, vs)),
              "scales must be float32 [S, H, C / 16]")
        _need(ks.stride() == vs.stride() and ks.stride(2) == 1, "scales' blocks must be dense, ks and vs alike")
        if acc is not None:
            _need(acc.dtype == torch.float32 and acc.shape == (s, h, c) and acc.device == k.device and acc.stride(2) == 1,
                  "acc must be float32 [S, H, C] with dense slots")
        self.tensors = (k, v, ks, vs, acc)      # keeps the memory alive
        self.device, self.index, self.shape = k.device, k.get_device(), (s, h, c, d)
        self.c = CCache(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), None if acc is None else acc.data_ptr(),
                        k.stride(0), k.stride(1), ks.stride(0), ks.stride(1), 0 if acc is None else acc.stride(0),
                        0 if acc is None else acc.stride(1), s, h, c, d)
        self.ref = ctypes.byref(self.c)


def empty(n_seq, n_kv_head, n_slots, head_dim, device="cuda", weights=True):
    """A cache of zeroed tensors with room for n_slots slots (rounded up to a multiple of 16)."""
    c = -(-n_slots // BLOCK) * BLOCK
    k, v = (torch.zeros(n_seq, n_kv_head, c, head_dim, dtype=torch.int8, device=device) for _ in range(2))
    ks, vs = (torch.zeros(n_seq, n_kv_head, c // BLOCK, device=device) for _ in range(2))
    return Cache(k, v, ks, vs, torch.zeros(n_seq, n_kv_head, c, device=device) if weights else None)


def rope_freqs(rot_dim, theta, scaling="none", factor=1.0, n_trained=0):
    """Frequencies of the rot_dim / 2 pairs, float64 (q3t_kv8_rope_freqs).  scaling: "none", "linear" (all divided by
    factor), "base" (a larger theta) or "turns" (the slow ones divided, the fast ones kept)."""
    _need(scaling in _SCALINGS, f"unknown scaling {scaling!r}")
    out = np.empty(max(int(rot_dim) // 2, 1), np.float64)
    _check(load_kv8_library().q3t_kv8_rope_freqs(int(rot_dim), float(theta), _SCALINGS[scaling], float(factor),
                                                 int(n_trained), out.ctypes.data), "rope_freqs")
    return out


def rope(xs, pos, freq, *, gains=None, outs=None, dtype=None, interleaved=False, mscale=1.0, eps=1e-6):
    """Rotates the first 2 * len(freq) dims of the rows of each tensor [T, heads, D] in xs (one to four, one launch) by
    pos [T] (int32), after an RMS norm with that tensor's gain where it has one.  outs: tensors to write (x itself: in
    place); without, new ones in `dtype` (default x's).  Returns the outputs."""
    n = len(xs)
    gains = gains or [None] * n
    if outs is None:
        outs = [torch.empty_like(x, dtype=dtype, memory_format=torch.contiguous_format) for x in xs]
    _need(1 <= n <= 4 and len(gains) == n and len(outs) == n, "1 to 4 tensors, as many gains and outputs")
    index = xs[0].get_device()
    t, d = xs[0].shape[0], xs[0].shape[-1]
    if freq.dtype is not torch.float64 or freq.get_device() != index or freq.dim() != 1 or not freq.is_contiguous():
        raise Kv8Error("freq must be contiguous float64 on the rows' GPU")
    rows = b""
    for x, y, g in zip(xs, outs, gains):
        shape = x.shape
        if len(shape) != 3 or shape[0] != t or shape[2] != d or y.shape != shape or index < 0 or x.get_device() != index or \
                y.get_device() != index:
            raise Kv8Error("rows must be [T, heads, D] on one GPU, outputs of the same shape")
        xt, yt, (xa, xb, xc), (ya, yb, yc) = _TYPES.get(x.dtype), _TYPES.get(y.dtype), x.stride(), y.stride()
        _need(xt is not None and yt is not None, "rows must be float32, float16 or bfloat16")
        _need((xc == 1 and yc == 1) or t == 0, "rows' dims must be dense")
        if g is not None and (g.dtype is not torch.float32 or g.shape != (d,) or g.get_device() != index or not g.is_contiguous()):
            raise Kv8Error("a gain must be contiguous float32 [D]")
        rows += _pack_rope(x.data_ptr(), y.data_ptr(), xa, xb, ya, yb, 0 if g is None else g.data_ptr(), shape[1], xt, yt)
    _check((_lib or load_kv8_library()).q3t_kv8_rope(index, rows, n, t, d, 2 * freq.shape[0], bool(interleaved),
                                                     _ints(pos, t, index, "pos"), 0, freq.data_ptr(), mscale, eps,
                                                     _stream(index)), "rope")
    return outs


def append(cache, k, v, start, n_new=None):
    """Stores rows k, v [S, n, H, D] (float32, float16 or bfloat16, alike) from slot start[s] on; n_new [S]: how many of
    a sequence's rows are rows (the rest is padding)."""
    s, h, _, d = cache.shape
    index, shape, stride, t = cache.index, k.shape, k.stride(), _TYPES.get(k.dtype)
    _need(start is not None, "start must be given")
    if len(shape) != 4 or shape[0] != s or shape[2] != h or shape[3] != d:
        raise Kv8Error(f"rows must be [{s}, n, {h}, {d}]")
    if shape != v.shape or k.dtype is not v.dtype or stride != v.stride() or k.get_device() != index or \
            v.get_device() != index or (stride[3] != 1 and shape[1]):
        raise Kv8Error("rows k and v must be alike, with dense dims, on the cache's GPU")
    _need(t is not None, "rows must be float32, float16 or bfloat16")
    _check((_lib or load_kv8_library()).q3t_kv8_append(index, cache.ref, k.data_ptr(), v.data_ptr(), t, stride[0], stride[1],
                                                       stride[2], shape[1], _ints(start, s, index, "start"), 0,
                                                       _ints(n_new, s, index, "n_new"), _stream(index)), "append")


def attend(cache, q, lens, *, scale=None, n_new=None, causal=True, weights=False, max_len=0, out=None, dtype=None):
    """Softmax attention of rows q [S, n, heads, D] (float16 or bfloat16) over a cache whose sequences have lens [S]
    slots, the rows' own (appended before) among them.  weights: cache.acc grows by the probabilities that each
    slot drew.  max_len: the longest sequence to size the call for (default: all slots).  out: where to write
    (default: a new tensor of `dtype`, by default q's); rows past n_new are left as they were."""
    s, h, _, d = cache.shape
    index, shape, stride = cache.index, q.shape, q.stride()
    if len(shape) != 4 or shape[0] != s or shape[3] != d or q.get_device() != index or (stride[3] != 1 and shape[1]):
        raise Kv8Error(f"q must be [{s}, n, heads, {d}] with dense dims, on the cache's GPU")
    if out is None:
        out = torch.empty_like(q, dtype=dtype, memory_format=torch.contiguous_format)
    _need(lens is not None, "lens must be given")
    ostride = out.stride()
    if out.shape != shape or out.get_device() != index or (ostride[3] != 1 and shape[1]):
        raise Kv8Error("out must have q's shape, with dense dims, on its GPU")
    qt, ot = _TYPES.get(q.dtype), _TYPES.get(out.dtype)
    _need(qt is not None and ot is not None, "q must be float16 or bfloat16, out one of these or float32")
    args = _pack_attend(q.data_ptr(), out.data_ptr(), stride[0], stride[1], stride[2], ostride[0], ostride[1], ostride[2],
                        qt, ot, shape[1], shape[2], _ints(lens, s, index, "lens"), 0, _ints(n_new, s, index, "n_new"),
                        max_len, bool(causal), d ** -0.5 if scale is None else scale, bool(weights))
    lib = _lib or load_kv8_library()
    need = _check(lib.q3t_kv8_attend_ws(cache.ref, args), "attend")
    # from torch's allocator on the current stream: reused only behind this call's kernels, and a captured graph's own
    ws = torch.empty(need, dtype=torch.uint8, device=cache.device) if need else None
    _check(lib.q3t_kv8_attend(index, cache.ref, args, ws.data_ptr() if need else None, need, _stream(index)), "attend")
    return out


def evict(cache, to, lens, *, n_keep, n_sink=0, n_recent=0):
    """Keeps n_keep slots of every sequence and head of `cache` (all of a shorter one) and writes them to `to`, in
    their order: the first n_sink, the last n_recent, and of the rest those that drew the most weight.  Returns (kept
    [S, H, n_keep] int32: the old slots, -1 behind them; the new lengths [S] int32)."""
    s, h = cache.shape[:2]
    index = cache.index
    _need(to.index == index, "both caches must be on one GPU")
    _need(n_keep >= 1, "n_keep must be at least 1")
    _need(lens is not None, "lens must be given")
    kept = torch.empty(s, h, n_keep, dtype=torch.int32, device=cache.device)
    left = torch.empty(s, dtype=torch.int32, device=cache.device)
    _check((_lib or load_kv8_library()).q3t_kv8_evict(index, cache.ref, to.ref, _ints(lens, s, index, "lens"), 0, n_keep, n_sink,
                                                      n_recent, kept.data_ptr(), left.data_ptr(), _stream(index)), "evict")
    return kept, left


def read(cache, start, n, *, dtype=torch.float32):
    """Values of slots start[s] .. + n (start None: 0 ..) of every head: (k, v), each [S, n, H, D] in `dtype`; 0 outside
    the cache."""
    s, h, _, d = cache.shape
    index = cache.index
    _need(dtype in _TYPES and n >= 0, "dtype must be float32, float16 or bfloat16, n not negative")
    k, v = (torch.empty(s, n, h, d, dtype=dtype, device=cache.device) for _ in range(2))
    _check((_lib or load_kv8_library()).q3t_kv8_read(index, cache.ref, _ints(start, s, index, "start"), 0, n, _TYPES[dtype],
                                                     k.data_ptr(), v.data_ptr(), _stream(index)), "read")
    return k, v

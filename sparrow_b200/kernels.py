"""Python mirror of `vmlm_ops::kernels` for the quantised-linear path.

Same operator names, argument order and meaning as the reference
(ops/src/kernels.rs in the shouzugzs-AI/Sparrow tree):

    gemm_nt_int8(a, q, scale, c, m, n, k)   ops/src/kernels.rs:1256-1287
    gemm_nt_bf16(a, b, c, m, n, k)          ops/src/kernels.rs:1199-1227

`a`, `q`/`b`, `scale` and `c` are host buffers (numpy arrays, contiguous, of
the stated element type and at least the stated length); `c` is overwritten.
The reference kernels check nothing and the VM calls exit(9) on misuse
(core/src/interp.rs:752-806); here a bad argument raises VmlmError (or
ValueError for a Python-side type or size mismatch) before any GPU work.

The `_dev` variants take device buffers: torch CUDA tensors (or raw device
addresses as ints) and an optional CUDA stream, and return without waiting.
"""
import ctypes

import numpy as np

from ._lib import Kv4, RopeTable, Slot, check, lib


def _host_ptr(x, dtype, count, name):
    if not isinstance(x, np.ndarray):
        raise ValueError(f"{name}: expected a numpy array, got {type(x).__name__}")
    if x.dtype != dtype:
        raise ValueError(f"{name}: expected {np.dtype(dtype).name}, got {x.dtype.name}")
    if not x.flags["C_CONTIGUOUS"]:
        raise ValueError(f"{name}: must be C-contiguous")
    if x.size < count:
        raise ValueError(f"{name}: needs {count} elements, has {x.size}")
    return ctypes.c_void_p(x.ctypes.data) if x.size else None


_dtype_names = {}  # torch dtype -> its name: str(dtype) costs more than all other checks of a tensor


def _dtype_name(dt):
    name = _dtype_names.get(dt)
    if name is None:
        name = _dtype_names[dt] = str(dt).replace("torch.", "")
    return name


def _dev_ptr(x, dtype_name, count, name):
    if x is None:
        return None
    if isinstance(x, int):
        return ctypes.c_void_p(x)
    if not getattr(x, "is_cuda", False):
        raise ValueError(f"{name}: expected a CUDA tensor or a device address")
    if _dtype_name(x.dtype) != dtype_name:
        raise ValueError(f"{name}: expected torch.{dtype_name}, got {x.dtype}")
    if not x.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    if x.numel() < count:
        raise ValueError(f"{name}: needs {count} elements, has {x.numel()}")
    return ctypes.c_void_p(x.data_ptr())


CUDA_STREAM_LEGACY = 1  # cudaStreamLegacy: the legacy default stream


def _stream_ptr(stream):
    """None -> the library's own stream. A torch stream whose handle is 0 is the
    legacy default stream, which the C ABI must receive as cudaStreamLegacy
    (a NULL handle there selects the library stream)."""
    if stream is None:
        return None
    h = stream if isinstance(stream, int) else stream.cuda_stream
    return ctypes.c_void_p(h if h else CUDA_STREAM_LEGACY)


# ------------------------------------------------------------------ setup

def init(device: int = 0) -> None:
    """Select the device for the host-pointer entry points (creates its context)."""
    check(lib().vmlm_init(device))


def shutdown() -> None:
    check(lib().vmlm_shutdown())


def register_weight(w: np.ndarray) -> None:
    """Keep a device copy of an immutable host weight (or scale) array."""
    if not isinstance(w, np.ndarray) or not w.flags["C_CONTIGUOUS"]:
        raise ValueError("register_weight: expected a C-contiguous numpy array")
    check(lib().vmlm_register_weight(ctypes.c_void_p(w.ctypes.data), w.nbytes))


def unregister_weight(w: np.ndarray) -> None:
    check(lib().vmlm_unregister_weight(ctypes.c_void_p(w.ctypes.data)))


def unregister_all() -> None:
    check(lib().vmlm_unregister_all())


def sync(stream=None) -> None:
    check(lib().vmlm_sync(_stream_ptr(stream)))


def launch_count() -> int:
    return int(lib().vmlm_launch_count())


def probe_mma_peak(kind: str, iters: int):
    """Dense tensor-core rate of the current device from back-to-back tcgen05.mma
    on shared-memory operands: kind "bf16" (kind::f16) or "int8" (kind::i8).
    Returns (TFLOP/s or TOP/s, kernel ms)."""
    code = {"bf16": 0, "int8": 1}[kind]
    tops, ms = ctypes.c_double(), ctypes.c_double()
    check(lib().vmlm_probe_mma_peak(code, int(iters), ctypes.byref(tops), ctypes.byref(ms)))
    return tops.value, ms.value


def profile_enable(on: bool) -> None:
    """Bracket each tensor-core GEMM launch with CUDA events (diagnostics)."""
    check(lib().vmlm_profile_enable(1 if on else 0))


def trace_enable(max_ctas: int) -> None:
    """Record per-CTA phase timestamps of each GEMM launch (0 disables)."""
    check(lib().vmlm_trace_enable(max_ctas))


def trace_take(n_ctas: int) -> np.ndarray:
    """The last traced launch: [n_ctas, 16] values (8 globaltimer stamps, 4 summed waits and
    3 summed split-tile phases in ns, then items * 65536 + tiles finished)."""
    out = np.zeros((n_ctas, 16), np.uint64)
    check(lib().vmlm_trace_take(ctypes.c_void_p(out.ctypes.data), out.size))
    return out


def profile_take():
    """(summed device ms, launches) of the GEMM launches recorded since the last take."""
    ms = ctypes.c_double(0.0)
    n = ctypes.c_uint64(0)
    check(lib().vmlm_profile_take(ctypes.byref(ms), ctypes.byref(n)))
    return ms.value, n.value


def profile_kernel() -> str:
    """Kernel and tile plan of the last profiled GEMM launch."""
    buf = ctypes.create_string_buffer(256)
    check(lib().vmlm_profile_kernel(buf, len(buf)))
    return buf.value.decode()


# ------------------------------------------------------- reference operators

def gemm_nt_int8(a, q, scale, c, m, n, k) -> None:
    """C[M,N] = (A[M,K] . f32(q[N,K])^T) * scale[N]  (ops/src/kernels.rs:1256-1287)."""
    check(lib().vmlm_gemm_nt_int8(
        _host_ptr(a, np.float32, m * k, "a"), _host_ptr(q, np.int8, n * k, "q"),
        _host_ptr(scale, np.float32, n, "scale"), _host_ptr(c, np.float32, m * n, "c"), m, n, k))


def gemm_nt_bf16(a, b, c, m, n, k) -> None:
    """C[M,N] = A[M,K] . widen(B_bf16[N,K])^T  (ops/src/kernels.rs:1199-1227); b holds bf16 bits as uint16."""
    check(lib().vmlm_gemm_nt_bf16(
        _host_ptr(a, np.float32, m * k, "a"), _host_ptr(b, np.uint16, n * k, "b"),
        _host_ptr(c, np.float32, m * n, "c"), m, n, k))


def gemm_i8i8(x, w, scale, c, acc, m, n, k) -> None:
    """int8 x int8 -> exact int32 acc[M,N]; C = f32(acc) * scale[N]. c or acc may be None."""
    check(lib().vmlm_gemm_i8i8(
        _host_ptr(x, np.int8, m * k, "x"), _host_ptr(w, np.int8, n * k, "w"),
        _host_ptr(scale, np.float32, n, "scale") if c is not None else None,
        _host_ptr(c, np.float32, m * n, "c") if c is not None else None,
        _host_ptr(acc, np.int32, m * n, "acc") if acc is not None else None, m, n, k))


def gemm_nt_f32(a, b, c, m, n, k, acc=False) -> None:
    """C[M,N] = A[M,K] . B[N,K]^T, plus the old C when acc  (ops/src/kernels.rs:987-1015)."""
    check(lib().vmlm_gemm_nt_f32(
        _host_ptr(a, np.float32, m * k, "a"), _host_ptr(b, np.float32, n * k, "b"),
        _host_ptr(c, np.float32, m * n, "c"), m, n, k, int(bool(acc))))


def gemm_f32(a, b, c, m, n, k, acc=False) -> None:
    """C[M,N] = A[M,K] . B[K,N], plus the old C when acc  (ops/src/kernels.rs:383-419)."""
    check(lib().vmlm_gemm_f32(
        _host_ptr(a, np.float32, m * k, "a"), _host_ptr(b, np.float32, k * n, "b"),
        _host_ptr(c, np.float32, m * n, "c"), m, n, k, int(bool(acc))))


# ----------------------------------------------------------- device variants

def gemm_nt_int8_dev(a, q, scale, c, m, n, k, stream=None) -> None:
    check(lib().vmlm_gemm_nt_int8_dev(
        _dev_ptr(a, "float32", m * k, "a"), _dev_ptr(q, "int8", n * k, "q"),
        _dev_ptr(scale, "float32", n, "scale"), _dev_ptr(c, "float32", m * n, "c"), m, n, k,
        _stream_ptr(stream)))


def gemm_nt_int8_dev_noalloc(a, q, scale, c, m, n, k, stream=None) -> None:
    """gemm_nt_int8_dev without any device allocation: its scratch is a fixed
    array inside the library (m <= 16, n <= 131072, k <= 16384). For callers
    that reserve all device memory up front and must not allocate per call.
    Calls that overlap on the GPU share that scratch and race.

    stream=None runs on the CUDA legacy default stream (the C entry point's
    NULL), not on the library stream that None selects for the other *_dev
    calls; pass a stream to order it with other work."""
    st = ctypes.c_void_p(CUDA_STREAM_LEGACY) if stream is None else _stream_ptr(stream)
    check(lib().vmlm_gemm_nt_int8_dev_noalloc(
        _dev_ptr(a, "float32", m * k, "a"), _dev_ptr(q, "int8", n * k, "q"),
        _dev_ptr(scale, "float32", n, "scale"), _dev_ptr(c, "float32", m * n, "c"), m, n, k, st))


def gemm_nt_bf16_dev(a, b, c, m, n, k, stream=None) -> None:
    """b: a bfloat16 (or int16/uint16 bit-pattern) CUDA tensor [n, k]."""
    if b is not None and not isinstance(b, int) and str(b.dtype) in ("torch.int16", "torch.uint16"):
        bptr = _dev_ptr(b, str(b.dtype)[6:], n * k, "b")
    else:
        bptr = _dev_ptr(b, "bfloat16", n * k, "b")
    check(lib().vmlm_gemm_nt_bf16_dev(
        _dev_ptr(a, "float32", m * k, "a"), bptr, _dev_ptr(c, "float32", m * n, "c"), m, n, k,
        _stream_ptr(stream)))


def gemm_i8i8_dev(x, w, scale, c, acc, m, n, k, stream=None) -> None:
    check(lib().vmlm_gemm_i8i8_dev(
        _dev_ptr(x, "int8", m * k, "x"), _dev_ptr(w, "int8", n * k, "w"),
        _dev_ptr(scale, "float32", n, "scale"), _dev_ptr(c, "float32", m * n, "c"),
        _dev_ptr(acc, "int32", m * n, "acc"), m, n, k, _stream_ptr(stream)))


def gemm_nt_f32_dev(a, b, c, m, n, k, acc=False, stream=None) -> None:
    check(lib().vmlm_gemm_nt_f32_dev(
        _dev_ptr(a, "float32", m * k, "a"), _dev_ptr(b, "float32", n * k, "b"),
        _dev_ptr(c, "float32", m * n, "c"), m, n, k, int(bool(acc)), _stream_ptr(stream)))


def gemm_f32_dev(a, b, c, m, n, k, acc=False, stream=None) -> None:
    check(lib().vmlm_gemm_f32_dev(
        _dev_ptr(a, "float32", m * k, "a"), _dev_ptr(b, "float32", k * n, "b"),
        _dev_ptr(c, "float32", m * n, "c"), m, n, k, int(bool(acc)), _stream_ptr(stream)))


# ------------------------------------------------ decode-step neighbours

def rmsnorm_gemm_nt_int8(a, g, eps, q, scale, c, m, n, k) -> None:
    """C = gemm_nt_int8(rmsnorm(a, g, eps), q, scale) (ops/src/kernels.rs:1346-1370, then :1256-1287)."""
    check(lib().vmlm_rmsnorm_gemm_nt_int8(
        _host_ptr(a, np.float32, m * k, "a"), _host_ptr(g, np.float32, k, "g"), float(eps),
        _host_ptr(q, np.int8, n * k, "q"), _host_ptr(scale, np.float32, n, "scale"),
        _host_ptr(c, np.float32, m * n, "c"), m, n, k))


def rmsnorm_gemm_nt_int8_dev(a, g, eps, q, scale, c, m, n, k, stream=None) -> None:
    check(lib().vmlm_rmsnorm_gemm_nt_int8_dev(
        _dev_ptr(a, "float32", m * k, "a"), _dev_ptr(g, "float32", k, "g"), float(eps),
        _dev_ptr(q, "int8", n * k, "q"), _dev_ptr(scale, "float32", n, "scale"),
        _dev_ptr(c, "float32", m * n, "c"), m, n, k, _stream_ptr(stream)))


def gemv_f32(a, b, c, m, k) -> None:
    """OP_GEMV (core/src/interp.rs:815-827): c[i] = sum_p a[i, p] * b[p]."""
    check(lib().vmlm_gemv_f32(_host_ptr(a, np.float32, m * k, "a"), _host_ptr(b, np.float32, k, "b"),
                              _host_ptr(c, np.float32, m, "c"), m, k))


def gemv_f32_dev(a, b, c, m, k, stream=None) -> None:
    check(lib().vmlm_gemv_f32_dev(_dev_ptr(a, "float32", m * k, "a"), _dev_ptr(b, "float32", k, "b"),
                                  _dev_ptr(c, "float32", m, "c"), m, k, _stream_ptr(stream)))


class Pool:
    """A .vmb program's constant pool, scratch regions and slot table in device
    memory (vmlm_pool_*; Vm::load, core/src/interp.rs:123-220)."""

    def __init__(self, image: bytes, weights: bytes = None):
        self._h = ctypes.c_void_p()
        img = bytes(image)
        w = bytes(weights) if weights is not None else None
        check(lib().vmlm_pool_load(img, len(img), w, len(w) if w is not None else 0, ctypes.byref(self._h)))

    def close(self) -> None:
        if self._h:
            check(lib().vmlm_pool_free(self._h))
            self._h = ctypes.c_void_p()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def info(self):
        """-> (n_const, n_slots, [const, act, state, grad] bytes)."""
        nc, ns = ctypes.c_size_t(), ctypes.c_size_t()
        rb = (ctypes.c_size_t * 4)()
        check(lib().vmlm_pool_info(self._h, ctypes.byref(nc), ctypes.byref(ns), rb))
        return nc.value, ns.value, list(rb)

    def region(self, r: int) -> int:
        p = ctypes.c_void_p()
        check(lib().vmlm_pool_region(self._h, r, ctypes.byref(p)))
        return p.value or 0

    def slot(self, i: int):
        """-> (device address, rows, cols, dtype, kind)."""
        s, kind = Slot(), ctypes.c_int()
        check(lib().vmlm_pool_slot(self._h, i, ctypes.byref(s), ctypes.byref(kind)))
        return s.ptr or 0, s.rows, s.cols, s.dtype, kind.value

    def layerb(self, delta: float) -> None:
        check(lib().vmlm_pool_layerb(self._h, ctypes.c_float(delta)))

    def layer_base(self) -> int:
        b = ctypes.c_size_t()
        check(lib().vmlm_pool_layer_base(self._h, ctypes.byref(b)))
        return b.value

    def find_const(self, name: str) -> int:
        i = ctypes.c_size_t()
        check(lib().vmlm_pool_find_const(self._h, name.encode(), ctypes.byref(i)))
        return i.value

    def find_slot(self, name: str) -> int:
        i = ctypes.c_size_t()
        check(lib().vmlm_pool_find_slot(self._h, name.encode(), ctypes.byref(i)))
        return i.value

    def gemm(self, ins: bytes, stream=None) -> None:
        """Run one 16-byte OP_GEMM instruction on the pool's slots."""
        assert len(ins) == 16
        check(lib().vmlm_pool_gemm(self._h, ins, _stream_ptr(stream)))


class Q8Call(ctypes.Structure):
    """vmlm_q8_call: one Q8 call of a batch (device pointers)."""
    _fields_ = [("a", ctypes.c_void_p), ("q", ctypes.c_void_p), ("scale", ctypes.c_void_p), ("c", ctypes.c_void_p),
                ("m", ctypes.c_size_t), ("n", ctypes.c_size_t), ("k", ctypes.c_size_t)]


def gemm_nt_int8_batch_dev(calls, stream=None) -> None:
    """Independent Q8 calls [(a, q, scale, c, m, n, k), ...] on CUDA tensors, as one grouped launch where they fit."""
    arr = (Q8Call * len(calls))()
    for i, (a, q, s, c, m, n, k) in enumerate(calls):
        arr[i] = Q8Call(_dev_ptr(a, "float32", m * k, "a"), _dev_ptr(q, "int8", n * k, "q"),
                        _dev_ptr(s, "float32", n, "scale"), _dev_ptr(c, "float32", m * n, "c"), m, n, k)
    check(lib().vmlm_gemm_nt_int8_batch_dev(arr, len(calls), _stream_ptr(stream)))


def set_host_pipeline(max_chunks: int) -> None:
    """Most row chunks a large host-pointer call is pipelined in (1 = off, 0 = default)."""
    check(lib().vmlm_set_host_pipeline(int(max_chunks)))


def gemm_nt_int4_gs(a, packed, scale, c, m, n, k, group, order=0) -> None:
    """int4 weights, a scale per group of columns (tests/src/quant.rs:298-362); packed
    [n, (k+1)//2] uint8, scale [n, ceil(k/group)]; order 1 = the AVX2 step as shipped."""
    gpr = (k + group - 1) // group if group else 0
    check(lib().vmlm_gemm_nt_int4_gs(
        _host_ptr(a, np.float32, m * k, "a"), _host_ptr(packed, np.uint8, n * ((k + 1) // 2), "packed"),
        _host_ptr(scale, np.float32, n * gpr, "scale"), _host_ptr(c, np.float32, m * n, "c"),
        m, n, k, group, int(order)))


def gemm_nt_int4_gs_dev(a, packed, scale, c, m, n, k, group, order=0, stream=None) -> None:
    gpr = (k + group - 1) // group if group else 0
    check(lib().vmlm_gemm_nt_int4_gs_dev(
        _dev_ptr(a, "float32", m * k, "a"), _dev_ptr(packed, "uint8", n * ((k + 1) // 2), "packed"),
        _dev_ptr(scale, "float32", n * gpr, "scale"), _dev_ptr(c, "float32", m * n, "c"),
        m, n, k, group, int(order), _stream_ptr(stream)))


def _idx_dev_ptr(idx, count):
    if idx is None or isinstance(idx, int):
        return _dev_ptr(idx, "int32", count, "idx")
    return _dev_ptr(idx, "uint32" if str(idx.dtype) == "torch.uint32" else "int32", count, "idx")


def gemm_nt_int8_outlier(a, q, scale, w, idx, c, m, n, k) -> None:
    """int8 plus f32 outlier columns (tests/src/quant.rs:524-565); idx uint32 column indices."""
    idx = np.ascontiguousarray(idx, np.uint32)
    check(lib().vmlm_gemm_nt_int8_outlier(
        _host_ptr(a, np.float32, m * k, "a"), _host_ptr(q, np.int8, n * k, "q"),
        _host_ptr(scale, np.float32, n, "scale"), _host_ptr(w, np.float32, n * k, "w") if idx.size else None,
        _host_ptr(idx, np.uint32, idx.size, "idx") if idx.size else None, idx.size,
        _host_ptr(c, np.float32, m * n, "c"), m, n, k))


def gemm_nt_int8_outlier_dev(a, q, scale, w, idx, n_idx, c, m, n, k, compact=False, stream=None) -> None:
    """w: the f32 weight [n, k] (compact False) or the gathered outlier columns [n, n_idx]."""
    check(lib().vmlm_gemm_nt_int8_outlier_dev(
        _dev_ptr(a, "float32", m * k, "a"), _dev_ptr(q, "int8", n * k, "q"), _dev_ptr(scale, "float32", n, "scale"),
        _dev_ptr(w, "float32", n * (n_idx if compact else k), "w") if n_idx else None, int(bool(compact)),
        _idx_dev_ptr(idx, n_idx) if n_idx else None, n_idx, _dev_ptr(c, "float32", m * n, "c"), m, n, k,
        _stream_ptr(stream)))


def gather_columns_dev(w, idx, n_idx, n, k, wo, stream=None) -> None:
    """wo[j, t] = w[j, idx[t]] (device tensors)."""
    check(lib().vmlm_gather_columns_dev(_dev_ptr(w, "float32", n * k, "w"), _idx_dev_ptr(idx, n_idx), n_idx, n, k,
                                        _dev_ptr(wo, "float32", n * n_idx, "wo"), _stream_ptr(stream)))


def emb(table, idx, out) -> None:
    """OP_EMB (core/src/interp.rs:1351-1420) for every index: out[t] = f32(table[idx[t]]);
    table: a [rows, cols] bf16-bit (uint16) or float32 array, idx: float32 row numbers."""
    rows, cols = table.shape
    dt = DT_BF16 if table.dtype == np.uint16 else DT_F32
    m = idx.size
    check(lib().vmlm_emb(_host_ptr(table, table.dtype, rows * cols, "table"), dt, rows, cols,
                         _host_ptr(idx, np.float32, m, "idx"), m, _host_ptr(out, np.float32, m * cols, "out")))


def emb_dev(table, idx, out, stream=None) -> None:
    """OP_EMB on CUDA tensors (bfloat16 / int16 bits or float32 table); a bad index is reported by sync()."""
    rows, cols = table.shape
    name = str(table.dtype)[6:]
    dt = DT_BF16 if name in ("bfloat16", "int16", "uint16") else DT_F32
    m = idx.numel()
    check(lib().vmlm_emb_dev(_dev_ptr(table, name, rows * cols, "table"), dt, rows, cols,
                             _dev_ptr(idx, "float32", m, "idx"), m, _dev_ptr(out, "float32", m * cols, "out"),
                             _stream_ptr(stream)))


# ------------------------------------- a 4-bit key/value cache for decode

_F32 = None  # torch.float32, once a tensor of it has been seen


def _rows_ptr(x, rows, width, name):
    """(address, row stride) of a [rows, >= width] float32 CUDA tensor whose rows may be slices of wider ones."""
    global _F32
    try:
        if not x.is_cuda or (x.dtype is not _F32 and _dtype_name(x.dtype) != "float32"):
            raise ValueError(f"{name}: expected a float32 CUDA tensor")
    except AttributeError:
        raise ValueError(f"{name}: expected a float32 CUDA tensor, got {type(x).__name__}") from None
    _F32 = x.dtype
    if x.dim() != 2:
        raise ValueError(f"{name}: expected a CUDA tensor of rows")
    (n, w), (ld, step) = x.shape, x.stride()
    if n < rows or w < width or (step != 1 and w > 1):
        raise ValueError(f"{name}: needs {rows} rows of {width} values with unit column stride, has {tuple(x.shape)}")
    return x.data_ptr(), ld if n > 1 else max(ld, w)


def _ptr(x, dtype_name, count, name):
    """_dev_ptr for the calls of a decode step, whose host time counts: a plain address."""
    if x is None or isinstance(x, int):
        return x
    try:
        if x.is_cuda and _dtype_name(x.dtype) == dtype_name and x.numel() >= count and x.is_contiguous():
            return x.data_ptr()
    except AttributeError:
        pass
    return _dev_ptr(x, dtype_name, count, name)  # says what is wrong


class Rope:
    """The rotation of a head's first 2 * cos.shape[1] columns: cos, sin [n_pos, rot/2] float32, pos [tokens] int32
    (vmlm_rope). `pos` may be set again for other tokens."""

    def __init__(self, cos, sin, pos, interleaved=False):
        n_pos, half = cos.shape
        self._keep = [cos, sin, pos]
        self.table = RopeTable(_dev_ptr(cos, "float32", n_pos * half, "cos"), _dev_ptr(sin, "float32", n_pos * half, "sin"),
                               _dev_ptr(pos, "int32", 0, "pos"), n_pos, 2 * half, int(bool(interleaved)))
        self.tokens = pos.numel()
        self.ref = ctypes.byref(self.table)

    def set_positions(self, pos) -> None:
        self.table.pos = _dev_ptr(pos, "int32", 0, "pos")
        self._keep[2], self.tokens = pos, pos.numel()


class Kv4Cache:
    """A 4-bit key/value cache over caller-owned CUDA tensors (vmlm_kv4): codes k, v uint8 [n_seq, n_kv, cap, d/2] and
    ks, vs float16 [n_seq, n_kv, cap, d/32, 2] (step, base). `Kv4Cache.empty` allocates them."""

    def __init__(self, k, v, ks, vs):
        n_seq, n_kv, cap, half = k.shape
        self.n_seq, self.n_kv, self.cap, self.d = n_seq, n_kv, cap, 2 * half
        n = n_seq * n_kv * cap
        if tuple(v.shape) != tuple(k.shape) or ks.numel() != n * half // 8 or vs.numel() != n * half // 8:
            raise ValueError("Kv4Cache: k, v, ks and vs differ in shape")
        self.k, self.v, self.ks, self.vs = k, v, ks, vs
        self.struct = Kv4(_dev_ptr(k, "uint8", n * half, "k"), _dev_ptr(v, "uint8", n * half, "v"),
                          _dev_ptr(ks, "float16", n * half // 8, "ks"), _dev_ptr(vs, "float16", n * half // 8, "vs"),
                          n_seq, n_kv, cap, 2 * half)
        self.ref = ctypes.byref(self.struct)

    @classmethod
    def empty(cls, n_seq, n_kv, cap, d, device="cuda"):
        import torch
        codes = [torch.empty((n_seq, n_kv, cap, d // 2), dtype=torch.uint8, device=device) for _ in range(2)]
        sb = [torch.empty((n_seq, n_kv, cap, d // 32, 2), dtype=torch.float16, device=device) for _ in range(2)]
        return cls(*codes, *sb)


def _rope_ref(rope, tokens):
    if rope is None:
        return None
    if rope.tokens < tokens:
        raise ValueError(f"rope: {rope.tokens} positions for {tokens} tokens")
    return rope.ref


def qk_norm_rope_dev(q, k, gq, gk, eps, rope, qo, ko, tokens, n_q, n_kv, d, stream=None) -> None:
    """RMSNorm of each query and key head (gains gq, gk [d] or None) and the rotation (rope or None), in one pass: q, qo
    [tokens, n_q * d], k, ko [tokens, n_kv * d], rows may be slices of wider ones; qo may be q, ko may be k."""
    pq, ldq = _rows_ptr(q, tokens, n_q * d, "q") if n_q else (None, 0)
    pqo, ldqo = _rows_ptr(qo, tokens, n_q * d, "qo") if n_q else (None, 0)
    pk, ldk = _rows_ptr(k, tokens, n_kv * d, "k") if n_kv else (None, 0)
    pko, ldko = _rows_ptr(ko, tokens, n_kv * d, "ko") if n_kv else (None, 0)
    check(lib().vmlm_qk_norm_rope_dev(pq, ldq, pk, ldk, _ptr(gq, "float32", d, "gq"), _ptr(gk, "float32", d, "gk"), eps,
                                      _rope_ref(rope, tokens), pqo, ldqo, pko, ldko, tokens, n_q, n_kv, d,
                                      _stream_ptr(stream)))


def kv4_append_dev(cache, k, v, length, m, q=None, qo=None, n_q=0, gq=None, gk=None, eps=0.0, rope=None,
                   stream=None) -> None:
    """Write the m new tokens of each sequence (rows b * m + t of k and v) to slots length[b] + t in 4 bits, the keys
    normalised and rotated where gk and rope are given, and the queries with them (q -> qo)."""
    tokens, d = cache.n_seq * m, cache.d
    pk, ldk = _rows_ptr(k, tokens, cache.n_kv * d, "k")
    pv, ldv = _rows_ptr(v, tokens, cache.n_kv * d, "v")
    pq, ldq = _rows_ptr(q, tokens, n_q * d, "q") if n_q else (None, 0)
    pqo, ldqo = _rows_ptr(qo, tokens, n_q * d, "qo") if n_q else (None, 0)
    check(lib().vmlm_kv4_append_dev(cache.ref, pq, ldq, pqo, ldqo, n_q, pk, ldk, pv, ldv, _ptr(gq, "float32", d, "gq"),
                                    _ptr(gk, "float32", d, "gk"), eps, _rope_ref(rope, tokens),
                                    _ptr(length, "int32", cache.n_seq, "length"), m, _stream_ptr(stream)))


def kv4_read_dev(cache, start, end, count, k, v, stream=None) -> None:
    """Rows start[b] .. start[b] + count - 1 of each sequence and kv head as the values they stand for: k, v float16
    [n_seq, n_kv, count, d]; rows at or behind end[b] are zeros."""
    n = cache.n_seq * cache.n_kv * count * cache.d
    check(lib().vmlm_kv4_read_dev(cache.ref, _ptr(start, "int32", cache.n_seq, "start"),
                                  _ptr(end, "int32", cache.n_seq, "end"), count, _ptr(k, "float16", n, "k"),
                                  _ptr(v, "float16", n, "v"), _stream_ptr(stream)))


def kv4_attn_dev(cache, q, length, out, m, n_q, scale, w_in=None, w_out=None, stream=None) -> None:
    """Attention of the m newest tokens of each sequence (rows b * m + t of q and out) over the cache; length[b] counts
    them. w_out [n_seq, n_kv, cap] (which may be w_in) receives w_in plus the weight that each slot got. out may not overlap
    q."""
    tokens, width = cache.n_seq * m, n_q * cache.d
    pq, ldq = _rows_ptr(q, tokens, width, "q")
    po, ldo = _rows_ptr(out, tokens, width, "out")
    slots = cache.n_seq * cache.n_kv * cache.cap
    check(lib().vmlm_kv4_attn_dev(cache.ref, pq, ldq, _ptr(length, "int32", cache.n_seq, "length"), po, ldo, m, n_q, scale,
                                  _ptr(w_in, "float32", slots, "w_in"), _ptr(w_out, "float32", slots, "w_out"),
                                  _stream_ptr(stream)))


def kv4_evict_dev(src, dst, w, length, keep, first, recent, idx, w_out, len_out, stream=None) -> None:
    """Copy the `keep` slots of each sequence and kv head with the most weight w [n_seq, n_kv, src.cap] (the first `first`
    and the last `recent` always among them) from src to dst, in slot order; idx, w_out [n_seq, n_kv, keep] and len_out
    [n_seq] say which they are. w_out may be None. No output may overlap an input: len_out is not length."""
    out = src.n_seq * src.n_kv * keep
    check(lib().vmlm_kv4_evict_dev(src.ref, dst.ref, _ptr(w, "float32", src.n_seq * src.n_kv * src.cap, "w"),
                                   _ptr(length, "int32", src.n_seq, "length"), keep, first, recent,
                                   _ptr(idx, "int32", out, "idx"), _ptr(w_out, "float32", out, "w_out"),
                                   _ptr(len_out, "int32", src.n_seq, "len_out"), _stream_ptr(stream)))


# ------------------------------------------------------ the OP_GEMM operator

DT_F32, DT_F16, DT_I8, DT_I32, DT_BF16 = 0, 1, 2, 3, 4  # core/src/format.rs:73-79
FL_ACC, FL_TRANS_B = 1, 2                                # trans/src/opcode.rs:303-304
_NP_DT = {"float32": DT_F32, "float16": DT_F16, "int8": DT_I8, "int32": DT_I32, "uint16": DT_BF16}


def slot(x, dtype=None):
    """A VM slot over a 2-D numpy array or CUDA tensor (uint16 / bfloat16 / int16 data is bf16)."""
    from ._lib import Slot
    if x is None:
        return None
    rows, cols = x.shape
    if isinstance(x, np.ndarray):
        if not x.flags["C_CONTIGUOUS"]:
            raise ValueError("slot: must be C-contiguous")
        ptr, dt = x.ctypes.data, _NP_DT.get(x.dtype.name, -1)
    else:
        if not x.is_contiguous():
            raise ValueError("slot: must be contiguous")
        name = str(x.dtype)[6:]
        ptr, dt = x.data_ptr(), DT_BF16 if name in ("bfloat16", "int16") else _NP_DT.get(name, -1)
    return Slot(ptr, rows, cols, dt if dtype is None else dtype)


def _slot_ref(s):
    return ctypes.byref(s) if s is not None else None


def op_gemm(fl, d, a, b, scale=None) -> None:
    """The VM's OP_GEMM (core/src/interp.rs:734-812) on host arrays: d = a . op(b) (+ d with FL_ACC)."""
    sd, sa, sb, ss = slot(d), slot(a), slot(b), slot(scale)
    check(lib().vmlm_op_gemm(fl, _slot_ref(sd), _slot_ref(sa), _slot_ref(sb), _slot_ref(ss)))


def op_gemm_dev(fl, d, a, b, scale=None, stream=None) -> None:
    """OP_GEMM on CUDA tensors, on `stream`."""
    sd, sa, sb, ss = slot(d), slot(a), slot(b), slot(scale)
    check(lib().vmlm_op_gemm_dev(fl, _slot_ref(sd), _slot_ref(sa), _slot_ref(sb), _slot_ref(ss),
                                 _stream_ptr(stream)))


# ---------------------------------------------------------- conveniences

def q8_linear(x: np.ndarray, q: np.ndarray, scale: np.ndarray) -> np.ndarray:
    """x[M,K] f32, q[N,K] int8, scale[N] f32 -> C[M,N] f32 through gemm_nt_int8."""
    m, k = x.shape
    n = q.shape[0]
    c = np.empty((m, n), np.float32)
    gemm_nt_int8(np.ascontiguousarray(x, np.float32), np.ascontiguousarray(q, np.int8),
                 np.ascontiguousarray(scale, np.float32), c, m, n, k)
    return c


def bf16_linear(x: np.ndarray, b_bits: np.ndarray) -> np.ndarray:
    """x[M,K] f32, b_bits[N,K] uint16 (bf16 bits) -> C[M,N] f32 through gemm_nt_bf16."""
    m, k = x.shape
    n = b_bits.shape[0]
    c = np.empty((m, n), np.float32)
    gemm_nt_bf16(np.ascontiguousarray(x, np.float32), np.ascontiguousarray(b_bits, np.uint16), c, m, n, k)
    return c

"""ctypes binding of libnvfp4_b200.so (the C ABI declared in include/nvfp4_b200.h).

Host-side helper for tests and benchmarks: it adds nothing to the data path -- every
method forwards raw device pointers to the C entry point of the same name.  There is
no CPU fallback: loading fails loudly when the CUDA library has not been built.
"""
import ctypes
import os
import struct

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libnvfp4_b200.so")

c_void_p, c_int, c_float, c_size_t = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t


class PeerExchange(ctypes.Structure):
    """nvfp4_peer_exchange (include/nvfp4_b200.h)."""
    _fields_ = [("peer", ctypes.c_void_p * 8), ("rank", ctypes.c_int), ("world", ctypes.c_int), ("slot_pairs", ctypes.c_int)]


class LinearDesc(ctypes.Structure):
    """nvfp4_linear_desc (include/nvfp4_b200.h)."""
    _fields_ = [("A", ctypes.c_void_p), ("swiglu_up", ctypes.c_void_p), ("a_row_stride", ctypes.c_longlong),
                ("k_valid", ctypes.c_int), ("M", ctypes.c_int), ("packed", ctypes.c_void_p), ("scale", ctypes.c_void_p),
                ("global_scale", ctypes.c_float), ("N", ctypes.c_int), ("K", ctypes.c_int), ("residual", ctypes.c_void_p),
                ("C", ctypes.c_void_p), ("px", ctypes.c_void_p), ("norm_weight", ctypes.c_void_p),
                ("norm_eps", ctypes.c_float), ("swiglu_epilogue", ctypes.c_int)]


class PeerExchange(ctypes.Structure):
    """nvfp4_peer_exchange of include/nvfp4_b200.h."""
    _fields_ = [("peer", c_void_p * 8), ("rank", c_int), ("world", c_int), ("slot_pairs", c_int)]


class QuantizedWeight(ctypes.Structure):
    """Layout of qwen_thor::core::QuantizedWeight (reference src/engine/layer.h:197-204)."""
    _fields_ = [("packed", c_void_p), ("scale", c_void_p), ("global_scale", c_float),
                ("input_scale", c_float), ("N", c_int), ("K", c_int)]


class KvCacheStruct(ctypes.Structure):
    """nvfp4_kv_cache of include/nvfp4_b200.h."""
    _fields_ = [("k", c_void_p), ("v", c_void_p), ("num_pages", c_int), ("page_size", c_int), ("kv_heads", c_int), ("head_dim", c_int),
                ("page_stride", ctypes.c_longlong), ("token_stride", ctypes.c_longlong), ("head_stride", ctypes.c_longlong)]


class PagedBatchStruct(ctypes.Structure):
    """nvfp4_paged_batch of include/nvfp4_b200.h."""
    _fields_ = [("cu_q", c_void_p), ("kv_len", c_void_p), ("block_table", c_void_p), ("table_stride", ctypes.c_longlong), ("table_cols", c_int),
                ("sequences", c_int), ("tokens", c_int), ("max_q_len", c_int)]


class KvAppendDesc(ctypes.Structure):
    """nvfp4_kv_append_desc of include/nvfp4_b200.h."""
    _fields_ = [(n, c_void_p) for n in ("cache", "batch", "q", "k", "v", "q_out")] + \
               [(n, ctypes.c_longlong) for n in ("q_stride", "q_head_stride", "k_stride", "k_head_stride", "v_stride", "v_head_stride",
                                                 "q_out_stride", "q_out_head_stride")] + \
               [(n, c_void_p) for n in ("q_norm", "k_norm", "inv_freq", "positions")] + [("q_heads", c_int), ("rot_dim", c_int), ("norm_eps", c_float)]


class PagedAttentionDesc(ctypes.Structure):
    """nvfp4_paged_attention_desc of include/nvfp4_b200.h."""
    _fields_ = [(n, c_void_p) for n in ("cache", "batch", "q", "gate", "out")] + \
               [(n, ctypes.c_longlong) for n in ("q_stride", "q_head_stride", "gate_stride", "gate_head_stride", "out_stride", "out_head_stride")] + \
               [("q_heads", c_int), ("scale", c_float)]


# name -> (restype, argtypes); every symbol include/nvfp4_b200.h declares.
SIGNATURES = {
    "nvfp4_create": (c_int, [c_int, c_size_t, ctypes.POINTER(c_void_p)]),
    "nvfp4_destroy": (c_int, [c_void_p]),
    "nvfp4_workspace_bytes": (c_int, [c_int, c_int, c_int, ctypes.POINTER(c_size_t)]),
    "nvfp4_status_string": (ctypes.c_char_p, [c_int]),
    "nvfp4_set_option": (c_int, [c_void_p, ctypes.c_char_p, c_int]),
    "nvfp4_get_option": (c_int, [c_void_p, ctypes.c_char_p, ctypes.POINTER(c_int)]),
    "nvfp4_linear": (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_float, c_int, c_int,
                             c_void_p, c_void_p, c_void_p]),
    "nvfp4_linear_decode_noalloc": (c_int, [c_void_p, c_int, c_void_p, c_void_p, c_float, c_int, c_int, c_void_p,
                                            c_void_p, c_void_p]),
    "nvfp4_noalloc_status": (c_int, [ctypes.POINTER(ctypes.c_uint), c_int]),
    "nvfp4_linear_f32": (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_float, c_int, c_int, c_void_p, c_void_p]),
    "nvfp4_linear_reduce_peers": (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_float, c_int, c_int, c_void_p, c_void_p,
                                          c_void_p, c_void_p]),
    "nvfp4_linear_ex": (c_int, [c_void_p, c_void_p, c_void_p]),
    "nvfp4_chain_create": (c_int, [c_void_p, c_void_p, c_int, ctypes.POINTER(c_void_p)]),
    "nvfp4_chain_run": (c_int, [c_void_p, c_void_p]),
    "nvfp4_chain_destroy": (c_int, [c_void_p]),
    "nvfp4_linear_dual": (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_float, c_void_p,
                                  c_void_p, c_float, c_int, c_int, c_void_p, c_void_p, c_void_p]),
    "nvfp4_dequant_bf16": (c_int, [c_void_p, c_void_p, c_void_p, c_float, c_int, c_int, c_void_p, c_void_p]),
    "nvfp4_scan_scales": (c_int, [c_void_p, c_void_p, c_int, c_int, ctypes.POINTER(ctypes.c_longlong), c_void_p]),
    "nvfp4_swiglu": (c_int, [c_void_p, c_void_p, c_void_p, c_int, c_int, c_void_p, c_void_p]),
    "nvfp4_swiglu_strided": (c_int, [c_void_p, c_void_p, c_void_p, c_int, c_int, ctypes.c_longlong, c_void_p,
                                     ctypes.c_longlong, c_void_p]),
    "nvfp4_linear_bf16": (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_int, c_int, c_void_p, c_void_p, c_void_p]),
    "nvfp4_rmsnorm": (c_int, [c_void_p, c_void_p, c_void_p, c_float, c_int, c_int, c_void_p, c_void_p]),
    "nvfp4_add_rmsnorm": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_float, c_int, c_int, c_void_p, c_void_p]),
    "nvfp4_swiglu_interleaved": (c_int, [c_void_p, c_void_p, c_int, c_int, ctypes.c_longlong, c_void_p, ctypes.c_longlong,
                                         c_void_p]),
    "nvfp4_kv_append": (c_int, [c_void_p, c_void_p, c_void_p]),
    "nvfp4_paged_attention": (c_int, [c_void_p, c_void_p, c_void_p]),
    "nvfp4_invoke_fp4_gemv": (None, [c_void_p, ctypes.POINTER(QuantizedWeight), c_void_p, c_void_p]),
    "nvfp4_invoke_fp4_gemv_add": (None, [c_void_p, ctypes.POINTER(QuantizedWeight), c_void_p, c_void_p,
                                         c_void_p]),
    "nvfp4_invoke_fp4_dual_gemv": (None, [c_void_p, ctypes.POINTER(QuantizedWeight),
                                          ctypes.POINTER(QuantizedWeight), c_void_p, c_void_p, c_void_p]),
    "nvfp4_invoke_fp4_gemm": (None, [c_void_p, ctypes.POINTER(QuantizedWeight), c_void_p, c_int, c_void_p]),
    "nvfp4_invoke_fp4_gemm_add": (None, [c_void_p, ctypes.POINTER(QuantizedWeight), c_void_p, c_void_p, c_int,
                                         c_void_p]),
    "nvfp4_init_fp4_cublaslt": (None, []),
    "nvfp4_cleanup_fp4_cublaslt": (None, []),
    "nvfp4_last_status": (c_int, []),
    "nvfp4_default_handle_workspace": (c_int, [c_size_t]),
    "nvfp4_linear_host": (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_float, c_int, c_int,
                                  c_void_p, c_void_p, c_void_p]),
    "nvfp4_launch_count": (c_int, [c_void_p, ctypes.POINTER(ctypes.c_ulonglong)]),
    "nvfp4_device_status": (c_int, [c_void_p, ctypes.POINTER(ctypes.c_uint)]),
}

_lib = None


def load():
    """Load the shared library and attach signatures.  Raises if it is missing."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `make -C {_HERE}` "
                "(or __graft_entry__.build()); there is no fallback path")
        lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = res, args
        _lib = lib
    return _lib


class Nvfp4Error(RuntimeError):
    def __init__(self, status):
        self.status = status
        super().__init__(f"nvfp4 status {status}: {load().nvfp4_status_string(status).decode()}")


def _ptr(t):
    """Device/host address of a torch tensor, an int, or None."""
    if t is None:
        return None
    if isinstance(t, int):
        return t
    return t.data_ptr()


_raw_stream = None


def _stream(stream, device=None):
    """Address of a stream; None: the current one of a device, by default of the current device."""
    if stream is None:
        global _raw_stream
        if _raw_stream is None:
            import torch
            torch.cuda.init()
            # the address alone, where torch gives it: building a Stream object takes 3 us of a call's 9
            get, dev = getattr(torch._C, "_cuda_getCurrentRawStream", None), getattr(torch._C, "_cuda_getDevice", None)
            _raw_stream = (lambda d: get(dev() if d is None else d)) if get and dev else (lambda d: torch.cuda.current_stream(d).cuda_stream)
        return _raw_stream(device)
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


class KvCache:
    """nvfp4_kv_cache over two BF16 tensors [pages, page size, heads, head dim] (order="token") or [pages, heads, page size, head dim]
    (order="head") of the same strides, the last one dense."""

    def __init__(self, k, v, order="token"):
        import torch
        token, head = (1, 2) if order == "token" else (2, 1)
        if order not in ("token", "head") or k.get_device() != v.get_device() or k.shape != v.shape or k.stride() != v.stride() or k.dim() != 4 or k.stride(3) != 1 or \
                any(t.dtype is not torch.bfloat16 for t in (k, v)):
            raise ValueError("k and v: 4-D BF16 tensors of a device and of the same shape and strides, the head's values dense; order 'token' or 'head'")
        self.keep = (k, v)
        self.types = (torch.bfloat16, torch.float32, torch.int32)      # of rows and norms, inv_freq, positions
        self.device = k.get_device()
        self.c = KvCacheStruct(k.data_ptr(), v.data_ptr(), k.shape[0], k.shape[token], k.shape[head], k.shape[3],
                               k.stride(0), k.stride(token), k.stride(head))
        self.address = ctypes.addressof(self.c)
        self.heads, self.dim = k.shape[head], k.shape[3]


class PagedBatch:
    """nvfp4_paged_batch: kv_len [sequences], block_table [sequences, columns] and cu_q [sequences + 1] (None: one new token per sequence)
    are int32 device tensors whose contents may change between calls; tokens (with cu_q the rows of q, k, v and out; without it one per
    sequence unless it says more) and max_q_len are bounds."""

    def __init__(self, kv_len, block_table, tokens=None, cu_q=None, max_q_len=1):
        import torch
        sequences = kv_len.shape[0]
        for t, dim in ((kv_len, 1), (block_table, 2), (cu_q, 1)):
            if t is not None and (t.dtype is not torch.int32 or t.dim() != dim or t.stride(-1) != 1 or t.get_device() != kv_len.get_device()):
                raise ValueError("kv_len [sequences], block_table [sequences, columns] and cu_q [sequences + 1] are dense int32 tensors of a device")
        if block_table.shape[0] != sequences or (cu_q is not None and cu_q.shape[0] != sequences + 1):
            raise ValueError("block_table has a row per sequence, cu_q an entry more than there are sequences")
        if cu_q is not None and tokens is None:             # rows behind `tokens` take part in nothing, and how many there are is on the device
            raise ValueError("cu_q comes with tokens")
        self.keep = (kv_len, block_table, cu_q)
        self.c = PagedBatchStruct(_ptr(cu_q), kv_len.data_ptr(), block_table.data_ptr(), block_table.stride(0), block_table.shape[1], sequences,
                                  sequences if tokens is None else tokens, max_q_len)
        self.address = ctypes.addressof(self.c)
        self.tokens = self.c.tokens
        self.device = kv_len.get_device()


# The descriptors of the calls on a paged cache as bytes: packing them takes a third of the time that filling a ctypes structure does.
_APPEND = struct.Struct("@6P8q4Piif4x")
_ATTENTION = struct.Struct("@5P6qif")
assert _APPEND.size == ctypes.sizeof(KvAppendDesc) and _ATTENTION.size == ctypes.sizeof(PagedAttentionDesc)
_NO_ROWS = (0, 0, 0, 0)


def _rows(t, tokens, dim, dtype, device):
    """Address, token stride, head stride and heads of a [tokens, heads, head dim] tensor."""
    n, heads, d = t.shape
    a, b, c = t.stride()
    if c != 1 or a == 0 or b == 0 or n < tokens or d != dim or t.dtype is not dtype or t.get_device() != device:       # a stride of 0 would mean dense
        raise ValueError("a BF16 tensor [tokens, heads, head dim] on the cache's device with the batch's tokens and the cache's head dim, whose heads are dense and that "
                         "repeats nothing")
    return t.data_ptr(), a, b, heads


_VECTORS = "norms are dense BF16 tensors of a head's values, inv_freq a dense FP32 one, positions a dense int32 one with a value a token, on the cache's device"


class Handle:
    """One library handle on one device (nvfp4_create / nvfp4_destroy)."""

    def __init__(self, device=0, workspace_bytes=64 << 20):
        self.lib = load()
        h = c_void_p()
        st = self.lib.nvfp4_create(device, workspace_bytes, ctypes.byref(h))
        if st:
            raise Nvfp4Error(st)
        self.h = h
        self.device = device

    def close(self):
        if getattr(self, "h", None):
            self.lib.nvfp4_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, st):
        if st:
            raise Nvfp4Error(st)

    def set_option(self, name, value):
        self._check(self.lib.nvfp4_set_option(self.h, name.encode(), value))

    def get_option(self, name):
        v = c_int()
        self._check(self.lib.nvfp4_get_option(self.h, name.encode(), ctypes.byref(v)))
        return v.value

    def launch_count(self):
        v = ctypes.c_ulonglong()
        self._check(self.lib.nvfp4_launch_count(self.h, ctypes.byref(v)))
        return v.value

    def device_status(self):
        v = ctypes.c_uint()
        self._check(self.lib.nvfp4_device_status(self.h, ctypes.byref(v)))
        return v.value

    def linear_ex(self, A, M, packed, scale, global_scale, N, K, C, residual=None, swiglu_up=None, a_row_stride=0,
                  k_valid=0, px=None, norm_weight=None, norm_eps=0.0, swiglu_epilogue=False, stream=None):
        """nvfp4_linear_ex: the linear layer with SwiGLU (A = gate half, swiglu_up = up half) or
        RMSNorm (norm_weight) formed while staging, a row stride, a zero-padded K, and an
        optional peer exchange."""
        d = LinearDesc(_ptr(A), _ptr(swiglu_up), a_row_stride, k_valid, M, _ptr(packed), _ptr(scale), global_scale, N, K,
                       _ptr(residual), _ptr(C), None if px is None else ctypes.addressof(px), _ptr(norm_weight), norm_eps, int(bool(swiglu_epilogue)))
        self._check(self.lib.nvfp4_linear_ex(self.h, ctypes.byref(d), _stream(stream)))

    def linear_f32(self, A, M, packed, scale, global_scale, N, K, C_f32, stream=None):
        self._check(self.lib.nvfp4_linear_f32(self.h, _ptr(A), M, _ptr(packed), _ptr(scale), global_scale, N, K,
                                              _ptr(C_f32), _stream(stream)))

    def linear_reduce_peers(self, A, M, packed, scale, global_scale, N, K, C, peers, rank, slot_pairs, residual=None,
                            stream=None, check=True):
        """nvfp4_linear_reduce_peers: `peers` = the world's exchange buffers as mapped into this process
        (device tensors or raw pointers), `rank` = this rank's place among them."""
        px = PeerExchange()
        for q, b in enumerate(peers):
            px.peer[q] = _ptr(b)
        px.rank, px.world, px.slot_pairs = rank, len(peers), slot_pairs
        st = self.lib.nvfp4_linear_reduce_peers(self.h, _ptr(A), M, _ptr(packed), _ptr(scale), global_scale, N, K,
                                                _ptr(residual), _ptr(C), ctypes.byref(px), _stream(stream))
        if check:
            self._check(st)
        return st

    def linear(self, A, M, packed, scale, global_scale, N, K, C, residual=None, stream=None, check=True):
        st = self.lib.nvfp4_linear(self.h, _ptr(A), M, _ptr(packed), _ptr(scale), global_scale, N, K,
                                   _ptr(residual), _ptr(C), _stream(stream))
        if check:
            self._check(st)
        return st

    def linear_dual(self, A, M, p1, s1, gs1, p2, s2, gs2, N, K, C1, C2, stream=None):
        self._check(self.lib.nvfp4_linear_dual(self.h, _ptr(A), M, _ptr(p1), _ptr(s1), gs1, _ptr(p2), _ptr(s2),
                                               gs2, N, K, _ptr(C1), _ptr(C2), _stream(stream)))

    def dequant(self, packed, scale, global_scale, N, K, out, stream=None):
        self._check(self.lib.nvfp4_dequant_bf16(self.h, _ptr(packed), _ptr(scale), global_scale, N, K,
                                                _ptr(out), _stream(stream)))

    def scan_scales(self, scale, N, K, stream=None):
        """Block-scale bytes 0x7F / 0xFF in a weight (480 to the reference, NaN to the tensor core); a weight
        that holds any stays off the tensor-core GEMV from here on.  Synchronises."""
        n = ctypes.c_longlong(0)
        self._check(self.lib.nvfp4_scan_scales(self.h, _ptr(scale), N, K, ctypes.byref(n), _stream(stream)))
        return n.value

    def swiglu(self, gate, up, M, I, out, stream=None):
        self._check(self.lib.nvfp4_swiglu(self.h, _ptr(gate), _ptr(up), M, I, _ptr(out), _stream(stream)))

    def swiglu_strided(self, gate, up, M, I, row_stride_in, out, row_stride_out, stream=None):
        self._check(self.lib.nvfp4_swiglu_strided(self.h, _ptr(gate), _ptr(up), M, I, row_stride_in, _ptr(out),
                                                  row_stride_out, _stream(stream)))

    def linear_bf16(self, A, M, W, N, K, C, residual=None, stream=None):
        self._check(self.lib.nvfp4_linear_bf16(self.h, _ptr(A), M, _ptr(W), N, K, _ptr(residual), _ptr(C), _stream(stream)))

    def rmsnorm(self, x, weight, eps, M, K, out, stream=None):
        self._check(self.lib.nvfp4_rmsnorm(self.h, _ptr(x), _ptr(weight), eps, M, K, _ptr(out), _stream(stream)))

    def add_rmsnorm(self, residual, bias, weight, eps, M, K, norm_out, stream=None):
        self._check(self.lib.nvfp4_add_rmsnorm(self.h, _ptr(residual), _ptr(bias), _ptr(weight), eps, M, K, _ptr(norm_out),
                                               _stream(stream)))

    def swiglu_interleaved(self, gate_up, M, I, row_stride_in, out, row_stride_out, stream=None):
        self._check(self.lib.nvfp4_swiglu_interleaved(self.h, _ptr(gate_up), M, I, row_stride_in, _ptr(out), row_stride_out,
                                                      _stream(stream)))

    def kv_append(self, cache, batch, q, k, v, q_out, q_norm=None, k_norm=None, norm_eps=1e-6, inv_freq=None, positions=None, stream=None):
        """nvfp4_kv_append: norms, rotation (of 2 * len(inv_freq) elements) and append.  q, k, v and q_out are [tokens, heads, head dim] tensors
        (views with strides are fine; q and q_out None: keys and values only)."""
        tokens, dim, device = batch.tokens, cache.dim, cache.device
        bf16, fp32, int32 = cache.types
        if q is not None and q_out is None:
            raise ValueError("q needs a q_out")
        qp, qt, qh, heads = _NO_ROWS if q is None else _rows(q, tokens, dim, bf16, device)
        op, ot, oh, out_heads = _NO_ROWS if q is None else _rows(q_out, tokens, dim, bf16, device)
        kp, kt, kh, k_heads = _rows(k, tokens, dim, bf16, device)
        vp, vt, vh, v_heads = _rows(v, tokens, dim, bf16, device)
        if heads != out_heads or k_heads != cache.heads or v_heads != cache.heads:
            raise ValueError("q and q_out have the same heads, k and v the cache's")
        if device != self.device or batch.device != device:
            raise ValueError("cache and batch are on the handle's device")
        qn = kn = freq = pos = rot_dim = 0
        if q_norm is not None:
            if q_norm.dtype is not bf16 or q_norm.numel() != dim or not q_norm.is_contiguous() or q_norm.get_device() != device:
                raise ValueError(_VECTORS)
            qn = q_norm.data_ptr()
        if k_norm is not None:
            if k_norm.dtype is not bf16 or k_norm.numel() != dim or not k_norm.is_contiguous() or k_norm.get_device() != device:
                raise ValueError(_VECTORS)
            kn = k_norm.data_ptr()
        if inv_freq is not None:
            if inv_freq.dtype is not fp32 or not inv_freq.is_contiguous() or inv_freq.get_device() != device:
                raise ValueError(_VECTORS)
            freq, rot_dim = inv_freq.data_ptr(), 2 * inv_freq.numel()
        if positions is not None:
            if positions.dtype is not int32 or positions.numel() < tokens or not positions.is_contiguous() or positions.get_device() != device:
                raise ValueError(_VECTORS)
            pos = positions.data_ptr()
        d = _APPEND.pack(cache.address, batch.address, qp, kp, vp, op, qt, qh, kt, kh, vt, vh, ot, oh, qn, kn, freq, pos, heads, rot_dim, norm_eps)
        self._check(self.lib.nvfp4_kv_append(self.h, d, _stream(stream, device)))

    def paged_attention(self, cache, batch, q, out, gate=None, scale=0.0, stream=None):
        """nvfp4_paged_attention: q, out and gate are [tokens, heads, head dim] tensors; scale 0 = 1 / sqrt(head dim)."""
        tokens, dim, device = batch.tokens, cache.dim, cache.device
        bf16 = cache.types[0]
        qp, qt, qh, heads = _rows(q, tokens, dim, bf16, device)
        op, ot, oh, out_heads = _rows(out, tokens, dim, bf16, device)
        gp, gt, gh, gate_heads = (0, 0, 0, heads) if gate is None else _rows(gate, tokens, dim, bf16, device)
        if not heads == out_heads == gate_heads:
            raise ValueError("q, out and gate have the same heads")
        if device != self.device or batch.device != device:
            raise ValueError("cache and batch are on the handle's device")
        d = _ATTENTION.pack(cache.address, batch.address, qp, gp, op, qt, qh, gt, gh, ot, oh, heads, scale)
        self._check(self.lib.nvfp4_paged_attention(self.h, d, _stream(stream, device)))

    def linear_host(self, A_host, M, packed, scale, global_scale, N, K, C_host, residual_host=None, stream=None):
        self._check(self.lib.nvfp4_linear_host(self.h, _ptr(A_host), M, _ptr(packed), _ptr(scale), global_scale,
                                               N, K, _ptr(residual_host), _ptr(C_host), _stream(stream)))


class Chain:
    """nvfp4_chain: a fixed sequence of linears (up to 8 tokens each) run by one launch.  `linears` is a list
    of dicts with the fields of nvfp4_linear_desc (A, M, packed, scale, global_scale, N, K, C and the
    optional residual, swiglu_up, a_row_stride, k_valid, px, norm_weight, norm_eps, swiglu_epilogue);
    tensors are given as torch tensors or raw addresses and must stay alive while the chain exists."""

    def __init__(self, handle, linears):
        self.handle = handle
        self.keep = linears
        arr = (LinearDesc * len(linears))()
        for d, l in zip(arr, linears):
            px = l.get("px")
            d.A, d.swiglu_up = _ptr(l["A"]), _ptr(l.get("swiglu_up"))
            d.a_row_stride, d.k_valid, d.M = l.get("a_row_stride", 0), l.get("k_valid", 0), l["M"]
            d.packed, d.scale, d.global_scale = _ptr(l["packed"]), _ptr(l["scale"]), l.get("global_scale", 1.0)
            d.N, d.K = l["N"], l["K"]
            d.residual, d.C = _ptr(l.get("residual")), _ptr(l["C"])
            d.px = None if px is None else ctypes.addressof(px)
            d.norm_weight, d.norm_eps = _ptr(l.get("norm_weight")), l.get("norm_eps", 0.0)
            d.swiglu_epilogue = int(bool(l.get("swiglu_epilogue", False)))
        c = c_void_p()
        st = handle.lib.nvfp4_chain_create(handle.h, arr, len(linears), ctypes.byref(c))
        if st:
            raise Nvfp4Error(st)
        self.c = c

    def run(self, stream=None):
        st = self.handle.lib.nvfp4_chain_run(self.c, _stream(stream))
        if st:
            raise Nvfp4Error(st)

    def close(self):
        if getattr(self, "c", None):
            self.handle.lib.nvfp4_chain_destroy(self.c)
            self.c = None

"""ctypes binding of libnihilus_b200.so (see include/nihilus_b200.h) plus small torch conveniences.

No fallback: if the shared library is absent this module raises at import, and every call below runs
the CUDA kernels through the C ABI.
"""
from __future__ import annotations

import ctypes as C
import os

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
# NHB_LIB names another build of the same library (experiments with compile-time knobs)
LIB_PATH = os.environ.get("NHB_LIB") or os.path.join(_HERE, "lib", "libnihilus_b200.so")

if not os.path.exists(LIB_PATH):
    raise ImportError(
        f"{LIB_PATH} is missing: build it with `python -m nihilus_b200.build` (nvcc, sm_100a). "
        "nihilus_b200 has no CPU or PyTorch fallback."
    )

lib = C.CDLL(LIB_PATH)

ACT_Q8, ACT_F32 = 0, 1
SQRT_IEEE, SQRT_X86_FAST = 0, 1
KERNEL_AUTO, KERNEL_GEMV_LDG, KERNEL_GEMV_STREAM, KERNEL_GEMM_TC, KERNEL_GEMV_ROWS = 0, 1, 2, 3, 4
OK, ERR_ARG, ERR_CUDA, ERR_NCCL, ERR_TIMEOUT, ERR_UNSUPPORTED, ERR_NOMEM = 0, -1, -2, -3, -4, -5, -6
KV_F16, KV_BF16 = 0, 1
ROPE_STYLES = {"pairs": 0, "halves": 1}

# every symbol include/nihilus_b200.h declares
EXPORTS = (
    "nhb_version", "nhb_arch", "nhb_last_error", "nhb_shard_rows", "nhb_repack_q8_0_host", "nhb_unpack_q8_0_host",
    "nhb_choose_kernel", "nhb_mul_mat_bytes", "nhb_mul_mat_flops", "nhb_ctx_create", "nhb_ctx_destroy", "nhb_ctx_set_stream",
    "nhb_sync", "nhb_ctx_set_gemv_max_m", "nhb_ctx_set_option", "nhb_ctx_launch_count", "nhb_memcpy_h2d", "nhb_memcpy_d2h",
    "nhb_weight_upload_q8_0", "nhb_weight_free", "nhb_weight_info_get", "nhb_weight_download_q8_0", "nhb_mul_mat",
    "nhb_mul_mat_batch", "nhb_mul_mat_host", "nhb_mul_mat_block_dots", "nhb_quantize_q8_0", "nhb_graph_begin", "nhb_graph_end",
    "nhb_graph_launch", "nhb_graph_free", "nhb_comm_unique_id", "nhb_comm_init", "nhb_all_gather", "nhb_all_gather_batch",
    "nhb_mul_mat_q8_0_noalloc", "nhb_noalloc_max_bytes", "nhb_noalloc_last_error", "nhb_device_alloc", "nhb_device_free", "nhb_symm_alloc", "nhb_symm_free", "nhb_symm_alloc_local", "nhb_all_gather_local", "nhb_sync_all", "nhb_wait_planner_create", "nhb_wait_planner_destroy", "nhb_wait_planner_add_region",
    "nhb_wait_planner_launch", "nhb_wait_planner_wait_all", "nhb_wait_planner_seq", "nhb_wait_planner_capture_begin", "nhb_wait_planner_capture_end",
    "nhb_wait_planner_replayed", "nhb_place_rows", "nhb_gemm_tile_plan",
    "nhb_rms_norm_mul", "nhb_rms_norm_mul_q8_0", "nhb_rms_norm_mul_mat_batch",
    "nhb_gguf_open", "nhb_gguf_last_error", "nhb_gguf_close", "nhb_gguf_tensor_count", "nhb_gguf_find", "nhb_gguf_tensor_get",
    "nhb_gguf_get_number", "nhb_gguf_get_string", "nhb_gguf_upload_q8_0", "nhb_gguf_read_f32",
    "nhb_chain_create", "nhb_chain_launch", "nhb_chain_free", "nhb_mul_mat_swiglu_add", "nhb_mul_mat_add", "nhb_swiglu",
    "nhb_get_rows_q8_0", "nhb_last_token_logits", "nhb_weight_save", "nhb_weight_load",
    "nhb_kv_reserve", "nhb_kv_fork", "nhb_kv_free", "nhb_kv_compact", "nhb_rope_kv_append", "nhb_attn_prompt", "nhb_attn_decode",
)


class WeightInfo(C.Structure):
    _fields_ = [("N", C.c_int64), ("K", C.c_int64), ("n0", C.c_int64), ("n1", C.c_int64), ("q", C.c_void_p), ("d", C.c_void_p),
                ("bytes_q8", C.c_int64)]


class GgufTensor(C.Structure):
    _fields_ = [("name", C.c_char_p), ("n_dims", C.c_int), ("dims", C.c_int64 * 4), ("type", C.c_int), ("bytes", C.c_int64),
                ("offset", C.c_int64), ("data", C.c_void_p)]


class MulMatOp(C.Structure):
    _fields_ = [("w", C.c_void_p), ("x", C.c_void_p), ("ldx", C.c_int64), ("y", C.c_void_p), ("ldy", C.c_int64), ("M", C.c_int64)]


class KvCacheStruct(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("table", C.c_void_p), ("lens", C.c_void_p), ("refs", C.c_void_p), ("n_layers", C.c_int64),
                ("n_pages", C.c_int64), ("kv_heads", C.c_int64), ("page_tokens", C.c_int64), ("head_dim", C.c_int64), ("max_seqs", C.c_int64),
                ("max_pages", C.c_int64), ("type", C.c_int)]


class RopeStruct(C.Structure):
    _fields_ = [("base", C.c_double), ("dims", C.c_int64), ("style", C.c_int), ("factors", C.c_void_p)]


def _sig(name, restype, *argtypes):
    fn = getattr(lib, name)
    fn.restype = restype
    fn.argtypes = list(argtypes)
    return fn


_vp, _i, _i64 = C.c_void_p, C.c_int, C.c_int64
_sig("nhb_version", _i)
_sig("nhb_gguf_open", _i, C.c_char_p, C.POINTER(_vp))
_sig("nhb_gguf_last_error", C.c_char_p)
_sig("nhb_gguf_close", _i, _vp)
_sig("nhb_gguf_tensor_count", _i64, _vp)
_sig("nhb_gguf_find", _i64, _vp, C.c_char_p)
_sig("nhb_gguf_tensor_get", _i, _vp, _i64, C.POINTER(GgufTensor))
_sig("nhb_gguf_get_number", _i, _vp, C.c_char_p, C.POINTER(C.c_double))
_sig("nhb_gguf_get_string", C.c_char_p, _vp, C.c_char_p)
_sig("nhb_gguf_upload_q8_0", _i, _vp, _vp, C.c_char_p, C.POINTER(_vp))
_sig("nhb_gguf_read_f32", _i, _vp, C.c_char_p, _vp, _i64)
_sig("nhb_rms_norm_mul", _i, _vp, _vp, _i64, _vp, C.c_float, _i, _vp, _i64, _i64, _i64)
_sig("nhb_rms_norm_mul_q8_0", _i, _vp, _vp, _i64, _vp, C.c_float, _i, _vp, _i64, _i64)
_sig("nhb_rms_norm_mul_mat_batch", _i, _vp, C.POINTER(MulMatOp), _i, _vp, C.c_float, _i, _i)
_sig("nhb_arch", _i)
_sig("nhb_last_error", C.c_char_p, _vp)
_sig("nhb_shard_rows", _i, _i64, _i, _i, C.POINTER(_i64), C.POINTER(_i64))
_sig("nhb_place_rows", _i, _i64, _i64, _i, _i, _i64, C.POINTER(_i64), C.POINTER(_i64))
_sig("nhb_gemm_tile_plan", _i, _i64, _i64, _i, C.POINTER(_i), C.POINTER(_i), C.POINTER(_i), C.POINTER(_i))
_sig("nhb_repack_q8_0_host", _i, _vp, _i64, _i64, _i64, _i64, _vp, _vp)
_sig("nhb_unpack_q8_0_host", _i, _vp, _vp, _i64, _i64, _vp)
_sig("nhb_choose_kernel", _i, _i64, _i64, _i64, _i)
_sig("nhb_mul_mat_bytes", _i64, _i64, _i64, _i64)
_sig("nhb_mul_mat_flops", _i64, _i64, _i64, _i64)
_sig("nhb_ctx_create", _i, C.POINTER(_vp), _i, _i, _i)
_sig("nhb_ctx_destroy", _i, _vp)
_sig("nhb_ctx_set_stream", _i, _vp, _vp)
_sig("nhb_sync", _i, _vp)
_sig("nhb_ctx_set_gemv_max_m", _i, _vp, _i)
_sig("nhb_ctx_set_option", _i, _vp, C.c_char_p, _i)
_sig("nhb_ctx_launch_count", C.c_longlong, _vp)
_sig("nhb_memcpy_h2d", _i, _vp, _vp, _vp, C.c_size_t)
_sig("nhb_memcpy_d2h", _i, _vp, _vp, _vp, C.c_size_t)
_sig("nhb_device_alloc", _i, _vp, C.c_size_t, C.POINTER(_vp))
_sig("nhb_device_free", _i, _vp, _vp)
_sig("nhb_symm_alloc", _i, _vp, C.c_size_t, C.POINTER(_vp))
_sig("nhb_symm_alloc_local", _i, C.POINTER(_vp), _i, C.c_size_t, C.POINTER(_vp))
_sig("nhb_all_gather_local", _i, C.POINTER(_vp), _i, C.POINTER(_vp), _i64, _i64, _i64)
_sig("nhb_sync_all", _i, C.POINTER(_vp), _i)
_sig("nhb_wait_planner_create", _vp, _i)
_sig("nhb_wait_planner_destroy", None, _vp)
_sig("nhb_wait_planner_add_region", _i, _vp, _vp, C.c_size_t)
_sig("nhb_wait_planner_launch", _i, _vp, C.POINTER(_vp), C.POINTER(C.c_size_t), _i, C.POINTER(_vp), C.POINTER(C.c_size_t), _i, _i, C.POINTER(_i), C.POINTER(_i))
_sig("nhb_wait_planner_wait_all", _i, _vp)
_sig("nhb_wait_planner_seq", C.c_longlong, _vp)
_sig("nhb_wait_planner_capture_begin", None, _vp)
_sig("nhb_wait_planner_capture_end", _i, _vp)
_sig("nhb_wait_planner_replayed", _i, _vp, _i)
_sig("nhb_symm_free", _i, _vp, _vp)
_sig("nhb_weight_upload_q8_0", _i, _vp, _vp, _i64, _i64, C.POINTER(_vp))
_sig("nhb_weight_free", _i, _vp, _vp)
_sig("nhb_weight_info_get", _i, _vp, C.POINTER(WeightInfo))
_sig("nhb_weight_download_q8_0", _i, _vp, _vp, _vp)
_sig("nhb_mul_mat", _i, _vp, _vp, _vp, _i64, _vp, _i64, _i64, _i, _i)
_sig("nhb_mul_mat_batch", _i, _vp, C.POINTER(MulMatOp), _i, _i, _i)
_sig("nhb_mul_mat_host", _i, _vp, _vp, _vp, _i64, _vp, _i64, _i64, _i, _i)
_sig("nhb_mul_mat_block_dots", _i, _vp, _vp, _vp, _i64, _i64, _vp)
_sig("nhb_quantize_q8_0", _i, _vp, _vp, _i64, _i64, _i64, _vp, _vp)
_sig("nhb_graph_begin", _i, _vp)
_sig("nhb_graph_end", _i, _vp, C.POINTER(_vp))
_sig("nhb_graph_launch", _i, _vp, _vp)
_sig("nhb_graph_free", _i, _vp, _vp)
_sig("nhb_comm_unique_id", _i, _vp)
_sig("nhb_comm_init", _i, _vp, _vp)
_sig("nhb_all_gather", _i, _vp, _vp, _i64, _i64, _i64)
_sig("nhb_mul_mat_q8_0_noalloc", _i, _vp, _vp, _i64, _i64, _vp, _i64, _vp, _i64, _i64, _vp)
_sig("nhb_noalloc_max_bytes", _i64)
_sig("nhb_noalloc_last_error", C.c_char_p)
_sig("nhb_all_gather_batch", _i, _vp, C.POINTER(_vp), C.POINTER(_i64), C.POINTER(_i64), C.POINTER(_i64), _i)
_sig("nhb_mul_mat_swiglu_add", _i, _vp, _vp, _vp, _vp, _i64, _vp, _i64, _vp, _i64, _i64)
_sig("nhb_mul_mat_add", _i, _vp, _vp, _vp, _i64, _vp, _i64, _vp, _i64, _i64)
_sig("nhb_swiglu", _i, _vp, _vp, _vp, _i64, _vp, _i64, _i64, _i64)
_sig("nhb_get_rows_q8_0", _i, _vp, _vp, _vp, _i64, _vp, _i64)
_sig("nhb_last_token_logits", _i, _vp, _vp, _vp, _i64, _i64, _vp, C.c_float, _i, _vp)
_sig("nhb_weight_save", _i, _vp, _vp, C.c_char_p)
_sig("nhb_weight_load", _i, _vp, C.c_char_p, _i64, _i64, C.POINTER(_vp))
_kvp = C.POINTER(KvCacheStruct)
_sig("nhb_kv_reserve", _i, _vp, _kvp, _vp, _vp, _i64)
_sig("nhb_kv_fork", _i, _vp, _kvp, _vp, _vp, _i64, _i)
_sig("nhb_kv_free", _i, _vp, _kvp, _vp, _i64)
_sig("nhb_kv_compact", _i, _vp, _kvp, _vp)
_sig("nhb_rope_kv_append", _i, _vp, _kvp, _i64, _vp, _i64, _i64, _vp, _i64, _vp, _i64, _i64, _vp, _vp, _i64, C.POINTER(RopeStruct), _vp, _i64)
_sig("nhb_attn_prompt", _i, _vp, _kvp, _i64, _vp, _i64, _i64, _i64, _vp, _vp, _i64, C.c_float, _vp, _i64)
_sig("nhb_attn_decode", _i, _vp, _kvp, _i64, _vp, _i64, _i64, _vp, _i64, _i64, C.c_float, _vp, _i64)
_sig("nhb_chain_create", _i, _vp, C.POINTER(MulMatOp), C.POINTER(_i), _i, C.POINTER(_vp))
_sig("nhb_chain_launch", _i, _vp, _vp)
_sig("nhb_chain_free", _i, _vp, _vp)


def _ld(t) -> int:
    """Leading dimension of a 2-D tensor; a single row may carry any stride (numpy's relaxed strides), which means nothing."""
    return t.stride(0) if t.shape[0] > 1 else max(int(t.stride(0)), int(t.shape[1]), 1)


def _tensor_from_ptr(ptr: int, nbytes: int, device: int, dtype):
    """A torch view of device memory this library owns (no copy; the caller keeps the allocation alive)."""
    import torch

    class _Cai:
        __cuda_array_interface__ = {"shape": (nbytes,), "typestr": "|u1", "data": (ptr, False), "version": 2}

    t = torch.as_tensor(_Cai(), device=f"cuda:{device}")
    return t.view(dtype)


class NhbError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"nihilus_b200 error {code}: {msg}")
        self.code = code


def last_error(ctx=None) -> str:
    s = lib.nhb_last_error(ctx)
    return s.decode() if s else ""


def _check(rc: int, ctx=None):
    if rc != OK:
        raise NhbError(rc, last_error(ctx))


def shard_rows(N: int, world: int, rank: int) -> tuple[int, int]:
    a, b = _i64(), _i64()
    _check(lib.nhb_shard_rows(N, world, rank, C.byref(a), C.byref(b)))
    return a.value, b.value


def place_rows(N: int, K: int, world: int, rank: int, replicate_below_bytes: int = 0) -> tuple[int, int]:
    a, b = _i64(), _i64()
    _check(lib.nhb_place_rows(N, K, world, rank, replicate_below_bytes, C.byref(a), C.byref(b)))
    return a.value, b.value


def gemm_tile_plan(rows: int, M: int, sms: int = 148) -> dict:
    sw, nt, lt, ct = _i(), _i(), _i(), _i()
    _check(lib.nhb_gemm_tile_plan(rows, M, sms, C.byref(sw), C.byref(nt), C.byref(lt), C.byref(ct)))
    return {"swapped": bool(sw.value), "tile_cols": nt.value, "lane_tiles": lt.value, "col_tiles": ct.value}


def repack_host(blocks: np.ndarray, n0: int = 0, n1: int | None = None):
    """uint8 [N, K/32, 34] -> (int8 [rows, K], uint16 [rows, K/32]) on the host (no GPU)."""
    blocks = np.ascontiguousarray(blocks, dtype=np.uint8)
    N, nb, _ = blocks.shape
    n1 = N if n1 is None else n1
    q = np.empty((max(n1 - n0, 0), nb * 32), dtype=np.int8)
    d = np.empty((max(n1 - n0, 0), nb), dtype=np.uint16)
    _check(lib.nhb_repack_q8_0_host(blocks.ctypes.data, N, nb * 32, n0, n1, q.ctypes.data, d.ctypes.data))
    return q, d


def unpack_host(q: np.ndarray, d: np.ndarray) -> np.ndarray:
    q = np.ascontiguousarray(q, dtype=np.int8)
    d = np.ascontiguousarray(d, dtype=np.uint16)
    rows, K = q.shape
    out = np.empty((rows, K // 32, 34), dtype=np.uint8)
    _check(lib.nhb_unpack_q8_0_host(q.ctypes.data, d.ctypes.data, rows, K, out.ctypes.data))
    return out


class Weight:
    def __init__(self, ctx: "Context", handle: int):
        self.ctx = ctx
        self.handle = handle
        info = WeightInfo()
        _check(lib.nhb_weight_info_get(handle, C.byref(info)))
        self.N, self.K, self.n0, self.n1 = info.N, info.K, info.n0, info.n1
        self.q_ptr, self.d_ptr, self.bytes_q8 = info.q, info.d, info.bytes_q8

    def save(self, path: str):
        """This shard's repacked planes as a cache file (nhb_weight_save)."""
        _check(lib.nhb_weight_save(self.ctx.handle, self.handle, os.fsencode(path)), self.ctx.handle)

    def download(self) -> np.ndarray:
        out = np.empty((self.n1 - self.n0, self.K // 32, 34), dtype=np.uint8)
        _check(lib.nhb_weight_download_q8_0(self.ctx.handle, self.handle, out.ctypes.data), self.ctx.handle)
        return out

    def free(self):
        if self.handle:
            lib.nhb_weight_free(self.ctx.handle, self.handle)
            self.handle = None


class Gguf:
    """A mapped GGUF model file (nhb_gguf_*): tensor table, scalar metadata, Q8_0 upload by tensor name."""

    def __init__(self, path: str):
        h = _vp()
        rc = lib.nhb_gguf_open(os.fsencode(path), C.byref(h))
        if rc != 0:
            raise NhbError(rc, (lib.nhb_gguf_last_error() or b"").decode())
        self.handle = h.value

    def close(self):
        if self.handle:
            lib.nhb_gguf_close(self.handle)
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    def __len__(self):
        return int(lib.nhb_gguf_tensor_count(self.handle))

    def tensor(self, key):
        """key: index or name -> dict(name, dims, type, bytes, offset)."""
        idx = key if isinstance(key, int) else int(lib.nhb_gguf_find(self.handle, key.encode()))
        t = GgufTensor()
        if idx < 0 or lib.nhb_gguf_tensor_get(self.handle, idx, C.byref(t)) != 0:
            raise KeyError(key)
        return {"name": t.name.decode(), "dims": tuple(t.dims[: max(t.n_dims, 1)]), "type": t.type, "bytes": t.bytes, "offset": t.offset,
                "data": t.data}

    def number(self, key: str):
        v = C.c_double()
        if lib.nhb_gguf_get_number(self.handle, key.encode(), C.byref(v)) != 0:
            raise KeyError(key)
        return v.value

    def string(self, key: str):
        v = lib.nhb_gguf_get_string(self.handle, key.encode())
        if v is None:
            raise KeyError(key)
        return v.decode()

    def read_f32(self, name: str) -> np.ndarray:
        t = self.tensor(name)
        out = np.empty(t["bytes"] // 4, dtype=np.float32)
        _check(lib.nhb_gguf_read_f32(self.handle, name.encode(), out.ctypes.data, out.size))
        return out.reshape(tuple(reversed(t["dims"])))

    def upload_q8_0(self, ctx: "Context", name: str) -> "Weight":
        h = _vp()
        _check(lib.nhb_gguf_upload_q8_0(ctx.handle, self.handle, name.encode(), C.byref(h)), ctx.handle)
        return Weight(ctx, h.value)


def _i32(t, what: str, device: int | None = None):
    """Pointer of a contiguous device int32 list (None stays None)."""
    if t is None:
        return None
    if t.dtype is not _torch_types()[0] or not t.is_contiguous() or (t.get_device() != device if device is not None else not t.is_cuda):
        raise NhbError(ERR_ARG, f"{what} must be a contiguous int32 tensor on the context's GPU")
    return t.data_ptr()


def _rows32(t, rows: int, width: int, what: str, device: int):
    """Pointer and leading dimension of f32 rows on the context's GPU."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or shape[0] != rows or shape[1] != width or (rows and width > 1 and stride[1] != 1) or t.dtype is not _torch_types()[1] or t.get_device() != device:
        raise NhbError(ERR_ARG, f"{what} must be {rows} f32 rows of {width} on the context's GPU")
    return t.data_ptr(), (stride[0] if rows > 1 else max(width, 1))  # (one row's stride says nothing)


def _torch_types():
    """(int32, float32) of torch, imported at the first use."""
    global _types
    if _types is None:
        import torch

        _types = (torch.int32, torch.float32)
    return _types


_types = None


def _torch_stream(device: int) -> int:
    """The handle of torch's current stream on a GPU."""
    global _current_stream
    if _current_stream is None:
        import torch

        torch.cuda.init()
        _current_stream = torch._C._cuda_getCurrentRawStream  # (a Stream object costs 3 us)
    # torch reports its default stream as handle 0, which nhb_ctx_set_stream reads as "the context's own
    # stream"; 1 is cudaStreamLegacy, the same default stream named explicitly
    return _current_stream(device) or 1


_current_stream = None


class KvCache:
    """The paged K/V cache over torch tensors (nhb_kv_cache): k, v [layers][pages][kv_heads][page_tokens][head_dim] f16 or bf16,
    table [max_seqs][max_pages], lens [max_seqs], refs [pages] int32.  It is made for these tensors: others take another KvCache."""

    def __setattr__(self, name, value):
        if name in ("k", "v", "table", "lens", "refs") and self.__dict__.get(name, value) is not value:
            raise NhbError(ERR_ARG, f"a KvCache is made for its tensors: {name} cannot be replaced")
        self.__dict__[name] = value

    def __init__(self, k, v, table, lens, refs):
        import torch

        types = {torch.float16: KV_F16, torch.bfloat16: KV_BF16}
        if k.dtype not in types or v.dtype != k.dtype or k.dim() != 5 or v.shape != k.shape or not (k.is_contiguous() and v.is_contiguous()) or not (k.is_cuda and v.is_cuda):
            raise NhbError(ERR_ARG, "k and v must be contiguous f16 or bf16 tensors [layers][pages][kv_heads][page_tokens][head_dim] on the GPU")
        if table.dim() != 2 or lens.shape != table.shape[:1] or refs.shape != k.shape[1:2]:
            raise NhbError(ERR_ARG, "table [max_seqs][max_pages], lens [max_seqs] and refs [pages] do not fit one another")
        if any(t.device != k.device for t in (v, table, lens, refs)):
            raise NhbError(ERR_ARG, "the cache's tensors lie on different devices")
        self.k, self.v, self.table, self.lens, self.refs = k, v, table, lens, refs
        self.layers, self.pages, self.kv_heads, self.page_tokens, self.head_dim = (int(x) for x in k.shape)
        self.max_seqs, self.max_pages = (int(x) for x in table.shape)
        self.struct = KvCacheStruct(k.data_ptr(), v.data_ptr(), _i32(table, "table"), _i32(lens, "lens"), _i32(refs, "refs"), self.layers, self.pages, self.kv_heads,
                                    self.page_tokens, self.head_dim, self.max_seqs, self.max_pages, types[k.dtype])
        self.ref = C.byref(self.struct)
        self.device = k.get_device()

    @classmethod
    def empty(cls, layers: int, pages: int, kv_heads: int, head_dim: int, max_seqs: int, max_tokens: int, page_tokens: int = 64, dtype=None, device: int = 0) -> "KvCache":
        """A cache that holds nothing; a sequence may grow to max_tokens."""
        import torch

        dev, dtype = f"cuda:{device}", dtype or torch.float16
        shape = (layers, pages, kv_heads, page_tokens, head_dim)
        table = torch.full((max_seqs, max(1, -(-max_tokens // page_tokens))), -1, dtype=torch.int32, device=dev)
        zeros = lambda n: torch.zeros(n, dtype=torch.int32, device=dev)  # noqa: E731
        return cls(torch.empty(shape, dtype=dtype, device=dev), torch.empty(shape, dtype=dtype, device=dev), table, zeros(max_seqs), zeros(pages))


class Rope:
    """Rotary embedding (nhb_rope): dims None rotates the whole head; factors: f32 [dims / 2] on the GPU or None."""

    def __init__(self, base: float = 500000.0, style: str = "pairs", dims: int | None = None, factors=None):
        self.base, self.style, self.dims, self.factors = float(base), style, dims, factors
        self._check()

    def __setattr__(self, name, value):
        self.__dict__[name] = value
        self.__dict__["_refs"] = {}  # structs by head size and GPU, of what is assigned now

    def _check(self):
        f = self.factors
        if self.style not in ROPE_STYLES:
            raise NhbError(ERR_ARG, f"unknown rotary style {self.style!r}")
        if f is not None and (f.dtype is not _torch_types()[1] or f.dim() != 1 or not f.is_contiguous() or not f.is_cuda):
            raise NhbError(ERR_ARG, "factors must be a contiguous f32 tensor on the GPU")

    def ref(self, head_dim: int, device: int | None = None):
        """The C struct for heads of this size, by reference; it follows what is assigned to the rotation.  device: the GPU that reads the factors."""
        made = self._refs.get((head_dim, device))
        if made is None:
            self._check()
            f, dims = self.factors, head_dim if self.dims is None else int(self.dims)
            if f is not None and device is not None and f.get_device() != device:
                raise NhbError(ERR_ARG, "factors lie on another GPU than the context")
            if f is not None and f.shape[0] < dims // 2:
                raise NhbError(ERR_ARG, "factors holds fewer than dims / 2 values")
            made = self._refs[(head_dim, device)] = C.byref(RopeStruct(self.base, dims, ROPE_STYLES[self.style], f.data_ptr() if f is not None else None))
        return made


def _check_cu(cu, n: int):
    if cu is not None and (cu.dim() != 1 or cu.shape[0] != n + 1):
        raise NhbError(ERR_ARG, "cu holds one offset more than there are list entries")


def _heads(width: int, cache: KvCache) -> int:
    if width % cache.head_dim:
        raise NhbError(ERR_ARG, "the rows are not a whole number of heads")
    return width // cache.head_dim


class Graph:
    def __init__(self, ctx: "Context", handle: int):
        self.ctx, self.handle = ctx, handle

    def launch(self):
        _check(lib.nhb_graph_launch(self.ctx.handle, self.handle), self.ctx.handle)

    def free(self):
        if self.handle:
            lib.nhb_graph_free(self.ctx.handle, self.handle)
            self.handle = None


class Chain:
    """A token's sequence of dependent stages as one persistent kernel (nhb_chain_*)."""

    def __init__(self, ctx: "Context", handle: int, keep):
        self.ctx, self.handle, self._keep = ctx, handle, keep  # the tensors the chain names stay alive with it

    def launch(self):
        _check(lib.nhb_chain_launch(self.ctx.handle, self.handle), self.ctx.handle)

    def free(self):
        if self.handle:
            lib.nhb_chain_free(self.ctx.handle, self.handle)
            self.handle = None
            self._keep = None


class Context:
    """One GPU, one row shard (rank of world)."""

    def __init__(self, device: int = 0, rank: int = 0, world: int = 1):
        h = _vp()
        _check(lib.nhb_ctx_create(C.byref(h), device, rank, world))
        self.handle = h.value
        self.device, self.rank, self.world = device, rank, world

    def close(self):
        if self.handle:
            lib.nhb_ctx_destroy(self.handle)
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    stream = None  # the handle last set (1: the legacy stream); None: the context's own stream
    capturing = False  # between graph_begin and graph_end

    def set_stream(self, cuda_stream: int | None):
        _check(lib.nhb_ctx_set_stream(self.handle, cuda_stream), self.handle)
        self.stream = cuda_stream or None

    def use_torch_stream(self):
        """Run on torch's current stream, so tensors made by torch and kernels launched here are ordered.  Cheap where the context is on it
        already: a program that changes torch's stream may call it in front of every step."""
        handle = _torch_stream(self.device)
        if handle != self.stream:
            self.set_stream(handle)

    def set_option(self, name: str, value: int):
        _check(lib.nhb_ctx_set_option(self.handle, name.encode(), value), self.handle)

    def sync(self):
        _check(lib.nhb_sync(self.handle), self.handle)

    @property
    def launches(self) -> int:
        return int(lib.nhb_ctx_launch_count(self.handle))

    def upload(self, blocks: np.ndarray) -> Weight:
        blocks = np.ascontiguousarray(blocks, dtype=np.uint8)
        N, nb, bb = blocks.shape
        assert bb == 34
        h = _vp()
        _check(lib.nhb_weight_upload_q8_0(self.handle, blocks.ctypes.data, N, nb * 32, C.byref(h)), self.handle)
        return Weight(self, h.value)

    def load_weight(self, path: str, N: int, K: int) -> Weight:
        """A weight from its cache file (nhb_weight_load): the planes go straight to the device."""
        h = _vp()
        _check(lib.nhb_weight_load(self.handle, os.fsencode(path), N, K, C.byref(h)), self.handle)
        return Weight(self, h.value)

    def get_rows(self, table: Weight, token_ids, y=None):
        """Token-embedding gather: token_ids torch cuda int32 [M] -> f32 [M, K]."""
        import torch

        M = token_ids.shape[0]
        if y is None:
            y = torch.zeros((M, table.K), dtype=torch.float32, device=token_ids.device)
        _check(lib.nhb_get_rows_q8_0(self.handle, table.handle, token_ids.data_ptr(), M, y.data_ptr(), _ld(y) if M else table.K), self.handle)
        return y

    def last_token_logits(self, w: Weight, hidden, norm_w, eps: float, sqrt_mode: int = SQRT_IEEE):
        import torch

        seq = hidden.shape[0]
        out = torch.zeros((1, w.N), dtype=torch.float32, device=hidden.device)
        _check(lib.nhb_last_token_logits(self.handle, w.handle, hidden.data_ptr(), _ld(hidden), seq, norm_w.data_ptr(), eps, sqrt_mode, out.data_ptr()), self.handle)
        return out

    # ---- device-pointer level (torch tensors supply the memory) ----
    def mul_mat(self, w: Weight, x, y=None, act_mode: int = ACT_Q8, kernel: int = KERNEL_AUTO):
        """x: torch cuda f32 [M, K] (row stride allowed) -> y f32 [M, N] (this shard's columns written)."""
        import torch

        M = x.shape[0]
        if y is None:
            y = torch.zeros((M, w.N), dtype=torch.float32, device=x.device)
        _check(lib.nhb_mul_mat(self.handle, w.handle, x.data_ptr(), _ld(x) if M > 0 else w.K, y.data_ptr(),
                               _ld(y) if M > 0 else max(w.N, 1), M, act_mode, kernel), self.handle)
        return y

    def mul_mat_batch(self, ops, act_mode: int = ACT_Q8, kernel: int = KERNEL_AUTO):
        """ops: list of (Weight, x, y) torch tensors."""
        arr = (MulMatOp * len(ops))()
        for i, (w, x, y) in enumerate(ops):
            arr[i] = MulMatOp(w.handle, x.data_ptr(), _ld(x), y.data_ptr(), _ld(y), x.shape[0])
        _check(lib.nhb_mul_mat_batch(self.handle, arr, len(ops), act_mode, kernel), self.handle)

    def mul_mat_host(self, w: Weight, x: np.ndarray, y: np.ndarray | None = None, act_mode: int = ACT_Q8, kernel: int = KERNEL_AUTO,
                     sync: bool = True) -> np.ndarray:
        x = np.ascontiguousarray(x, dtype=np.float32)
        if x.ndim == 1:
            x = x[None, :]
        M = x.shape[0]
        if y is None:
            y = np.zeros((M, w.N), dtype=np.float32)
        _check(lib.nhb_mul_mat_host(self.handle, w.handle, x.ctypes.data, x.shape[1], y.ctypes.data, max(w.N, 1), M, act_mode, kernel),
               self.handle)
        if sync:
            self.sync()
        return y

    def mul_mat_swiglu_add(self, w: Weight, gate, up, residual=None, y=None):
        """y = W . quantise(silu(gate) * up) [+ residual] (the FFN tail of a block)."""
        import torch

        M = gate.shape[0]
        if y is None:
            y = torch.zeros((M, w.N), dtype=torch.float32, device=gate.device)
        _check(lib.nhb_mul_mat_swiglu_add(self.handle, w.handle, gate.data_ptr(), up.data_ptr(), _ld(gate) if M else w.K,
                                          residual.data_ptr() if residual is not None else None, _ld(residual) if residual is not None and M else max(w.N, 1),
                                          y.data_ptr(), _ld(y) if M else max(w.N, 1), M), self.handle)
        return y

    def mul_mat_add(self, w: Weight, x, residual, y=None):
        """y = W . quantise(x) + residual (attn_output and the residual stream)."""
        import torch

        M = x.shape[0]
        if y is None:
            y = torch.zeros((M, w.N), dtype=torch.float32, device=x.device)
        _check(lib.nhb_mul_mat_add(self.handle, w.handle, x.data_ptr(), _ld(x) if M else w.K, residual.data_ptr(), _ld(residual) if M else max(w.N, 1),
                                   y.data_ptr(), _ld(y) if M else max(w.N, 1), M), self.handle)
        return y

    def swiglu(self, gate, up):
        import torch

        M, K = gate.shape
        h = torch.empty((M, K), dtype=torch.float32, device=gate.device)
        _check(lib.nhb_swiglu(self.handle, gate.data_ptr(), up.data_ptr(), _ld(gate) if M else K, h.data_ptr(), K, M, K), self.handle)
        return h

    def block_dots(self, w: Weight, x):
        import torch

        M = x.shape[0]
        out = torch.zeros((M, w.n1 - w.n0, w.K // 32), dtype=torch.int32, device=x.device)
        _check(lib.nhb_mul_mat_block_dots(self.handle, w.handle, x.data_ptr(), x.stride(0), M, out.data_ptr()), self.handle)
        return out

    def quantize(self, x):
        import torch

        M, K = x.shape
        q = torch.empty((M, K), dtype=torch.int8, device=x.device)
        d = torch.empty((M, K // 32), dtype=torch.float32, device=x.device)
        _check(lib.nhb_quantize_q8_0(self.handle, x.data_ptr(), x.stride(0), M, K, q.data_ptr(), d.data_ptr()), self.handle)
        return q, d

    # ---- rms_norm x norm-weight ----
    def rms_norm_mul(self, x, norm_w, eps: float, sqrt_mode: int = SQRT_IEEE, y=None):
        import torch

        M, K = x.shape
        if y is None:
            y = torch.empty((M, K), dtype=torch.float32, device=x.device)
        _check(lib.nhb_rms_norm_mul(self.handle, x.data_ptr(), x.stride(0) if M > 0 else K, norm_w.data_ptr(), eps, sqrt_mode, y.data_ptr(),
                                    y.stride(0) if M > 0 else K, M, K), self.handle)
        return y

    def rms_norm_mul_q8_0(self, x, norm_w, eps: float, sqrt_mode: int = SQRT_IEEE):
        """Returns the rows as 34-byte Q8_0 blocks: uint8 [M][K/32][34]."""
        import torch

        M, K = x.shape
        out = torch.empty((M, K // 32, 34), dtype=torch.uint8, device=x.device)
        _check(lib.nhb_rms_norm_mul_q8_0(self.handle, x.data_ptr(), x.stride(0) if M > 0 else K, norm_w.data_ptr(), eps, sqrt_mode,
                                         out.data_ptr(), M, K), self.handle)
        return out

    def rms_norm_mul_mat_batch(self, ops, norm_w, eps: float, sqrt_mode: int = SQRT_IEEE, kernel: int = KERNEL_AUTO):
        """ops: list of (Weight, x, y); x is the row before the norm, the same tensor in every op."""
        arr = (MulMatOp * len(ops))()
        for i, (w, x, y) in enumerate(ops):
            arr[i] = MulMatOp(w.handle, x.data_ptr(), _ld(x), y.data_ptr(), _ld(y), x.shape[0])
        _check(lib.nhb_rms_norm_mul_mat_batch(self.handle, arr, len(ops), norm_w.data_ptr(), eps, sqrt_mode, kernel), self.handle)

    def memcpy_h2d(self, dst_ptr: int, src_ptr: int, nbytes: int):
        _check(lib.nhb_memcpy_h2d(self.handle, dst_ptr, src_ptr, nbytes), self.handle)

    def memcpy_d2h(self, dst_ptr: int, src_ptr: int, nbytes: int):
        _check(lib.nhb_memcpy_d2h(self.handle, dst_ptr, src_ptr, nbytes), self.handle)

    def chain(self, stages) -> Chain:
        """stages: list of stages, each a list of (Weight, x, y); every stage may read the outputs of the one before."""
        flat = [op for st in stages for op in st]
        arr = (MulMatOp * max(len(flat), 1))()
        for i, (w, x, y) in enumerate(flat):
            arr[i] = MulMatOp(w.handle, x.data_ptr(), _ld(x), y.data_ptr(), _ld(y), x.shape[0])
        counts = (_i * max(len(stages), 1))(*[len(st) for st in stages])
        h = _vp()
        _check(lib.nhb_chain_create(self.handle, arr, counts, len(stages), C.byref(h)), self.handle)
        return Chain(self, h.value, flat)

    # ---- the paged K/V cache and the attention over it (seqs, cu: device int32; see nhb_kv_cache) ----
    def _kv(self, cache: KvCache):
        if cache.device != self.device:
            raise NhbError(ERR_ARG, "the cache lies on another GPU than the context")
        return cache.ref

    def _zeros(self, like, rows: int, width: int):
        """A new output of zeros.  torch fills it on its own current stream: on another one the context must not come before the fill (a capture
        runs nothing now, and is replayed after it)."""
        import torch

        out = like.new_zeros((rows, width))
        if out.is_cuda and not self.capturing and _torch_stream(self.device) != self.stream and not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream(out.device).synchronize()
        return out

    def kv_reserve(self, cache: KvCache, seqs, cu=None):
        """Room for cu[i + 1] - cu[i] new tokens (cu None: one) of every listed sequence."""
        n = seqs.numel()
        _check_cu(cu, n)
        _check(lib.nhb_kv_reserve(self.handle, self._kv(cache), _i32(seqs, "seqs", self.device), _i32(cu, "cu", self.device), n), self.handle)

    def kv_fork(self, cache: KvCache, parents, children, deep: bool = False):
        if parents.shape != children.shape:
            raise NhbError(ERR_ARG, "as many children as parents")
        _check(lib.nhb_kv_fork(self.handle, self._kv(cache), _i32(parents, "parents", self.device), _i32(children, "children", self.device), children.numel(), int(deep)), self.handle)

    def kv_free(self, cache: KvCache, seqs):
        _check(lib.nhb_kv_free(self.handle, self._kv(cache), _i32(seqs, "seqs", self.device), seqs.numel()), self.handle)

    def kv_compact(self, cache: KvCache, live=None):
        """live: int32 [1] or None; receives the number of pages in use."""
        if live is not None and live.numel() < 1:
            raise NhbError(ERR_ARG, "live has no room for a number")
        _check(lib.nhb_kv_compact(self.handle, self._kv(cache), _i32(live, "live", self.device)), self.handle)

    def rope_kv_append(self, cache: KvCache, layer: int, q, k, v, seqs, cu=None, rope: Rope | None = None, q_out=None):
        """Rotates q into q_out (None: a new tensor; may be q) and stores rotated k and v as the sequences' last tokens."""
        M, width = q.shape
        n = seqs.numel()
        if q_out is None:
            q_out = self._zeros(q, M, width)
        _check_cu(cu, n)
        kw = cache.kv_heads * cache.head_dim
        (qp, ldq), (kp, ldk), (vp, ldv) = _rows32(q, M, width, "q", self.device), _rows32(k, M, kw, "k", self.device), _rows32(v, M, kw, "v", self.device)
        op, ldo = _rows32(q_out, M, width, "q_out", self.device)
        _check(lib.nhb_rope_kv_append(self.handle, self._kv(cache), layer, qp, ldq, _heads(width, cache), kp, ldk, vp, ldv, M, _i32(seqs, "seqs", self.device), _i32(cu, "cu", self.device), n,
                                      rope.ref(cache.head_dim, self.device) if rope is not None else None, op, ldo), self.handle)
        return q_out

    def attn_prompt(self, cache: KvCache, layer: int, q, seqs, cu, scale: float, out=None):
        """Causal attention of packed prompt rows (nhb_attn_prompt): q f32 [M][heads * head_dim] -> out."""
        M, width = q.shape
        n = seqs.numel()
        if out is None:
            out = self._zeros(q, M, width)
        _check_cu(cu, n)
        (qp, ldq), (op, ldo) = _rows32(q, M, width, "q", self.device), _rows32(out, M, width, "out", self.device)
        _check(lib.nhb_attn_prompt(self.handle, self._kv(cache), layer, qp, ldq, _heads(width, cache), M, _i32(seqs, "seqs", self.device), _i32(cu, "cu", self.device), n, scale, op, ldo), self.handle)
        return out

    def attn_decode(self, cache: KvCache, layer: int, q, seqs, scale: float, shared: int = 0, out=None):
        """Attention of one row per listed sequence over all its keys; `shared` leading tokens are common to the batch (nhb_attn_decode)."""
        n, width = q.shape
        if out is None:
            out = self._zeros(q, n, width)
        if seqs.numel() != n:
            raise NhbError(ERR_ARG, "one row of q per listed sequence")
        (qp, ldq), (op, ldo) = _rows32(q, n, width, "q", self.device), _rows32(out, n, width, "out", self.device)
        _check(lib.nhb_attn_decode(self.handle, self._kv(cache), layer, qp, ldq, _heads(width, cache), _i32(seqs, "seqs", self.device), n, shared, scale, op, ldo), self.handle)
        return out

    # ---- graphs ----
    def graph_begin(self):
        _check(lib.nhb_graph_begin(self.handle), self.handle)
        self.capturing = True

    def graph_end(self) -> Graph:
        h = _vp()
        self.capturing = False
        _check(lib.nhb_graph_end(self.handle, C.byref(h)), self.handle)
        return Graph(self, h.value)

    # ---- multi-GPU ----
    @staticmethod
    def comm_unique_id() -> bytes:
        buf = C.create_string_buffer(128)
        _check(lib.nhb_comm_unique_id(buf))
        return buf.raw

    def comm_init(self, uid: bytes):
        buf = C.create_string_buffer(uid, 128)
        _check(lib.nhb_comm_init(self.handle, buf), self.handle)

    def symm_empty(self, shape, dtype=None):
        """A zeroed torch tensor in symmetric memory (collective: same call, same order, on every rank)."""
        import torch

        dtype = dtype or torch.float32
        n = 1
        for d in shape:
            n *= int(d)
        nbytes = max(n, 1) * torch.empty((), dtype=dtype).element_size()
        p = _vp()
        _check(lib.nhb_symm_alloc(self.handle, nbytes, C.byref(p)), self.handle)
        return _tensor_from_ptr(p.value, nbytes, self.device, dtype).view(*shape) if n else torch.empty(shape, dtype=dtype, device=f"cuda:{self.device}")

    def all_gather(self, y):
        M, N = y.shape
        _check(lib.nhb_all_gather(self.handle, y.data_ptr(), y.stride(0), M, N), self.handle)

    def all_gather_batch(self, ys):
        n = len(ys)
        ptrs = (_vp * n)(*[y.data_ptr() for y in ys])
        ld = (_i64 * n)(*[y.stride(0) for y in ys])
        ms = (_i64 * n)(*[y.shape[0] for y in ys])
        ns = (_i64 * n)(*[y.shape[1] for y in ys])
        _check(lib.nhb_all_gather_batch(self.handle, ptrs, ld, ms, ns, n), self.handle)


# ---- one process driving several GPUs: ctxs[i] is rank i of a world of len(ctxs) ----
def _handles(ctxs):
    return (_vp * len(ctxs))(*[c.handle for c in ctxs])


def symm_empty_local(ctxs, shape, dtype=None):
    """One zeroed torch tensor per context, the same symmetric allocation on every context's device."""
    import torch

    dtype = dtype or torch.float32
    n = 1
    for d in shape:
        n *= int(d)
    nbytes = max(n, 1) * torch.empty((), dtype=dtype).element_size()
    out = (_vp * len(ctxs))()
    _check(lib.nhb_symm_alloc_local(_handles(ctxs), len(ctxs), nbytes, out), ctxs[0].handle)
    return [_tensor_from_ptr(out[i], nbytes, c.device, dtype).view(*shape) for i, c in enumerate(ctxs)]


def all_gather_local(ctxs, ys):
    M, N = ys[0].shape
    ptrs = (_vp * len(ys))(*[y.data_ptr() for y in ys])
    _check(lib.nhb_all_gather_local(_handles(ctxs), len(ctxs), ptrs, ys[0].stride(0), M, N), ctxs[0].handle)


def sync_all(ctxs):
    _check(lib.nhb_sync_all(_handles(ctxs), len(ctxs)), ctxs[0].handle)


class WaitPlanner:
    """The wait decisions of the fused all-gather without a GPU (nhb_wait_planner_*): buffers are (address, bytes) pairs."""

    def __init__(self, peer_window: int = 4):
        self.handle = lib.nhb_wait_planner_create(peer_window)

    def add_region(self, base: int, nbytes: int):
        _check(lib.nhb_wait_planner_add_region(self.handle, base, nbytes))

    def launch(self, reads, writes, delivers: bool):
        """reads / writes: lists of (address, bytes).  Returns (waits, lag)."""
        ri = (_vp * max(len(reads), 1))(*[a for a, _ in reads])
        rb = (C.c_size_t * max(len(reads), 1))(*[b for _, b in reads])
        wi = (_vp * max(len(writes), 1))(*[a for a, _ in writes])
        wb = (C.c_size_t * max(len(writes), 1))(*[b for _, b in writes])
        waits, lag = _i(), _i()
        _check(lib.nhb_wait_planner_launch(self.handle, ri, rb, len(reads), wi, wb, len(writes), int(delivers), C.byref(waits), C.byref(lag)))
        return bool(waits.value), lag.value

    def wait_all(self) -> bool:
        return bool(lib.nhb_wait_planner_wait_all(self.handle))

    def capture_begin(self):
        lib.nhb_wait_planner_capture_begin(self.handle)

    def capture_end(self) -> int:
        return int(lib.nhb_wait_planner_capture_end(self.handle))

    def replayed(self, recording: int):
        _check(lib.nhb_wait_planner_replayed(self.handle, recording))

    @property
    def seq(self) -> int:
        return int(lib.nhb_wait_planner_seq(self.handle))

    def close(self):
        if self.handle:
            lib.nhb_wait_planner_destroy(self.handle)
            self.handle = None

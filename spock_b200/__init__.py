"""spock_b200: B200 (sm_100a) Gated DeltaNet hot path behind a C ABI.

Host-side mirror of spock's DeltaNet entry points over libspock_b200.so
(include/spock_b200.h). PyTorch provides device memory and streams only; every
computation runs in this package's own CUDA kernels. There is no CPU fallback:
if the library or a B200 is missing, calls raise SpockError.

Reference interfaces mirrored here:
  DeltaNetChunkConfig / Inputs / Outputs, run_deltanet_chunk_rule
      src/runtime/deltanet_chunk.hpp:8-40 (same field names, layouts and the
      same "fields must be non-zero" / size-mismatch errors)
  chunk_prefill        batched device-tensor form used by
                       DecodeSession::gpu_chunk_prefill_from_gpu_collect
                       (src/runtime/vk_session.cpp:4466-4828)
  deltanet_decode_step fused conv_l2_qk + recurrent_gbeta_norm_gate
                       (src/runtime/vk_session.cpp:2878-2883, 3213-3218)
"""
import ctypes
import os
import struct
import warnings
from dataclasses import dataclass, field
from typing import List, Optional

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libspock_b200.so")

SPOCK_OK = 0
SPOCK_ERR_INVALID = -1
SPOCK_ERR_UNSUPPORTED = -2
SPOCK_ERR_CUDA = -3
SPOCK_ERR_ALLOC = -4
SPOCK_ERR_TIMEOUT = -5
F32, F16, BF16 = 0, 1, 2

EXPORTED = ["spock_create", "spock_destroy", "spock_last_error", "spock_sync",
            "spock_kernel_launch_count", "spock_selftest_wait_timeout", "spock_chunk_prefill", "spock_chunk_last_to_fp16",
            "spock_deltanet_decode_step", "spock_deltanet_recurrent", "spock_chunk_prefill_noalloc",
            "spock_model_create", "spock_model_destroy", "spock_model_last_error", "spock_model_set_weight",
            "spock_model_reset", "spock_model_step", "spock_model_generate", "spock_model_load_artifact",
            "spock_model_prefill", "spock_noalloc_sync", "spock_model_sync",
            "spock_rms_norm", "spock_matvec", "spock_argmax", "spock_attention_decode", "spock_attention_prefill",
            "spock_paged_attention_prep", "spock_paged_attention", "spock_paged_attention_workspace",
            "spock_deltanet_decode_span", "spock_draft_verify", "spock_draft_verify_workspace"]


class SpockError(RuntimeError):
    def __init__(self, code, msg):
        super().__init__(f"[{code}] {msg}")
        self.code = code


class ChunkDesc(ctypes.Structure):
    _fields_ = [("batch", ctypes.c_int64), ("num_heads", ctypes.c_int64), ("seq_len", ctypes.c_int64),
                ("key_dim", ctypes.c_int64), ("value_dim", ctypes.c_int64), ("chunk_size", ctypes.c_int64),
                ("dtype_in", ctypes.c_int32), ("dtype_out", ctypes.c_int32),
                ("use_qk_l2norm", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class DnLayer(ctypes.Structure):
    _fields_ = [("num_heads", ctypes.c_int32), ("key_dim", ctypes.c_int32), ("value_dim", ctypes.c_int32),
                ("conv_kernel", ctypes.c_int32), ("conv_weight", ctypes.c_void_p),
                ("a_log_bias", ctypes.c_void_p), ("norm_weight", ctypes.c_void_p),
                ("eps", ctypes.c_float), ("reserved", ctypes.c_int32)]


class PagedKv(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("page_stride", ctypes.c_int64),
                ("pos_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64), ("page_table", ctypes.c_void_p),
                ("table_stride", ctypes.c_int64), ("kv_len", ctypes.c_void_p), ("table_width", ctypes.c_int32),
                ("num_pages", ctypes.c_int32), ("page_size", ctypes.c_int32), ("kv_heads", ctypes.c_int32),
                ("head_dim", ctypes.c_int32), ("dtype", ctypes.c_int32)]


_LIB = None


def build(force=False):
    from . import builder as _b
    lib_path = _b.build(force=force)
    _b.build_apps(force=force)
    try:
        _b.build_binding(force=force)
    except (ImportError, OSError, RuntimeError) as e:  # the library and the wrappers do without
        _no_binding(e)
    return lib_path


def lib():
    """Loads libspock_b200.so (building it in-tree when absent or stale)."""
    global _LIB
    if _LIB is None:
        if not os.path.exists(LIB_PATH):
            build()
        L = ctypes.CDLL(LIB_PATH)
        vp, i64, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32
        L.spock_create.argtypes = [ctypes.c_int, ctypes.POINTER(vp)]
        L.spock_destroy.argtypes = [vp]
        L.spock_last_error.argtypes = [vp]
        L.spock_last_error.restype = ctypes.c_char_p
        L.spock_sync.argtypes = [vp, vp]
        L.spock_kernel_launch_count.restype = ctypes.c_uint64
        L.spock_selftest_wait_timeout.argtypes = [vp, ctypes.c_uint32, vp]
        L.spock_chunk_prefill.argtypes = [vp, ctypes.POINTER(ChunkDesc)] + [vp] * 9
        L.spock_chunk_prefill_noalloc.argtypes = [ctypes.POINTER(ChunkDesc)] + [vp] * 9
        L.spock_noalloc_sync.argtypes = [vp]
        L.spock_rms_norm.argtypes = [vp, vp, vp, vp, i64, i32, ctypes.c_float, vp]
        L.spock_matvec.argtypes = [vp, i32, i32, vp, i32, i32, vp, i64, vp, vp, vp]
        L.spock_argmax.argtypes = [vp, vp, i64, i64, vp, vp]
        L.spock_attention_decode.argtypes = [vp, i32, vp, vp, vp, ctypes.c_float, ctypes.c_float, vp, vp, i32, i64,
                                             vp, vp]
        L.spock_attention_prefill.argtypes = [vp, i32, vp, vp, vp, ctypes.c_float, ctypes.c_float, vp, vp, i32, i64,
                                              i32, vp, vp]
        L.spock_chunk_last_to_fp16.argtypes = [vp, i64, i64, i64, i64, vp, vp, vp]
        L.spock_deltanet_decode_step.argtypes = [vp, ctypes.POINTER(DnLayer), i64] + [vp] * 9
        L.spock_deltanet_recurrent.argtypes = [vp, i64, i32, i32, i32] + [vp] * 8
        f32, szp = ctypes.c_float, ctypes.POINTER(ctypes.c_size_t)
        L.spock_paged_attention_prep.argtypes = [vp, vp, i32, vp, i64, vp, i64, i32, i32, vp, vp, f32, vp, i64, i32,
                                                 vp, vp]
        L.spock_paged_attention.argtypes = [vp, vp, i32, vp, i64, i32, vp, i64, i64, vp, i64, i64, f32, vp, vp,
                                            ctypes.c_size_t, vp]
        L.spock_paged_attention_workspace.argtypes = [vp, i32, i32, i32, szp]
        L.spock_deltanet_decode_span.argtypes = [vp, vp, i32, vp, vp, i64, vp, i64, vp, vp, i64, vp, i64] + [vp] * 6
        L.spock_draft_verify.argtypes = [vp, i32, vp, i64, i64, i64, i32, vp, vp, vp, i64] + [vp] * 6 + [
            ctypes.c_size_t, vp]
        L.spock_draft_verify_workspace.argtypes = [vp, i64, i64, i32, szp]
        _LIB = L
    return _LIB


def _ptr(t):
    if t is None:
        return None
    import torch
    if not t.is_cuda:
        raise SpockError(SPOCK_ERR_INVALID, "expected a CUDA tensor")
    if not t.is_contiguous():
        raise SpockError(SPOCK_ERR_INVALID, "expected a contiguous tensor")
    return ctypes.c_void_p(t.data_ptr())


def _dtype_code(dt):
    import torch
    return {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}[dt]


class Context:
    """One per GPU (spock_ctx). Replaces VulkanDevice (src/runtime/vk_device.hpp:29-117)."""

    _by_device = {}

    def __init__(self, device=0):
        L = lib()
        h = ctypes.c_void_p()
        rc = L.spock_create(int(device), ctypes.byref(h))
        if rc != SPOCK_OK:
            raise SpockError(rc, L.spock_last_error(None).decode())
        self.h = h
        self.device = device
        self.ws_bytes = {}  # workspace sizes by shape

    @classmethod
    def get(cls, device=0):
        if device not in cls._by_device:
            cls._by_device[device] = Context(device)
        return cls._by_device[device]

    def check(self, rc):
        if rc != SPOCK_OK:
            raise SpockError(rc, lib().spock_last_error(self.h).decode())

    def sync(self, stream=None):
        self.check(lib().spock_sync(self.h, _stream(stream)))

    def selftest_wait_timeout(self, polls=256, stream=None):
        """Launches the failure-detection self-test (a bounded device wait that
        must give up); the following sync() raises SpockError(SPOCK_ERR_TIMEOUT)."""
        self.check(lib().spock_selftest_wait_timeout(self.h, int(polls), _stream(stream)))

    def close(self):
        if self.h:
            lib().spock_destroy(self.h)
            self.h = None


def _stream(stream):
    import torch
    if stream is None:
        stream = torch.cuda.current_stream()
    return ctypes.c_void_p(stream.cuda_stream)


def chunk_prefill(q, k, v, g, beta, initial_state=None, out_dtype=None, use_qk_l2norm=False,
                  chunk_size=64, out=None, final_state=None, ctx=None, stream=None):
    """Batched chunked gated delta rule on device tensors.

    q, k [B,H,S,K] and v [B,H,S,V] (fp32/fp16/bf16, same dtype); g, beta [B,H,S]
    fp32; initial_state [B,H,K,V] fp32 or None. Returns (core_attn_out [B,H,S,V]
    in out_dtype (default: q's dtype), final_state [B,H,K,V] fp32).
    """
    import torch
    B, H, S, K = q.shape
    V = v.shape[-1]
    out_dtype = out_dtype or q.dtype
    ctx = ctx or Context.get(q.device.index or 0)
    if out is None:
        out = torch.empty((B, H, S, V), dtype=out_dtype, device=q.device)
    if final_state is None:
        final_state = torch.empty((B, H, K, V), dtype=torch.float32, device=q.device)
    d = ChunkDesc(B, H, S, K, V, chunk_size, _dtype_code(q.dtype), _dtype_code(out_dtype),
                  int(bool(use_qk_l2norm)), 0)
    ctx.check(lib().spock_chunk_prefill(ctx.h, ctypes.byref(d), _ptr(q), _ptr(k), _ptr(v), _ptr(g),
                                        _ptr(beta), _ptr(initial_state), _ptr(out), _ptr(final_state),
                                        _stream(stream)))
    return out, final_state


def chunk_last_to_fp16(core_out, ctx=None, stream=None):
    """Last token of core_attn_out [B,H,S,V] fp32 -> fp16 [B,H*V] by truncation (FTZ)."""
    import torch
    B, H, S, V = core_out.shape
    ctx = ctx or Context.get(core_out.device.index or 0)
    out = torch.empty((B, H * V), dtype=torch.float16, device=core_out.device)
    ctx.check(lib().spock_chunk_last_to_fp16(ctx.h, B, H, S, V, _ptr(core_out), _ptr(out), _stream(stream)))
    return out


MV_STORE, MV_RESIDUAL, MV_SILU_GATE, MV_ARGMAX = 0, 1, 2, 3


def rms_norm(x, w, eps=1e-6, out=None, ctx=None, stream=None):
    """rms_norm.comp on fp16 rows x [rows, 1024] with (1+w) weights w [1024] fp16."""
    import torch
    ctx = ctx or Context.get(x.device.index or 0)
    out = torch.empty_like(x) if out is None else out
    ctx.check(lib().spock_rms_norm(ctx.h, _ptr(x), _ptr(w), _ptr(out), x.shape[0], x.shape[1], eps, _stream(stream)))
    return out


def matvec(w, x, epilogue=MV_STORE, residual=None, exact=False, out=None, ctx=None, stream=None):
    """matvec.comp over rows x [rows, in] with fp16 W [out(, x2 for SILU_GATE), in] and a fused epilogue;
    ARGMAX returns int32 token ids [rows]."""
    import torch
    ctx = ctx or Context.get(x.device.index or 0)
    rows, n_in = x.shape
    n_out = w.shape[0] // 2 if epilogue == MV_SILU_GATE else w.shape[0]
    if out is None:
        out = (torch.empty(rows, dtype=torch.int32, device=x.device) if epilogue == MV_ARGMAX
               else torch.empty((rows, n_out), dtype=torch.float16, device=x.device))
    ctx.check(lib().spock_matvec(ctx.h, int(epilogue), int(bool(exact)), _ptr(w), n_out, n_in, _ptr(x), rows,
                                 _ptr(out), _ptr(residual), _stream(stream)))
    return out


def argmax(logits, ctx=None, stream=None):
    """argmax.comp per row of fp16 logits [rows, n] -> int32 [rows] (lowest index among ties)."""
    import torch
    ctx = ctx or Context.get(logits.device.index or 0)
    out = torch.empty(logits.shape[0], dtype=torch.int32, device=logits.device)
    ctx.check(lib().spock_argmax(ctx.h, _ptr(logits), logits.shape[0], logits.shape[1], _ptr(out), _stream(stream)))
    return out


def attention_decode(proj, q_norm, k_norm, pos, kv_cache, eps=1e-6, theta=1e7, exact=False, ctx=None, stream=None):
    """One gated-attention decode token per sequence: proj [rows, 5120] fp16, pos int32 [rows],
    kv_cache [rows, max_seq, 2, 2, 256] fp16 (row pos written) -> out [rows, 2048] fp16."""
    import torch
    ctx = ctx or Context.get(proj.device.index or 0)
    rows = proj.shape[0]
    out = torch.empty((rows, 2048), dtype=torch.float16, device=proj.device)
    ctx.check(lib().spock_attention_decode(ctx.h, int(bool(exact)), _ptr(proj), _ptr(q_norm), _ptr(k_norm), eps, theta,
                                           _ptr(pos), _ptr(kv_cache), kv_cache.shape[1], rows, _ptr(out),
                                           _stream(stream)))
    return out


def attention_prefill(proj, q_norm, k_norm, pos, kv_cache, eps=1e-6, theta=1e7, exact=False, ctx=None, stream=None):
    """Gated attention over `len` prompt tokens per sequence: proj [batch, len, 5120] fp16, pos int32 [batch]
    (first prompt position), kv_cache [batch, max_seq, 2, 2, 256] fp16 -> out [batch, len, 2048] fp16."""
    import torch
    ctx = ctx or Context.get(proj.device.index or 0)
    B, T = proj.shape[0], proj.shape[1]
    out = torch.empty((B, T, 2048), dtype=torch.float16, device=proj.device)
    ctx.check(lib().spock_attention_prefill(ctx.h, int(bool(exact)), _ptr(proj), _ptr(q_norm), _ptr(k_norm), eps,
                                            theta, _ptr(pos), _ptr(kv_cache), kv_cache.shape[1], B, T, _ptr(out),
                                            _stream(stream)))
    return out


@dataclass
class DeltaNetLayer:
    """Per-layer constants (spock_dn_layer). Tensors are device tensors."""
    conv_weight: object   # fp16 [conv_dim, conv_kernel]
    a_log_bias: object    # fp32 [num_heads, 2]
    norm_weight: object   # fp32 [value_dim]
    num_heads: int = 16
    key_dim: int = 128
    value_dim: int = 128
    conv_kernel: int = 4
    eps: float = 1e-6

    def c_struct(self):
        return DnLayer(self.num_heads, self.key_dim, self.value_dim, self.conv_kernel,
                       _ptr(self.conv_weight), _ptr(self.a_log_bias), _ptr(self.norm_weight),
                       self.eps, 0)


def deltanet_decode_step(layer, qkv, conv_state, state, a, b, z, out=None, core_raw=None, ctx=None,
                         stream=None):
    """One decode token through a DeltaNet mixer core; qkv, conv_state, state updated in place."""
    import torch
    B = qkv.shape[0]
    ctx = ctx or Context.get(qkv.device.index or 0)
    if out is None:
        out = torch.empty((B, layer.num_heads * layer.value_dim), dtype=torch.float16, device=qkv.device)
    st = layer.c_struct()
    ctx.check(lib().spock_deltanet_decode_step(ctx.h, ctypes.byref(st), B, _ptr(qkv), _ptr(conv_state),
                                               _ptr(state), _ptr(a), _ptr(b), _ptr(z), _ptr(out),
                                               _ptr(core_raw), _stream(stream)))
    return out


def deltanet_recurrent(q, k, v, g, beta, state, num_heads=16, key_dim=128, value_dim=128, ctx=None,
                       stream=None):
    """Unfused recurrent update (deltanet_recurrent.comp contract); state updated in place."""
    import torch
    B = q.shape[0]
    ctx = ctx or Context.get(q.device.index or 0)
    out = torch.empty((B, num_heads * value_dim), dtype=torch.float16, device=q.device)
    ctx.check(lib().spock_deltanet_recurrent(ctx.h, B, num_heads, key_dim, value_dim, _ptr(q), _ptr(k),
                                             _ptr(v), _ptr(g), _ptr(beta), _ptr(state), _ptr(out),
                                             _stream(stream)))
    return out


_BINDING = None  # the module; False where it cannot be had


def _no_binding(why):
    warnings.warn("spock_b200: %s; calls of the ragged steps take some 10 us longer on the host" % why)


def _binding():
    """The ragged steps' short way into the library (csrc/binding.cpp), built in-tree when absent; None where it cannot
    be built or loaded: the wrappers then make their checks themselves."""
    global _BINDING
    if _BINDING is None:
        lib()
        import importlib.machinery
        import importlib.util
        import torch  # noqa: F401  (its libraries are loaded first)
        from . import builder
        try:
            path = builder.build_binding()
            loader = importlib.machinery.ExtensionFileLoader("spock_b200._binding", path)
            spec = importlib.util.spec_from_file_location("spock_b200._binding", path, loader=loader)
            module = importlib.util.module_from_spec(spec)
            loader.exec_module(module)
            _BINDING = module
        except (ImportError, OSError, RuntimeError) as e:
            _no_binding(e)
            _BINDING = False
    return _BINDING or None


# ---- ragged steps: several new tokens per sequence, packed rows ----------------
# `start` int32 [batch + 1]: sequence b owns rows start[b] .. start[b + 1] - 1 of
# every row-shaped tensor. All tensors of a call are on one device; the work goes
# to that device's current stream unless `stream` is given. Starts, lengths, page
# tables and token ids are checked on the device: Context.sync() raises for one
# that was out of range.

def _bad(msg):
    raise SpockError(SPOCK_ERR_INVALID, msg)


def _refuse(first, tensors):
    """Says which of the (name, tensor, dtype, ndim, contiguous) entries a call cannot take."""
    dev = first.device
    for name, t, dtype, ndim, contiguous in tensors:
        if t is None:
            continue
        if t.device != dev:
            _bad(f"{name}: expected a tensor on {dev}")
        if t.dtype != dtype:
            _bad(f"{name}: expected {dtype}, got {t.dtype}")
        if t.dim() != ndim:
            _bad(f"{name}: expected {ndim} dimensions, got {t.dim()}")
        if contiguous and not t.is_contiguous():
            _bad(f"{name}: expected a contiguous tensor")
        if not contiguous and t.shape[-1] > 1 and t.stride(-1) != 1:
            _bad(f"{name}: expected a contiguous last dimension")
    _bad("expected CUDA tensors")


def _checked(d, r):
    """A result of the binding: a status that is not SPOCK_OK raises."""
    if type(r) is int:
        Context.get(d).check(r)
    return r


# The wrappers' own checks. The binding makes them first; what it does not take
# (a named stream, an argument to refuse) goes on here. `d` is the device index.
def _rows(t, dtype, ndim, d):
    """A tensor of contiguous rows (any strides before the last dimension)."""
    return t.dtype is dtype and t.dim() == ndim and t.get_device() == d and (t.stride(-1) == 1 or t.shape[-1] <= 1)


def _whole(t, dtype, ndim, d):
    """A contiguous tensor."""
    return t.dtype is dtype and t.dim() == ndim and t.get_device() == d and t.is_contiguous()


def _stream_of(d, stream):
    """The stream's handle; None: device d's current stream."""
    if stream is not None:
        if stream.device.index != d:
            _bad(f"stream: expected one of cuda:{d}, got one of {stream.device}")
        return stream.cuda_stream
    import torch
    return torch._C._cuda_getCurrentRawStream(d)


def _new(shape, dtype, like, stream):
    """An uninitialised tensor for work on `stream` (None: the current one)."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    import torch
    # From the allocator's blocks of `stream`: one of the current stream's may still be in use by work queued there.
    with torch.cuda.stream(stream):
        t = like.new_empty(shape, dtype=dtype)
    t.record_stream(torch.cuda.current_stream(like.device))  # where the caller may read it
    return t


def _row_stride(t):
    """Elements from one row to the next (any value does for a single row)."""
    return t.stride(0) if t.shape[0] > 1 else (t.shape[-1] + 7) // 8 * 8 if t.dim() == 2 else t.shape[1] * t.shape[2]


_PAGED = struct.Struct("@PPqqqPqPiiiiii")  # spock_paged_kv


def _paged_kv(k_pages, v_pages, page_table, kv_len, batch):
    """spock_paged_kv over pages [num_pages, page_size, kv_heads, head_dim] (any strides, head_dim contiguous)."""
    import torch
    st, dt = k_pages.stride(), k_pages.dtype
    if k_pages.shape != v_pages.shape or st != v_pages.stride():
        _bad("k_pages and v_pages must have the same shape and strides")
    width = page_table.shape[1]
    if batch < 1 or page_table.shape[0] != batch or kv_len.shape[0] != batch:
        _bad("start, page_table and kv_len disagree on the batch")
    if dt is not torch.float16 and dt is not torch.bfloat16:
        raise SpockError(SPOCK_ERR_UNSUPPORTED, "the cache is fp16 or bf16")
    pages, page, heads, dim = k_pages.shape
    table_stride = page_table.stride(0)
    # strides of dimensions of one element say nothing
    return _PAGED.pack(k_pages.data_ptr(), v_pages.data_ptr(), st[0] if pages > 1 else page * heads * dim,
                       st[1] if page > 1 else heads * dim, st[2] if heads > 1 else dim, page_table.data_ptr(),
                       table_stride if batch > 1 or table_stride > width else width, kv_len.data_ptr(), width, pages,
                       page, heads, dim, F16 if dt is torch.float16 else BF16), heads, dim


def _workspace(ctx, query, key, like, stream):
    """A workspace tensor from the caching allocator (so a captured graph keeps its own)."""
    import torch
    n = ctx.ws_bytes.get(key)
    if n is None:
        size = ctypes.c_size_t()
        ctx.check(query(ctx.h, *key[1:], ctypes.byref(size)))
        n = size.value
        if len(ctx.ws_bytes) < 1024:  # sizes only, by shape
            ctx.ws_bytes[key] = n
    return _new((n,), torch.uint8, like, stream), n


def paged_attention_prep(proj, start, k_pages, v_pages, page_table, kv_len, rope=None, q_norm=None, k_norm=None,
                         gated=True, eps=1e-6, q_out=None, stream=None):
    """Projected rows -> rotated queries, K and V stored into the pages (spock_paged_attention_prep).

    proj [total, (q_heads * (2 if gated else 1) + 2 * kv_heads) * head_dim] fp16/bf16 (q | gate per head, then k, v);
    k_pages, v_pages [num_pages, page_size, kv_heads, head_dim], written in place; page_table int32 [batch, width];
    kv_len int32 [batch], the new tokens included; rope fp32 [positions, rotary / 2, 2] (cos, sin) or None;
    q_norm, k_norm [head_dim] ((1 + w) RMSNorm) or None. Returns q [total, q_heads, head_dim]."""
    import torch
    d = proj.get_device()
    short = _binding() if d >= 0 and stream is None else None
    if short is not None:
        r = short.paged_attention_prep(Context.get(d).h.value, proj, start, k_pages, v_pages, page_table, kv_len,
                                       rope, q_norm, k_norm, gated, eps, q_out)
        if r is not None:
            return _checked(d, r)
    i32, f32, dt = torch.int32, torch.float32, k_pages.dtype
    if not (d >= 0 and _rows(proj, dt, 2, d) and _whole(start, i32, 1, d) and _rows(k_pages, dt, 4, d) and
            _rows(v_pages, dt, 4, d) and _rows(page_table, i32, 2, d) and _whole(kv_len, i32, 1, d) and
            (rope is None or _whole(rope, f32, 3, d)) and (q_norm is None or _whole(q_norm, dt, 1, d)) and
            (k_norm is None or _whole(k_norm, dt, 1, d)) and (q_out is None or _whole(q_out, dt, 3, d))):
        _refuse(proj, (("proj", proj, dt, 2, False), ("start", start, i32, 1, True),
                       ("k_pages", k_pages, dt, 4, False), ("v_pages", v_pages, dt, 4, False),
                       ("page_table", page_table, i32, 2, False), ("kv_len", kv_len, i32, 1, True),
                       ("rope", rope, f32, 3, True), ("q_norm", q_norm, dt, 1, True),
                       ("k_norm", k_norm, dt, 1, True), ("q_out", q_out, dt, 3, True)))
    ctx, batch = Context.get(d), start.shape[0] - 1
    kv, kv_heads, dim = _paged_kv(k_pages, v_pages, page_table, kv_len, batch)
    (total, width), per = proj.shape, 2 if gated else 1
    heads = width // dim - 2 * kv_heads
    q_heads = heads // per
    if width % dim or heads <= 0 or heads % per:
        _bad("proj: the row is not q heads (with gates), k heads and v heads")
    if (q_norm is not None and q_norm.shape[0] != dim) or (k_norm is not None and k_norm.shape[0] != dim):
        _bad("q_norm and k_norm have head_dim elements")
    if rope is not None and rope.shape[2] != 2:
        _bad("rope: expected [positions, rotary / 2, 2]")
    if q_out is None:
        q_out = _new((total, q_heads, dim), dt, proj, stream)
    elif q_out.shape != (total, q_heads, dim):
        _bad("q_out: expected [total, q_heads, head_dim]")
    ctx.check(lib().spock_paged_attention_prep(
        ctx.h, kv, batch, start.data_ptr(), total, proj.data_ptr(), _row_stride(proj), q_heads, int(bool(gated)), None if q_norm is None else q_norm.data_ptr(),
        None if k_norm is None else k_norm.data_ptr(), eps, None if rope is None else rope.data_ptr(),
        0 if rope is None else rope.shape[0], 0 if rope is None else 2 * rope.shape[1], q_out.data_ptr(),
        _stream_of(d, stream)))
    return q_out


def paged_attention(q, start, k_pages, v_pages, page_table, kv_len, scale, gate=None, out=None, workspace=None,
                    stream=None):
    """Causal attention of each sequence's new tokens over its pages (spock_paged_attention).

    q [total, q_heads, head_dim] and gate (or None), any row and head strides (positive ones for q); scale positive
    and finite; the cache as in paged_attention_prep.
    Token t of n sees positions 0 .. kv_len - n + t. Returns out [total, q_heads, head_dim]: softmax(scale q k) v,
    times sigmoid(gate); rows behind start[batch] are left as they are. `workspace`: a uint8 tensor of
    the caller's instead of one from the caching allocator."""
    import torch
    d = q.get_device()
    short = _binding() if d >= 0 and stream is None else None
    if short is not None:
        r = short.paged_attention(Context.get(d).h.value, q, start, k_pages, v_pages, page_table, kv_len, scale,
                                  gate, out, workspace)
        if r is not None:
            return _checked(d, r)
    i32, dt = torch.int32, k_pages.dtype
    if not (d >= 0 and _rows(q, dt, 3, d) and _whole(start, i32, 1, d) and _rows(k_pages, dt, 4, d) and
            _rows(v_pages, dt, 4, d) and _rows(page_table, i32, 2, d) and _whole(kv_len, i32, 1, d) and
            (gate is None or _rows(gate, dt, 3, d)) and (out is None or _whole(out, dt, 3, d)) and
            (workspace is None or _whole(workspace, torch.uint8, 1, d))):
        _refuse(q, (("q", q, dt, 3, False), ("start", start, i32, 1, True), ("k_pages", k_pages, dt, 4, False),
                    ("v_pages", v_pages, dt, 4, False), ("page_table", page_table, i32, 2, False),
                    ("kv_len", kv_len, i32, 1, True), ("gate", gate, dt, 3, False), ("out", out, dt, 3, True),
                    ("workspace", workspace, torch.uint8, 1, True)))
    ctx, batch, shape = Context.get(d), start.shape[0] - 1, q.shape
    kv, kv_heads, dim = _paged_kv(k_pages, v_pages, page_table, kv_len, batch)
    total, q_heads, q_dim = shape
    if q_dim != dim:
        _bad("q: expected head_dim elements per head")
    if gate is not None and gate.shape != shape:
        _bad("gate: expected the shape of q")
    if out is None:
        out = _new(shape, dt, q, stream)
    elif out.shape != shape:
        _bad("out: expected the shape of q")
    if workspace is None:
        workspace, n = _workspace(ctx, lib().spock_paged_attention_workspace, ("attn", q_heads, kv_heads, dim), q,
                                  stream)
    else:
        n = workspace.shape[0]
    g = gate is not None
    ctx.check(lib().spock_paged_attention(
        ctx.h, kv, batch, start.data_ptr(), total, q_heads, q.data_ptr(), _row_stride(q),
        q.stride(1) if q_heads > 1 else dim, gate.data_ptr() if g else None, _row_stride(gate) if g else 0,
        (gate.stride(1) if q_heads > 1 else dim) if g else 0, scale, out.data_ptr(), workspace.data_ptr(), n,
        _stream_of(d, stream)))
    return out


def deltanet_decode_span(layer, qkv, conv_state, state, a, b, z, start, counts=None, state_out=None, conv_out=None,
                         out=None, stream=None):
    """One or more tokens per sequence through a DeltaNet mixer core (spock_deltanet_decode_span).

    qkv [total, 3 * heads * 128], a and b [total, heads], z [total, heads * 128] fp16 (any row stride); conv_state
    [batch, 3 * heads * 128, 4] fp16, state [batch, heads, 128, 128] fp32, both only read. With `out` (or when nothing
    else is asked for) the gated outputs [total, heads * 128] are written and returned; with state_out and conv_out
    (which may be state and conv_state) the state after each sequence's first counts[b] rows (None: all)."""
    import torch
    d = qkv.get_device()
    short = _binding() if d >= 0 and stream is None else None
    if short is not None:
        r = short.deltanet_decode_span(Context.get(d).h.value, layer.num_heads, layer.key_dim, layer.value_dim,
                                       layer.conv_kernel, layer.eps, layer.conv_weight, layer.a_log_bias,
                                       layer.norm_weight, qkv, conv_state, state, a, b, z, start, counts,
                                       state_out, conv_out, out)
        if r is not None:
            return _checked(d, r)
    f16, f32, i32 = torch.float16, torch.float32, torch.int32
    cw = layer.conv_weight
    if not (d >= 0 and _rows(qkv, f16, 2, d) and _rows(a, f16, 2, d) and _rows(b, f16, 2, d) and
            (z is None or _rows(z, f16, 2, d)) and _whole(conv_state, f16, 3, d) and _whole(state, f32, 4, d) and
            _whole(start, i32, 1, d) and (counts is None or _whole(counts, i32, 1, d)) and
            (state_out is None or _whole(state_out, f32, 4, d)) and (conv_out is None or _whole(conv_out, f16, 3, d)) and
            (out is None or _whole(out, f16, 2, d)) and _whole(cw, cw.dtype, cw.dim(), d) and
            _whole(layer.a_log_bias, f32, 2, d) and _whole(layer.norm_weight, f32, 1, d)):
        _refuse(qkv, (("qkv", qkv, f16, 2, False), ("a", a, f16, 2, False), ("b", b, f16, 2, False),
                      ("z", z, f16, 2, False), ("conv_state", conv_state, f16, 3, True),
                      ("state", state, f32, 4, True), ("start", start, i32, 1, True),
                      ("counts", counts, i32, 1, True), ("state_out", state_out, f32, 4, True),
                      ("conv_out", conv_out, f16, 3, True), ("out", out, f16, 2, True),
                      ("conv_weight", cw, cw.dtype, cw.dim(), True),
                      ("a_log_bias", layer.a_log_bias, f32, 2, True), ("norm_weight", layer.norm_weight, f32, 1, True)))
    ctx = Context.get(d)
    h, total, batch = layer.num_heads, qkv.shape[0], start.shape[0] - 1
    inner = h * layer.value_dim
    if out is None and state_out is None:
        out = _new((total, inner), f16, qkv, stream)
    shapes = ((qkv, (total, 3 * inner)), (a, (total, h)), (b, (total, h)), (z, (total, inner)),
              (conv_state, (batch, 3 * inner, 4)), (conv_out, (batch, 3 * inner, 4)),
              (state, (batch, h, 128, 128)), (state_out, (batch, h, 128, 128)), (out, (total, inner)),
              (counts, (batch,)), (layer.a_log_bias, (h, 2)), (layer.norm_weight, (layer.value_dim,)))
    for t, shape in shapes:
        if t is not None and t.shape != shape:
            _bad(f"expected a tensor of shape {shape}, got {tuple(t.shape)}")
    if cw.numel() != 3 * inner * layer.conv_kernel or cw.element_size() != 2:
        _bad("conv_weight: expected fp16 [conv_dim, conv_kernel]")
    if total > 1 and a.stride(0) != b.stride(0):
        _bad("a and b must have the same row stride")
    st = layer.c_struct()
    p = lambda t: None if t is None else t.data_ptr()
    ctx.check(lib().spock_deltanet_decode_span(
        ctx.h, ctypes.byref(st), batch, start.data_ptr(), p(counts), total, qkv.data_ptr(), _row_stride(qkv),
        a.data_ptr(), b.data_ptr(), _row_stride(a), p(z), 0 if z is None else _row_stride(z), conv_state.data_ptr(),
        state.data_ptr(), p(conv_out), p(state_out), p(out), _stream_of(d, stream)))
    return out if out is not None else (state_out, conv_out)


def draft_verify(logits, tokens, start, u_accept, u_sample, temperature=None, draft_probs=None, emitted=None,
                 out_tokens=None, workspace=None, stream=None):
    """Acceptance of drafted tokens from given random numbers (spock_draft_verify).

    logits [total, vocab] fp32/fp16/bf16: a sequence's rows are its last accepted token and its drafts; tokens int32
    [total], the input token of each row; u_accept fp32 [total], u_sample fp32 [batch]; temperature fp32 [batch] (0:
    greedy) or None (1.0); draft_probs fp32 [total, vocab], row i the distribution that row i + 1's token was drawn
    from, or None for drafts without one. Returns (emitted int32 [batch], out_tokens int32 [total]): the accepted
    drafts, the next token, then -1."""
    import torch
    d = logits.get_device()
    short = _binding() if d >= 0 and stream is None else None
    if short is not None:
        r = short.draft_verify(Context.get(d).h.value, logits, tokens, start, u_accept, u_sample, temperature,
                               draft_probs, emitted, out_tokens, workspace)
        if r is not None:
            return _checked(d, r)
    f32, i32, dt = torch.float32, torch.int32, logits.dtype
    if dt not in (f32, torch.float16, torch.bfloat16):
        raise SpockError(SPOCK_ERR_UNSUPPORTED, "logits are fp32, fp16 or bf16")
    if not (d >= 0 and _rows(logits, dt, 2, d) and _whole(tokens, i32, 1, d) and _whole(start, i32, 1, d) and
            _whole(u_accept, f32, 1, d) and _whole(u_sample, f32, 1, d) and
            (temperature is None or _whole(temperature, f32, 1, d)) and
            (draft_probs is None or _rows(draft_probs, f32, 2, d)) and (emitted is None or _whole(emitted, i32, 1, d)) and
            (out_tokens is None or _whole(out_tokens, i32, 1, d)) and
            (workspace is None or _whole(workspace, torch.uint8, 1, d))):
        _refuse(logits, (("logits", logits, dt, 2, False), ("tokens", tokens, i32, 1, True),
                         ("start", start, i32, 1, True), ("u_accept", u_accept, f32, 1, True),
                         ("u_sample", u_sample, f32, 1, True), ("temperature", temperature, f32, 1, True),
                         ("draft_probs", draft_probs, f32, 2, False), ("emitted", emitted, i32, 1, True),
                         ("out_tokens", out_tokens, i32, 1, True), ("workspace", workspace, torch.uint8, 1, True)))
    ctx = Context.get(d)
    (total, vocab), batch = logits.shape, start.shape[0] - 1
    if (tokens.shape[0] != total or u_accept.shape[0] != total or u_sample.shape[0] != batch or
            (temperature is not None and temperature.shape[0] != batch) or
            (draft_probs is not None and draft_probs.shape != logits.shape) or
            (emitted is not None and emitted.shape[0] != batch) or
            (out_tokens is not None and out_tokens.shape[0] != total)):
        _bad("tokens, u_accept and out_tokens have a value per row, u_sample, temperature and emitted one per sequence")
    if emitted is None:
        emitted = _new((batch,), i32, logits, stream)
    if out_tokens is None:
        out_tokens = _new((total,), i32, logits, stream)
    if workspace is None:
        workspace, n = _workspace(ctx, lib().spock_draft_verify_workspace, ("verify", total, vocab, batch), logits,
                                  stream)
    else:
        n = workspace.shape[0]
    p = lambda t: None if t is None else t.data_ptr()
    ctx.check(lib().spock_draft_verify(
        ctx.h, _dtype_code(logits.dtype), logits.data_ptr(), logits.stride(0) if total > 1 else vocab, total, vocab,
        batch, start.data_ptr(), tokens.data_ptr(), p(draft_probs),
        0 if draft_probs is None else draft_probs.stride(0) if total > 1 else vocab, p(temperature),
        u_accept.data_ptr(), u_sample.data_ptr(), emitted.data_ptr(), out_tokens.data_ptr(), workspace.data_ptr(), n,
        _stream_of(d, stream)))
    return emitted, out_tokens


# ---- reference-shaped API (host vectors in, host vectors out) ----------------

@dataclass
class DeltaNetChunkConfig:
    num_heads: int = 0
    sequence_length: int = 0
    key_dim: int = 0
    value_dim: int = 0
    chunk_size: int = 64
    use_qk_l2norm: bool = True


@dataclass
class DeltaNetChunkInputs:
    query: List[float] = field(default_factory=list)   # [head][token][dim]
    key: List[float] = field(default_factory=list)
    value: List[float] = field(default_factory=list)
    g: List[float] = field(default_factory=list)       # [head][token]
    beta: List[float] = field(default_factory=list)
    initial_state: List[float] = field(default_factory=list)  # [head][key][value] or empty


@dataclass
class DeltaNetChunkOutputs:
    core_attn_out: np.ndarray = None   # flat [head][token][value]
    final_state: np.ndarray = None     # flat [head][key][value]


def run_deltanet_chunk_rule(config: DeltaNetChunkConfig, inputs: DeltaNetChunkInputs,
                            device=0) -> DeltaNetChunkOutputs:
    """Drop-in for spock::runtime::run_deltanet_chunk_rule on the GPU (fp32 in, fp32 out)."""
    import torch
    c = config
    if min(c.num_heads, c.sequence_length, c.key_dim, c.value_dim, c.chunk_size) <= 0:
        raise SpockError(SPOCK_ERR_INVALID, "DeltaNet chunk config fields must be non-zero")
    H, S, K, V = c.num_heads, c.sequence_length, c.key_dim, c.value_dim

    def checked(x, n, name):
        a = np.asarray(x, dtype=np.float32).reshape(-1)
        if a.size != n:
            raise SpockError(SPOCK_ERR_INVALID, f"{name} size mismatch: expected {n}, got {a.size}")
        return a

    dev = torch.device("cuda", device)
    t = lambda a, shape: torch.from_numpy(a.reshape(shape)).to(dev)
    q = t(checked(inputs.query, H * S * K, "query"), (1, H, S, K))
    k = t(checked(inputs.key, H * S * K, "key"), (1, H, S, K))
    v = t(checked(inputs.value, H * S * V, "value"), (1, H, S, V))
    g = t(checked(inputs.g, H * S, "g"), (1, H, S))
    b = t(checked(inputs.beta, H * S, "beta"), (1, H, S))
    init = None
    if len(inputs.initial_state):
        init = t(checked(inputs.initial_state, H * K * V, "initial_state"), (1, H, K, V))
    out, st = chunk_prefill(q, k, v, g, b, initial_state=init, out_dtype=torch.float32,
                            use_qk_l2norm=c.use_qk_l2norm, chunk_size=c.chunk_size)
    return DeltaNetChunkOutputs(out.reshape(-1).cpu().numpy(), st.reshape(-1).cpu().numpy())


# ---- full-model decode session ------------------------------------------------

class ModelDesc(ctypes.Structure):
    _fields_ = [("num_layers", ctypes.c_int32), ("vocab", ctypes.c_int32), ("max_batch", ctypes.c_int32),
                ("max_seq", ctypes.c_int32), ("rms_eps", ctypes.c_float), ("rope_theta", ctypes.c_float),
                ("exact", ctypes.c_int32), ("reserved", ctypes.c_int32)]


def _model_lib():
    L = lib()
    if not getattr(L, "_model_types", False):
        vp = ctypes.c_void_p
        L.spock_model_create.argtypes = [vp, ctypes.POINTER(ModelDesc), ctypes.POINTER(vp)]
        L.spock_model_destroy.argtypes = [vp]
        L.spock_model_last_error.argtypes = [vp]
        L.spock_model_last_error.restype = ctypes.c_char_p
        L.spock_model_set_weight.argtypes = [vp, ctypes.c_char_p, vp, ctypes.c_size_t]
        L.spock_model_load_artifact.argtypes = [vp, ctypes.c_char_p]
        L.spock_model_reset.argtypes = [vp, ctypes.c_int32]
        L.spock_model_step.argtypes = [vp, vp, vp, vp, vp]
        L.spock_model_generate.argtypes = [vp, vp, ctypes.c_int32, ctypes.c_int32, vp, vp]
        L.spock_model_prefill.argtypes = [vp, vp, ctypes.c_int32, vp, vp, vp]
        L.spock_model_sync.argtypes = [vp, vp]
        L._model_types = True
    return L


class Model:
    """Qwen3.5-0.8B-layout decode session on one GPU (spock_model): the B200
    form of DecodeSession (src/runtime/vk_session.hpp:22-46) for a batch of
    independent sequences. Weights are uploaded by the reference's role names."""

    def __init__(self, num_layers=24, vocab=248320, max_batch=1, max_seq=2048, eps=1e-6, theta=1e7,
                 ctx=None, device=0, exact=False):
        self.L = _model_lib()
        self.ctx = ctx or Context.get(device)
        self.device = device
        self.exact = bool(exact)
        d = ModelDesc(num_layers, vocab, max_batch, max_seq, eps, theta, int(bool(exact)), 0)
        h = ctypes.c_void_p()
        rc = self.L.spock_model_create(self.ctx.h, ctypes.byref(d), ctypes.byref(h))
        if rc != SPOCK_OK:
            raise SpockError(rc, "spock_model_create failed")
        self.h = h
        self.max_batch = max_batch

    def _check(self, rc):
        if rc != SPOCK_OK:
            raise SpockError(rc, self.L.spock_model_last_error(self.h).decode())

    def set_weights(self, weights):
        for role, arr in weights.items():
            arr = np.ascontiguousarray(arr)
            self._check(self.L.spock_model_set_weight(self.h, role.encode(), arr.ctypes.data, arr.nbytes))

    def load_artifact(self, repack_dir):
        """Loads a repacked text artifact (text_repack_manifest.json + text_weights.bin)."""
        self._check(self.L.spock_model_load_artifact(self.h, os.fsencode(repack_dir)))

    def sync(self, stream=None):
        """Waits for the stream; raises SpockError(SPOCK_ERR_TIMEOUT) when one of this
        model's kernels reported a bounded wait that gave up (spock_model_sync)."""
        self._check(self.L.spock_model_sync(self.h, _stream(stream)))

    def reset(self, batch):
        self.batch = batch
        self._check(self.L.spock_model_reset(self.h, batch))

    def step(self, tokens, stream=None):
        """tokens: int32 CUDA tensor [batch] -> (next tokens [batch], final-normed hidden fp16 [batch,1024])."""
        import torch
        out = torch.empty_like(tokens)
        hid = torch.empty((tokens.shape[0], 1024), dtype=torch.float16, device=tokens.device)
        self._check(self.L.spock_model_step(self.h, _ptr(tokens), _ptr(out), _ptr(hid), _stream(stream)))
        return out, hid

    def prefill(self, prompt, stream=None):
        """prompt: int32 CUDA tensor [batch, len] -> (next tokens [batch], final-normed hidden of the
        last prompt token fp16 [batch, 1024]). Layer-major: every layer over the whole prompt."""
        import torch
        prompt = prompt.contiguous()
        out = torch.empty((prompt.shape[0],), dtype=torch.int32, device=prompt.device)
        hid = torch.empty((prompt.shape[0], 1024), dtype=torch.float16, device=prompt.device)
        self._check(self.L.spock_model_prefill(self.h, _ptr(prompt), prompt.shape[1], _ptr(out), _ptr(hid),
                                               _stream(stream)))
        return out, hid

    def generate(self, prompt, n_new, stream=None):
        """prompt: int32 CUDA tensor [batch, len] -> greedy tokens [batch, n_new] (layer-major prefill,
        then graph-replayed decode steps)."""
        import torch
        out = torch.empty((prompt.shape[0], n_new), dtype=torch.int32, device=prompt.device)
        self._check(self.L.spock_model_generate(self.h, _ptr(prompt), prompt.shape[1], n_new, _ptr(out),
                                                _stream(stream)))
        return out

    def close(self):
        if self.h:
            self.L.spock_model_destroy(self.h)
            self.h = None

"""clutor-b200: the Clutor engine's MoE feed-forward block on B200 (sm_100a), through the C ABI of include/clb200.h.

This module is the Python view of that ABI (ctypes), used by the tests and bench.py; C host code (the reference engine)
calls the same entry points directly. There is no CPU path: importing works anywhere, but every entry point needs the
built library (python -m clutor_b200.build) and a CUDA device, and fails loudly without them.
"""
from __future__ import annotations

import ctypes as C
import os
import re
import struct

import numpy as np

from . import synth

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libclutor_b200.so")
HEADER = os.path.join(os.path.dirname(HERE), "include", "clb200.h")

T_F32, T_F16, T_Q8_0, T_Q4_K, T_Q6_K, T_BF16 = 0, 1, 8, 12, 14, 30


class CLW(C.Structure):
    """clb200_w == the reference's cl_w (c/src/forward.h:18)."""
    _fields_ = [("p", C.c_void_p), ("type", C.c_uint32), ("rows", C.c_int), ("cols", C.c_int)]


class MoELayer(C.Structure):
    """clb200_moe_layer (include/clb200.h)."""
    _fields_ = [("ffn_norm_f", C.c_void_p), ("router_f", C.c_void_p), ("gate", CLW), ("up", CLW), ("down", CLW),
                ("gate_slab", C.c_uint64), ("up_slab", C.c_uint64), ("down_slab", C.c_uint64),
                ("n_embd", C.c_int), ("n_ff_exp", C.c_int), ("n_expert", C.c_int), ("n_used", C.c_int),
                ("norm_topk", C.c_int), ("resid_scale", C.c_float), ("rms_eps", C.c_float)]


class Q8K(C.Structure):
    _fields_ = [("d", C.c_float), ("qs", C.c_int8 * 256), ("bsums", C.c_int16 * 16)]


class XQ(C.Structure):
    _fields_ = [("b", C.c_void_p), ("n", C.c_int)]


class MV(C.Structure):
    """clb200_mv == the reference's cl_mv (c/src/quant.h:31-34)."""
    _fields_ = [("type", C.c_uint32), ("w", C.c_void_p), ("rows", C.c_int), ("cols", C.c_int), ("xf", C.c_void_p),
                ("xq", C.c_void_p), ("out", C.c_void_p), ("nb", C.c_int), ("xf_stride", C.c_size_t),
                ("out_stride", C.c_size_t)]


SUPPORTS = C.CFUNCTYPE(C.c_int, C.c_uint32)
MATVEC = C.CFUNCTYPE(None, C.POINTER(MV), C.c_int)


class Backend(C.Structure):
    """clb200_backend_t == the reference's cl_backend (c/src/backend.h:9-13)."""
    _fields_ = [("name", C.c_char_p), ("supports", SUPPORTS), ("matvec_batch", MATVEC)]


class CacheStats(C.Structure):
    """clb200_cache_stats == the reference's cl_cache_stats (c/src/cache.h:14-17)."""
    _fields_ = [(n, C.c_uint64) for n in ("hits", "misses", "stage_hits", "inserts", "evictions", "admit_rejects",
                                         "stage_inserts", "stage_wasted", "aging_resets")] + [("window_slots", C.c_uint32)]

    def as_dict(self) -> dict:
        return {n: getattr(self, n) for n, _ in self._fields_}


LRU, WTINYLFU, ADAPTIVE = 0, 1, 2


class StoreStats(C.Structure):
    """clb200_store_stats (the reference's cl_xs_stats, c/src/xs.h:14-17, with copy_ns for read_ns)."""
    _fields_ = [(n, C.c_uint64) for n in ("accesses", "hits", "stage_hits", "misses", "bypass", "prefetch_issued",
                                         "prefetch_late", "prefetch_wasted", "admit_rejects", "evictions", "demand_bytes",
                                         "prefetch_bytes", "copy_ns", "wait_ns", "pred_total", "pred_hit")]

    def as_dict(self) -> dict:
        return {n: getattr(self, n) for n, _ in self._fields_}


_lib: C.CDLL | None = None


class Smart(C.Structure):
    """clb200_smart (the layout of the reference's cl_smart, c/src/route.h:14)."""
    _fields_ = [("enabled", C.c_int), ("J", C.c_int), ("M", C.c_int), ("tau", C.c_double)]


class RouteResult(C.Structure):
    """clb200_route_result (the layout of cl_route_result, c/src/route.h:16-22)."""
    _fields_ = [("selected", C.c_int * 32), ("k", C.c_int), ("substituted", C.c_int), ("dropped_mass", C.c_double),
                ("max_delta", C.c_double)]

    def as_dict(self) -> dict:
        return {"selected": list(self.selected[:self.k]), "substituted": self.substituted,
                "dropped_mass": self.dropped_mass, "max_delta": self.max_delta}


class SmartStats(C.Structure):
    _fields_ = [("substituted", C.c_uint64), ("expert_slots", C.c_uint64), ("dropped_mass", C.c_double),
                ("max_delta", C.c_double)]

    def as_dict(self) -> dict:
        return {f: getattr(self, f) for f, _ in self._fields_}


class KvStruct(C.Structure):
    """clb200_kv (include/clb200.h)."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("type", C.c_uint32), ("n_pages", C.c_int), ("page_size", C.c_int),
                ("n_kv", C.c_int), ("head_dim", C.c_int), ("page_stride", C.c_int64), ("slot_stride", C.c_int64),
                ("head_stride", C.c_int64), ("table", C.c_void_p), ("table_stride", C.c_int), ("table_width", C.c_int),
                ("n_seq", C.c_int), ("q_start", C.c_void_p), ("kv_len", C.c_void_p)]


class QkStruct(C.Structure):
    """clb200_qk (include/clb200.h)."""
    _fields_ = [("T", C.c_int), ("n_head", C.c_int), ("src_type", C.c_uint32), ("q", C.c_void_p), ("k", C.c_void_p),
                ("v", C.c_void_p), ("q_stride", C.c_int64), ("k_stride", C.c_int64), ("v_stride", C.c_int64),
                ("norm", C.c_int), ("q_norm", C.c_void_p), ("k_norm", C.c_void_p), ("eps", C.c_float), ("rope", C.c_void_p),
                ("n_pos", C.c_int), ("pairs", C.c_int), ("out", C.c_void_p), ("out_stride", C.c_int64)]


class AttnStruct(C.Structure):
    """clb200_attn (include/clb200.h)."""
    _fields_ = [("T", C.c_int), ("n_head", C.c_int), ("max_q", C.c_int), ("q", C.c_void_p), ("q_stride", C.c_int64),
                ("out", C.c_void_p), ("out_type", C.c_uint32), ("out_stride", C.c_int64), ("scale", C.c_float),
                ("window", C.c_int), ("sinks", C.c_int), ("work", C.c_void_p), ("work_bytes", C.c_size_t)]


class SamplingStruct(C.Structure):
    """clb200_sampling (include/clb200.h)."""
    _fields_ = [("rows", C.c_int), ("vocab", C.c_int), ("type", C.c_uint32), ("logits", C.c_void_p), ("stride", C.c_int64),
                ("u", C.c_void_p), ("temperature", C.c_void_p), ("top_k", C.c_void_p), ("top_p", C.c_void_p),
                ("min_p", C.c_void_p), ("token", C.c_void_p), ("prob", C.c_void_p)]


QK_NORM_NONE, QK_NORM_ROW, QK_NORM_HEAD = 0, 1, 2


def header_functions() -> list[str]:
    """Names of the functions include/clb200.h declares."""
    text = open(HEADER).read()
    return sorted(set(re.findall(r"^\s*(?:const\s+)?[\w\s\*]+?\b(clb200_\w+)\s*\(", text, re.M)))


def lib() -> C.CDLL:
    """The CUDA library; raises if it is not built (there is no fallback)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is not built: run `python -m clutor_b200.build` (no CPU fallback exists)")
        L = C.CDLL(LIB_PATH)
        L.clb200_open.restype = C.c_void_p
        L.clb200_open.argtypes = [C.c_int, C.c_char_p, C.c_size_t]
        L.clb200_close.argtypes = [C.c_void_p]
        L.clb200_device.argtypes = [C.c_void_p]
        L.clb200_moe_ffn.argtypes = [C.c_void_p, C.POINTER(MoELayer), C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_char_p, C.c_size_t]
        L.clb200_layer_bind.argtypes = [C.c_void_p, C.POINTER(MoELayer), C.c_int, C.c_char_p, C.c_size_t]
        L.clb200_moe_ffn_dev.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p, C.c_char_p, C.c_size_t]
        L.clb200_status.argtypes = [C.c_void_p, C.c_char_p, C.c_size_t]
        L.clb200_layer_release.argtypes = [C.c_void_p, C.c_int]
        L.clb200_moe_ffn_decode_noalloc.argtypes = [C.POINTER(MoELayer), C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                                                    C.c_char_p, C.c_size_t]
        L.clb200_moe_dispatch.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p,
                                          C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_char_p, C.c_size_t]
        L.clb200_device_bytes.restype = C.c_uint64
        L.clb200_device_bytes.argtypes = [C.c_void_p]
        L.clb200_set_trace.argtypes = [C.c_void_p, C.c_void_p]
        L.clb200_set_exact.argtypes = [C.c_void_p, C.c_int]
        L.clb200_set_option.argtypes = [C.c_void_p, C.c_int, C.c_int]
        L.clb200_backend.restype = C.POINTER(Backend)
        L.clb200_cache_new.restype = C.c_void_p
        L.clb200_cache_new.argtypes = [C.c_uint32, C.c_uint32, C.c_uint32, C.c_int, C.c_uint32]
        L.clb200_cache_free.argtypes = [C.c_void_p]
        L.clb200_cache_access.argtypes = [C.c_void_p, C.c_uint32, C.POINTER(C.c_int)]
        L.clb200_cache_stage.argtypes = [C.c_void_p, C.c_uint32]
        for f in ("pin", "unpin", "abandon"):
            getattr(L, f"clb200_cache_{f}").argtypes = [C.c_void_p, C.c_int]
        L.clb200_cache_find.argtypes = [C.c_void_p, C.c_uint32]
        L.clb200_cache_freq.argtypes = [C.c_void_p, C.c_uint32]
        L.clb200_cache_freq.restype = C.c_uint32
        L.clb200_cache_count.argtypes = [C.c_void_p]
        L.clb200_cache_count.restype = C.c_uint32
        L.clb200_cache_total_slots.argtypes = [C.c_void_p]
        L.clb200_cache_total_slots.restype = C.c_uint32
        L.clb200_cache_segment.argtypes = [C.c_void_p, C.c_int]
        L.clb200_cache_slot_key.argtypes = [C.c_void_p, C.c_int]
        L.clb200_cache_slot_key.restype = C.c_uint32
        L.clb200_cache_get_stats.argtypes = [C.c_void_p]
        L.clb200_cache_get_stats.restype = CacheStats
        L.clb200_store_open.restype = C.c_void_p
        L.clb200_store_open.argtypes = [C.c_void_p, C.POINTER(MoELayer), C.c_int, C.c_uint64, C.c_int, C.c_int, C.c_char_p, C.c_size_t]
        L.clb200_store_close.argtypes = [C.c_void_p]
        L.clb200_store_load_layer.argtypes = [C.c_void_p, C.c_int, C.POINTER(MoELayer), C.c_char_p, C.c_size_t]
        L.clb200_store_cache_slots.argtypes = [C.c_void_p]
        L.clb200_store_cache_slots.restype = C.c_uint32
        L.clb200_store_slot_bytes.argtypes = [C.c_void_p]
        L.clb200_store_slot_bytes.restype = C.c_uint64
        L.clb200_store_get_stats.argtypes = [C.c_void_p]
        L.clb200_store_get_stats.restype = StoreStats
        L.clb200_store_reset_stats.argtypes = [C.c_void_p]
        L.clb200_store_set_prefetch.argtypes = [C.c_void_p, C.c_int]
        L.clb200_store_set_prefetch_n.argtypes = [C.c_void_p, C.c_int]
        L.clb200_store_set_prefetch_depth.argtypes = [C.c_void_p, C.c_int]
        L.clb200_store_log.argtypes = [C.c_void_p, C.c_int]
        L.clb200_store_read_log.argtypes = [C.c_void_p, C.c_void_p, C.c_int64]
        L.clb200_store_read_log.restype = C.c_int64
        L.clb200_store_request.argtypes = [C.c_void_p, C.c_int, C.c_int]
        L.clb200_store_wait.argtypes = [C.c_void_p, C.c_int]
        L.clb200_store_wait.restype = C.c_void_p
        L.clb200_store_release.argtypes = [C.c_void_p, C.c_int, C.c_void_p]
        L.clb200_store_resident.argtypes = [C.c_void_p, C.c_int, C.c_int]
        L.clb200_store_prefetch.argtypes = [C.c_void_p, C.c_int, C.c_int]
        L.clb200_moe_ffn_stored.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                                            C.c_char_p, C.c_size_t]
        L.clb200_moe_experts_stored.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                                                C.c_void_p, C.c_char_p, C.c_size_t]
        L.clb200_route.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p, C.c_char_p,
                                   C.c_size_t]
        L.clb200_route_dev.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_int,
                                       C.c_void_p, C.c_void_p]
        L.clb200_store_set_smart.argtypes = [C.c_void_p, C.c_void_p, C.c_char_p, C.c_size_t]
        L.clb200_store_smart_stats.argtypes = [C.c_void_p]
        L.clb200_store_smart_stats.restype = SmartStats
        L.clb200_store_route.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_char_p, C.c_size_t]
        serving = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_char_p, C.c_size_t]
        L.clb200_qk_rope.argtypes = serving
        L.clb200_attention.argtypes = serving
        L.clb200_attention_work.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p]
        L.clb200_attention_work.restype = C.c_size_t
        L.clb200_sample.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_char_p, C.c_size_t]
        L.clb200_store_failed.argtypes = [C.c_void_p]
        L.clb200_store_inject_fill_failure.argtypes = [C.c_void_p, C.c_int]
        _lib = L
    return _lib


class ClutorError(RuntimeError):
    pass


def _ptr(a) -> int:
    if a is None:
        return 0
    if isinstance(a, np.ndarray):
        assert a.flags["C_CONTIGUOUS"]
        return a.ctypes.data
    return a.data_ptr()   # torch tensor


def _stream(stream) -> int:
    """The cudaStream_t for a call on torch tensors: the given torch stream, else torch's current stream (so the call is
    ordered with the torch work that made its inputs and will read its outputs)."""
    import torch
    st = (stream if stream is not None else torch.cuda.current_stream()).cuda_stream
    return st or CUDA_STREAM_LEGACY   # torch's default stream is the legacy stream; 0 would mean the context's own stream


CUDA_STREAM_LEGACY = 1   # cudaStreamLegacy


def layer_struct(layer) -> MoELayer:
    """A clb200_moe_layer over a synth.HostLayer (numpy, host pointers) or synth.DeviceLayer (torch, device pointers)."""
    s = MoELayer()
    s.ffn_norm_f, s.router_f = _ptr(layer.ffn_norm), _ptr(layer.router)
    E, FF = layer.E, layer.FF
    s.gate = CLW(_ptr(layer.gate), layer.gate_type, FF, E)
    s.up = CLW(_ptr(layer.up), layer.up_type, FF, E)
    s.down = CLW(_ptr(layer.down), layer.down_type, E, FF)
    s.gate_slab, s.up_slab, s.down_slab = layer.gate_slab, layer.up_slab, layer.down_slab
    s.n_embd, s.n_ff_exp, s.n_expert, s.n_used = E, FF, layer.NE, layer.K
    s.norm_topk, s.resid_scale, s.rms_eps = layer.norm_topk, layer.resid_scale, layer.rms_eps
    return s


class Context:
    """A clb200 context on one CUDA device (clb200_open). One host thread at a time uses it, as in C."""

    def __init__(self, device: int = 0):
        self._err = C.create_string_buffer(512)
        self.handle = lib().clb200_open(device, self._err, 512)
        if not self.handle:
            raise ClutorError(self._err.value.decode())
        self.device = lib().clb200_device(self.handle)   # device -1: the current one
        self._keep: list = []
        self._c_qk, self._c_attention, self._c_sample = lib().clb200_qk_rope, lib().clb200_attention, lib().clb200_sample
        self._work_bytes: dict = {}

    def close(self) -> None:
        if self.handle:
            lib().clb200_close(self.handle)
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, rc: int) -> None:
        if rc:
            raise ClutorError(self._err.value.decode())

    def moe_ffn(self, layer: "synth.HostLayer", x: np.ndarray):
        """The host-pointer entry point (clb200_moe_ffn): returns (x_out, sel, wt); x is not modified."""
        x = np.ascontiguousarray(x, dtype=np.float32).copy()
        T = x.shape[0]
        sel = np.zeros((T, layer.K), np.int32)
        wt = np.zeros((T, layer.K), np.float32)
        s = layer_struct(layer)
        self._check(lib().clb200_moe_ffn(self.handle, C.byref(s), _ptr(x), T, _ptr(sel), _ptr(wt), self._err, 512))
        return x, sel, wt

    def moe_ffn_inplace(self, s: MoELayer, x: np.ndarray, sel: np.ndarray, wt: np.ndarray) -> None:
        """clb200_moe_ffn on caller buffers (x updated in place), with a prebuilt layer struct: no copies on the Python side
        (for timing the host entry point from pinned memory)."""
        self._check(lib().clb200_moe_ffn(self.handle, C.byref(s), _ptr(x), x.shape[0], _ptr(sel), _ptr(wt), self._err, 512))

    def bind(self, layer, on_device: bool | None = None) -> int:
        """Registers a layer (clb200_layer_bind); device tensors are used in place, host arrays are uploaded."""
        if on_device is None:
            on_device = not isinstance(layer.gate, np.ndarray)
        s = layer_struct(layer)
        h = lib().clb200_layer_bind(self.handle, C.byref(s), 1 if on_device else 0, self._err, 512)
        if h < 0:
            raise ClutorError(self._err.value.decode())
        self._keep.append(layer)
        return h

    def release(self, handle: int) -> None:
        """Frees a bound layer's device copy (clb200_layer_release)."""
        if lib().clb200_layer_release(self.handle, handle):
            raise ClutorError(f"no layer {handle}")

    def moe_ffn_dev(self, handle: int, x, sel=None, wt=None, stream=None) -> None:
        """The device entry point (clb200_moe_ffn_dev) on torch CUDA tensors; asynchronous on `stream` (a torch stream)."""
        T = x.shape[0]
        st = _stream(stream)
        self._check(lib().clb200_moe_ffn_dev(self.handle, handle, _ptr(x), T, _ptr(sel), _ptr(wt), C.c_void_p(st), self._err, 512))

    def status(self) -> None:
        self._check(lib().clb200_status(self.handle, self._err, 512))

    def dispatch(self, sel, wt, n_expert: int, stream=None):
        """clb200_moe_dispatch on torch CUDA tensors sel [T, K] int32 and wt [T, K] float32. Returns device tensors
        (todo [n_expert + 1], offsets [n_expert + 1], pos_token [T * K], pos_wt [T * K]); asynchronous."""
        import torch
        T, K = sel.shape
        todo = torch.full((n_expert + 1,), -1, dtype=torch.int32, device=sel.device)
        offsets = torch.full((n_expert + 1,), -1, dtype=torch.int32, device=sel.device)
        pos_token = torch.full((T * K,), -1, dtype=torch.int32, device=sel.device)
        pos_wt = torch.zeros((T * K,), dtype=torch.float32, device=sel.device)
        self._check(lib().clb200_moe_dispatch(self.handle, T, n_expert, K, _ptr(sel), _ptr(wt), _ptr(todo), _ptr(offsets),
                                              _ptr(pos_token), _ptr(pos_wt), C.c_void_p(_stream(stream)), self._err, 512))
        return todo, offsets, pos_token, pos_wt

    def device_bytes(self) -> int:
        return int(lib().clb200_device_bytes(self.handle))

    def set_exact(self, on: bool) -> None:
        """clb200_set_exact: batched expert products on the integer path only (bit-exact), or on the tensor cores."""
        lib().clb200_set_exact(self.handle, int(on))

    OPT_DECODE_KERNEL, OPT_TEST_SPECULATION_MISS, OPT_TEST_STALL_WAIT, OPT_COOPERATIVE, OPT_PROMPT_ATTENTION = 1, 2, 3, 4, 5

    def set_option(self, option: int, value: int) -> None:
        """clb200_set_option: OPT_DECODE_KERNEL (0 expert-group kernel where it fits, 1 grid-wide kernel, the default) or
        the OPT_TEST_SPECULATION_MISS test hook."""
        if lib().clb200_set_option(self.handle, option, int(value)):
            raise ClutorError(f"option {option} = {value} refused")

    def set_trace(self, buf=None) -> None:
        """Phase trace of the one-token kernel (clb200_set_trace): buf is a torch uint64/int64 CUDA tensor of 32 entries per
        SM, or None to stop."""
        lib().clb200_set_trace(self.handle, _ptr(buf))


    def route(self, logits: np.ndarray, K: int, smart: tuple | None = None, resident: np.ndarray | None = None) -> dict | None:
        """cl_route on the GPU (clb200_route): logits [E] float32 (host); smart = (J, M, tau) or None; resident [E] bytes
        or None. Returns the result as a dict, or None when the arguments are out of range (as cl_route's -1)."""
        lg = np.ascontiguousarray(logits, np.float32)
        res = None if resident is None else np.ascontiguousarray(resident, np.uint8)
        sm = Smart(1, *smart) if smart else None
        out = RouteResult()
        rc = lib().clb200_route(self.handle, lg.ctypes.data, lg.shape[0], K, C.addressof(sm) if sm else None,
                                None if res is None else res.ctypes.data, C.addressof(out), self._err, 512)
        if rc < 0:
            return None
        self._check(rc)
        return out.as_dict()

    def route_dev(self, logits, K: int, smart: tuple | None, resident, out, resident_stride: int = 0, stream=None) -> int:
        """clb200_route_dev on torch CUDA tensors: logits [T, E] float32, resident uint8 or None, out a uint8 tensor of
        T * 152 bytes (clb200_route_result each). Returns the C return code."""
        sm = Smart(1, *smart) if smart else None
        T, E = logits.shape
        return lib().clb200_route_dev(self.handle, _ptr(logits), T, E, K, C.addressof(sm) if sm else None,
                                      None if resident is None else _ptr(resident), resident_stride, _ptr(out),
                                      C.c_void_p(_stream(stream)))

    def qk_rope(self, q, k, v, pages: "KvPages", q_start, kv_len, rope, *, q_norm=None, k_norm=None,
                norm: int = QK_NORM_HEAD, pairs: bool = False, eps: float = 1e-6, out=None, stream=None):
        """clb200_qk_rope on torch CUDA tensors: q [T, n_head, head_dim], k and v [T, n_kv, head_dim] (float32 or the cache's
        type; rows any stride apart) are normalised, turned by position and, k and v, stored into `pages`; q_start [n_seq + 1]
        and kv_len [n_seq] int32; rope [n_pos, head_dim] float32 (cosines, then sines). Returns the turned q, [T, n_head,
        head_dim] of the cache's type (`out`, or a new tensor); asynchronous."""
        try:
            T, H, D = q.shape
        except ValueError:
            raise ClutorError(f"q {tuple(q.shape)}: [T, n_head, head_dim]") from None
        KV, dt, f32 = pages.n_kv, q.dtype, _float32
        rows = T, KV, D
        if k.shape != rows or v.shape != rows or D != pages.head_dim:
            raise ClutorError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not fit a cache of "
                              f"{KV} heads of {pages.head_dim}")
        if k.dtype is not dt or v.dtype is not dt:
            raise ClutorError("q, k and v must have one type")
        device = self.device
        if not (pages.device == device == q.get_device() == k.get_device() == v.get_device() == rope.get_device()):
            self._on_device(pages.k, q, k, v, rope)
        if rope.dtype is not f32 or rope.dim() != 2 or rope.shape[1] != D or not rope.is_contiguous():
            raise ClutorError("rope must be a contiguous float32 [n_pos, head_dim] tensor")
        qn = kn = 0
        if norm:
            one = norm == QK_NORM_HEAD
            if q_norm is None or k_norm is None or not (q_norm.get_device() == device == k_norm.get_device()):
                self._on_device(q_norm, k_norm)
            if q_norm is None or k_norm is None or q_norm.dtype is not f32 or k_norm.dtype is not f32 or \
                    q_norm.numel() != (D if one else H * D) or k_norm.numel() != (D if one else KV * D) or \
                    not q_norm.is_contiguous() or not k_norm.is_contiguous():
                raise ClutorError("the norm's weights must be contiguous float32 tensors of head_dim elements, or for the "
                                  "whole row of its heads' elements")
            qn, kn = q_norm.data_ptr(), k_norm.data_ptr()
        st = self._raw_stream(stream)
        if out is None:
            out = _new((T, H, D), dtype=pages.dtype, device=q.device) if stream is None else _empty((T, H, D), pages.dtype, q.device, stream)
            out_row = H * D
        elif out.shape != (T, H, D) or out.dtype is not pages.dtype or out.get_device() != device:
            raise ClutorError(f"out must be {[T, H, D]} of {pages.dtype} on cuda:{device}")
        else:
            out_row = _rows(out, T, H, D)
        try:
            args = _QK.pack(T, H, _dtype(dt), q.data_ptr(), k.data_ptr(), v.data_ptr(), _rows(q, T, H, D), _rows(k, T, KV, D),
                            _rows(v, T, KV, D), norm, qn, kn, eps, rope.data_ptr(), rope.shape[0], 1 if pairs else 0, out.data_ptr(), out_row)
        except struct.error as e:
            raise ClutorError(f"an argument is out of range: {e}") from None
        if self._c_qk(self.handle, pages.pack(q_start, kv_len), args, st, self._err, 512):
            raise ClutorError(self._err.value.decode())
        return out

    def attention(self, q, pages: "KvPages", q_start, kv_len, *, max_q: int | None = None, scale: float | None = None,
                  window: int = 0, sinks: int = 0, out=None, out_dtype=None, stream=None):
        """clb200_attention on torch CUDA tensors: q [T, n_head, head_dim] of the cache's type, the new rows of sequences whose
        keys and values (the new ones included) are in `pages`; max_q bounds the new rows of a sequence (default: T, which is
        right but takes the kernel for chunks: give 1 where every sequence has one new row); scale defaults to head_dim ** -0.5. Returns [T, n_head, head_dim] (`out`, or a new tensor of out_dtype, by default q's type);
        asynchronous. The call's workspace is allocated for the stream, so calls may overlap on the device."""
        try:
            T, H, D = q.shape
        except ValueError:
            raise ClutorError(f"q {tuple(q.shape)}: [T, n_head, head_dim]") from None
        dt = q.dtype
        if D != pages.head_dim or dt is not pages.dtype:
            raise ClutorError(f"q {tuple(q.shape)} of {dt} does not fit a {pages.dtype} cache of head_dim {pages.head_dim}")
        device = self.device
        if pages.device != device or q.get_device() != device:
            self._on_device(pages.k, q)
        st = self._raw_stream(stream)
        if out is None:
            odt, out_row = out_dtype or dt, H * D
            out = _like(q) if odt is dt and stream is None and q.is_contiguous() else _empty((T, H, D), odt, q.device, stream)
        elif out.shape != (T, H, D) or (out_dtype is not None and out.dtype is not out_dtype) or out.get_device() != device:
            raise ClutorError(f"out must be {[T, H, D]} of {out_dtype or out.dtype} on cuda:{device}")
        else:
            odt, out_row = out.dtype, _rows(out, T, H, D)
        kv = pages.pack(q_start, kv_len)
        if max_q is None:
            max_q = T
        if scale is None:
            scale = D ** -0.5
        # the workspace depends on the heads, their size and whether few or many rows share a key/value head
        key = H, pages.n_kv, D, max_q
        size = self._work_bytes.get(key)
        qp, qr, op, ot = q.data_ptr(), _rows(q, T, H, D), out.data_ptr(), _dtype(odt)
        if size is None:
            try:
                args = _ATTN.pack(T, H, max_q, qp, qr, op, ot, out_row, scale, window, sinks, 0, 0)
            except struct.error as e:
                raise ClutorError(f"an argument is out of range: {e}") from None
            size = self._work_bytes[key] = lib().clb200_attention_work(self.handle, kv, args)
        if stream is None and size:
            work = _new(size, dtype=_uint8, device=q.device)
        else:
            work = _empty(size, _uint8, q.device, stream) if size else None   # 0: the call says what is wrong
        try:
            args = _ATTN.pack(T, H, max_q, qp, qr, op, ot, out_row, scale, window, sinks, work.data_ptr() if size else 0, size)
        except struct.error as e:
            raise ClutorError(f"an argument is out of range: {e}") from None
        if self._c_attention(self.handle, kv, args, st, self._err, 512):
            self._work_bytes.pop(key, None)
            raise ClutorError(self._err.value.decode())
        return out

    def sample(self, logits, u, temperature=None, top_k=None, top_p=None, min_p=None, *, token=None, prob=None, stream=None):
        """clb200_sample on torch CUDA tensors: one token for each row of logits [rows, vocab] (float32, float16 or bfloat16)
        from u [rows] float32 in [0, 1) and, each None or [rows], temperature, top_p, min_p (float32) and top_k (int32).
        Returns (token [rows] int32, prob [rows] float32); asynchronous."""
        if _new is None:
            _use_torch()
        try:
            R, V = logits.shape
        except ValueError:
            raise ClutorError(f"logits {tuple(logits.shape)}: [rows, vocab]") from None
        step, along = logits.stride()
        if V > 1 and along != 1:
            raise ClutorError("a row's logits must lie next to one another")
        self._on_device(logits, u, temperature, top_k, top_p, min_p, token, prob)
        f32, i32 = _float32, _int32
        for t, d in ((u, f32), (temperature, f32), (top_k, i32), (top_p, f32), (min_p, f32), (token, i32), (prob, f32)):
            if t is not None and (t.dtype is not d or t.shape != (R,) or not t.is_contiguous()):
                raise ClutorError(f"u, temperature, top_p, min_p, prob (float32) and top_k, token (int32) must be contiguous tensors "
                                  f"of {R} elements: got {d} wanted, {t.dtype} {tuple(t.shape)}")
        st = self._raw_stream(stream)
        if token is None:
            token = _empty(R, i32, logits.device, stream)
        if prob is None:
            prob = _empty(R, f32, logits.device, stream)
        args = _SAMPLING.pack(R, V, _dtype(logits.dtype), logits.data_ptr(), step, u.data_ptr(),
                              0 if temperature is None else temperature.data_ptr(), 0 if top_k is None else top_k.data_ptr(),
                              0 if top_p is None else top_p.data_ptr(), 0 if min_p is None else min_p.data_ptr(), token.data_ptr(),
                              prob.data_ptr())
        if self._c_sample(self.handle, args, st, self._err, 512):
            raise ClutorError(self._err.value.decode())
        return token, prob

    def _on_device(self, *tensors) -> None:
        """Raises unless every tensor given lies on this context's device."""
        d = self.device
        for t in tensors:
            if t is not None and t.get_device() != d:
                raise ClutorError(f"a tensor is on {t.device}, the context on cuda:{d}")

    def _raw_stream(self, stream) -> int:
        """The cudaStream_t of a torch stream, or of the device's current one."""
        return (_current_stream(self.device) if stream is None else stream.cuda_stream) or CUDA_STREAM_LEGACY


# the argument structs above as byte layouts: packing one costs a third of making a ctypes structure, and these calls are made
# once a layer of every token. A call's bytes are its own: the library runs without Python's lock, so that another thread may
# pack the next call's meanwhile.
_KV = struct.Struct("@PPIiiiiqqqPiiiPP0q")
_QK = struct.Struct("@iiIPPPqqqiPPfPiiPq0q")
_ATTN = struct.Struct("@iiiPqPIqfiiPN0q")
_SAMPLING = struct.Struct("@iiIPqPPPPPPP0q")
_TYPES: dict = {}   # torch types to ggml type ids
# of torch, which is imported when the first of these calls is prepared: its types, its allocator, and the raw handle of a current stream
_float32 = _int32 = _uint8 = _new = _like = _current_stream = None


def _use_torch() -> None:
    global _float32, _int32, _uint8, _new, _like, _current_stream
    if _new is None:
        try:
            import torch
        except ImportError:   # the calls on host arrays do without
            return
        _TYPES.update({torch.float32: T_F32, torch.float16: T_F16, torch.bfloat16: T_BF16})
        _float32, _int32, _uint8, _new, _like = torch.float32, torch.int32, torch.uint8, torch.empty, torch.empty_like
        _current_stream = torch._C._cuda_getCurrentRawStream


def _empty(shape, dtype, device, stream):
    """A new tensor whose memory belongs to `stream`, or to the current stream if that is None."""
    if stream is None:
        return _new(shape, dtype=dtype, device=device)
    import torch
    with torch.cuda.stream(stream):
        return _new(shape, dtype=dtype, device=device)


def _dtype(d) -> int:
    """The ggml type id of a torch type."""
    t = _TYPES.get(d)
    if t is None:
        raise ClutorError(f"{d} is not float32, float16 or bfloat16")
    return t


def _rows(t, T: int, H: int, D: int) -> int:
    """The stride of the rows of t, a [T, H, D] tensor; the heads of a row must follow one another."""
    a, b, c = t.stride()
    if c != 1 or (b != D and H > 1):
        raise ClutorError(f"the heads of a row must follow one another (strides {t.stride()} of {tuple(t.shape)})")
    return a if T > 1 else max(a, H * D)


class KvPages:
    """A paged key/value cache on the device (clb200_kv): k and v [n_pages, page_size, n_kv, head_dim] float16 or bfloat16 (the
    same strides, head_dim contiguous), table [n_seq, width] int32: the pages of each sequence in order, a row in memory for each
    (sequences that share pages name them in their own rows)."""

    __slots__ = ("k", "v", "table", "n_pages", "page_size", "n_kv", "head_dim", "dtype", "device", "_fixed")

    def __init__(self, k, v, table):
        _use_torch()
        strides, shape, dt = k.stride(), k.shape, k.dtype
        if len(shape) != 4 or shape != v.shape or dt is not v.dtype or strides != v.stride() or strides[3] != 1:
            raise ClutorError("k and v must be [n_pages, page_size, n_kv, head_dim] tensors of one type and layout")
        kind = _TYPES.get(dt)
        if kind != T_F16 and kind != T_BF16:
            raise ClutorError(f"the cache is {dt}: it must be float16 or bfloat16")
        n_seq, width = table.shape if table.dim() == 2 else (0, 0)
        row, along = table.stride() if table.dim() == 2 else (0, 0)
        if table.dim() != 2 or table.dtype is not _int32 or (width > 1 and along != 1):
            raise ClutorError("table must be an int32 [n_seq, width] tensor")
        if n_seq > 1 and row < width:   # the kernels step from row to row by at least a row's ids
            raise ClutorError(f"the rows of table share memory ({row} ids apart, {width} each): it must hold a row for each sequence")
        self.device = device = k.get_device()
        if device < 0 or v.get_device() != device or table.get_device() != device:
            raise ClutorError("k, v and table must lie on one CUDA device")
        self.k, self.v, self.table, self.dtype = k, v, table, dt
        self.n_pages, self.page_size, self.n_kv, self.head_dim = shape
        self._fixed = (k.data_ptr(), v.data_ptr(), kind, *shape, *strides[:3], table.data_ptr(), max(row, width), width, n_seq)

    def pack(self, q_start, kv_len) -> bytes:
        """The clb200_kv of one call's sequences."""
        n_seq, i32, device = self._fixed[-1], _int32, self.device
        if q_start.dtype is not i32 or kv_len.dtype is not i32 or q_start.shape != (n_seq + 1,) or kv_len.shape != (n_seq,) or \
                not q_start.is_contiguous() or not kv_len.is_contiguous() or q_start.get_device() != device or kv_len.get_device() != device:
            raise ClutorError(f"q_start and kv_len must be contiguous int32 tensors of {n_seq + 1} and {n_seq} elements on cuda:{device}")
        return _KV.pack(*self._fixed, q_start.data_ptr(), kv_len.data_ptr())


def backend() -> Backend:
    """The "b200" cl_backend struct (clb200_backend)."""
    return lib().clb200_backend().contents


def matvec(type_: int, w: np.ndarray, rows: int, cols: int, xf: np.ndarray | None = None, xq: np.ndarray | None = None):
    """One cl_mv job through the backend's matvec_batch (host pointers, like the reference's seam). xf [nb, cols] float32;
    xq: numpy array of Q8K structured dtype [nb, cols/256]. Returns out [nb, rows]."""
    nb = (xf.shape[0] if xf is not None and xf.ndim == 2 else (xq.shape[0] if xq is not None and xq.ndim == 2 else 1))
    out = np.zeros((nb, rows), np.float32)
    xqs = None
    if xq is not None:
        xq = np.ascontiguousarray(xq.reshape(nb, -1))
        xqs = (XQ * nb)(*[XQ(xq[b].ctypes.data, cols) for b in range(nb)])
    xf_c = None if xf is None else np.ascontiguousarray(xf.reshape(nb, cols), dtype=np.float32)
    job = MV(type_, _ptr(np.ascontiguousarray(w)), rows, cols, _ptr(xf_c), C.addressof(xqs) if xqs is not None else 0,
             _ptr(out), nb, cols, rows)
    be = backend()
    be.matvec_batch(C.byref(job), 1)
    return out


class ExpertCache:
    """The expert-cache policy (clb200_cache_*): which expert holds which HBM slot. Host code; needs no GPU."""

    def __init__(self, cache_slots: int, stage_slots: int, universe: int, policy: int = WTINYLFU, window_pct: int = 0):
        self.L = lib()
        self.h = self.L.clb200_cache_new(cache_slots, stage_slots, universe, policy, window_pct)
        if not self.h:
            raise ValueError("clb200_cache_new refused the sizes")

    def close(self) -> None:
        if self.h:
            self.L.clb200_cache_free(self.h)
            self.h = None

    def __del__(self):
        self.close()

    def access(self, key: int) -> tuple[int, int]:
        slot = C.c_int(-1)
        r = self.L.clb200_cache_access(self.h, key, C.byref(slot))
        return r, slot.value

    def stage(self, key: int) -> int:
        return self.L.clb200_cache_stage(self.h, key)

    def pin(self, slot: int) -> None:
        self.L.clb200_cache_pin(self.h, slot)

    def unpin(self, slot: int) -> None:
        self.L.clb200_cache_unpin(self.h, slot)

    def abandon(self, slot: int) -> None:
        self.L.clb200_cache_abandon(self.h, slot)

    def find(self, key: int) -> int:
        return self.L.clb200_cache_find(self.h, key)

    def freq(self, key: int) -> int:
        return self.L.clb200_cache_freq(self.h, key)

    def count(self) -> int:
        return self.L.clb200_cache_count(self.h)

    def total_slots(self) -> int:
        return self.L.clb200_cache_total_slots(self.h)

    def segment(self, slot: int) -> int:
        return self.L.clb200_cache_segment(self.h, slot)

    def stats(self) -> dict:
        return self.L.clb200_cache_get_stats(self.h).as_dict()


class Store:
    """The HBM expert store (clb200_store_*): every layer's experts in pinned host memory, a cache budget of them in HBM."""

    def __init__(self, ctx: "Context", shape, n_layer: int, cache_bytes: int, stage_slots: int, policy: int = WTINYLFU):
        self.ctx, self.L = ctx, lib()
        self._err = C.create_string_buffer(512)
        self._shape = layer_struct(shape)
        self.h = self.L.clb200_store_open(ctx.handle, C.byref(self._shape), n_layer, cache_bytes, stage_slots, policy, self._err, 512)
        if not self.h:
            raise ClutorError(self._err.value.decode())
        self.K = shape.K

    def close(self) -> None:
        if self.h:
            self.L.clb200_store_close(self.h)
            self.h = None

    def load_layer(self, i: int, layer) -> None:
        s = layer_struct(layer)
        if self.L.clb200_store_load_layer(self.h, i, C.byref(s), self._err, 512):
            raise ClutorError(self._err.value.decode())

    def cache_slots(self) -> int:
        return self.L.clb200_store_cache_slots(self.h)

    def slot_bytes(self) -> int:
        return self.L.clb200_store_slot_bytes(self.h)

    def stats(self) -> dict:
        return self.L.clb200_store_get_stats(self.h).as_dict()

    def reset_stats(self) -> None:
        self.L.clb200_store_reset_stats(self.h)

    PREFETCH_OFF, PREFETCH_PREV, PREFETCH_AHEAD = 0, 1, 2

    def set_prefetch_depth(self, depth: int) -> None:
        self.L.clb200_store_set_prefetch_depth(self.h, int(depth))

    def prefetch(self, layer: int, expert: int) -> None:
        """Stages one expert (clb200_store_prefetch, the reference's cl_xs_prefetch)."""
        self.L.clb200_store_prefetch(self.h, int(layer), int(expert))

    def set_prefetch(self, mode: int, n: int = 0, depth: int | None = None) -> None:
        """mode 0 off, 1 prev (the previous token's choice), 2 ahead (the next layer's router on this x); n experts staged per
        prediction (0: n_used); depth: prefetch fills in flight at once."""
        self.L.clb200_store_set_prefetch(self.h, int(mode))
        self.L.clb200_store_set_prefetch_n(self.h, int(n))
        if depth is not None:
            self.L.clb200_store_set_prefetch_depth(self.h, int(depth))

    def log(self, on: bool) -> None:
        self.L.clb200_store_log(self.h, int(on))

    def read_log(self) -> np.ndarray:
        n = self.L.clb200_store_read_log(self.h, None, 0)
        out = np.zeros(n, np.int64)
        self.L.clb200_store_read_log(self.h, out.ctypes.data, n)
        return out.reshape(-1, 3)

    def moe_ffn(self, layer: int, x, stream=None):
        """One token of `layer` through the store; x a device tensor [n_embd], updated in place. Returns (sel, wt)."""
        sel = np.zeros(self.K, np.int32)
        wt = np.zeros(self.K, np.float32)
        if self.L.clb200_moe_ffn_stored(self.ctx.handle, self.h, layer, _ptr(x), sel.ctypes.data, wt.ctypes.data,
                                        stream if isinstance(stream, int) else _stream(stream), self._err, 512):
            raise ClutorError(self._err.value.decode())
        return sel, wt

    def set_smart(self, smart: tuple | None) -> None:
        """SMART-ROUTE in moe_ffn / route (clb200_store_set_smart): (J, M, tau), or None for plain routing."""
        sm = Smart(1, *smart) if smart else None
        if self.L.clb200_store_set_smart(self.h, C.addressof(sm) if sm else None, self._err, 512):
            raise ClutorError(self._err.value.decode())

    def smart_stats(self) -> dict:
        return self.L.clb200_store_smart_stats(self.h).as_dict()

    def route(self, layer: int, logits: np.ndarray) -> dict:
        """Routing of `layer` from host logits against the store's resident set (clb200_store_route)."""
        lg = np.ascontiguousarray(logits, np.float32)
        out = RouteResult()
        if self.L.clb200_store_route(self.ctx.handle, self.h, layer, lg.ctypes.data, C.addressof(out), self._err, 512):
            raise ClutorError(self._err.value.decode())
        return out.as_dict()

    def failed(self) -> bool:
        return bool(self.L.clb200_store_failed(self.h))

    def inject_fill_failure(self, n: int) -> None:
        """Test hook: the n-th fill from now copies nothing and fails (clb200_store_inject_fill_failure)."""
        self.L.clb200_store_inject_fill_failure(self.h, n)

    def resident(self, layer: int, expert: int) -> bool:
        return bool(self.L.clb200_store_resident(self.h, layer, expert))

    def experts(self, layer: int, x, sel: np.ndarray, wt: np.ndarray, next_pred: np.ndarray | None = None, stream=None):
        """The experts of a given routing (host arrays) through the store; x a device tensor, updated in place."""
        sel = np.ascontiguousarray(sel, np.int32)
        wt = np.ascontiguousarray(wt, np.float32)
        nxt = None if next_pred is None else np.ascontiguousarray(next_pred, np.int32)
        if self.L.clb200_moe_experts_stored(self.ctx.handle, self.h, layer, _ptr(x), sel.ctypes.data, wt.ctypes.data,
                                            None if nxt is None else nxt.ctypes.data,
                                            stream if isinstance(stream, int) else _stream(stream), self._err, 512):
            raise ClutorError(self._err.value.decode())

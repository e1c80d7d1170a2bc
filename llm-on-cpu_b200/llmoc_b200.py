"""ctypes binding of libllmoc_b200.so (C ABI: include/llmoc_b200.h).

Loads the in-tree sm_100a library and exposes its entry points to Python
callers (tests, bench.py, a ctypes-based host).  Device buffers are passed
as integer addresses or as objects with ``data_ptr()`` (torch tensors).
Importing this module never falls back to anything: a missing library
raises at import time.
"""
from __future__ import annotations

import ctypes as C
import os
import re
import struct
from typing import Optional, Sequence

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libllmoc_b200.so")
HEADER = os.path.join(os.path.dirname(HERE), "include", "llmoc_b200.h")

if not os.path.exists(LIB_PATH):
    raise ImportError(f"{LIB_PATH} is not built; run `make -C {HERE}` (or __graft_entry__.build())")
lib = C.CDLL(LIB_PATH)

OK = 0
STATUS = {0: "OK", 1: "INVALID", 2: "NO_DEVICE", 3: "CUDA", 4: "NO_MEMORY", 5: "NOT_ENABLED",
          6: "UNSUPPORTED", 7: "WORKSPACE", 8: "TIMEOUT"}
SCHEME_GPTQ_ASYM = 1
SCHEME_AWQ_SYM = 2
ROUTER_SOFTMAX = 0
ROUTER_SIGMOID_BIAS = 1
DTYPE_F32 = 0
DTYPE_BF16 = 1


class Int4View(C.Structure):
    _fields_ = [("qweight", C.c_void_p), ("scales", C.c_void_p), ("zeros", C.c_void_p),
                ("scales_f32", C.c_void_p), ("M", C.c_int32), ("K", C.c_int32),
                ("group_size", C.c_int32), ("scheme", C.c_uint32), ("awq_zp", C.c_int32)]


class MoeExpertInt4(C.Structure):
    _fields_ = [("gate", C.POINTER(Int4View)), ("up", C.POINTER(Int4View)),
                ("down", C.POINTER(Int4View)), ("weight", C.c_float)]


class LayerDesc(C.Structure):
    _fields_ = [("hidden", C.c_int32), ("inter", C.c_int32), ("n_experts", C.c_int32),
                ("topk", C.c_int32), ("group_size", C.c_int32), ("scheme", C.c_int32),
                ("awq_zp", C.c_int32), ("router", C.c_int32), ("routed_scaling", C.c_float),
                ("has_shared", C.c_int32), ("shared_scale", C.c_float)]


class QlwcLayerInfo(C.Structure):
    _fields_ = [("hidden", C.c_int32), ("inter", C.c_int32), ("n_experts", C.c_int32),
                ("group_size", C.c_int32), ("scheme", C.c_int32), ("has_router", C.c_int32),
                ("has_shared", C.c_int32), ("has_shared_gate", C.c_int32), ("has_bias", C.c_int32)]


class RouteViews(C.Structure):
    _fields_ = [("logits", C.c_void_p), ("ids", C.c_void_p), ("weights", C.c_void_p),
                ("offsets", C.c_void_p), ("sorted", C.c_void_p), ("inverse", C.c_void_p),
                ("n_active", C.c_void_p), ("error_flag", C.c_void_p)]


class NormDesc(C.Structure):
    _fields_ = [("hidden", C.c_int32), ("post", C.c_int32), ("pre", C.c_int32), ("weight_dtype", C.c_int32),
                ("post_weight", C.c_void_p), ("post_bias", C.c_void_p), ("pre_weight", C.c_void_p),
                ("pre_bias", C.c_void_p), ("weight_offset", C.c_float), ("eps", C.c_float),
                ("block_scale", C.c_float), ("residual_scale", C.c_float), ("gate_act", C.c_int32)]


class NormIO(C.Structure):
    _fields_ = [("block", C.c_void_p), ("ld_block", C.c_int64), ("residual", C.c_void_p), ("ld_residual", C.c_int64),
                ("residual_out", C.c_void_p), ("ld_residual_out", C.c_int64), ("norm_out", C.c_void_p),
                ("ld_norm_out", C.c_int64), ("gate", C.c_void_p), ("gate_row_stride", C.c_int64),
                ("gate_col_stride", C.c_int64), ("block_dtype", C.c_int32), ("residual_dtype", C.c_int32),
                ("norm_dtype", C.c_int32), ("gate_dtype", C.c_int32)]


class BeamDesc(C.Structure):
    _fields_ = [("batch", C.c_int32), ("beams", C.c_int32), ("vocab", C.c_int32), ("n_out", C.c_int32),
                ("eos_token", C.c_int32)]


class ReorderTensor(C.Structure):
    _fields_ = [("src", C.c_void_p), ("dst", C.c_void_p), ("src_stride", C.c_int64), ("dst_stride", C.c_int64),
                ("seg_stride", C.c_int64), ("seg_bytes", C.c_int64), ("n_seg", C.c_int32)]


_vp, _i, _sz, _f = C.c_void_p, C.c_int, C.c_size_t, C.c_float
_SIGS = {
    "llmoc_cuda_probe_available": (_i, []),
    "llmoc_cuda_enabled": (_i, []),
    "llmoc_cuda_status": (C.c_char_p, []),
    "llmoc_cuda_device_count": (_i, []),
    "llmoc_cuda_enable": (_i, [_sz]),
    "llmoc_cuda_disable": (None, []),
    "llmoc_cuda_vram_used": (_sz, []),
    "llmoc_cuda_vram_budget": (_sz, []),
    "llmoc_cuda_set_vram_budget": (None, [_sz]),
    "llmoc_cuda_device_mem_info": (_i, [C.POINTER(_sz), C.POINTER(_sz)]),
    "llmoc_cuda_host_register": (_i, [_vp, _sz]),
    "llmoc_cuda_host_unregister": (_i, [_vp]),
    "llmoc_last_error": (C.c_char_p, []),
    "llmoc_try_gemm_int4": (_i, [_vp, C.POINTER(Int4View), _vp]),
    "llmoc_try_gemm_int4_argmax": (_i, [_vp, C.POINTER(Int4View), C.POINTER(C.c_int32), C.POINTER(C.c_float)]),
    "llmoc_collective_create": (_i, [_i, _i, C.c_size_t, _i, C.POINTER(_vp), _vp]),
    "llmoc_collective_connect": (_i, [_vp, _vp]),
    "llmoc_collective_connect_local": (_i, [_vp, C.POINTER(_vp)]),
    "llmoc_collective_destroy": (None, [_vp]),
    "llmoc_collective_world_size": (_i, [_vp]),
    "llmoc_collective_error": (_i, [_vp]),
    "llmoc_collective_set_wait_cycles": (_i, [_vp, C.c_longlong]),
    "llmoc_collective_start": (_i, [_vp, _i, _vp, C.c_size_t, _i, _vp]),
    "llmoc_collective_finish": (_i, [_vp, _i, _vp, C.c_size_t, _i, _i, _vp]),
    "llmoc_collective_alltoall": (_i, [_vp, _vp, _vp, C.c_size_t, _vp]),
    "llmoc_collective_allreduce_sum": (_i, [_vp, _vp, C.c_size_t, _i, _vp]),
    "llmoc_collective_broadcast": (_i, [_vp, _vp, C.c_size_t, _i, _vp]),
    "llmoc_try_gemm_int4_batch": (_i, [_vp, _i, C.POINTER(Int4View), _vp]),
    "llmoc_try_gemm_int4_multi": (_i, [_vp, C.POINTER(C.POINTER(Int4View)), C.POINTER(_vp), _i]),
    "llmoc_try_gemm_int4_batch_multi": (_i, [_vp, _i, C.POINTER(C.POINTER(Int4View)),
                                             C.POINTER(_vp), _i]),
    "llmoc_prefetch_int4_weight": (_i, [C.POINTER(Int4View)]),
    "llmoc_pin_int4_weight": (_i, [C.POINTER(Int4View)]),
    "llmoc_try_dequant_int4_matrix": (_i, [C.POINTER(Int4View), _vp]),
    "llmoc_try_moe_ffn_int4": (_i, [_vp, _i, _i, C.POINTER(MoeExpertInt4), _i, C.POINTER(Int4View),
                                    C.POINTER(Int4View), C.POINTER(Int4View), _f, _vp]),
    "llmoc_moe_layer_create": (_i, [C.POINTER(LayerDesc), _vp, _vp, C.POINTER(Int4View),
                                    C.POINTER(Int4View), _i, C.POINTER(_vp)]),
    "llmoc_moe_layer_create_device": (_i, [C.POINTER(LayerDesc), _vp, _vp, C.POINTER(Int4View),
                                           C.POINTER(Int4View), _i, C.POINTER(_vp)]),
    "llmoc_moe_layer_destroy": (None, [_vp]),
    "llmoc_moe_layer_weight_bytes": (_sz, [_vp]),
    "llmoc_expert_storage_bytes": (_sz, [_i, _i, _i, _i]),
    "llmoc_moe_workspace_bytes": (_sz, [_vp, _i]),
    "llmoc_moe_forward": (_i, [_vp, _vp, _i, _vp, _vp, _sz, _vp]),
    "llmoc_moe_layer_set_shared_gate": (_i, [_vp, _vp, _i]),
    "llmoc_qlwc_describe": (_i, [C.c_char_p, C.c_char_p, _i, C.POINTER(QlwcLayerInfo)]),
    "llmoc_qlwc_moe_layers": (_i, [C.c_char_p, C.c_char_p, C.POINTER(C.c_int32), _i]),
    "llmoc_moe_layer_create_qlwc": (_i, [C.c_char_p, C.c_char_p, _i, C.POINTER(LayerDesc), _i, C.POINTER(_vp)]),
    "llmoc_moe_forward_residual": (_i, [_vp, _vp, _i, _vp, _vp, _vp, _sz, _vp]),
    "llmoc_moe_route_views": (_i, [_vp, _i, _vp, _sz, C.POINTER(RouteViews)]),
    "llmoc_moe_route": (_i, [_vp, _vp, _i, _vp, _sz, _vp]),
    "llmoc_moe_dequant": (_i, [_vp, _i, _i, _vp, _vp]),
    "llmoc_quantize_awq_sym": (_i, [_vp, _i, _i, _i, _i, _vp, _vp, _vp]),
    "llmoc_kernel_launch_count": (C.c_uint64, []),
    "llmoc_moe_layer_set_wait_cycles": (_i, [_vp, C.c_longlong]),
    "llmoc_moe_set_stage_timing": (_i, [_vp, _i]),
    "llmoc_moe_forward_noalloc": (_i, [_vp, _vp, _i, _vp, _vp]),
    "llmoc_moe_noalloc_capacity": (_sz, []),
    "llmoc_moe_noalloc_status": (_i, [_vp, _i, _vp]),
    "llmoc_moe_stage_times": (_i, [_vp, C.POINTER(C.c_float), C.POINTER(_i)]),
    "llmoc_moe_layer_create_ep": (_i, [C.POINTER(LayerDesc), _vp, _vp, C.POINTER(Int4View),
                                       C.POINTER(Int4View), _i, _i, _i, _i, C.POINTER(_vp)]),
    "llmoc_moe_ep_source_workspace_bytes": (_sz, [_vp, _i]),
    "llmoc_moe_ep_owner_workspace_bytes": (_sz, [_vp, _i]),
    "llmoc_moe_ep_dispatch": (_i, [_vp, _vp, _i, _vp, _sz, _vp, _vp, _vp, _vp]),
    "llmoc_moe_ep_experts": (_i, [_vp, _vp, _vp, _i, _vp, _vp, _sz, _vp]),
    "llmoc_moe_ep_experts_padded": (_i, [_vp, _vp, _vp, _i, _i, _vp, _vp, _sz, _vp]),
    "llmoc_moe_ep_combine": (_i, [_vp, _vp, _i, _vp, _vp, _vp, _sz, _vp]),
    "llmoc_ep_ipc_handle_bytes": (_sz, []),
    "llmoc_ep_transport_create": (_i, [_i, _i, _i, _i, _i, _i, C.POINTER(_vp), _vp]),
    "llmoc_ep_transport_connect": (_i, [_vp, _vp]),
    "llmoc_ep_transport_connect_local": (_i, [_vp, C.POINTER(_vp)]),
    "llmoc_ep_transport_destroy": (None, [_vp]),
    "llmoc_ep_transport_error": (_i, [_vp]),
    "llmoc_ep_transport_set_wait_cycles": (_i, [_vp, C.c_longlong]),
    "llmoc_ep_p2p_workspace_bytes": (_sz, [_vp, _vp, _i]),
    "llmoc_ep_p2p_send": (_i, [_vp, _vp, _vp, _i, C.c_uint32, _vp, _sz, _vp]),
    "llmoc_ep_p2p_serve": (_i, [_vp, _vp, _i, C.c_uint32, _vp, _sz, _vp]),
    "llmoc_int4_linear_create": (_i, [C.POINTER(Int4View), _i, _i, _i, C.POINTER(_vp)]),
    "llmoc_int4_linear_destroy": (None, [_vp]),
    "llmoc_int4_linear_weight_bytes": (_sz, [_vp]),
    "llmoc_int4_linear_status": (_i, [_vp, _vp]),
    "llmoc_int4_linear_forward": (_i, [_vp, _vp, C.c_int64, _i, _vp, C.c_int64, _vp, C.c_int64, _i, _vp]),
    "llmoc_norm_residual": (_i, [C.POINTER(NormDesc), _vp, _i, _i, _vp]),  # io: a NormIO by reference or its bytes
    "llmoc_moe_block_workspace_bytes": (_sz, [_vp, _i]),
    "llmoc_moe_forward_block": (_i, [_vp, C.POINTER(NormDesc), C.POINTER(NormDesc), _vp, _i, _vp, _sz,
                                     _vp]),
    "llmoc_beam_workspace_bytes": (_sz, [C.POINTER(BeamDesc)]),
    "llmoc_beam_select": (_i, [C.POINTER(BeamDesc), _vp, C.c_int64, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz, _i,
                               _vp]),
    "llmoc_beam_reorder": (_i, [C.POINTER(ReorderTensor), _i, _vp, _i, _i, _i, _i, _vp]),
    "llmoc_ep_p2p_finish": (_i, [_vp, _vp, _vp, _i, _vp, C.c_uint32, _vp, _sz, _vp]),
}
for _name, (_res, _args) in _SIGS.items():
    _fn = getattr(lib, _name)
    _fn.restype = _res
    _fn.argtypes = _args


def header_symbols(path: str = HEADER) -> list:
    """Every function the C header declares."""
    txt = open(path).read()
    return sorted(set(re.findall(r"LLMOC_API\s+[\w\s\*]+?\b(llmoc_\w+)\s*\(", txt)))


def ptr(x) -> Optional[int]:
    if x is None:
        return None
    if isinstance(x, int):
        return x
    if hasattr(x, "data_ptr"):
        return int(x.data_ptr())
    if hasattr(x, "ctypes"):
        return int(x.ctypes.data)
    raise TypeError(f"cannot take the address of {type(x)}")


def last_error() -> str:
    return (lib.llmoc_last_error() or b"").decode()


class LlmocError(RuntimeError):
    pass


def check(status: int, what: str) -> None:
    if status != OK:
        raise LlmocError(f"{what}: {STATUS.get(status, status)}: {last_error()}")


def stream_ptr(stream) -> Optional[int]:
    """cudaStream_t of a torch stream (or an int / None)."""
    if stream is None or isinstance(stream, int):
        return stream
    return int(stream.cuda_stream)


def view(q, scales, zeros, M: int, K: int, group_size: int, scheme: int = SCHEME_AWQ_SYM,
         awq_zp: int = 7) -> Int4View:
    """An Int4View over host (numpy) or device (torch / int) buffers."""
    return Int4View(ptr(q), ptr(scales), ptr(zeros) if zeros is not None else None, None, M, K,
                    group_size, scheme, awq_zp)


def view_of(w) -> Int4View:
    """Int4View of an oracle.orc.Int4Weight-like object (host numpy arrays)."""
    return view(w.q, w.scales, w.zeros, w.M, w.K, w.group_size, w.scheme, w.awq_zp)


class MoeLayer:
    """A device-resident MoE layer (llmoc_moe_layer_*)."""

    def __init__(self, handle: int, desc: LayerDesc, device: int = 0):
        self.handle = handle
        self.desc = desc
        self.device = device

    @classmethod
    def create(cls, desc: LayerDesc, router_w, bias, experts: Sequence[Int4View],
               shared: Optional[Sequence[Int4View]], device: int = 0, on_device: bool = False):
        n = len(experts)
        arr = (Int4View * n)(*experts)
        sh = (Int4View * 3)(*shared) if shared is not None else None
        h = C.c_void_p()
        fn = lib.llmoc_moe_layer_create_device if on_device else lib.llmoc_moe_layer_create
        check(fn(C.byref(desc), ptr(router_w), ptr(bias), arr, sh, device, C.byref(h)),
              "llmoc_moe_layer_create")
        return cls(h.value, desc, device)

    @classmethod
    def from_host(cls, layer, device: int = 0) -> "MoeLayer":
        """From an oracle.orc.MoeLayer (host numpy weights)."""
        e0 = layer.experts[0].gate
        desc = LayerDesc(layer.H, layer.I, layer.E, layer.topk, e0.group_size, e0.scheme,
                         e0.awq_zp if e0.awq_zp > 0 else 7, layer.router, layer.routed_scaling,
                         1 if layer.shared is not None else 0, layer.shared_scale)
        views = []
        for ex in layer.experts:
            views += [view_of(ex.gate), view_of(ex.up), view_of(ex.down)]
        sh = None
        if layer.shared is not None:
            sh = [view_of(layer.shared.gate), view_of(layer.shared.up), view_of(layer.shared.down)]
        dev = cls.create(desc, layer.router_w, layer.bias, views, sh, device)
        if getattr(layer, "shared_gate_w", None) is not None:
            dev.set_shared_gate(layer.shared_gate_w)
        return dev

    @classmethod
    def from_qlwc(cls, path: str, prefix: str, layer: int, desc: "LayerDesc", device: int = 0) -> "MoeLayer":
        """Layer `layer` of a QLWC file (llmoc_moe_layer_create_qlwc)."""
        h = C.c_void_p()
        check(lib.llmoc_moe_layer_create_qlwc(path.encode(), prefix.encode(), layer, C.byref(desc), device,
                                              C.byref(h)), "llmoc_moe_layer_create_qlwc")
        return cls(h.value, desc, device)

    def set_shared_gate(self, gate_row, on_device: bool = False) -> None:
        """Per-token shared-expert weight sigmoid(gate_row . x) (bf16 [hidden])."""
        check(lib.llmoc_moe_layer_set_shared_gate(self.handle, ptr(gate_row), 1 if on_device else 0),
              "llmoc_moe_layer_set_shared_gate")

    def close(self) -> None:
        if self.handle:
            lib.llmoc_moe_layer_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def kk(self) -> int:
        return self.desc.topk + self.desc.has_shared

    @property
    def n_exp(self) -> int:
        return self.desc.n_experts + self.desc.has_shared

    def weight_bytes(self) -> int:
        return int(lib.llmoc_moe_layer_weight_bytes(self.handle))

    def workspace_bytes(self, T: int) -> int:
        return int(lib.llmoc_moe_workspace_bytes(self.handle, T))

    def forward(self, X, T: int, Y, ws, ws_bytes: int, stream=None) -> None:
        check(lib.llmoc_moe_forward(self.handle, ptr(X), T, ptr(Y), ptr(ws), ws_bytes,
                                    stream_ptr(stream)), "llmoc_moe_forward")

    def forward_residual(self, X, T: int, R, Y, ws, ws_bytes: int, stream=None) -> None:
        """Y = R + MoE(X) (R may be Y, and both may be X)."""
        check(lib.llmoc_moe_forward_residual(self.handle, ptr(X), T, ptr(R), ptr(Y), ptr(ws), ws_bytes,
                                             stream_ptr(stream)), "llmoc_moe_forward_residual")

    def block_workspace_bytes(self, T: int) -> int:
        return int(lib.llmoc_moe_block_workspace_bytes(self.handle, T))

    def forward_block(self, before: "ResidualNorm", after: "ResidualNorm", T: int, residual, residual_out, norm_out,
                      ws, ws_bytes: int, gate=None, stream=None) -> None:
        """The MoE block on its residual stream: before's pre norm, the layer,
        then after's post norm, gate, scales, residual add and pre norm."""
        for norm in (before, after):
            if norm.device != self.device:
                raise LlmocError(f"llmoc_moe_forward_block: a norm on cuda:{norm.device}, the layer on cuda:{self.device}")
        io = after.io(T, None, residual, residual_out, norm_out, gate)
        check(lib.llmoc_moe_forward_block(self.handle, C.byref(before.desc), C.byref(after.desc), io, T,
                                          _workspace(ws, ws_bytes, self.device), ws_bytes, stream_ptr(stream)),
              "llmoc_moe_forward_block")

    def route(self, X, T: int, ws, ws_bytes: int, stream=None) -> None:
        check(lib.llmoc_moe_route(self.handle, ptr(X), T, ptr(ws), ws_bytes, stream_ptr(stream)),
              "llmoc_moe_route")

    def route_views(self, T: int, ws, ws_bytes: int) -> RouteViews:
        v = RouteViews()
        check(lib.llmoc_moe_route_views(self.handle, T, ptr(ws), ws_bytes, C.byref(v)),
              "llmoc_moe_route_views")
        return v

    STAGES = ("router", "topk", "permute", "gate_up", "down", "combine")

    def set_wait_cycles(self, cycles: int) -> None:
        """Budget (SM clocks) of each barrier wait of the fused one-token forward."""
        check(lib.llmoc_moe_layer_set_wait_cycles(self.handle, int(cycles)), "llmoc_moe_layer_set_wait_cycles")

    def set_stage_timing(self, enable: bool) -> None:
        check(lib.llmoc_moe_set_stage_timing(self.handle, int(enable)), "llmoc_moe_set_stage_timing")

    def stage_times(self):
        """(dict stage -> summed ms, number of timed calls); clears the record."""
        ms = (C.c_float * 6)()
        n = C.c_int()
        check(lib.llmoc_moe_stage_times(self.handle, ms, C.byref(n)), "llmoc_moe_stage_times")
        return dict(zip(self.STAGES, [float(v) for v in ms])), n.value

    def dequant(self, expert: int, proj: int, out, stream=None) -> None:
        check(lib.llmoc_moe_dequant(self.handle, expert, proj, ptr(out), stream_ptr(stream)),
              "llmoc_moe_dequant")


def quantize_awq_sym(W, M: int, K: int, gs: int, bf16_scale: bool, q, scales, stream=None) -> None:
    check(lib.llmoc_quantize_awq_sym(ptr(W), M, K, gs, int(bf16_scale), ptr(q), ptr(scales),
                                     stream_ptr(stream)), "llmoc_quantize_awq_sym")


# ------------------------------------------- operators around the MoE layer
#
# Tensors are torch tensors on the operator's device; row strides are taken
# from them, and a tensor of another device, type or shape is refused here,
# before the library sees its address.

_DT = {}  # torch.dtype -> LLMOC_DTYPE_*, filled on first use (this module does not import torch)


def _dtype(x, what: str) -> int:
    d = _DT.get(x.dtype)
    if d is None:
        d = {"torch.float32": DTYPE_F32, "torch.bfloat16": DTYPE_BF16}.get(str(x.dtype))
        if d is None:
            raise LlmocError(f"{what}: {x.dtype} is not supported (bfloat16 or float32)")
        _DT[x.dtype] = d
    return d


_KINDS = ("torch.float32", "torch.int32", "torch.uint8")
_KIND = {}


def _kind(x) -> int:
    """Index of the tensor's type in _KINDS (-1: another)."""
    k = _KIND.get(x.dtype)
    if k is None:
        k = _KIND[x.dtype] = _KINDS.index(str(x.dtype)) if str(x.dtype) in _KINDS else -1
    return k


def _device(x, device: int, what: str) -> int:
    """The address of a cuda:`device` tensor."""
    if x.get_device() != device:
        raise LlmocError(f"{what} is on {x.device}, not on cuda:{device}")
    return x.data_ptr()


def _workspace(ws, ws_bytes: int, device: int):
    """The address of a workspace: ws_bytes of a contiguous tensor on
    cuda:`device`, or a raw device address."""
    if ws is None or isinstance(ws, int):
        return ws
    if ws.get_device() != device:
        raise LlmocError(f"the workspace is on {ws.device}, not on cuda:{device}")
    if not ws.is_contiguous() or ws.numel() * ws.element_size() < ws_bytes:
        raise LlmocError(f"the workspace is no contiguous tensor of {ws_bytes} bytes")
    return ws.data_ptr()


def _rows(x, rows: int, cols: int, device: int, what: str):
    """(address, row stride) of a [>= rows, cols] tensor with adjacent columns."""
    shape, stride = x.shape, x.stride()
    if len(shape) == 2:
        (n, c), (ld, step) = shape, stride
        if n >= rows and c == cols and (step == 1 or cols == 1) and x.get_device() == device:
            return x.data_ptr(), ld if rows > 1 or ld > cols else cols
    if len(shape) != 2 or shape[0] < rows or shape[1] != cols:
        raise LlmocError(f"{what}: shape {tuple(shape)}, not [{rows}, {cols}]")
    if stride[1] != 1 and cols > 1:
        raise LlmocError(f"{what}: columns are not adjacent in memory")
    raise LlmocError(f"{what} is on {x.device}, not on cuda:{device}")


class Int4Linear:
    """Dense INT4 weights resident on one device (llmoc_int4_linear_*):
    Y = X . W^T (+ R) for bf16 rows, asynchronous on a stream."""

    def __init__(self, handle: int, M: int, K: int, device: int):
        self.handle, self.M, self.K, self.device = handle, M, K, device

    @classmethod
    def create(cls, views: Sequence[Int4View], device: int = 0, on_device: bool = False) -> "Int4Linear":
        """From one view, or from several that share their input (stacked rows).
        Host buffers, or with on_device buffers of that device."""
        arr = (Int4View * len(views))(*views)
        h = C.c_void_p()
        check(lib.llmoc_int4_linear_create(arr, len(views), device, 1 if on_device else 0, C.byref(h)),
              "llmoc_int4_linear_create")
        return cls(h.value, sum(v.M for v in views), views[0].K, device)

    def forward(self, X, T: int, Y, R=None, stream=None) -> None:
        """Y[T, M] (bf16 or fp32) = X[T, K] (bf16) . W^T (+ R[T, M] bf16; R may be Y)."""
        if self.handle is None:
            raise LlmocError("llmoc_int4_linear_forward: the weights are closed")
        if T == 0:
            return
        dev = self.device
        x, ldx = _rows(X, T, self.K, dev, "X")
        y, ldy = _rows(Y, T, self.M, dev, "Y")
        r, ldr = (None, 0) if R is None else _rows(R, T, self.M, dev, "R")
        if _dtype(X, "X") != DTYPE_BF16 or (R is not None and _dtype(R, "R") != DTYPE_BF16):
            raise LlmocError("llmoc_int4_linear_forward: X and R are bfloat16")
        st = lib.llmoc_int4_linear_forward(self.handle, x, ldx, T, r, ldr, y, ldy, _dtype(Y, "Y"), stream_ptr(stream))
        if st:
            check(st, "llmoc_int4_linear_forward")

    def status(self, stream=None) -> None:
        """Synchronizes the stream; raises if a bounded wait of a forward gave up since the last call."""
        check(lib.llmoc_int4_linear_status(self.handle, stream_ptr(stream)), "llmoc_int4_linear_status")

    def weight_bytes(self) -> int:
        return int(lib.llmoc_int4_linear_weight_bytes(self.handle))

    def close(self) -> None:
        if self.handle:
            lib.llmoc_int4_linear_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


_NORM_IO = struct.Struct("PqPqPqPqPqqiiii").pack  # a NormIO's bytes, without the cost of filling one
assert struct.calcsize("PqPqPqPqPqqiiii") == C.sizeof(NormIO)


class ResidualNorm:
    """The norm after a block, its gate and scale, the residual add and the
    norm before the next block, in one pass (llmoc_norm_residual)."""

    KINDS = {"none": 0, "rms": 1, "layer": 2}
    ACTS = {"none": 0, "sigmoid": 1}

    def __init__(self, hidden: int, post: str = "none", post_weight=None, post_bias=None, pre: str = "none",
                 pre_weight=None, pre_bias=None, weight_offset: float = 0.0, eps: float = 1e-6,
                 block_scale: float = 1.0, residual_scale: float = 1.0, gate_act: str = "none", device: int = 0):
        self.hidden, self.device = hidden, device
        self._keep = [w for w in (post_weight, post_bias, pre_weight, pre_bias) if w is not None]
        for w in self._keep:
            if w.dim() != 1 or w.shape[0] != hidden or (hidden > 1 and w.stride(0) != 1):
                raise LlmocError(f"norm weight: shape {tuple(w.shape)}, not a contiguous [{hidden}]")
            if w.dtype != self._keep[0].dtype:
                raise LlmocError("norm weights differ in type")

        def at(w):
            return None if w is None else _device(w, device, "norm weight")

        self.desc = NormDesc(hidden, self.KINDS[post], self.KINDS[pre],
                             _dtype(self._keep[0], "norm weight") if self._keep else DTYPE_F32, at(post_weight),
                             at(post_bias), at(pre_weight), at(pre_bias), weight_offset, eps, block_scale,
                             residual_scale, self.ACTS[gate_act])
        self._desc = C.byref(self.desc)

    def io(self, T: int, block, residual, residual_out, norm_out, gate) -> bytes:
        """The operands as a llmoc_norm_io."""
        H, dev = self.hidden, self.device
        b = r = ro = no = 0
        ldb = ldr = ldro = ldno = 0
        bdt = rdt = ndt = DTYPE_BF16
        if block is not None:
            (b, ldb), bdt = _rows(block, T, H, dev, "block"), _dtype(block, "block")
        if residual_out is not None:
            (ro, ldro), rdt = _rows(residual_out, T, H, dev, "residual_out"), _dtype(residual_out, "residual_out")
        if residual is not None:
            (r, ldr), rdt = _rows(residual, T, H, dev, "residual"), _dtype(residual, "residual")
            if residual_out is not None and residual.dtype != residual_out.dtype:
                raise LlmocError("residual and residual_out differ in type")
        if norm_out is not None:
            (no, ldno), ndt = _rows(norm_out, T, H, dev, "norm_out"), _dtype(norm_out, "norm_out")
        g, gr, gc, gdt = 0, 0, 0, DTYPE_BF16
        if gate is not None:  # [T, H], [1, H], [T, 1] or [1, 1]
            if gate.dim() != 2 or (gate.shape[0] != 1 and gate.shape[0] < T) or gate.shape[1] not in (1, H):
                raise LlmocError(f"gate: shape {tuple(gate.shape)}, not [{T} or 1, {H} or 1]")
            g, gdt = _device(gate, dev, "gate"), _dtype(gate, "gate")
            gr = gate.stride(0) if gate.shape[0] > 1 else 0
            gc = gate.stride(1) if gate.shape[1] > 1 else 0
        return _NORM_IO(b, ldb, r, ldr, ro, ldro, no, ldno, g, gr, gc, bdt, rdt, ndt, gdt)

    def forward(self, T: int, block, residual, residual_out, norm_out, gate=None, stream=None) -> None:
        """residual_out = residual_scale * residual + block_scale * act(gate) *
        post(block), norm_out = pre(that); any operand may be None where the
        desc needs none."""
        io = self.io(T, block, residual, residual_out, norm_out, gate)
        st = lib.llmoc_norm_residual(self._desc, io, T, self.device, stream_ptr(stream))
        if st:
            check(st, "llmoc_norm_residual")


class BeamSearch:
    """Selection over beams and vocabulary (llmoc_beam_select) for one shape."""

    def __init__(self, batch: int, beams: int, vocab: int, n_out: int, eos_token: int = -1, device: int = 0):
        self.desc = BeamDesc(batch, beams, vocab, n_out, eos_token)
        self.device = device
        self._desc = C.byref(self.desc)
        self._rows, self._kept, self._n_rows, self._vocab = (batch, beams), (batch, n_out), batch * beams, vocab

    def workspace_bytes(self) -> int:
        return int(lib.llmoc_beam_workspace_bytes(C.byref(self.desc)))

    def _plain(self, x, shape, kind: int, what: str):
        if _KIND.get(x.dtype) == kind and x.shape == shape and x.is_contiguous() and x.get_device() == self.device:
            return x.data_ptr()
        if x.shape != shape or _kind(x) != kind or not x.is_contiguous():
            raise LlmocError(f"{what}: not a contiguous {_KINDS[kind]} tensor of shape {shape}")
        if x.get_device() != self.device:
            raise LlmocError(f"{what} is on {x.device}, not on cuda:{self.device}")
        return x.data_ptr()

    def select(self, logits, scores, parent, token, out_scores, ws, ws_bytes: int, finished=None, finished_out=None,
               stream=None) -> None:
        """logits [batch * beams, vocab] (bf16 or fp32), scores [batch, beams]
        fp32, finished [batch, beams] uint8 -> parent, token (int32),
        out_scores (fp32), finished_out (uint8), all [batch, n_out]."""
        rows, kept = self._rows, self._kept
        x, ld = _rows(logits, self._n_rows, self._vocab, self.device, "logits")
        st = lib.llmoc_beam_select(
            self._desc, x, ld, _dtype(logits, "logits"), self._plain(scores, rows, 0, "scores"),
            None if finished is None else self._plain(finished, rows, 2, "finished"),
            self._plain(parent, kept, 1, "parent"), self._plain(token, kept, 1, "token"),
            self._plain(out_scores, kept, 0, "out_scores"),
            None if finished_out is None else self._plain(finished_out, kept, 2, "finished_out"),
            _workspace(ws, ws_bytes, self.device), ws_bytes, self.device, stream_ptr(stream))
        if st:
            check(st, "llmoc_beam_select")


class BeamReorder:
    """The beams' states gathered by parent (llmoc_beam_reorder) for one set of
    tensors, whose addresses are taken here: src[i] [batch, beams, ...] and
    dst[i] [batch, n_out, ...], contiguous, or [batch * rows, ...]; dst[i] may
    be src[i] when n_out = beams.  With `used`, only the first `used` indices
    of dimension `dim` of a row move (a cache filled up to that length)."""

    def __init__(self, src: Sequence, dst: Sequence, batch: int, beams: int, n_out: int, device: int = 0,
                 dim: int = 0, used: Optional[int] = None):
        if len(src) != len(dst):
            raise LlmocError("BeamReorder: as many destinations as sources")
        self.batch, self.beams, self.n_out, self.device = batch, beams, n_out, device
        self._keep = (list(src), list(dst))
        self.tensors = (ReorderTensor * max(1, len(src)))()
        self.dim, self.n = dim, len(src)
        self._row = []
        for i, (s, d) in enumerate(zip(src, dst)):
            n = [1, 1]
            for j, (x, rows) in enumerate(((s, beams), (d, n_out))):
                if not x.is_contiguous() or x.numel() % max(1, batch * rows):
                    raise LlmocError(f"BeamReorder: tensor {i} is not a contiguous block of {batch} x {rows} rows")
                n[j] = x.numel() // max(1, batch * rows)
            shape, to = [tuple(x.shape[2:]) if x.dim() > 1 and tuple(x.shape[:2]) == (batch, rows) else tuple(x.shape[1:])
                         for x, rows in ((s, beams), (d, n_out))]
            if n[0] != n[1] or s.dtype != d.dtype:
                raise LlmocError(f"BeamReorder: rows of tensor {i} differ in size or type")
            self._row.append((shape, to, s.element_size(), n[0]))
            size = n[0] * s.element_size()
            self.tensors[i] = ReorderTensor(_device(s, device, f"src[{i}]"), _device(d, device, f"dst[{i}]"), size, size,
                                            0, size, 1)
        if used is not None:
            self.set_used(used)

    def set_used(self, used: int) -> None:
        """Move only the first `used` indices of dimension `dim` of every row from now on."""
        for i, (shape, to, _, _) in enumerate(self._row):
            if not 0 <= self.dim < len(shape) or not 0 <= used <= shape[self.dim]:
                raise LlmocError(f"BeamReorder: {used} of dimension {self.dim} of rows {shape}")
            if shape != to:
                raise LlmocError(f"BeamReorder: rows of tensor {i} differ in shape")
        for i, (shape, _, es, n) in enumerate(self._row):
            inner = es
            for v in shape[self.dim + 1:]:
                inner *= v
            whole = inner * shape[self.dim]
            t = self.tensors[i]
            t.n_seg, t.seg_stride, t.seg_bytes = max(1, n * es // whole if whole else 1), whole, inner * used

    def run(self, parent, stream=None) -> None:
        """parent [batch, n_out] int32 on the device (outside [0, beams): that row stays)."""
        if parent.shape != (self.batch, self.n_out) or _kind(parent) != 1 or not parent.is_contiguous():
            raise LlmocError(f"parent: not a contiguous int32 tensor of shape {(self.batch, self.n_out)}")
        st = lib.llmoc_beam_reorder(self.tensors, self.n, _device(parent, self.device, "parent"), self.batch,
                                    self.beams, self.n_out, self.device, stream_ptr(stream))
        if st:
            check(st, "llmoc_beam_reorder")


def launch_count() -> int:
    return int(lib.llmoc_kernel_launch_count())


class EpLayerShard(MoeLayer):
    """One rank's shard of an expert-parallel layer (llmoc_moe_layer_create_ep):
    routed experts e with e % world == rank, plus the router and shared expert."""

    def __init__(self, handle: int, desc: LayerDesc, rank: int, world: int, device: int = 0):
        super().__init__(handle, desc, device)
        self.rank, self.world = rank, world

    @classmethod
    def create_ep(cls, desc: LayerDesc, router_w, bias, experts: Sequence[Int4View],
                  shared: Optional[Sequence[Int4View]], rank: int, world: int, device: int = 0,
                  on_device: bool = False):
        n = len(experts)
        arr = (Int4View * n)(*experts)
        sh = (Int4View * 3)(*shared) if shared is not None else None
        h = C.c_void_p()
        check(lib.llmoc_moe_layer_create_ep(C.byref(desc), ptr(router_w), ptr(bias), arr, sh, device, rank, world,
                                            1 if on_device else 0, C.byref(h)), "llmoc_moe_layer_create_ep")
        return cls(h.value, desc, rank, world, device)

    @classmethod
    def from_host_ep(cls, layer, rank: int, world: int, device: int = 0) -> "EpLayerShard":
        e0 = layer.experts[0].gate
        desc = LayerDesc(layer.H, layer.I, layer.E, layer.topk, e0.group_size, e0.scheme,
                         e0.awq_zp if e0.awq_zp > 0 else 7, layer.router, layer.routed_scaling,
                         1 if layer.shared is not None else 0, layer.shared_scale)
        views = []
        for ex in layer.experts:
            views += [view_of(ex.gate), view_of(ex.up), view_of(ex.down)]
        sh = None
        if layer.shared is not None:
            sh = [view_of(layer.shared.gate), view_of(layer.shared.up), view_of(layer.shared.down)]
        dev = cls.create_ep(desc, layer.router_w, layer.bias, views, sh, rank, world, device)
        if getattr(layer, "shared_gate_w", None) is not None:
            dev.set_shared_gate(layer.shared_gate_w)
        return dev

    @property
    def e_loc(self) -> int:
        return self.desc.n_experts // self.world

    def source_workspace_bytes(self, T: int) -> int:
        return int(lib.llmoc_moe_ep_source_workspace_bytes(self.handle, T))

    def owner_workspace_bytes(self, rows: int) -> int:
        return int(lib.llmoc_moe_ep_owner_workspace_bytes(self.handle, rows))

    def dispatch(self, X, T, ws, ws_bytes, send_rows, send_expert, send_counts, stream=None) -> None:
        check(lib.llmoc_moe_ep_dispatch(self.handle, ptr(X), T, ptr(ws), ws_bytes, ptr(send_rows), ptr(send_expert),
                                        ptr(send_counts), stream_ptr(stream)), "llmoc_moe_ep_dispatch")

    def experts(self, rows, expert, n, out_rows, ws, ws_bytes, stream=None, n_hint=None) -> None:
        """n rows of owner-local expert ids; with n_hint, the fixed-capacity
        layout (ids outside the shard's experts are empty slots, n_hint the
        occupied slots expected: llmoc_moe_ep_experts_padded)."""
        if n_hint is None:
            check(lib.llmoc_moe_ep_experts(self.handle, ptr(rows), ptr(expert), n, ptr(out_rows), ptr(ws),
                                           ws_bytes, stream_ptr(stream)), "llmoc_moe_ep_experts")
        else:
            check(lib.llmoc_moe_ep_experts_padded(self.handle, ptr(rows), ptr(expert), n, n_hint, ptr(out_rows),
                                                  ptr(ws), ws_bytes, stream_ptr(stream)),
                  "llmoc_moe_ep_experts_padded")

    def combine(self, X, T, ret_rows, Y, ws, ws_bytes, stream=None) -> None:
        check(lib.llmoc_moe_ep_combine(self.handle, ptr(X), T, ptr(ret_rows), ptr(Y), ptr(ws), ws_bytes,
                                       stream_ptr(stream)), "llmoc_moe_ep_combine")


class EpTransport:
    """This rank's end of the NVLink expert-parallel transport
    (llmoc_ep_transport_*): buffers for `world` ranks of a layer with `hidden`
    and `topk`, up to max_tokens tokens per rank and step."""

    def __init__(self, world: int, rank: int, hidden: int, max_tokens: int, topk: int, device: int = 0,
                 export: bool = True):
        self.world, self.rank, self.max_tokens = world, rank, max_tokens
        h = C.c_void_p()
        self.ipc = (C.c_char * int(lib.llmoc_ep_ipc_handle_bytes()))() if export else None
        check(lib.llmoc_ep_transport_create(world, rank, hidden, max_tokens, topk, device, C.byref(h),
                                            C.cast(self.ipc, C.c_void_p) if export else None),
              "llmoc_ep_transport_create")
        self.handle = h.value
        self.seq = 0

    def connect(self, handles: bytes) -> None:
        """handles: every rank's IPC handle, in rank order."""
        buf = C.create_string_buffer(handles, len(handles))
        check(lib.llmoc_ep_transport_connect(self.handle, C.cast(buf, C.c_void_p)), "llmoc_ep_transport_connect")

    @staticmethod
    def connect_local(transports) -> None:
        """Every rank of the world in this process (tests)."""
        arr = (C.c_void_p * len(transports))(*[t.handle for t in transports])
        for t in transports:
            check(lib.llmoc_ep_transport_connect_local(t.handle, arr), "llmoc_ep_transport_connect_local")

    def error(self) -> int:
        return int(lib.llmoc_ep_transport_error(self.handle))

    def workspace_bytes(self, shard, T: int) -> int:
        return int(lib.llmoc_ep_p2p_workspace_bytes(shard.handle, self.handle, T))

    def send(self, shard, X, T: int, seq: int, ws, ws_bytes: int, stream=None) -> None:
        check(lib.llmoc_ep_p2p_send(shard.handle, self.handle, ptr(X), T, seq, ptr(ws), ws_bytes,
                                    stream_ptr(stream)), "llmoc_ep_p2p_send")

    def serve(self, shard, T: int, seq: int, ws, ws_bytes: int, stream=None) -> None:
        check(lib.llmoc_ep_p2p_serve(shard.handle, self.handle, T, seq, ptr(ws), ws_bytes, stream_ptr(stream)),
              "llmoc_ep_p2p_serve")

    def finish(self, shard, X, T: int, Y, seq: int, ws, ws_bytes: int, stream=None) -> None:
        check(lib.llmoc_ep_p2p_finish(shard.handle, self.handle, ptr(X), T, ptr(Y), seq, ptr(ws), ws_bytes,
                                      stream_ptr(stream)), "llmoc_ep_p2p_finish")

    def close(self) -> None:
        if self.handle:
            lib.llmoc_ep_transport_destroy(self.handle)
            self.handle = None


class Collective:
    """This rank's end of the NVLink collectives (llmoc_collective_*), the
    contracts::ICollective operations between the GPUs of a box."""

    ALLTOALL, ALLREDUCE_SUM, BROADCAST = 0, 1, 2
    F32, BF16 = 0, 1

    def __init__(self, world: int, rank: int, max_bytes: int, device: int = 0, export: bool = True):
        self.world, self.rank = world, rank
        h = C.c_void_p()
        self.ipc = (C.c_char * int(lib.llmoc_ep_ipc_handle_bytes()))() if export else None
        check(lib.llmoc_collective_create(world, rank, max_bytes, device, C.byref(h),
                                          C.cast(self.ipc, C.c_void_p) if export else None),
              "llmoc_collective_create")
        self.handle = h.value

    def connect(self, handles: bytes) -> None:
        """handles: every rank's IPC handle, in rank order."""
        buf = C.create_string_buffer(handles, len(handles))
        check(lib.llmoc_collective_connect(self.handle, C.cast(buf, C.c_void_p)), "llmoc_collective_connect")

    @staticmethod
    def connect_local(colls) -> None:
        """Every rank of the world in this process (tests)."""
        arr = (C.c_void_p * len(colls))(*[c.handle for c in colls])
        for c in colls:
            check(lib.llmoc_collective_connect_local(c.handle, arr), "llmoc_collective_connect_local")

    def world_size(self) -> int:
        return int(lib.llmoc_collective_world_size(self.handle))

    def error(self) -> int:
        return int(lib.llmoc_collective_error(self.handle))

    def start(self, op: int, src, nbytes: int, root: int = 0, stream=None) -> None:
        check(lib.llmoc_collective_start(self.handle, op, ptr(src), nbytes, root, stream_ptr(stream)),
              "llmoc_collective_start")

    def finish(self, op: int, dst, nbytes: int, dtype: int = 0, root: int = 0, stream=None) -> None:
        check(lib.llmoc_collective_finish(self.handle, op, ptr(dst), nbytes, dtype, root, stream_ptr(stream)),
              "llmoc_collective_finish")

    def alltoall(self, send, recv, chunk_bytes: int, stream=None) -> None:
        check(lib.llmoc_collective_alltoall(self.handle, ptr(send), ptr(recv), chunk_bytes, stream_ptr(stream)),
              "llmoc_collective_alltoall")

    def allreduce_sum(self, inout, nbytes: int, dtype: int, stream=None) -> None:
        check(lib.llmoc_collective_allreduce_sum(self.handle, ptr(inout), nbytes, dtype, stream_ptr(stream)),
              "llmoc_collective_allreduce_sum")

    def broadcast(self, buf, nbytes: int, root: int, stream=None) -> None:
        check(lib.llmoc_collective_broadcast(self.handle, ptr(buf), nbytes, root, stream_ptr(stream)),
              "llmoc_collective_broadcast")

    def close(self) -> None:
        if self.handle:
            lib.llmoc_collective_destroy(self.handle)
            self.handle = None


def qlwc_moe_layers(path: str, prefix: str) -> list:
    """Layer numbers of the QLWC file's MoE layers, ascending."""
    n = int(lib.llmoc_qlwc_moe_layers(path.encode(), prefix.encode(), None, 0))
    if n < 0:
        raise LlmocError("llmoc_qlwc_moe_layers: " + last_error())
    arr = (C.c_int32 * max(1, n))()
    lib.llmoc_qlwc_moe_layers(path.encode(), prefix.encode(), arr, n)
    return list(arr[:n])


def qlwc_describe(path: str, prefix: str, layer: int) -> QlwcLayerInfo:
    info = QlwcLayerInfo()
    check(lib.llmoc_qlwc_describe(path.encode(), prefix.encode(), layer, C.byref(info)), "llmoc_qlwc_describe")
    return info
